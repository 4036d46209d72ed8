"""Rotary positions, stores into 8 bits, read-backs and attention together, as a server uses them through PagedCache: prompts, steps, pieces of
different lengths, forks, cuts, compaction.  Attention is checked in 64 bits against the numbers that the cache holds (read back in fp32 from codes
and scales), those against the keys and values that were stored."""
import math

import pytest
import torch

from flame_amd import functional
from flame_amd.paged_cache import PagedCache
from flame_amd.rotary import Rotary
from tests.test_gpu_rotary import close, reference as turned

pytestmark = pytest.mark.gpu
H, HKV, D, PAGE, BLOCK, LAYERS = 8, 2, 64, 32, 8, 2


def rand(*shape):
    return torch.randn(shape, device="cuda").to(torch.bfloat16)


def numbers(cache, layer, seq):
    """k, v [HKV, tokens, D] in 64 bits of a sequence, from the codes and scales themselves"""
    out = []
    for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        pages = cache.pages(seq)
        x = c[layer].view(torch.uint8)[pages].view(c.dtype).double() * s[layer][pages].double().repeat_interleave(BLOCK, 2)[..., None]
        out.append(x.transpose(0, 1).reshape(HKV, -1, D)[:, :cache.length(seq)])
    return out


def attended(q, k, v):
    """q [H, n, D] of the last n tokens: (O, bound)"""
    keep = torch.ones((q.shape[1], k.shape[1]), dtype=torch.bool, device="cuda").tril(k.shape[1] - q.shape[1])
    k, v = (x.repeat_interleave(H // HKV, 0) for x in (k, v))
    p = torch.softmax((q.double() @ k.transpose(1, 2) * D ** -0.5).masked_fill(~keep, -math.inf), -1)
    return p @ v, p @ v.abs()


class Life:
    def __init__(self, dtype):
        self.cache = PagedCache(LAYERS, 60, PAGE, HKV, D, dtype=dtype, block=BLOCK)
        self.rope = Rotary(D, base=500000.0, scaling="bands", factor=8.0, original_length=8192)
        self.said = {}                 # of every sequence and layer: lists of keys and values, as they were stored
        self.dtype = dtype

    def step(self, seqs, counts, share=True):
        cache, n = self.cache, sum(counts)
        before = [cache.length(s) for s in seqs]
        batch = cache.extend(seqs, counts, share_prefix=share)
        held = cache.held(seqs)
        assert batch.past.tolist() == before
        for layer in range(LAYERS):
            q, k, v = rand(n, H, D), rand(n, HKV, D), rand(n, HKV, D)
            plain = k
            q, k = functional.rotary(self.rope, q, k, cu_seqlens=batch.cu, start=batch.past)
            pos = torch.cat([torch.arange(a, a + m) for a, m in zip(before, counts)])
            close(k, *turned(plain, pos, self.rope), torch.bfloat16)
            cache.store(layer, k, v, batch)
            outs = [cache.attend_rows(layer, q, batch, held)]
            if len(set(counts)) == 1:
                outs.append(cache.attend(layer, q.view(len(seqs), counts[0], H, D).transpose(1, 2), batch).transpose(1, 2).reshape(n, H, D))
            at = 0
            read = cache.load(layer, held)
            for s, m, rows in zip(seqs, counts, held.cu.tolist()):
                said = self.said.setdefault((s, layer), ([], []))
                said[0].extend(k[at:at + m])
                said[1].extend(v[at:at + m])
                kk, vv = numbers(cache, layer, s)
                for mine, wanted, scale, back in ((kk, said[0], cache.k_scale, read[0]), (vv, said[1], cache.v_scale, read[1])):
                    x = torch.stack(wanted, 1).double()
                    step = scale[layer][cache.pages(s)].transpose(0, 1).reshape(HKV, -1).double().repeat_interleave(BLOCK, 1)[:, :x.shape[1], None]
                    # int8: less than a step of the block's last scale; e4m3: rounded twice at most, by a sixteenth and half of the smallest step
                    off = (mine - x).abs()
                    assert (off <= (step if self.dtype == torch.int8 else x.abs() / 8 + step * 2.0 ** -9)).all()
                    assert torch.equal(back[rows:rows + x.shape[1]].transpose(0, 1), mine.float().to(torch.bfloat16))
                # attend_rows attends to the numbers rounded to bf16: a relative 2^-9 of every key and value more
                want, mass = attended(q[at:at + m].transpose(0, 1), kk, vv)
                kb, vb = (x.float().to(torch.bfloat16).double() for x in (kk, vv))
                want_b, mass_b = attended(q[at:at + m].transpose(0, 1), kb, vb)
                assert ((outs[0][at:at + m].transpose(0, 1).double() - want_b).abs() <= 2.0 ** -7 * mass_b).all()
                if len(outs) > 1:
                    assert ((outs[1][at:at + m].transpose(0, 1).double() - want).abs() <= 2.0 ** -7 * mass).all()
                at += m
        return batch


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_a_server_s_life(dtype):
    life = Life(dtype)
    cache = life.cache
    prompts = [cache.new() for _ in range(4)]
    life.step(prompts, [75, 130, 16, 1])
    life.step(prompts, [1] * 4)
    life.step(prompts, [9, 1, 40, 3])                       # pieces of different lengths
    answers = [prompts[1]] + [cache.fork(prompts[1]) for _ in range(5)]
    for a in answers[1:]:
        for layer in range(LAYERS):
            life.said[a, layer] = tuple(list(x) for x in life.said[prompts[1], layer])
    for n in (1, 3, 1):
        assert int(life.step(answers, [n] * 6).prefix_len) == 128
    life.step(answers, [1] * 6, share=False)
    for a in answers:                                      # refused drafts
        cache.cut(a, cache.length(a) - 2)
        for layer in range(LAYERS):
            life.said[a, layer] = tuple(x[:-2] for x in life.said[a, layer])
    life.step(answers, [2] * 6)
    cache.free(answers[1:4] + [prompts[0]])
    assert cache.compact() > 0
    life.step([answers[0], answers[4], answers[5], prompts[2], prompts[3]], [1] * 5)
    life.step([answers[0], prompts[2]], [1, 30])


def test_reading_a_bf16_cache_back():
    """Pieces of prompts against a bf16 cache: exactly the packed attention over what was stored."""
    cache = PagedCache(1, 40, PAGE, HKV, D)
    seqs = [cache.new() for _ in range(3)]
    ks, vs = [[] for _ in seqs], [[] for _ in seqs]
    for counts in ([40, 3, 100], [1, 64, 5]):
        batch = cache.extend(seqs, counts)
        held = cache.held(seqs)
        q, k, v = rand(sum(counts), H, D), rand(sum(counts), HKV, D), rand(sum(counts), HKV, D)
        cache.store(0, k, v, batch)
        for i in range(3):
            a, b = int(batch.cu[i]), int(batch.cu[i + 1])
            ks[i].append(k[a:b])
            vs[i].append(v[a:b])
        o = cache.attend_rows(0, q, batch, held)
        flat = lambda x: torch.cat([t for s in x for t in s])
        assert torch.equal(o, functional.sdpa_packed(q, flat(ks), flat(vs), batch.cu, held.cu, is_causal=True))
        got = cache.load(0, held)
        assert torch.equal(got[0], flat(ks)) and torch.equal(got[1], flat(vs))


def test_no_rows():
    cache = PagedCache(1, 4, PAGE, HKV, D, dtype=torch.int8, block=BLOCK)
    s = cache.new()
    batch, held = cache.extend([s], [0]), cache.held([s])
    cache.store(0, rand(0, HKV, D), rand(0, HKV, D), batch)
    assert cache.attend_rows(0, rand(0, H, D), batch, held).shape == (0, H, D)
    k, v = cache.load(0, held)
    assert k.shape == v.shape == (0, HKV, D)
