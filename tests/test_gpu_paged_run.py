"""The operators of packed sequences and of the paged cache together, as a server uses them: prompts through packed attention,
their keys into pages, forks, steps of single and of drafted tokens with a shared prefix, cuts, frees and compaction; and the
decoding step in captured graphs.  Checked against 64-bit attention over plain lists of every sequence's keys."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
H, HKV, D, PAGE, LAYERS = 8, 2, 64, 16, 2


def rand(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(torch.bfloat16)


def attended(q, keys, values, N):
    """q [H, N, D] of the last N tokens on lists of rows [HKV, D]: (O, bound)."""
    k, v = (torch.stack(x, 1).double() for x in (keys, values))
    keep = torch.ones((N, k.shape[1]), dtype=torch.bool, device="cuda").tril(k.shape[1] - N)
    k, v = (x.repeat_interleave(H // HKV, 0) for x in (k, v))
    s = (q.double() @ k.transpose(1, 2) * D ** -0.5).masked_fill(~keep, -math.inf)
    p = torch.softmax(s, -1)
    return p @ v, 2.0 ** -7 * (p @ v.abs())


class Said:
    """Every sequence's keys and values per layer, as lists."""

    def __init__(self):
        self.k, self.v = [[] for _ in range(LAYERS)], [[] for _ in range(LAYERS)]

    def copy(self):
        s = Said()
        s.k, s.v = [list(x) for x in self.k], [list(x) for x in self.v]
        return s

    def cut(self, n):
        self.k, self.v = [x[:n] for x in self.k], [x[:n] for x in self.v]


def step(g, cache, said, seqs, N, share=True):
    batch = cache.extend(seqs, [N] * len(seqs), share_prefix=share)
    for layer in range(LAYERS):
        k, v, q = rand(g, N * len(seqs), HKV, D), rand(g, N * len(seqs), HKV, D), rand(g, len(seqs), H, N, D)
        cache.store(layer, k, v, batch)
        o = cache.attend(layer, q, batch)
        for i, s in enumerate(seqs):
            said[s].k[layer] += list(k[i * N:(i + 1) * N])
            said[s].v[layer] += list(v[i * N:(i + 1) * N])
            want, bound = attended(q[i], said[s].k[layer], said[s].v[layer], N)
            assert ((o[i].double() - want).abs() <= bound).all(), (layer, i)
    return batch


def test_a_server_s_life():
    from flame_amd import functional
    from flame_amd.paged_cache import PagedCache
    g = torch.Generator(device="cuda").manual_seed(1)
    cache, said = PagedCache(LAYERS, 120, PAGE, HKV, D), {}
    # prompts of different lengths in one packed call per layer
    lens = [75, 130, 16, 1]
    prompts = [cache.new() for _ in lens]
    batch = cache.extend(prompts, lens)
    said.update({s: Said() for s in prompts})
    for layer in range(LAYERS):
        q, k, v = rand(g, sum(lens), H, D), rand(g, sum(lens), HKV, D), rand(g, sum(lens), HKV, D)
        o = functional.sdpa_packed(q, k, v, batch.cu, is_causal=True)
        cache.store(layer, k, v, batch)
        for i, s in enumerate(prompts):
            a, b = int(batch.cu[i]), int(batch.cu[i + 1])
            said[s].k[layer], said[s].v[layer] = list(k[a:b]), list(v[a:b])
            want, bound = attended(q[a:b].transpose(0, 1), said[s].k[layer], said[s].v[layer], b - a)
            assert ((o[a:b].transpose(0, 1).double() - want).abs() <= bound).all()
    # one token each, no common beginning
    assert step(g, cache, said, prompts, 1).prefix_table is None
    # eight answers to the second prompt: its whole pages are read once
    answers = [prompts[1]] + [cache.fork(prompts[1]) for _ in range(7)]
    said.update({s: said[prompts[1]].copy() for s in answers[1:]})
    for n in (1, 1, 3, 1):
        assert int(step(g, cache, said, answers, n).prefix_len) == 128
    # the same without a prefix, and with other sequences in the batch
    step(g, cache, said, answers, 1, share=False)
    step(g, cache, said, answers[:3] + [prompts[0]], 2)
    # drafted tokens that are refused, then others in their place
    step(g, cache, said, answers, 4)
    for s in answers:
        n = cache.length(s) - 3
        cache.cut(s, n)
        said[s].cut(n)
    step(g, cache, said, answers, 2)
    # most answers end; what is left moves together and goes on
    cache.free(answers[1:6])
    cache.free([prompts[0]])
    used = len(cache._users) - cache.free_pages
    assert cache.compact() > 0
    left = [answers[0], answers[6], answers[7], prompts[2], prompts[3]]
    assert all(p < used for s in left for p in cache.pages(s))
    step(g, cache, said, left, 1)
    step(g, cache, said, left[:3], 1)


def test_decoding_step_in_graphs():
    """Two captured steps with workspaces of their own, replayed one after the other and eager work in between; the lengths and
    tables in the captured buffers change from replay to replay."""
    from flame_amd import capi
    g = torch.Generator(device="cuda").manual_seed(2)
    B, pages, page = 5, 200, 16
    kc, vc = rand(g, pages, HKV, page, D), rand(g, pages, HKV, page, D)
    prefix = torch.arange(100, 120, dtype=torch.int32, device="cuda")
    steps = []
    for i in range(2):
        st = dict(q=rand(g, B, H, 1, D), k=rand(g, B, HKV, D), v=rand(g, B, HKV, D), table=torch.arange(B * 10, dtype=torch.int32, device="cuda").view(B, 10) + 50 * i,
                  start=torch.tensor([3, 0, 100, 159, 40], dtype=torch.int32, device="cuda"), plen=torch.tensor([300], dtype=torch.int32, device="cuda"),
                  cu=torch.arange(B + 1, dtype=torch.int32, device="cuda"), out=torch.empty((B, H, 1, D), dtype=torch.bfloat16, device="cuda"),
                  ws=torch.empty(capi.paged_workspace_bytes(B, H, HKV, 1, D, page, 10, 20), dtype=torch.uint8, device="cuda"))
        st["len"] = st["start"] + 1
        steps.append(st)

    def run(st, out, ws):
        capi.kv_store(st["k"], st["v"], kc, vc, st["table"], st["cu"], st["start"])
        return capi.attn_paged_fwd(st["q"], kc, vc, st["table"], st["len"], 0.125, prefix, st["plen"], want_lse=True, out=out, workspace=ws)[1]

    graphs = []
    for st in steps:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(st, st["out"], st["ws"])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            st["lse"] = run(st, st["out"], st["ws"])
        graphs.append(graph)
    for rep in range(4):
        for st in steps:
            st["q"].copy_(rand(g, B, H, 1, D))
            st["k"].copy_(rand(g, B, HKV, D))
            st["start"].copy_(torch.randint(0, 160, (B,), device="cuda", generator=g, dtype=torch.int32))
            st["len"].copy_(st["start"] + 1)
            st["plen"].fill_([300, 0, 1, 17][rep])
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for st in steps:
            out = torch.empty_like(st["out"])
            lse = run(st, out, torch.empty_like(st["ws"]))
            torch.cuda.synchronize()
            assert torch.equal(out, st["out"]) and torch.equal(lse, st["lse"])


def test_copies_in_a_graph_keep_their_pairs():
    from flame_amd import capi
    g = torch.Generator(device="cuda").manual_seed(3)
    kc, vc = rand(g, 2, 30, HKV, 16, D), rand(g, 2, 30, HKV, 16, D)
    src, dst = [1, 2, 1], [10, 11, 12]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        capi.kv_copy_pages(kc, vc, [0], [29])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        capi.kv_copy_pages(kc, vc, src, dst)
    src[:], dst[:] = [5, 5, 5], [20, 21, 22]
    for rep in range(3):
        kc[:, 1], kc[:, 2], vc[:, 1] = rep + 1.0, -rep - 1.0, 0.5 * rep
        graph.replay()
        torch.cuda.synchronize()
        assert bool((kc[:, [10, 12]] == rep + 1).all()) and bool((kc[:, 11] == -rep - 1).all()) and bool((vc[:, 10] == 0.5 * rep).all())


def test_python_refusals_on_the_device():
    from flame_amd import capi, functional
    g = torch.Generator(device="cuda").manual_seed(4)
    kc, q = rand(g, 6, HKV, 16, D), rand(g, 3, H, 1, D)
    table, n = torch.zeros((3, 2), dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    ok = (q, kc, kc, table, n)
    functional.sdpa_paged(*ok)
    for i, bad in ((0, q[:2]), (0, q[..., :32]), (0, q[:, :3]), (1, kc.float()), (1, kc[:5]), (2, kc.cpu()), (3, table[:2]), (3, table.long()), (3, table.t()), (3, table[:, :0]),
                   (4, n[:2]), (4, n.long())):
        with pytest.raises(AssertionError):
            functional.sdpa_paged(*(bad if j == i else t for j, t in enumerate(ok)))
    with pytest.raises(AssertionError):
        functional.sdpa_paged(*ok, prefix_table=n)
    with pytest.raises(AssertionError):
        functional.sdpa_paged(*ok, prefix_table=n[:0], prefix_len=n[:1])
    with pytest.raises(RuntimeError, match="no backward"):
        functional.sdpa_paged(q.clone().requires_grad_(True), kc, kc, table, n)
    with torch.no_grad():
        functional.sdpa_paged(q.clone().requires_grad_(True), kc, kc, table, n)
    assert functional.sdpa_paged(q.float(), kc, kc, table, n).dtype == torch.float32
    with pytest.raises(capi.FlameAttnError):
        capi.attn_paged_fwd(q, kc, kc, table.repeat(1, 40), n, 0.1, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(capi.FlameAttnError):
        capi.kv_copy_pages(kc, kc.clone(), [0, 1], [1, 2])
    with pytest.raises(OverflowError):
        capi.kv_copy_pages(kc, kc.clone(), [2 ** 40], [1])
    with pytest.raises(TypeError):
        capi.kv_copy_pages(kc, kc.clone(), ["a"], [1])
