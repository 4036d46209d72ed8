"""What autograd is told by the calls that write into a cache or have no derivative: gradients and tangents that would be lost are
refused, and a graph that holds what is overwritten raises in its backward."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from flame_amd import capi, functional

D, HKV, PAGE = 64, 2, 16


def inputs(device):
    rand = lambda *s: torch.randn(s).to(torch.bfloat16).to(device)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)
    return dict(k=rand(5, HKV, D), v=rand(5, HKV, D), kc=rand(4, HKV, PAGE, D), vc=rand(4, HKV, PAGE, D), table=ints([2], [3]), cu=ints(0, 2, 5), start=ints(0, 3))


def store(x):
    capi.kv_store(x["k"], x["v"], x["kc"], x["vc"], x["table"], x["cu"], x["start"])


def copies(x):
    capi.kv_copy_pages(x["kc"], x["vc"], [0], [1])


@pytest.mark.parametrize("call,names", [(store, ("k", "v", "kc", "vc")), (copies, ("kc", "vc"))])
def test_lost_gradients_are_refused(call, names):
    for name in names:
        x = inputs("cpu")
        x[name].requires_grad_(True)
        with pytest.raises(RuntimeError, match="no backward"):
            call(x)
        with torch.no_grad(), pytest.raises(AssertionError, match="GPU"):       # the next check: no tensor is on one
            call(x)


@pytest.mark.parametrize("recorded", [False, True])
@pytest.mark.parametrize("call,names", [(store, ("k", "v", "kc", "vc")), (copies, ("kc", "vc"))])
def test_lost_tangents_are_refused(call, names, recorded):
    for name in names:
        x = inputs("cpu")
        with fwad.dual_level():
            x[name] = fwad.make_dual(x[name].requires_grad_(recorded), torch.ones_like(x[name]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(x)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call(x)


@pytest.mark.gpu
@pytest.mark.parametrize("call", [store, copies])
def test_graphs_that_hold_the_cache(call):
    """The keys of a recorded graph are a view of the cache (of another page, too: views share one version, as with torch's own writes)."""
    x = inputs("cuda")
    q = torch.randn(PAGE, HKV, D, device="cuda").to(torch.bfloat16).requires_grad_(True)
    bounds = torch.tensor([0, PAGE], dtype=torch.int32, device="cuda")
    for held in ("kc", "vc"):
        o = functional.sdpa_packed(q, x["kc"][0].transpose(0, 1), x["vc"][0].transpose(0, 1), bounds)
        versions = {n: x[n]._version for n in ("kc", "vc", "k", "v")}
        call(x)
        assert x["kc"]._version > versions["kc"] and x["vc"]._version > versions["vc"]
        assert x["k"]._version == versions["k"] and x["v"]._version == versions["v"]
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            o.sum().backward()
    q.grad = None
    functional.sdpa_packed(q, x["kc"][0].transpose(0, 1), x["vc"][0].transpose(0, 1), bounds).sum().backward()       # nothing is written in between
    assert q.grad is not None


@pytest.mark.gpu
def test_only_calls_that_write_count():
    """No pairs, refused pairs: nothing was written."""
    x = inputs("cuda")
    version = x["kc"]._version
    capi.kv_copy_pages(x["kc"], x["vc"], [], [])
    with pytest.raises(capi.FlameAttnError):
        capi.kv_copy_pages(x["kc"], x["vc"], [0, 1], [2, 2])
    assert x["kc"]._version == version
    layers = x["kc"][None].contiguous()
    capi.kv_copy_pages(layers, layers.clone(), [0], [1])
    assert layers._version == 1 and torch.equal(layers[0, 0], layers[0, 1])


@pytest.mark.gpu
def test_caches_of_inference_mode():
    """Their tensors have no version; the calls work inside and outside of the mode, with weights that require a gradient around."""
    with torch.inference_mode():
        x = inputs("cuda")
        store(x)
        copies(x)
    store(x)
    copies(x)
    want = x["k"][:2].transpose(0, 1)
    assert torch.equal(x["kc"][2, :, :2], want) and torch.equal(x["kc"][1], x["kc"][0])
    y = inputs("cuda")
    version = y["kc"]._version
    with torch.inference_mode():
        store(y)
    assert y["kc"]._version > version
    y["k"].requires_grad_(True)
    with torch.no_grad():
        store(y)


@pytest.mark.parametrize("recorded", [False, True])
def test_forward_mode_of_the_attention_calls(recorded):
    """There is no forward-mode derivative, and a result without a tangent would mean a derivative of zero."""
    x = inputs("cpu")
    q = torch.randn(2, 4, 1, D).to(torch.bfloat16)
    paged = [q, x["kc"], x["vc"], x["table"], torch.tensor([3, 4], dtype=torch.int32)]
    packed = [torch.randn(5, 4, D).to(torch.bfloat16), x["k"], x["v"], x["cu"]]
    for call, args in ((functional.sdpa_paged, paged), (functional.sdpa_packed, packed)):
        for which in range(3):
            with fwad.dual_level():
                dual = list(args)
                dual[which] = fwad.make_dual(dual[which].clone().requires_grad_(recorded), torch.ones_like(dual[which]))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(*dual)
                with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                    call(*dual)


def test_gradients_of_paged_attention():
    x = inputs("cpu")
    args = [torch.randn(2, 4, 1, D).to(torch.bfloat16), x["kc"], x["vc"], x["table"], torch.tensor([3, 4], dtype=torch.int32)]
    for which in range(3):
        leaves = list(args)
        leaves[which] = leaves[which].clone().requires_grad_(True)
        with pytest.raises(RuntimeError, match="no backward"):
            functional.sdpa_paged(*leaves)


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [torch.enable_grad, torch.no_grad, torch.inference_mode])
def test_layers_of_a_cache_share_its_version(mode):
    from flame_amd.paged_cache import PagedCache
    c = PagedCache(2, 8, PAGE, HKV, D)
    a = c.new()
    batch = c.extend([a], [5])
    k, v = torch.randn(2, 5, HKV, D, device="cuda").to(torch.bfloat16)
    before = c.k._version, c.v._version
    with mode():
        c.store(1, k, v, batch)
    assert c.k._version > before[0] and c.v._version > before[1]
    fork, before = c.fork(a), c.k._version
    with mode():
        c.extend([a, fork], [1, 1])                 # copies the shared page
    assert c.k._version > before and torch.equal(c.k[1, c.pages(fork)[0], :, :5], c.k[1, c.pages(a)[0], :, :5])
