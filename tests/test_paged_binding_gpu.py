"""What the decoder operators' Python calls make of autograd's tensors: nothing that needs a derivative is taken, nothing written unseen."""
import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _inputs():
    k, v, table, q_start, kv_len = (t.to(DEV) for t in R.make_batch([3], [20], 16, 2, 64, torch.bfloat16))
    bf = dict(device=DEV, dtype=torch.bfloat16)
    return dict(q=torch.ones(3, 4, 64, **bf), new=torch.ones(3, 2, 64, **bf), k=k, v=v, batch=(table, q_start, kv_len), freq=R.inv_freq(32).to(DEV), pos=torch.arange(3, device=DEV),
                out=torch.zeros(3, 4, 64, **bf))


def _calls():
    """Every operand of every call that may be of a floating type: name, and the call with that operand changed by `f`."""
    from llcompiler_b200.executor import kv_append, paged_attention, rotary
    turn = lambda d: rotary(d["q"], d["pos"], d["freq"], out=d["out"])
    write = lambda d: kv_append(d["new"], d["new_v"], d["k"], d["v"], *d["batch"], q=d["q"], inv_freq=d["freq"], q_out=d["out"])
    read = lambda d: paged_attention(d["q"], d["k"], d["v"], *d["batch"], out=d["out"])
    return [("rotary", turn, ("q", "freq", "out")), ("kv_append", write, ("new", "new_v", "k", "v", "q", "freq", "out")), ("paged_attention", read, ("q", "k", "v", "out"))]


CASES = [("rotary", n) for n in ("q", "freq", "out")] + [("kv_append", n) for n in ("new", "new_v", "k", "v", "q", "freq", "out")] + [("paged_attention", n) for n in ("q", "k", "v", "out")]


def _call_with(which, name, change):
    call = {w: c for w, c, _ in _calls()}[which]
    d = _inputs()
    d["new_v"] = d["new"].clone()
    d[name] = change(d[name])
    return lambda: call(d)


@pytest.mark.parametrize("which,name", CASES)
def test_operands_that_require_a_gradient_are_refused(which, name):
    call = _call_with(which, name, lambda t: t.clone().requires_grad_())
    with pytest.raises(ValueError, match="requires a gradient"):
        call()
    with torch.no_grad():                                     # nobody asks for it there
        call()


@pytest.mark.parametrize("which,name", CASES)
def test_operands_with_a_forward_mode_tangent_are_refused(which, name):
    """A dual tensor does not require a gradient; its tangent would be lost.  Other tensors are taken inside a dual level."""
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        call = _call_with(which, name, lambda t: fwd.make_dual(t.clone(), torch.ones_like(t)))
        with pytest.raises(ValueError, match="tangent"):
            call()
        _call_with(which, name, lambda t: t)()


@pytest.mark.parametrize("which,name", [("rotary", "out"), ("kv_append", "k"), ("kv_append", "v"), ("kv_append", "out"), ("paged_attention", "out")])
def test_a_graph_that_saved_what_a_call_writes_raises(which, name):
    call = {w: c for w, c, _ in _calls()}[which]
    d = _inputs()
    d["new_v"] = d["new"].clone()
    d[name] = d[name].abs() + 1
    w = torch.ones_like(d[name], requires_grad=True)
    (w * d[name]).sum().backward()                            # as long as nothing is written
    graph = (w * d[name]).sum()
    with torch.no_grad():
        call(d)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        graph.backward()


def test_nothing_else_counts_as_written():
    d = _inputs()
    d["new_v"] = d["new"].clone()
    before = {n: t._version for n, t in d.items() if isinstance(t, torch.Tensor)}
    from llcompiler_b200.executor import kv_append, paged_attention, rotary
    made = [rotary(d["q"], d["pos"], d["freq"]), paged_attention(d["q"], d["k"], d["v"], *d["batch"])]
    assert {n: t._version for n, t in d.items() if isinstance(t, torch.Tensor)} == before
    made.append(kv_append(d["new"], d["new_v"], d["k"], d["v"], *d["batch"], q=d["q"], inv_freq=d["freq"]))
    assert all(t._version == 0 for t in made)
    assert {n for n, t in d.items() if isinstance(t, torch.Tensor) and t._version != before[n]} == {"k", "v"}
    with torch.inference_mode():                              # tensors without a counter are written all the same
        x = torch.ones(3, 4, 64, device=DEV, dtype=torch.bfloat16)
        assert rotary(x, d["pos"], d["freq"], out=x) is x


def test_caches_that_repeat_their_elements_are_read_but_not_written():
    from llcompiler_b200.executor import kv_append, paged_attention
    d = _inputs()
    for k, v in ((d["k"][:, :, :1].expand(-1, -1, 2, -1), d["v"]), (d["k"], d["v"][:1].expand(d["v"].shape))):
        with pytest.raises(ValueError):
            kv_append(d["new"], d["new"], k, v, *d["batch"])
        host = [t.cpu() for t in (d["q"], k, v, *d["batch"])]
        want, size, largest = R.attention(*host, R.scale_of(64), 0, 0)
        off = (paged_attention(d["q"], k, v, *d["batch"]).double().cpu() - want).abs()
        assert (off <= R.attention_tolerance(want, size, largest, torch.bfloat16)).all()


def test_the_device_status_is_healthy_after_the_calls():
    from llcompiler_b200.executor import device_status
    for _, call, _ in _calls():
        d = _inputs()
        d["new_v"] = d["new"].clone()
        call(d)
        assert device_status() == 0 and device_status(torch.cuda.current_device()) == 0


def test_a_module_that_calls_them_is_compiled_in_pieces():
    """The package's backend compiles what lies between the calls, which run as they are."""
    from llcompiler_b200.compiler import LLCompiler
    from llcompiler_b200.executor import kv_append, paged_attention
    d = _inputs()
    torch.manual_seed(0)

    class Layer(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.qkv, self.out = torch.nn.Linear(256, 512), torch.nn.Linear(256, 256)

        def forward(self, x):
            y = self.qkv(x).view(-1, 8, 64).to(torch.bfloat16)
            q = kv_append(y[:, 4:6], y[:, 6:], d["k"], d["v"], *d["batch"], q=y[:, :4], inv_freq=d["freq"])
            return self.out(paged_attention(q, d["k"], d["v"], *d["batch"]).reshape(-1, 256).float())

    layer, x = Layer().to(DEV), torch.randn(3, 256, device=DEV)
    torch._dynamo.reset()
    with torch.no_grad():
        want = layer(x)
        got = torch.compile(layer, backend=LLCompiler())(x)
    # the projections may differ in their last bits, so that q, k, v and the context round to the neighbouring bf16 number: a step of 2^-8 each
    assert float((got - want).norm() / want.norm()) < 4 * 2.0 ** -8
