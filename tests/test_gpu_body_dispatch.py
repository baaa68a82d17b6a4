"""GPU: the native dispatch of the body operators gives the registered ops' results and gradients bit for bit
and leaves to them whatever has to see the op; captured graphs, other streams, compilation, checkpointing."""
from __future__ import annotations

import pytest
import torch
import torch._dynamo.compiled_autograd
import torch.utils.checkpoint
from torch.library import CustomOpDef
from torch.utils._python_dispatch import TorchDispatchMode

import body_reference as R
from sihc_hip import _native, body

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def normal(*shape, dtype=torch.float32, seed=[0]):
    seed[0] += 1
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed[0])).to(dtype).cuda()


def cases():
    """(op, its tensors that may need a gradient, how its arguments are made of them, how many outputs have one)"""
    def linear(act, gate, residual, dtype, outer=24):
        wide = 2 * outer if act == "swiglu" else outer
        leaves = [normal(3, 7, 40, dtype=dtype), normal(wide, 40, dtype=dtype), normal(wide, dtype=dtype)]
        if gate:
            leaves.append(normal(3, 2, outer, dtype=dtype)[:, 1])
        if residual:
            leaves.append(normal(3, 7, outer, dtype=dtype))

        def arguments(t):
            return (t[0], t[1], t[2], act, t[3] if gate else None, t[-1] if residual else None)

        return body._linear_act, leaves, arguments, 1

    yield linear("none", False, False, BF16)
    yield linear("none", True, False, torch.float32)
    yield linear("silu", False, True, BF16)
    yield linear("swiglu", True, True, BF16)
    yield linear("swiglu", False, False, torch.float32)
    at = torch.arange(10, dtype=torch.int32).reshape(5, 2).cuda()
    qkv = normal(2, 5, 9, 24, dtype=BF16)
    yield (body._qk_norm_rotary, [qkv[:, :, :4], qkv[:, :, 4:6], normal(24), normal(24)],
           lambda t: (*t, at, [12, 12], 1e4, 1e-6), 2)
    yield (body._qk_norm_rotary, [normal(2, 5, 4, 24), normal(2, 5, 1, 24), normal(24), normal(24)],
           lambda t: (*t, at.float(), (8, 4), 100, 0), 2)
    yield body._axis_rotary, [qkv], lambda t: (t[0], at, [12, 10], 1e4, False), 1
    seed = torch.tensor([77], device="cuda")
    yield body._dropout, [normal(3, 50)], lambda t: (t[0], 0.3, seed, 5, None), 1
    yield body._dropout, [normal(3, 50, dtype=BF16), normal(3, 50, dtype=BF16)], lambda t: (t[0], 0.3, seed, 5, t[1]), 1


def passed(leaves, arguments, count, call):
    leaves = [t.detach().requires_grad_() for t in leaves]
    out = call(*arguments(leaves))
    out = out if isinstance(out, tuple) else (out,)
    grads = torch.autograd.grad(out[:count], leaves, [torch.full_like(o, 0.5) for o in out[:count]])
    return [t.detach() for t in out] + list(grads)


def equal(a, b):
    return len(a) == len(b) and all(x.dtype == y.dtype and torch.equal(x, y) for x, y in zip(a, b))


def test_same_bits_as_the_registered_ops(monkeypatch):
    for op, leaves, arguments, count in cases():
        taken = []
        load = op._sihc_load
        monkeypatch.setattr(op, "_sihc_entry", None)
        monkeypatch.setattr(op, "_sihc_load", lambda: (lambda e: lambda *a: taken.append(e(*a)) or taken[-1])(load()))
        native = passed(leaves, arguments, count, op)
        assert taken and taken[0] is not NotImplemented, op
        assert equal(native, passed(leaves, arguments, count, lambda *a: CustomOpDef.__call__(op, *a))), op
        with torch.no_grad():
            again = op(*arguments(leaves))
        again = list(again) if isinstance(again, tuple) else [again]
        assert equal(again, native[:len(again)])
        monkeypatch.undo()


def test_the_result_alone_is_the_same():
    for op, leaves, arguments, _ in cases():
        if op is body._linear_act:
            with torch.no_grad():
                want = op(*arguments(leaves))[0]
                got = body._linear_act_result(*arguments(leaves))
                slow = CustomOpDef.__call__(body._linear_act_result, *arguments(leaves))
            assert torch.equal(got, want) and torch.equal(slow, want)


def test_only_the_gradients_that_are_asked_for():
    for op, leaves, arguments, count in cases():
        whole = passed(leaves, arguments, count, op)[-len(leaves):]
        for i in range(len(leaves)):
            for call in (op, lambda *a: CustomOpDef.__call__(op, *a)):
                some = [t.detach().requires_grad_(j == i) for j, t in enumerate(leaves)]
                out = call(*arguments(some))
                out = (out if isinstance(out, tuple) else (out,))[:count]
                (got,) = torch.autograd.grad(out, some[i], [torch.full_like(o, 0.5) for o in out])
                assert torch.equal(got, whole[i]), (op, i)


def test_modes_hooks_and_bad_arguments_reach_the_registered_ops():
    seen = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    for op, leaves, arguments, count in cases():
        seen.clear()
        with Watch():
            op(*arguments(leaves))
        assert any(op._qualname.replace("::", ".") in name for name in seen), (op, seen)
        with pytest.raises((ValueError, RuntimeError)):
            op(*arguments([t.double() for t in leaves]))

        def shrink(t):  # an unpack hook that gives back something else: refused, never launched
            return t[..., :0] if t.numel() > 1 else t.int()

        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, shrink):
            with pytest.raises((ValueError, RuntimeError)):
                passed(leaves, arguments, count, op)


def test_entries_are_the_modules_own():
    for name in ("linear_act", "linear_act_result", "qk_norm_rotary", "axis_rotary", "dropout"):
        assert _native.module().entry(name, f"sihc::{name}") is not None


def test_second_use_of_an_input_and_double_gradients():
    x = normal(4, 16, dtype=BF16).requires_grad_()
    w = normal(16, 16, dtype=BF16)
    y = body.linear_act(x, w, residual=x)  # one input twice
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    (want,) = torch.autograd.grad(body.linear_act(x, w), x, torch.ones_like(y))
    assert torch.equal(dx, want + 1)
    y = body.linear_act(x, w, None, "silu")
    (dx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises((RuntimeError, NotImplementedError)):  # the gradient's own gradient has no rule
        torch.autograd.grad(dx.sum(), x)


def test_empty_batches():
    for dtype in (BF16, torch.float32):
        x, w, b = (t.requires_grad_() for t in (torch.empty(0, 5, 8, device="cuda", dtype=dtype), normal(6, 8, dtype=dtype),
                                                normal(6, dtype=dtype)))
        gate = torch.empty(0, 3, device="cuda", dtype=dtype).requires_grad_()
        y = body.linear_act(x, w, b, "swiglu", gate)
        assert y.shape == (0, 5, 3)
        dx, dw, db, dg = torch.autograd.grad(y, (x, w, b, gate), torch.ones_like(y))
        assert dx.shape == x.shape and dg.shape == gate.shape and not dw.any() and not db.any()
        x = torch.empty(2, 0, 8, device="cuda", dtype=dtype)  # images without rows: a gate without terms
        gate = normal(2, 6, dtype=dtype).requires_grad_()
        (dg,) = torch.autograd.grad(body.linear_act(x, w, b, "none", gate).sum(), gate)
        assert dg.shape == gate.shape and not dg.any()
        q = torch.empty(2, 0, 4, 8, device="cuda", dtype=dtype).requires_grad_()
        wq = normal(8, dtype=dtype).requires_grad_()
        at = torch.empty(0, 1, device="cuda", dtype=torch.int32)
        out = body.qk_norm_rotary(q, q[:, :, :2], wq, wq, at, (8,))
        assert [t.shape[2] for t in out] == [4, 2]
        assert not torch.autograd.grad(out[0].sum() + out[1].sum(), wq)[0].any()
        assert body.axis_rotary(q, at, (8,)).shape == q.shape
        assert body.dropout(x, 0.5, torch.tensor([1], device="cuda")).shape == x.shape


def steps():
    """A training pass through each operator, on tensors that keep their places."""
    for op, leaves, arguments, count in cases():
        leaves = [t.detach().clone().requires_grad_() for t in leaves]

        def step(leaves=leaves, op=op, arguments=arguments, count=count):
            out = op(*arguments(leaves))
            out = (out if isinstance(out, tuple) else (out,))[:count]
            return [o.detach() for o in out] + list(torch.autograd.grad(out, leaves, [torch.ones_like(o) for o in out]))

        yield leaves, step


def test_captured_graphs_replay_the_eager_results():
    for leaves, step in steps():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = step()
        for turn in range(4):
            with torch.no_grad():
                for t in leaves:
                    t.add_(0.25 * turn)
            want = [t.clone() for t in step()]  # eager work between the replays
            graph.replay()
            torch.cuda.synchronize()
            assert equal(kept, want)


def test_a_replayed_mask_follows_its_seed():
    x, seed = torch.ones(1000, device="cuda"), torch.tensor([1], device="cuda")
    body.dropout(x, 0.5, seed)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = body.dropout(x, 0.5, seed, 9)
    for value in (1, 5, -1, 5):
        seed.fill_(value)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.cpu() != 0, R.mask(1000, 0.5, value, 9))


def test_a_seed_that_changed_before_the_backward_is_noticed():
    x, seed = torch.ones(64, device="cuda", requires_grad=True), torch.tensor([1], device="cuda")
    y = body.dropout(x, 0.5, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_two_streams_at_once():
    pairs = [(step(), step) for _, step in steps()]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i, (_, step) in enumerate(pairs * 3):
        with torch.cuda.stream(streams[i % 2]):
            got.append(step())
    torch.cuda.synchronize()
    for i, values in enumerate(got):
        assert equal(values, pairs[i % len(pairs)][0])


PUBLIC = {
    "linear": lambda t: body.linear_act(t[0], t[1], t[2], "silu", None, t[0]),
    "heads": lambda t: torch.cat(body.qk_norm_rotary(t[0].view(3, 8, 4, 4), t[0].view(3, 8, 4, 4), t[3], t[3], t[4], (4,)), 2),
    "rotary": lambda t: body.axis_rotary(t[0].view(3, 8, 4, 4), t[4], (4,)),
    "dropout": lambda t: body.dropout(t[0], 0.4, t[5], 2, t[0]),
}


def public(name):
    call = PUBLIC[name]
    fixed = [torch.arange(8, dtype=torch.int32, device="cuda").reshape(8, 1), torch.tensor([3], device="cuda")]
    leaves = [normal(3, 8, 16), normal(16, 16), normal(16), normal(4)]
    if name == "rotary" or name == "dropout":
        leaves = leaves[:1]
        return (lambda *t: call([t[0], None, None, None, *fixed])), leaves
    if name == "heads":
        return (lambda x, w: call([x, None, None, w, *fixed])), [leaves[0], leaves[3]]
    return (lambda x, w, b: call([x, w, b])), leaves[:3]


def grads_of(call, values):
    leaves = [v.clone().requires_grad_() for v in values]
    out = call(*leaves)
    return [out.detach(), *torch.autograd.grad(out, leaves, torch.ones_like(out))]


@pytest.mark.parametrize("name", PUBLIC)
def test_compiled(name):
    call, values = public(name)
    want = grads_of(call, values)
    torch._dynamo.reset()
    assert equal(grads_of(torch.compile(call, fullgraph=True, backend="aot_eager"), values), want)


@pytest.mark.parametrize("name", PUBLIC)
def test_compiled_autograd(name):
    call, values = public(name)
    want = grads_of(call, values)
    leaves = [v.clone().requires_grad_() for v in values]
    out = call(*leaves)
    torch._dynamo.reset()
    with torch._dynamo.compiled_autograd._enable(torch.compile(backend="eager")):
        torch.autograd.backward(out, torch.ones_like(out))
    assert equal([out.detach(), *(t.grad for t in leaves)], want)


@pytest.mark.parametrize("reentrant", [False, True])
@pytest.mark.parametrize("name", PUBLIC)
def test_checkpointing(name, reentrant):
    call, values = public(name)
    want = grads_of(call, values)
    leaves = [v.clone().requires_grad_() for v in values]
    out = torch.utils.checkpoint.checkpoint(call, *leaves, use_reentrant=reentrant)
    torch.autograd.backward(out, torch.ones_like(out))
    assert equal([out.detach(), *(t.grad for t in leaves)], want)


@pytest.mark.parametrize("name", PUBLIC)
def test_gradients_against_differences(name):
    """Central differences in fp32 along one direction: of a smooth function of values of size 1 over h = 2^-6,
    off by h^2 / 6 of the third derivative (below 1 here, times the direction's entries) and by the results'
    rounding, 2^-20 of the sum's terms, over 2 h."""
    call, values = public(name)
    grads = grads_of(call, values)[1:]
    h = 2.0 ** -6
    for i, v in enumerate(values):
        direction = normal(*v.shape)
        ends = []
        with torch.no_grad():
            for sign in (1, -1):
                moved = list(values)
                moved[i] = v + sign * h * direction
                ends.append(call(*moved).double())
        slope = float((ends[0] - ends[1]).sum()) / (2 * h)
        want = float((grads[i].double() * direction.double()).sum())
        terms = float(ends[0].abs().sum())
        third = h * h / 6 * 40 * float(direction.abs().pow(3).sum()) * max(1.0, float(values[-1].abs().max()))
        assert abs(slope - want) <= third + terms * 2.0 ** -20 / h, (name, i, slope, want)


EXTREMES = [2.0 ** 70, 2.0 ** -60, 2.0 ** 126]


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("size", EXTREMES)
def test_norms_of_values_whose_squares_leave_fp32(size, dtype):
    x = (normal(2, 3, 5, 40) * 0.25).to(dtype)
    x[:, :, 1::2] *= size
    w = normal(40)
    at = torch.arange(3, dtype=torch.int32, device="cuda").reshape(3, 1)
    eps = 0.0
    grad = normal(2, 3, 5, 40, dtype=dtype)
    lx, lw = x.clone().requires_grad_(), w.clone().requires_grad_()
    out, _ = body.qk_norm_rotary(lx, lx.detach(), lw, w, at, (40,), 1e4, eps)
    dx, dw = torch.autograd.grad(out, (lx, lw), grad)
    want = R.heads(x, w, at, (40,), 1e4, eps, grad)
    R.check(out, *want[0], f"{size}")
    # (a gradient of size 1 / x below fp32's smallest normal value is a flush to zero, or is rounded there)
    R.check(dx, want[1][0], want[1][1] + 2.0 ** -125, f"gradient {size}")
    R.check(dw, *want[2], f"gradient of the weight {size}")


def test_a_row_that_is_not_finite_stays_alone():
    x, w = normal(70, 96, dtype=BF16), normal(200, 96, dtype=BF16)
    want = body.linear_act(x, w, None, "silu")
    bad = x.clone()
    bad[7, 3], bad[33, 5] = float("nan"), float("inf")
    got = body.linear_act(bad, w, None, "silu")
    keep = torch.ones(70, dtype=torch.bool)
    keep[[7, 33]] = False
    assert torch.equal(got[keep], want[keep]) and got[7].isnan().all() and not got[33].isfinite().all()
    h = normal(2, 4, 6, 40, dtype=BF16)
    at, one = torch.zeros(4, 1, dtype=torch.int32, device="cuda"), torch.ones(40, device="cuda")
    want, _ = body.qk_norm_rotary(h, h, one, one, at, (40,))
    bad = h.clone()
    bad[1, 2, 3, 4] = float("nan")
    got, _ = body.qk_norm_rotary(bad, bad, one, one, at, (40,))
    keep = torch.ones(2, 4, 6, dtype=torch.bool)
    keep[1, 2, 3] = False
    assert torch.equal(got[keep], want[keep]) and got[1, 2, 3].isnan().all()


def test_offsets_past_32_bits():
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    rows, inner, outer = 2 ** 26 + 77, 40, 40  # 2.7e9 elements each way
    x = torch.zeros(rows, inner, device="cuda", dtype=BF16)
    w, b = normal(outer, inner, dtype=BF16), normal(outer, dtype=BF16)
    x[-300:] = normal(300, inner, dtype=BF16)
    y = body.linear_act(x, w, b)
    want = body.linear_act(x[-300:].contiguous(), w, b)
    assert torch.equal(y[-300:], want) and torch.equal(y[0], b)
    del y
    q = x[: 2 ** 26].view(1, 2 ** 22, 16, 40)
    at = torch.zeros(2 ** 22, 1, device="cuda", dtype=torch.int32)
    q[:, -3:] = normal(1, 3, 16, 40, dtype=BF16)
    at[-3:] = 1000
    y = body.axis_rotary(q, at, (40,))
    assert torch.equal(y[:, -3:], body.axis_rotary(q[:, -3:].contiguous(), at[-3:].contiguous(), (40,)))


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_tensors_that_start_anywhere(dtype):
    """Packed views one element into their storage: no access is aligned to more than an element."""
    def moved(t):
        whole = torch.empty(t.numel() + 1, device="cuda", dtype=t.dtype)
        whole[1:] = t.reshape(-1)
        return whole[1:].view(t.shape)

    for size, act in (((2, 40, 64, 72), "swiglu"), ((3, 1, 200, 40), "silu"), ((4, 300, 512, 600), "none")):
        batch, tokens, inner, outer = size
        wide = 2 * outer if act == "swiglu" else outer
        t = [normal(batch, tokens, inner, dtype=dtype), normal(wide, inner, dtype=dtype) * inner ** -0.5,
             normal(wide, dtype=dtype), normal(batch, outer, dtype=dtype), normal(batch, tokens, outer, dtype=dtype)]
        results = []
        for values in (t, [moved(v) for v in t]):
            leaves = [v.detach().requires_grad_() for v in values]
            y = body.linear_act(*leaves[:3], act, *leaves[3:])
            results.append([y.detach(), *torch.autograd.grad(y, leaves, torch.ones_like(y))])
        assert equal(*results)
    x, seed = normal(5, 1003, dtype=dtype), torch.tensor([4], device="cuda")
    assert torch.equal(body.dropout(moved(x), 0.3, seed, 1, moved(x)), body.dropout(x, 0.3, seed, 1, x))


@pytest.mark.parametrize("name", PUBLIC)
def test_vmap(name):
    call, values = public(name)
    with torch.no_grad():
        want = [call(factor * values[0], *values[1:]) for factor in (1, 2)]
        got = torch.func.vmap(lambda t: call(t, *values[1:]))(torch.stack([values[0], 2 * values[0]]))
    assert equal(list(got), want)


@pytest.mark.parametrize("name", PUBLIC)
def test_subclasses_and_modes_in_the_backward(name):
    call, values = public(name)
    want, seen = grads_of(call, values), []

    class Log(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    leaves = [v.clone().requires_grad_() for v in values]
    out = call(*leaves)
    with Log():
        got = torch.autograd.grad(out, leaves, torch.ones_like(out))
    assert any("sihc" in s for s in seen) and equal(list(got), want[1:])

    class Sub(torch.Tensor):
        pass

    with torch.no_grad():
        out = call(values[0].as_subclass(Sub), *values[1:])
        assert isinstance(out, Sub) and torch.equal(out.as_subclass(torch.Tensor), want[0])
        assert torch.equal(call(torch.nn.Parameter(values[0]), *values[1:]), want[0])


def test_a_large_product_is_captured_at_its_first_call():
    """Kernels with more than 64 KB of LDS have it allowed at their first launch, which a capture may hold."""
    x, w = normal(4096, 520, dtype=BF16), normal(2064, 520, dtype=BF16) * 0.05
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = body.linear_act(x, w, None, "swiglu")
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, body.linear_act(x, w, None, "swiglu"))
