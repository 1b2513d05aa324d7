"""The sequence operators as they are used: together in a mixing block, in CUDA graphs, on large layouts, with small and
large values, at the sizes where one kernel takes over from another."""
import os
import sys

import pytest

import sequence_reference as R
from test_gpu_sequence import Case, norm_ir, normal, ptr, stream

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_mixing_block_example(V):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import sequence_mixing
    finally:
        sys.path.pop(0)
    tokens_off, state_off, losses = sequence_mixing.run(length=300, heads=4, say=lambda *_: None)
    # two runs of bf16 arithmetic, each with three roundings to 2^-8 after another (attention, projection, sum)
    assert tokens_off <= 2.0 ** -8
    # the keys and values of both come from matrix products of other shapes: a bf16 rounding may fall the other way
    assert state_off <= 2.0 ** -8
    assert all(b < a for a, b in zip(losses, losses[1:]))


@pytest.mark.parametrize("dtype", ["F32", "BF16"])
@pytest.mark.parametrize("rows,features", [(3000, 1024), (1300, 2048), (2400, 4096), (1201, 8192), (700, 16384), (9000, 64), (5000, 520),
                                           (1500, 3001)])
def test_layer_norm_many_rows(V, ctx, rows, features, dtype):
    """Rows enough for several to a group, at every width of group."""
    t = R.TYPES[dtype]
    x, dy = normal(1, rows, features, dtype=t, std=1.5, mean=0.5), normal(2, rows, features, dtype=t)
    w, b = normal(3, features, dtype=t, std=0.3, mean=1.0), normal(4, features, dtype=t)
    ir = norm_ir(V, ctx, rows, features, dtype, dtype)
    y, mean, rstd = torch.empty_like(x), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    ctx.execute_layer_norm(ir, ptr(x), ptr(y), ptr(w), ptr(b), ptr(mean), ptr(rstd), stream=stream())
    tol = R.norm_tolerance(dtype, features)
    assert R.rel(y, R.layer_norm(x, w, b, 1e-5)[0]) <= tol
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    ws = torch.empty(ir.backward_workspace_bytes, dtype=torch.uint8, device="cuda")
    args = (ptr(x), ptr(mean), ptr(rstd), ptr(dy), ptr(w), ptr(dx), ptr(dw), ptr(db), ptr(ws))
    ctx.execute_layer_norm_backward(ir, *args, stream=stream())
    gx, gw, gb = R.layer_norm_grad(x, w, mean, rstd, dy)
    terms = torch.linalg.vector_norm(dy.double() * w.double() * rstd.double()[:, None])
    assert float(torch.linalg.vector_norm(dx.double() - gx)) <= tol * float(terms)
    ptol = R.norm_tolerance(dtype, rows)
    assert R.rel(dw, gw) <= 2 * ptol and R.rel(db, gb) <= 2 * ptol
    first = [v.clone() for v in (dx, dw, db)]
    ctx.execute_layer_norm_backward(ir, *args, stream=stream())
    assert all(torch.equal(a, b) for a, b in zip(first, (dx, dw, db)))


@pytest.mark.parametrize("dtype", ["F16", "BF16", "F32"])
@pytest.mark.parametrize("small", [1e-4, 3e-6])
def test_attention_small_values(V, ctx, dtype, small):
    """Gradients of a late training step: values near and below the least normal f16 keep the accuracy of their type."""
    c = Case(V, ctx, [300], 2, 2, 64, 64, dtype)
    for t in (c.k, c.do):
        t.mul_(small)
    c.s0.mul_(small)
    c.ds.mul_(small * small if dtype != "F16" else small)
    if dtype == "F16":
        # results below 2^-24 are not representable: scale the partner up
        c.q.mul_(100.0)
        c.v.mul_(100.0)
    o, s = c.forward()
    want = [R.attention(c.q[b], c.k[b], c.v[b], c.g, c.scale, c.s0[b]) for b in range(1)]
    f32 = R.attention_tolerance("F32", 300)
    assert R.rel(s[0], want[0][1]) <= f32
    # half a unit of the type, or of its subnormals where the values are that small
    floor = {"F16": 2.0 ** -25, "BF16": 0.0, "F32": 0.0}[dtype]
    size = float(torch.linalg.vector_norm(want[0][0])) / want[0][0].numel() ** 0.5
    assert R.rel(o[0], want[0][0]) <= R.attention_tolerance(dtype, 300) + 2 * floor / size
    grads = c.backward()
    exact = R.attention_grad(c.q[0], c.k[0], c.v[0], c.g, c.scale, c.do[0], c.s0[0], c.ds[0])
    assert R.rel(grads[3][0], exact[3]) <= f32
    for x, w in zip(grads[:3], exact):
        size = float(torch.linalg.vector_norm(w)) / w.numel() ** 0.5
        assert R.rel(x[0], w) <= R.attention_tolerance(dtype, 300) + 2 * floor / size


@pytest.mark.parametrize("dtype,length", [("BF16", 260), ("F32", 130), ("BF16", 1)])
def test_attention_offsets_past_32_bits(V, ctx, dtype, length):
    """Rows so far apart that element offsets pass 2^31 (and byte offsets 2^32)."""
    stride = (1 << 31) // 128 + 8  # elements between tokens; from one token: between heads
    t = R.TYPES[dtype]
    if length > 1:
        base = torch.empty(stride * (length - 1) + 2 * 64, dtype=t, device="cuda")
        view = base.as_strided((1, length, 2, 64), (0, stride, 64, 1))
        strides = (0, stride, 64)
    else:
        stride = (1 << 31) + 8
        base = torch.empty(stride + 64, dtype=t, device="cuda")
        view = base.as_strided((1, 1, 2, 64), (0, 64, stride, 1))
        strides = (0, 64, stride)
    c = Case(V, ctx, [length], 2, 2, 64, 64, dtype)
    view.copy_(c.v)
    cfg = c.cfg.with_value_strides(*strides)
    c.build(cfg)
    o, s = torch.empty_like(c.do), torch.empty_like(c.s0)
    ctx.execute_linear_attention(c.ir, ptr(c.q), ptr(c.k), base.data_ptr(), ptr(c.g), ptr(o), ptr(c.s0), ptr(s), stream=stream())
    c.compare_forward(o, s)
    # and results written that far
    c.build(c.cfg.with_output_strides(*strides))
    ctx.execute_linear_attention(c.ir, ptr(c.q), ptr(c.k), ptr(c.v), ptr(c.g), base.data_ptr(), ptr(c.s0), ptr(s), stream=stream())
    c.compare_forward(view.clone(), s)
    del base, view


def test_layer_norm_rows_past_32_bits(V, ctx):
    rows, features, stride = 40, 256, (1 << 31) // 32 + 8
    base = torch.empty(stride * (rows - 1) + features, dtype=torch.bfloat16, device="cuda")
    view = base.as_strided((rows, features), (stride, 1))
    x = normal(1, rows, features, dtype=torch.bfloat16)
    view.copy_(x)
    ir = norm_ir(V, ctx, rows, features, "BF16", "BF16", xs=stride)
    y = torch.empty_like(x)
    ctx.execute_layer_norm(ir, base.data_ptr(), ptr(y), stream=stream())
    assert R.rel(y, R.layer_norm(x, None, None, 1e-5)[0]) <= R.norm_tolerance("BF16", features)


@pytest.mark.parametrize("dtype", ["BF16", "F16", "F32"])
def test_attention_segments(V, ctx, dtype):
    """Few heads and a long sequence: segments side by side, with and without states, forwards and backwards."""
    c = Case(V, ctx, [4000], 2, 1, 64, 64, dtype)
    assert c.build().workspace_bytes > 0
    c.check_forward()
    c.check_forward(state=False)
    c.check_backward()
    c = Case(V, ctx, [2500, 1, 0, 900], 2, 2, 128, 64, dtype, packed=True)
    assert c.build().workspace_bytes > 0
    c.check_forward()
    c.check_backward()
    # a state in place
    whole = c.s0.clone()
    o = torch.empty_like(c.do)
    ctx.execute_linear_attention(c.build(), ptr(c.q), ptr(c.k), ptr(c.v), ptr(c.g), ptr(o), ptr(whole), ptr(whole),
                                 ptr(c.offsets), stream=stream())
    o2, s2 = c.forward()
    assert torch.equal(o, o2) and torch.equal(whole, s2)


def test_operators_in_a_graph(V, ctx):
    """Calls with a workspace of their own can be captured and replayed on new data."""
    c = Case(V, ctx, [600] * 2, 4, 2, 64, 64, "BF16")
    ir = c.build()
    rows = 2 * 600
    nir = norm_ir(V, ctx, rows, 256, "BF16", "BF16")
    o, s, y = torch.empty_like(c.do), torch.empty_like(c.s0), torch.empty_like(c.do)
    grads = [torch.empty_like(x) for x in (c.q, c.k, c.v)]
    ws = torch.empty(max(ir.workspace_bytes, ir.backward_workspace_bytes, 16), dtype=torch.uint8, device="cuda")

    def calls():
        ctx.execute_linear_attention(ir, ptr(c.q), ptr(c.k), ptr(c.v), ptr(c.g), ptr(o), ptr(c.s0), ptr(s),
                                     workspace_ptr=ptr(ws), stream=stream())
        ctx.execute_layer_norm(nir, ptr(o), ptr(y), stream=stream())
        ctx.execute_linear_attention_backward(ir, ptr(c.q), ptr(c.k), ptr(c.v), ptr(c.g), ptr(c.do), *(ptr(x) for x in grads),
                                              workspace_ptr=ptr(ws), stream=stream())

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            calls()
    torch.cuda.synchronize()
    for k in range(2):
        c.q.copy_(normal(50 + k, *c.q.shape, dtype=c.t))
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in (o, s, y, *grads)]
        with torch.cuda.stream(side):
            calls()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (o, s, y, *grads)))


def test_operators_follow_one_another(V, ctx):
    """A chain of calls in which each reads what the one before wrote, many times over, with torch's kernels between."""
    rows, width = 512, 4 * 64
    c = Case(V, ctx, [256] * 2, 4, 4, 64, 64, "BF16")
    ir, nir = c.build(), norm_ir(V, ctx, rows, width, "BF16", "BF16")

    def chain(wait):
        x = c.q.clone()
        for _ in range(20):
            y, o = torch.empty_like(x), torch.empty_like(x)
            ctx.execute_layer_norm(nir, ptr(x), ptr(y), stream=stream())
            if wait:
                torch.cuda.synchronize()
            ctx.execute_linear_attention(ir, ptr(y), ptr(y), ptr(y), ptr(c.g), ptr(o), stream=stream())
            if wait:
                torch.cuda.synchronize()
            ctx.execute_layer_norm(nir, ptr(o), ptr(x), stream=stream())
            x = x * 0.5 + y * 0.5
            if wait:
                torch.cuda.synchronize()
        return x

    assert torch.equal(chain(False), chain(True))
