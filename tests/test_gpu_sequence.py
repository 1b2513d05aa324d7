"""Layer normalisation and linear attention on the GPU against their definitions in 64 bits."""
import itertools
import math

import numpy as np
import pytest

import sequence_reference as R

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def stream():
    return torch.cuda.current_stream().cuda_stream or 1


def normal(seed, *shape, dtype=torch.float32, std=1.0, mean=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dtype)


def ptr(t):
    return 0 if t is None else t.data_ptr()


# ---- layer normalisation ----------------------------------------------------------------

NORM_SIZES = [(1, 1), (3, 1), (5, 2), (7, 31), (64, 32), (9, 33), (33, 64), (130, 96), (17, 255), (6, 256), (11, 1000),
              (300, 1023), (257, 1024), (19, 2047), (70, 2048), (9, 4096), (5, 4100), (3, 8192), (700, 8200), (4, 16384), (2, 16411),
              (3, 40000)]


def norm_ir(V, ctx, rows, features, dtype, param, **strides):
    cfg = V.LayerNormConfig(rows, features).with_element_type(V.ElementType[dtype])
    cfg = cfg.with_parameter_type(V.ElementType[param])
    if strides.get("xs"):
        cfg = cfg.with_input_row_stride(strides["xs"])
    if strides.get("ys"):
        cfg = cfg.with_output_row_stride(strides["ys"])
    return V.LayerNormIr.build(cfg, ctx.device_profile())


def strided(t, stride, shift=0):
    """The rows of t at a row stride, `shift` elements behind an aligned address; the gaps hold NaN."""
    rows, features = t.shape
    base = torch.full((rows * stride + shift,), float("nan"), dtype=t.dtype, device="cuda")
    view = base[shift:shift + rows * stride].view(rows, stride)[:, :features]
    view.copy_(t)
    return view


@pytest.mark.parametrize("dtype,param", [("F32", "F32"), ("F16", "F16"), ("BF16", "BF16"), ("BF16", "F32")])
@pytest.mark.parametrize("rows,features", NORM_SIZES)
def test_layer_norm(V, ctx, rows, features, dtype, param):
    t, pt = R.TYPES[dtype], R.TYPES[param]
    x = normal(1, rows, features, dtype=t, std=1.5, mean=0.5)
    w, b = normal(2, features, dtype=pt, std=0.3, mean=1.0), normal(3, features, dtype=pt, std=0.2)
    dy = normal(4, rows, features, dtype=t)
    ir = norm_ir(V, ctx, rows, features, dtype, param)
    y, mean, rstd = torch.empty_like(x), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    ctx.execute_layer_norm(ir, ptr(x), ptr(y), ptr(w), ptr(b), ptr(mean), ptr(rstd), stream=stream())
    want, m, r = R.layer_norm(x, w, b, 1e-5)
    tol = R.norm_tolerance(dtype, features)
    f32 = R.norm_tolerance("F32", features)
    assert R.rel(y, want) <= tol
    assert float((mean.double() - m).abs().max()) <= f32 * (float(x.double().abs().max()) + 1)
    # the variance's relative error, against a variance that may be small beside the values
    assert float(((rstd.double() - r) / r).abs().max()) <= f32 * 4
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    ctx.execute_layer_norm_backward(ir, ptr(x), ptr(mean), ptr(rstd), ptr(dy), ptr(w), ptr(dx), ptr(dw), ptr(db),
                                    stream=stream())
    gx, gw, gb = R.layer_norm_grad(x, w, mean, rstd, dy)
    # dx is a difference: its rounding error is that of its terms
    terms = torch.linalg.vector_norm(dy.double() * w.double() * rstd.double()[:, None])
    assert float(torch.linalg.vector_norm(dx.double() - gx)) <= tol * float(terms)
    ptol = R.norm_tolerance(param, rows)
    for got, exact, scale in ((dw, gw, None), (db, gb, None)):
        size = torch.sqrt((dy.double() ** 2).sum(0)) * math.sqrt(max(1.0, 3.0))
        assert float(torch.linalg.vector_norm(got.double() - exact)) <= ptol * float(
            torch.linalg.vector_norm(exact)) + R.norm_tolerance("F32", rows) * float(torch.linalg.vector_norm(size))


@pytest.mark.parametrize("dtype", ["F32", "BF16"])
@pytest.mark.parametrize("features,xs,ys,shift", [(64, 72, 80, 0), (96, 97, 96, 0), (1024, 1032, 1024, 3), (4096, 4096, 4104, 1),
                                                  (1000, 1001, 1003, 5), (20000, 20001, 20000, 0)])
def test_layer_norm_strides_and_addresses(V, ctx, dtype, features, xs, ys, shift):
    """Row strides and odd addresses give the bits that dense rows give."""
    t, rows = R.TYPES[dtype], 13
    x, dy = normal(5, rows, features, dtype=t), normal(6, rows, features, dtype=t)
    w, b = normal(7, features, dtype=t), normal(8, features, dtype=t)
    want, m, r = R.layer_norm(x, w, b, 1e-5)
    ir = norm_ir(V, ctx, rows, features, dtype, dtype, xs=xs, ys=ys)
    xv, yv = strided(x, xs, shift), strided(torch.zeros_like(x), ys, shift)
    wv, bv = strided(w[None], features + 1, shift)[0], strided(b[None], features + 1, shift)[0]
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    whole = yv._base.clone()
    ctx.execute_layer_norm(ir, ptr(xv), ptr(yv), ptr(wv), ptr(bv), ptr(mean), ptr(rstd), stream=stream())
    tol = R.norm_tolerance(dtype, features)
    assert R.rel(yv, want) <= tol
    gaps = torch.isnan(whole)
    assert bool(torch.isnan(yv._base[gaps]).all())
    dyv, dxv = strided(dy, ys, shift), strided(torch.zeros_like(x), xs, shift)
    dw, db = torch.empty_like(w), torch.empty_like(b)
    whole = dxv._base.clone()
    ctx.execute_layer_norm_backward(ir, ptr(xv), ptr(mean), ptr(rstd), ptr(dyv), ptr(wv), ptr(dxv), ptr(dw), ptr(db),
                                    stream=stream())
    gx, gw, gb = R.layer_norm_grad(x, w, mean, rstd, dy)
    terms = torch.linalg.vector_norm(dy.double() * w.double() * rstd.double()[:, None])
    assert float(torch.linalg.vector_norm(dxv.double() - gx)) <= tol * float(terms)
    assert bool(torch.isnan(dxv._base[torch.isnan(whole)]).all())
    assert R.rel(dw, gw) <= R.norm_tolerance(dtype, rows) * 4
    assert R.rel(db, gb) <= R.norm_tolerance(dtype, rows) * 4


@pytest.mark.parametrize("dtype", ["F32", "F16", "BF16"])
@pytest.mark.parametrize("features,gap,shift", [(2, 2, 2), (66, 0, 0), (130, 2, 2), (257, 0, 0), (258, 2, 6), (546, 0, 2), (1025, 0, 0),
                                                (1026, 4, 2), (1230, 0, 0), (2050, 2, 2), (4097, 1, 0), (4098, 2, 2), (8190, 0, 2),
                                                (8194, 2, 2), (1537, 0, 0), (2561, 0, 0), (5119, 0, 0), (5121, 1, 0), (6145, 0, 0),
                                                (10242, 2, 2), (12290, 0, 2), (16386, 0, 2)])
def test_layer_norm_pairs(V, ctx, dtype, features, gap, shift):
    """Rows that pairs of elements divide, at addresses that hold pairs but not sixteen bytes, and widths beside those."""
    test_layer_norm_strides_and_addresses(V, ctx, dtype, features, features + gap, features + 2 * gap, shift)


@pytest.mark.parametrize("features", [64, 1023, 4096, 20000])
def test_layer_norm_optional_tensors_and_in_place(V, ctx, features):
    rows = 37
    x, dy = normal(1, rows, features), normal(2, rows, features)
    w = normal(3, features, mean=1.0)
    ir = norm_ir(V, ctx, rows, features, "F32", "F32")
    tol = R.norm_tolerance("F32", features)
    y = torch.empty_like(x)
    ctx.execute_layer_norm(ir, ptr(x), ptr(y), stream=stream())
    assert R.rel(y, R.layer_norm(x, None, None, 1e-5)[0]) <= tol
    z, mean, rstd = x.clone(), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    ctx.execute_layer_norm(ir, ptr(z), ptr(z), ptr(w), 0, ptr(mean), ptr(rstd), stream=stream())
    assert R.rel(z, R.layer_norm(x, w, None, 1e-5)[0]) <= tol
    # dx alone, weight gradients alone, and dx in dy's place give the same as all together
    full = [torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)]
    call = lambda g, dx, dw, db: ctx.execute_layer_norm_backward(  # noqa: E731
        ir, ptr(x), ptr(mean), ptr(rstd), ptr(g), ptr(w), ptr(dx), ptr(dw), ptr(db), stream=stream())
    call(dy, *full)
    alone = torch.empty_like(x)
    call(dy, alone, None, None)
    assert torch.equal(alone, full[0])
    only = [torch.empty_like(w), torch.empty_like(w)]
    call(dy, None, *only)
    assert R.rel(only[0], full[1]) <= tol and R.rel(only[1], full[2]) <= tol
    one = torch.empty_like(w)
    call(dy, None, one, None)
    assert torch.equal(one, only[0])
    place = dy.clone()
    again = [torch.empty_like(w), torch.empty_like(w)]
    call(place, place, *again)
    assert torch.equal(place, full[0]) and torch.equal(again[0], full[1]) and torch.equal(again[1], full[2])


def test_layer_norm_rows_do_not_touch_one_another(V, ctx):
    """A row of NaN or infinity stays its own; a constant row normalises to the bias."""
    rows, features = 9, 512
    x = normal(1, rows, features)
    x[2], x[5, 7], x[7] = float("nan"), float("inf"), 4.25
    b = normal(2, features)
    ir = norm_ir(V, ctx, rows, features, "F32", "F32")
    y = torch.empty_like(x)
    ctx.execute_layer_norm(ir, ptr(x), ptr(y), 0, ptr(b), stream=stream())
    fine = [0, 1, 3, 4, 6, 8]
    assert R.rel(y[fine], R.layer_norm(x[fine], None, b, 1e-5)[0]) <= R.norm_tolerance("F32", features)
    assert bool(torch.isnan(y[2]).all()) and bool(torch.isnan(y[5]).all())
    assert torch.equal(y[7], b)


def test_layer_norm_large_mean(V, ctx):
    """Values far from zero: the variance comes from centred values, not from a difference of squares."""
    rows, features = 40, 4096
    x = normal(1, rows, features) + 3000.0
    ir = norm_ir(V, ctx, rows, features, "F32", "F32")
    y = torch.empty_like(x)
    ctx.execute_layer_norm(ir, ptr(x), ptr(y), stream=stream())
    # the mean's own rounding (2^-24 of 3000 at most a few times) is an error of each value
    assert R.rel(y, R.layer_norm(x, None, None, 1e-5)[0]) <= 2.0 ** -24 * 3000 * 8


def test_layer_norm_gradient_against_differences(V, ctx):
    rows, features, eps = 6, 48, 1e-3
    x, w, b = normal(1, rows, features), normal(2, features, mean=1.0), normal(3, features)
    dy = normal(4, rows, features)
    ir = norm_ir(V, ctx, rows, features, "F32", "F32")
    y, mean, rstd = torch.empty_like(x), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    ctx.execute_layer_norm(ir, ptr(x), ptr(y), ptr(w), ptr(b), ptr(mean), ptr(rstd), stream=stream())
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    ctx.execute_layer_norm_backward(ir, ptr(x), ptr(mean), ptr(rstd), ptr(dy), ptr(w), ptr(dx), ptr(dw), ptr(db),
                                    stream=stream())
    loss = lambda x, w, b: float((R.layer_norm(x, w, b, 1e-5)[0] * dy.double()).sum())  # noqa: E731
    at = [t.double() for t in (x, w, b)]
    for k, grad in enumerate((dx, dw, db)):
        d = normal(10 + k, *grad.shape).double()
        up, down = list(at), list(at)
        up[k], down[k] = at[k] + eps * d, at[k] - eps * d
        slope = (loss(*up) - loss(*down)) / (2 * eps)
        size = float(torch.linalg.vector_norm(grad.double()) * torch.linalg.vector_norm(d))
        assert abs(slope - float((grad.double() * d).sum())) <= 1e-5 * size  # eps^2 times third derivatives, and f32


# ---- linear attention -----------------------------------------------------------------

class Case:
    """Tensors of one linear attention call, packed or [batch, token, head, dim]."""

    def __init__(self, V, ctx, lengths, heads, kv_heads, dk, dv, dtype, packed=False, decay=None, seed=0, scale=None,
                 layout="dense"):
        self.V, self.ctx, self.lengths, self.heads, self.kv, self.dk, self.dv = V, ctx, lengths, heads, kv_heads, dk, dv
        self.dtype, self.packed, self.t = dtype, packed, R.TYPES[dtype]
        self.scale = dk ** -0.5 if scale is None else scale
        n, most = len(lengths), max(max(lengths), 1)
        lead = (sum(lengths),) if packed else (n, lengths[0])
        make = lambda s, h, d: self.place(normal(seed + s, *lead, h, d, dtype=self.t), layout)  # noqa: E731
        self.q, self.k, self.v = make(1, heads, dk), make(2, kv_heads, dk), make(3, kv_heads, dv)
        self.do = self.place(normal(seed + 4, *lead, heads, dv, dtype=self.t), layout)
        self.s0, self.ds = normal(seed + 5, n, heads, dk, dv, std=2.0), normal(seed + 6, n, heads, dk, dv)
        if decay is None:
            self.g = torch.log1p(-torch.exp2(-(1 + 7 * torch.arange(heads, device="cuda") / max(1, heads - 1)))).float()
        else:
            self.g = torch.tensor([decay[h % len(decay)] for h in range(heads)], device="cuda")
        cfg = V.LinearAttentionConfig(most, heads, dk, dv).with_batch_count(n).with_key_value_heads(kv_heads)
        cfg = cfg.with_element_type(V.ElementType[dtype]).with_scale(self.scale)
        self.offsets = None
        if packed:
            cfg = cfg.with_packed_tokens(sum(lengths))
            self.offsets = torch.tensor([0] + list(lengths), device="cuda").cumsum(0)
        if layout != "dense":
            cfg = cfg.with_query_strides(*self.strides(self.q)).with_key_strides(*self.strides(self.k))
            cfg = cfg.with_value_strides(*self.strides(self.v)).with_output_strides(*self.strides(self.do))
        self.cfg, self.layout = cfg, layout

    @staticmethod
    def place(x, layout):
        if layout == "dense":
            return x
        if layout == "heads":  # [batch, head, token, dim] in memory
            y = torch.full_like(x.transpose(-2, -3).contiguous(), float("nan")).transpose(-2, -3)
        else:  # rows inside wider rows, at an odd address
            wide = torch.full((*x.shape[:-2], x.shape[-2] + 1, x.shape[-1] + 3), float("nan"), dtype=x.dtype,
                              device="cuda")
            y = wide[..., 1:, 1:1 + x.shape[-1]]
        y.copy_(x)
        return y

    def strides(self, x):
        return (0 if self.packed else x.stride(0)), x.stride(-3), x.stride(-2)

    def empty(self, like):
        out = self.place(torch.zeros_like(like, memory_format=torch.contiguous_format), self.layout)
        out.fill_(float("nan"))
        return out

    def build(self, cfg=None):
        self.ir = self.V.LinearAttentionIr.build(cfg or self.cfg, self.ctx.device_profile())
        return self.ir

    def sequence(self, x, b):
        if not self.packed:
            return x[b]
        start = sum(self.lengths[:b])
        return x[start:start + self.lengths[b]]

    def forward(self, state=True, final=True):
        self.build()
        o = self.empty(self.do)
        s = torch.full_like(self.s0, float("nan")) if final else None
        self.ctx.execute_linear_attention(self.ir, ptr(self.q), ptr(self.k), ptr(self.v), ptr(self.g), ptr(o),
                                          ptr(self.s0 if state else None), ptr(s), ptr(self.offsets), stream=stream())
        return o, s

    def check_forward(self, state=True):
        o, s = self.forward(state)
        self.compare_forward(o, s, state)

    def compare_forward(self, o, s, state=True):
        want_o, want_s = self.empty(self.do).double(), torch.empty_like(self.s0, dtype=torch.float64)
        for b, n in enumerate(self.lengths):
            got = R.attention(*(self.sequence(x, b) for x in (self.q, self.k, self.v)), self.g, self.scale,
                              self.s0[b] if state else None)
            self.sequence(want_o, b).copy_(got[0])
            want_s[b] = got[1]
        n = max(self.lengths)
        assert R.rel(o, want_o) <= R.attention_tolerance(self.dtype, n)
        if s is not None:
            assert R.rel(s, want_s) <= R.attention_tolerance("F32", n)

    def backward(self, state=True):
        self.build()
        out = [self.empty(x) for x in (self.q, self.k, self.v)] + [torch.full_like(self.s0, float("nan"))]
        self.ctx.execute_linear_attention_backward(
            self.ir, ptr(self.q), ptr(self.k), ptr(self.v), ptr(self.g), ptr(self.do), *(ptr(x) for x in out[:3]),
            initial_state_ptr=ptr(self.s0 if state else None), final_state_gradient_ptr=ptr(self.ds if state else None),
            initial_state_gradient_ptr=ptr(out[3]), sequence_offsets_ptr=ptr(self.offsets), stream=stream())
        return out

    def check_backward(self, state=True):
        out = self.backward(state)
        want = [self.empty(x).double() for x in (self.q, self.k, self.v)] + [torch.empty_like(self.s0).double()]
        for b, n in enumerate(self.lengths):
            got = R.attention_grad(*(self.sequence(x, b) for x in (self.q, self.k, self.v)), self.g, self.scale,
                                   self.sequence(self.do, b), self.s0[b] if state else None,
                                   self.ds[b] if state else None)
            for w, x in zip(want[:3], got):
                self.sequence(w, b).copy_(x)
            want[3][b] = got[3]
        n = max(self.lengths)
        for x, w in zip(out[:3], want):
            assert R.rel(x, w) <= R.attention_tolerance(self.dtype, n)
        assert R.rel(out[3], want[3]) <= R.attention_tolerance("F32", n)


LENGTHS = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200, 256, 257, 500]


@pytest.mark.parametrize("dtype", ["F32", "F16", "BF16"])
@pytest.mark.parametrize("length", LENGTHS)
def test_attention_lengths(V, ctx, length, dtype):
    c = Case(V, ctx, [length] * 2, 4, 2, 64, 64, dtype, seed=length)
    c.check_forward(state=True)
    c.check_forward(state=False)
    c.check_backward(state=True)


DIMS = [(1, 1), (3, 5), (8, 16), (16, 8), (33, 20), (40, 64), (64, 40), (64, 96), (80, 80), (96, 128), (128, 64), (128, 128),
        (130, 127), (200, 72), (72, 200), (256, 256)]


@pytest.mark.parametrize("dtype", ["F32", "F16", "BF16"])
@pytest.mark.parametrize("dk,dv", DIMS)
def test_attention_dims(V, ctx, dk, dv, dtype):
    for length in (1, 150):
        c = Case(V, ctx, [length], 3, 3, dk, dv, dtype, seed=dk + dv)
        c.check_forward()
        c.check_backward()


@pytest.mark.parametrize("dtype", ["F32", "F16", "BF16"])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 5), (4, 1), (6, 3), (12, 4)])
def test_attention_heads(V, ctx, heads, kv_heads, dtype):
    for dim in (24, 128):
        c = Case(V, ctx, [140] * 3, heads, kv_heads, dim, dim, dtype)
        c.check_forward()
        c.check_backward()
        c.check_backward(state=False)


@pytest.mark.parametrize("dtype", ["F32", "F16", "BF16"])
@pytest.mark.parametrize("lengths", [[1], [0, 3, 0], [5, 0, 1, 300, 0, 129, 128, 2], [700, 1, 1, 64], [0, 0]])
def test_attention_packed(V, ctx, lengths, dtype):
    for kv_heads, dim in ((4, 64), (2, 128)):
        c = Case(V, ctx, lengths, 4, kv_heads, dim, dim, dtype, packed=True)
        c.check_forward()
        c.check_forward(state=False)
        c.check_backward()


@pytest.mark.parametrize("dtype", ["F32", "F16", "BF16"])
@pytest.mark.parametrize("layout", ["heads", "odd"])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_attention_layouts(V, ctx, dim, layout, dtype):
    for packed in (False, True):
        c = Case(V, ctx, [190, 190] if not packed else [150, 1, 90], 4, 2, dim, dim, dtype, packed=packed, layout=layout)
        c.check_forward()
        c.check_backward()
    c = Case(V, ctx, [1] * 3, 4, 2, dim, dim, dtype, layout=layout)
    c.check_forward()


DECAYS = [[0.0], [-1e-4, -0.5, -3.0], [-30.0, -90.0, -1000.0], [-math.inf, 0.0, -2.0]]


@pytest.mark.parametrize("dtype", ["F32", "F16", "BF16"])
@pytest.mark.parametrize("decay", DECAYS, ids=["none", "mixed", "strong", "infinite"])
def test_attention_decays(V, ctx, decay, dtype):
    for length in (1, 300):
        for dim in (16, 128):
            c = Case(V, ctx, [length], 3, 3, dim, dim, dtype, decay=decay)
            c.check_forward()
            c.check_backward()


@pytest.mark.parametrize("dtype", ["F32", "BF16"])
def test_attention_long(V, ctx, dtype):
    c = Case(V, ctx, [5003], 2, 1, 128, 64, dtype)
    c.check_forward()
    c.check_backward()


@pytest.mark.parametrize("dtype", ["F32", "F16", "BF16"])
def test_attention_prompt_then_steps(V, ctx, dtype):
    """A prompt, then its further tokens one at a time through a pool of states, in place, against the whole at once."""
    c = Case(V, ctx, [160] * 3, 4, 2, 64, 64, dtype)
    pool = normal(9, 5, 4, 64, 64)
    keep = pool.clone()
    slots = torch.tensor([4, 0, 2], dtype=torch.int32, device="cuda")
    pool[slots.long()] = c.s0
    outs = []

    def part(a, n):
        cfg = V.LinearAttentionConfig(n, 4, 64, 64).with_batch_count(3).with_key_value_heads(2).with_state_slots(5)
        cfg = cfg.with_element_type(V.ElementType[dtype])
        q, k, v = (x[:, a:a + n] for x in (c.q, c.k, c.v))
        cfg = cfg.with_query_strides(*c.strides(q)).with_key_strides(*c.strides(k)).with_value_strides(*c.strides(v))
        ir = V.LinearAttentionIr.build(cfg, ctx.device_profile())
        o = torch.empty(3, n, 4, 64, dtype=c.t, device="cuda")
        ctx.execute_linear_attention(ir, ptr(q), ptr(k), ptr(v), ptr(c.g), ptr(o), ptr(pool), ptr(pool),
                                     state_slots_ptr=ptr(slots), stream=stream())
        outs.append(o)

    part(0, 140)
    for t in range(140, 160):
        part(t, 1)
    c.compare_forward(torch.cat(outs, 1), pool[slots.long()])
    assert torch.equal(pool[1], keep[1]) and torch.equal(pool[3], keep[3])


@pytest.mark.parametrize("length", [1, 200])
def test_attention_slots_outside(V, ctx, length):
    """A sequence whose slot is not in the pool starts from zero and keeps nothing; the others are untouched by it."""
    c = Case(V, ctx, [length] * 4, 2, 2, 64, 64, "BF16")
    pool = normal(9, 3, 2, 64, 64)
    before = pool.clone()
    slots = torch.tensor([-1, 2, 3, 1 << 30], dtype=torch.int32, device="cuda")
    c.build(c.cfg.with_state_slots(3))
    o = torch.empty_like(c.do)
    ctx.execute_linear_attention(c.ir, ptr(c.q), ptr(c.k), ptr(c.v), ptr(c.g), ptr(o), ptr(pool), ptr(pool),
                                 state_slots_ptr=ptr(slots), stream=stream())
    for b in range(4):
        s0 = before[2] if b == 1 else None
        want, state = R.attention(c.q[b], c.k[b], c.v[b], c.g, c.scale, s0)
        assert R.rel(o[b], want) <= R.attention_tolerance("BF16", length)
        if b == 1:
            assert R.rel(pool[2], state) <= R.attention_tolerance("F32", length)
    assert torch.equal(pool[:2], before[:2])


def test_attention_offsets_outside(V, ctx):
    """Offsets past the rows, running backwards or longer than the stated length read and write nothing outside."""
    c = Case(V, ctx, [100, 60, 40], 2, 2, 64, 64, "BF16", packed=True)
    cfg = c.cfg
    cfg._s.length = 50  # shorter than the first two sequences
    c.build(cfg)
    offsets = torch.tensor([-7, 90, 60, 1 << 40], device="cuda")
    o = torch.full_like(c.do, float("nan"))
    s = torch.full_like(c.s0, float("nan"))
    ctx.execute_linear_attention(c.ir, ptr(c.q), ptr(c.k), ptr(c.v), ptr(c.g), ptr(o), 0, ptr(s), ptr(offsets),
                                 stream=stream())
    tol = R.attention_tolerance("BF16", 50)
    want, state = R.attention(c.q[:50], c.k[:50], c.v[:50], c.g, c.scale)
    assert R.rel(o[:50], want) <= tol and R.rel(s[0], state) <= R.attention_tolerance("F32", 50)
    assert bool(torch.isnan(o[50:60]).all()) and float(s[1].abs().max()) == 0.0
    want, state = R.attention(c.q[60:110], c.k[60:110], c.v[60:110], c.g, c.scale)
    assert R.rel(o[60:110], want) <= tol and R.rel(s[2], state) <= R.attention_tolerance("F32", 50)
    assert bool(torch.isnan(o[110:]).all())


@pytest.mark.parametrize("dtype", ["F32", "F16", "BF16"])
def test_attention_neighbours_stay_apart(V, ctx, dtype):
    """NaN and infinity in one packed sequence do not reach another, and not the tokens before them."""
    c = Case(V, ctx, [70, 130, 131], 2, 2, 128, 128, dtype, packed=True)
    clean, _ = c.forward()
    start = 70 + 100
    c.k[start], c.v[start, 0, 5], c.q[start + 3] = float("nan"), float("inf"), float("nan")
    o, s = c.forward()
    assert torch.equal(o[:start], clean[:start]) and torch.equal(o[200:], clean[200:])
    assert bool(torch.isnan(o[start:200]).all())
    assert bool(torch.isfinite(s[0]).all()) and bool(torch.isfinite(s[2]).all()) and not bool(torch.isfinite(s[1]).any())


@pytest.mark.parametrize("dtype", ["F32", "F16", "BF16"])
@pytest.mark.parametrize("part", [-1.0, 0.9975, 0.9946])
def test_attention_lowest_values_stay_behind(V, ctx, dtype, part):
    """Values at the ends of the type's range do not reach the tokens before them."""
    c = Case(V, ctx, [150], 2, 2, 64, 96, dtype)
    clean, _ = c.forward()
    start = 83
    c.v[0, start:start + 3, 1, 5:40] = part * torch.finfo(c.v.dtype).max
    o, _ = c.forward()
    assert torch.equal(o[0, :start], clean[0, :start]) and torch.equal(o[:, :, 0], clean[:, :, 0])


@pytest.mark.parametrize("dtype,big", [("F16", 60.0), ("BF16", 3e4)])
def test_attention_large_scores(V, ctx, dtype, big):
    """Scores beyond the range of half precision, weighed down by small values again."""
    c = Case(V, ctx, [140], 2, 2, 128, 128, dtype, scale=1.0, decay=[-0.01])
    c.q.mul_(big)
    c.k.mul_(big)
    c.v.mul_(1.0 / (big * big))
    c.s0.mul_(1.0 / big)
    c.check_forward()


def test_attention_wanted_gradients(V, ctx):
    """Any subset of the gradients gives the bits of all together."""
    for kv in (2, 1):
        c = Case(V, ctx, [150], 2, kv, 64, 64, "BF16")
        full = c.backward()
        for wanted in itertools.product((0, 1), repeat=4):
            out = [torch.full_like(x, float("nan")) for x in full]
            give = [ptr(x) if w else 0 for x, w in zip(out, wanted)]
            ctx.execute_linear_attention_backward(
                c.ir, ptr(c.q), ptr(c.k), ptr(c.v), ptr(c.g), ptr(c.do), *give[:3], initial_state_ptr=ptr(c.s0),
                final_state_gradient_ptr=ptr(c.ds), initial_state_gradient_ptr=give[3], stream=stream())
            for x, y, w in zip(out, full, wanted):
                if w:
                    assert R.rel(x, y) <= (0.0 if x is not out[3] else R.attention_tolerance("F32", 150))
                else:
                    assert bool(torch.isnan(x).all())


def test_attention_gradient_state_in_place(V, ctx):
    c = Case(V, ctx, [150] * 2, 2, 2, 64, 64, "BF16")
    full = c.backward()
    out = [torch.empty_like(x) for x in full[:3]]
    ds = c.ds.clone()
    c.ctx.execute_linear_attention_backward(
        c.ir, ptr(c.q), ptr(c.k), ptr(c.v), ptr(c.g), ptr(c.do), *(ptr(x) for x in out), initial_state_ptr=ptr(c.s0),
        final_state_gradient_ptr=ptr(ds), initial_state_gradient_ptr=ptr(ds), stream=stream())
    assert torch.equal(ds, full[3])
    for x, y in zip(out, full):
        assert torch.equal(x, y)


def test_attention_gradient_against_differences(V, ctx):
    c = Case(V, ctx, [23], 2, 1, 12, 9, "F32")
    grads = c.backward()
    at = [t.double() for t in (c.q[0], c.k[0], c.v[0], c.s0[0])]

    def loss(q, k, v, s0):
        o, s = R.attention(q, k, v, c.g, c.scale, s0)
        return float((o * c.do[0].double()).sum() + (s * c.ds[0].double()).sum())

    for n, grad in enumerate(x[0] for x in grads):
        d = normal(40 + n, *grad.shape).double()
        up, down = list(at), list(at)
        up[n], down[n] = at[n] + 1e-3 * d, at[n] - 1e-3 * d
        slope = (loss(*up) - loss(*down)) / 2e-3  # the loss is linear in each argument: no truncation error
        size = float(torch.linalg.vector_norm(grad.double()) * torch.linalg.vector_norm(d))
        assert abs(slope - float((grad.double() * d).sum())) <= 2e-6 * size


def test_attention_is_the_exponential_convolution(V, ctx):
    """With q = k = 1 the operator is the causal convolution with l^n: the FFT engine computes the same."""
    n, channels, log_decay = 200, 8, -0.05
    m = 512
    dev = ctx.device_profile()
    x = np.zeros((channels, m), dtype=np.complex64)
    x[:, :n] = np.random.default_rng(3).standard_normal((channels, n))
    kernel = np.zeros(m, dtype=np.complex64)
    kernel[:n] = np.exp(log_decay * np.arange(n))
    fwd = V.TransformIr.build(V.FftConfig([m]), V.Direction.FORWARD, dev)
    spectrum = ctx.execute_transform(fwd, kernel)
    cfg = V.FftConfig([m]).with_batch_count(channels).with_convolution(True).with_inverse_normalization(True)
    conv = V.ConvolutionIr.build_from_spectrum(cfg, spectrum, dev)
    want = ctx.execute_convolution(conv, x).reshape(channels, m)[:, :n].real
    one = torch.ones(1, n, 1, 1, device="cuda")
    v = torch.from_numpy(x[:, :n].real.T.copy()).cuda().view(1, n, 1, channels)
    g = torch.full((1,), log_decay, device="cuda")
    o = torch.empty_like(v)
    ir = V.LinearAttentionIr.build(V.LinearAttentionConfig(n, 1, 1, channels), dev)
    ctx.execute_linear_attention(ir, ptr(one), ptr(one), ptr(v), ptr(g), ptr(o), stream=stream())
    torch.cuda.synchronize()
    assert R.rel(o.view(n, channels).T.cpu(), torch.from_numpy(want.copy())) <= 2e-6 + R.attention_tolerance("F32", n)


def test_repeats_and_streams(V, ctx):
    """Equal inputs give equal bits, on the default stream, another stream and the context's own."""
    c = Case(V, ctx, [1500] * 2, 4, 2, 128, 128, "BF16")
    o, s = c.forward()
    grads = c.backward()
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        o2, s2 = c.forward()
        grads2 = c.backward()
    torch.cuda.synchronize()
    assert torch.equal(o, o2) and torch.equal(s, s2) and all(torch.equal(x, y) for x, y in zip(grads, grads2))
    o3 = torch.empty_like(o)
    torch.cuda.synchronize()
    ctx.execute_linear_attention(c.ir, ptr(c.q), ptr(c.k), ptr(c.v), ptr(c.g), ptr(o3), ptr(c.s0))
    ctx.synchronize()
    assert torch.equal(o, o3)


# ---- refusals ------------------------------------------------------------------------------

def refuses(V, variant, call):
    with pytest.raises(V.VkFftError) as e:
        call()
    assert e.value.variant == variant


def test_execution_refusals(V, ctx):
    c = Case(V, ctx, [8], 2, 2, 16, 16, "BF16")
    ir = c.build()
    o = torch.empty_like(c.do)
    run = lambda **kw: ctx.execute_linear_attention(ir, **{**dict(query_ptr=ptr(c.q), key_ptr=ptr(c.k), value_ptr=ptr(c.v),  # noqa: E731
                                                    log_decay_ptr=ptr(c.g), output_ptr=ptr(o), stream=1), **kw})
    for name in ("query_ptr", "key_ptr", "value_ptr", "log_decay_ptr", "output_ptr"):
        refuses(V, "ValueOutOfRange", lambda: run(**{name: 0}))
        refuses(V, "ValueOutOfRange", lambda: run(**{name: ptr(c.q) + 1}))
    refuses(V, "ValueOutOfRange", lambda: run(initial_state_ptr=ptr(c.s0) + 2))
    refuses(V, "ValueOutOfRange", lambda: run(final_state_ptr=ptr(c.s0) + 2))
    refuses(V, "ValueOutOfRange", lambda: run(state_slots_ptr=ptr(c.s0) + 2))
    packed = V.LinearAttentionIr.build(c.cfg.with_packed_tokens(8), ctx.device_profile())
    refuses(V, "ValueOutOfRange", lambda: ctx.execute_linear_attention(packed, ptr(c.q), ptr(c.k), ptr(c.v), ptr(c.g), ptr(o)))
    n = norm_ir(V, ctx, 4, 8, "F32", "F32")
    x = torch.zeros(4, 8, device="cuda")
    refuses(V, "ValueOutOfRange", lambda: ctx.execute_layer_norm(n, 0, ptr(x)))
    refuses(V, "ValueOutOfRange", lambda: ctx.execute_layer_norm(n, ptr(x), 0))
    refuses(V, "ValueOutOfRange", lambda: ctx.execute_layer_norm(n, ptr(x) + 2, ptr(x)))
    refuses(V, "ValueOutOfRange", lambda: ctx.execute_layer_norm(n, ptr(x), ptr(x), ptr(x) + 1))
    refuses(V, "ValueOutOfRange", lambda: ctx.execute_layer_norm_backward(n, ptr(x), 0, ptr(x), ptr(x)))
    run()  # refusals leave the context usable
    torch.cuda.synchronize()
    assert bool(torch.isfinite(o.float()).all())


def test_empty_calls(V, ctx):
    """Packed rows of no token: states pass through, null tensors are accepted."""
    cfg = V.LinearAttentionConfig(4, 2, 32, 32).with_batch_count(3).with_packed_tokens(0)
    ir = V.LinearAttentionIr.build(cfg, ctx.device_profile())
    offsets, g = torch.zeros(4, dtype=torch.int64, device="cuda"), torch.zeros(2, device="cuda")
    s0 = normal(1, 3, 2, 32, 32)
    s = torch.empty_like(s0)
    ctx.execute_linear_attention(ir, 0, 0, 0, ptr(g), 0, ptr(s0), ptr(s), ptr(offsets), stream=stream())
    assert torch.equal(s, s0)
    ds0 = torch.empty_like(s0)
    ctx.execute_linear_attention_backward(ir, 0, 0, 0, ptr(g), 0, final_state_gradient_ptr=ptr(s0),
                                          initial_state_gradient_ptr=ptr(ds0), sequence_offsets_ptr=ptr(offsets),
                                          stream=stream())
    assert torch.equal(ds0, s0)
