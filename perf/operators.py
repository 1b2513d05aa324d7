"""Timing cases of the sequence operators: layer normalisation and decayed linear attention.

A case names an operator ("op"), its sizes and its element type.  run() computes it either in
plain elementary torch operations in 32 bits (own = False) or through the framework's own entry
points (own = True); exact() evaluates the definition in 64 bits.

Operators
  norm       y = (x - mean) rstd w + b, with mean and rstd kept for the backward pass
  norm_grad  dx, dw, db of it
  mix        linear attention with one decay per head over whole sequences: S_t = l S_{t-1} + k_t v_t^T,
             o_t = scale S_t^T q_t, and the state after the last token
  mix_step   the same for one new token of each sequence
  mix_grad   dq, dk, dv (and the initial state's gradient)
"""
import math
import os
import sys

import torch

own = False

EPSILON = 1e-5
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- cases -----------------------------------------------------------------------------

def _norm(name, op, rows, features, dtype):
    return {"name": name, "op": op, "rows": rows, "features": features, "dtype": dtype}


def _mix(name, op, batch, length, heads, kv_heads, key_dim, value_dim, dtype, state=False, packed=False):
    return {"name": name, "op": op, "batch": batch, "length": length, "heads": heads, "kv_heads": kv_heads,
            "key_dim": key_dim, "value_dim": value_dim, "dtype": dtype, "state": state, "packed": packed}


def listed():
    return [
        # the norm in front of a mixer while eight sequences generate: latency
        _norm("norm, 8 tokens", "norm", 8, 4096, "bf16"),
        # the same norm over four prompts of 4096 tokens
        _norm("norm, prompts", "norm", 16384, 4096, "bf16"),
        # a training step's norm
        _norm("norm gradient", "norm_grad", 8192, 4096, "bf16"),
        # an odd width and an odd number of rows, whose rows start at odd addresses
        _norm("norm gradient, odd", "norm_grad", 4099, 1023, "f32"),
        # one prompt of ordinary length
        _mix("mix, prompt", "mix", 1, 8192, 16, 16, 128, 128, "bf16"),
        # prompts of many lengths packed behind one another, key/value heads shared by four query heads
        _mix("mix, packed prompts", "mix", 13, 2048, 16, 4, 64, 64, "bf16", state=True, packed=True),
        # short odd sequences in single precision
        _mix("mix, odd f32", "mix", 2, 1023, 8, 8, 64, 96, "f32", state=True),
        # a long document continued from a kept state
        _mix("mix, long", "mix", 1, 65537, 8, 8, 128, 128, "bf16", state=True),
        # one sequence generating: latency
        _mix("mix step, 1 sequence", "mix_step", 1, 1, 16, 16, 128, 128, "bf16", state=True),
        # a full serving batch: the states' bytes
        _mix("mix step, 256 sequences", "mix_step", 256, 1, 16, 16, 128, 128, "bf16", state=True),
        # a training step's mixer
        _mix("mix gradient", "mix_grad", 2, 4096, 16, 16, 128, 128, "bf16"),
        # the same in half precision with shared heads, an odd length and a carried state
        _mix("mix gradient, f16", "mix_grad", 4, 1000, 12, 4, 64, 64, "f16", state=True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    while True:
        op = rng.choice(("norm", "norm_grad", "mix", "mix_step", "mix_grad"))
        dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
        if op in ("norm", "norm_grad"):
            features = _log_int(rng, 64, 16384)
            if rng.random() < 0.5:
                features = max(64, features // 64 * 64)
            case = {"op": op, "rows": _log_int(rng, 4, 60000), "features": features, "dtype": dtype}
        else:
            kv_heads = rng.choice((1, 2, 4, 8, 16))
            heads = kv_heads * rng.choice((1, 1, 1, 2, 4))
            dims = (32, 64, 64, 80, 128, 128, 128)
            key_dim = rng.choice(dims)
            value_dim = key_dim if rng.random() < 0.7 else rng.choice(dims)
            if op == "mix_step":
                batch, length, state, packed = _log_int(rng, 1, 256), 1, True, False
            else:
                batch, state = _log_int(rng, 1, 16), rng.random() < 0.5
                length = _log_int(rng, 17, 65537 if op == "mix" else 8192)
                packed = op == "mix" and rng.random() < 0.4
            case = {"op": op, "batch": batch, "length": length, "heads": heads, "kv_heads": kv_heads,
                    "key_dim": key_dim, "value_dim": value_dim, "dtype": dtype, "state": state, "packed": packed}
        w = work(case)
        if w["bytes"] <= 3.0e8 and w["flops"] <= 3.4e10 and heads_fit(case):
            return case


def heads_fit(case):
    return "heads" not in case or case["heads"] <= 32


def _lengths(case):
    """Lengths of a packed case's sequences: the longest, then a ragged spread, one of a single token, one empty."""
    if not case["packed"]:
        return [case["length"]] * case["batch"]
    n = case["batch"]
    out = [max(1, case["length"] * (n - b) * 31 // (n * 31 + 7 * (b % 3))) for b in range(n)]
    out[0] = case["length"]
    if n > 2:
        out[n // 2], out[n // 2 - 1] = 1, 0
    return out


def work(case):
    size = torch.empty(0, dtype=TYPES[case["dtype"]]).element_size()
    if "rows" in case:
        rows, features = case["rows"], case["features"]
        if case["op"] == "norm":
            return {"bytes": (2 * rows * features + 2 * features) * size + 8 * rows, "flops": 8 * rows * features}
        return {"bytes": (3 * rows * features + 3 * features) * size + 8 * rows, "flops": 14 * rows * features}
    tokens, h, g, dk, dv = sum(_lengths(case)), case["heads"], case["kv_heads"], case["key_dim"], case["value_dim"]
    states = case["batch"] * h * dk * dv * 4
    if case["op"] == "mix_grad":
        n = tokens * (2 * h * dk + 2 * g * dk + 2 * g * dv + h * dv) * size
        # dq, dk and dv each read a state from both sides, which two recurrences keep up
        return {"bytes": n + (3 * states if case["state"] else 0), "flops": tokens * h * dk * dv * 10}
    n = tokens * (h * dk + g * dk + g * dv + h * dv) * size
    return {"bytes": n + states * (2 if case["state"] else 1), "flops": tokens * h * dk * dv * 4}


# ---- inputs ------------------------------------------------------------------------------

def _package():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(root, "vkfft-rs_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import vkfft_rs
    return vkfft_rs


_context = []


def _open(V):
    """The program's one execution context."""
    if not _context:
        c = V.CudaExecutionContext(0)
        _context.append((c, c.device_profile()))
    return _context[0]


def _inputs(case, seed):
    rnd = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, to=dtype):
        return (torch.randn(*shape, generator=rnd, device="cuda") * std + mean).to(to)

    s = {"case": case}
    if "rows" in case:
        rows, features = case["rows"], case["features"]
        # residual-stream rows: an offset, and rows of different scale
        s["x"] = (torch.randn(rows, features, generator=rnd, device="cuda")
                  * (0.5 + torch.rand(rows, 1, generator=rnd, device="cuda") * 2) + 0.3).to(dtype)
        s["w"], s["b"] = normal(features, std=0.2, mean=1.0), normal(features, std=0.1)
        if case["op"] == "norm_grad":
            s["dy"] = normal(rows, features, std=0.05)
            x = s["x"].float()  # the statistics that the forward pass left behind
            s["mean"] = x.mean(-1)
            s["rstd"] = torch.rsqrt((x - s["mean"][:, None]).square().mean(-1) + EPSILON)
        return s
    b, t, h, g, dk, dv = (case[n] for n in ("batch", "length", "heads", "kv_heads", "key_dim", "value_dim"))
    lengths = _lengths(case)
    lead = (sum(lengths),) if case["packed"] else (b, t)
    s["q"], s["k"], s["v"] = normal(*lead, h, dk), normal(*lead, g, dk), normal(*lead, g, dv)
    # per-head decays 1 - 2^-n, from a memory of about 16 tokens to one of about 4000
    n = 4 + 8 * torch.arange(h, device="cuda", dtype=torch.float64) / max(1, h - 1)
    s["log_decay"] = torch.log1p(-torch.exp2(-n)).float()
    s["scale"] = dk ** -0.5
    s["lengths"] = lengths
    if case["packed"]:
        s["offsets"] = torch.tensor([0] + lengths, device="cuda").cumsum(0)
    if case["state"]:
        s["s0"] = normal(b, h, dk, dv, std=3.0, to=torch.float32)
    if case["op"] == "mix_grad":
        s["do"] = normal(*lead, h, dv, std=0.1)
        if case["state"]:
            s["ds"] = normal(b, h, dk, dv, std=0.1, to=torch.float32)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:  # the handle of these sizes and the output buffers that a program keeps; the inputs above are the same
        _plan(s)
    return s


def _plan(s):
    V, case = _package(), s["case"]
    s["ctx"], device = _open(V)
    kind = {"f32": V.ElementType.F32, "f16": V.ElementType.F16, "bf16": V.ElementType.BF16}[case["dtype"]]
    if "rows" in case:
        cfg = V.LayerNormConfig(case["rows"], case["features"]).with_element_type(kind).with_parameter_type(kind)
        s["ir"] = V.LayerNormIr.build(cfg.with_epsilon(EPSILON), device)
        names = {"norm": ("x",), "norm_grad": ("x", "w", "b")}[case["op"]]
        s["out"] = [torch.empty_like(s[n]) for n in names]
        if case["op"] == "norm":
            s["out"] += [torch.empty(case["rows"], device="cuda") for _ in range(2)]
    else:
        cfg = V.LinearAttentionConfig(case["length"], case["heads"], case["key_dim"], case["value_dim"])
        cfg = cfg.with_batch_count(case["batch"]).with_key_value_heads(case["kv_heads"])
        cfg = cfg.with_element_type(kind).with_scale(s["scale"])
        if case["packed"]:
            cfg = cfg.with_packed_tokens(sum(s["lengths"]))
        s["ir"] = V.LinearAttentionIr.build(cfg, device)
        states = (case["batch"], case["heads"], case["key_dim"], case["value_dim"])
        if case["op"] == "mix_grad":
            s["out"] = [torch.empty_like(s[n]) for n in ("q", "k", "v") + (("s0",) if case["state"] else ())]
        else:
            s["out"] = [torch.empty(*s["q"].shape[:-1], case["value_dim"], dtype=s["q"].dtype, device="cuda"),
                        torch.empty(states, device="cuda")]
    need = s["ir"].backward_workspace_bytes if case["op"].endswith("grad") else s["ir"].workspace_bytes
    s["workspace"] = torch.empty(need, dtype=torch.uint8, device="cuda") if need else None


# ---- one pass ----------------------------------------------------------------------------

def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _run_own(s):
    op, ctx, ir, out = s["case"]["op"], s["ctx"], s["ir"], s["out"]
    stream = torch.cuda.current_stream().cuda_stream or 1  # 1: the legacy default stream
    if op == "norm":
        ctx.execute_layer_norm(ir, s["x"].data_ptr(), out[0].data_ptr(), s["w"].data_ptr(), s["b"].data_ptr(),
                               out[1].data_ptr(), out[2].data_ptr(), stream=stream)
        return {"y": out[0], "mean": out[1], "rstd": out[2]}
    ws = _ptr(s["workspace"])
    if op == "norm_grad":
        ctx.execute_layer_norm_backward(ir, s["x"].data_ptr(), s["mean"].data_ptr(), s["rstd"].data_ptr(),
                                        s["dy"].data_ptr(), s["w"].data_ptr(), out[0].data_ptr(), out[1].data_ptr(),
                                        out[2].data_ptr(), workspace_ptr=ws, stream=stream)
        return {"dx": out[0], "dw": out[1], "db": out[2]}
    if op == "mix_grad":
        ctx.execute_linear_attention_backward(
            ir, s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["log_decay"].data_ptr(),
            s["do"].data_ptr(), out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(),
            initial_state_ptr=_ptr(s.get("s0")), final_state_gradient_ptr=_ptr(s.get("ds")),
            initial_state_gradient_ptr=_ptr(out[3] if len(out) > 3 else None), workspace_ptr=ws, stream=stream)
        return dict(zip(("dq", "dk", "dv", "ds0"), out))
    ctx.execute_linear_attention(
        ir, s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["log_decay"].data_ptr(), out[0].data_ptr(),
        initial_state_ptr=_ptr(s.get("s0")), final_state_ptr=out[1].data_ptr(),
        sequence_offsets_ptr=_ptr(s.get("offsets")), workspace_ptr=ws, stream=stream)
    return {"o": out[0], "state": out[1]}


CHUNK = 128


def _core(q, k, v, g):
    """scale-free, state-free decayed attention of [B, T, H, D] float tensors, by chunks of 128 tokens:
    inside a chunk the masked products, between chunks the decayed sums of the chunks' states."""
    b, t, h, _ = q.shape
    c = min(CHUNK, t)
    n = -(-t // c)
    pad = (0, 0, 0, 0, 0, n * c - t)
    q, k, v = (torch.nn.functional.pad(x, pad).view(b, n, c, h, -1).permute(0, 3, 1, 2, 4) for x in (q, k, v))
    i = torch.arange(c, device=q.device)
    ahead = i[:, None] - i[None, :]
    decay = torch.where(ahead >= 0, torch.exp(g[:, None, None] * ahead.clamp(min=0)), 0.0)
    out = (q @ k.transpose(-1, -2) * decay[None, :, None]) @ v
    if n > 1:
        local = (k * torch.exp(g[:, None] * (c - 1 - i))[None, :, None, :, None]).transpose(-1, -2) @ v
        m = torch.arange(n, device=q.device)
        gap = m[:, None] - 1 - m[None, :]
        between = torch.where(gap >= 0, torch.exp(g[:, None, None] * (c * gap.clamp(min=0))), 0.0)
        entering = (between @ local.flatten(-2)).view(local.shape)
        out = out + torch.exp(g[:, None] * (i + 1))[None, :, None, :, None] * (q @ entering)
    return out.permute(0, 2, 3, 1, 4).reshape(b, n * c, h, -1)[:, :t]


def _shared(x, heads):
    """Each key/value head repeated for the query heads that share it, in 32 bits."""
    return x.float().repeat_interleave(heads // x.shape[-2], dim=-2)


def _plain_mix(s):
    case, g, scale = s["case"], s["log_decay"], s["scale"]
    heads, t = case["heads"], case["length"]
    q, k, v = s["q"].float(), _shared(s["k"], heads), _shared(s["v"], heads)
    at = torch.arange(t, device=q.device)
    if case["packed"]:
        count = s["offsets"][1:] - s["offsets"][:-1]
        live = at < count[:, None]
        index = (s["offsets"][:-1, None] + at).clamp(max=q.shape[0] - 1)
        q, k, v = (torch.where(live[:, :, None, None], x[index], 0.0) for x in (q, k, v))
    else:
        count = torch.full((case["batch"],), t, device=q.device)
        live = None
    out = scale * _core(q, k, v, g)
    # the state after the last token of each sequence
    left = (count[:, None] - 1 - at).clamp(min=0)
    state = torch.einsum("bthk,bth,bthv->bhkv", k, torch.exp(left[:, :, None] * g), v)
    if case["state"]:
        out = out + scale * torch.exp((at[:, None] + 1) * g)[None, :, :, None] * torch.einsum(
            "bthk,bhkv->bthv", q, s["s0"])
        state = state + torch.exp(count[:, None] * g)[:, :, None, None] * s["s0"]
    if live is not None:
        out = out[live]
    return {"o": out.to(s["q"].dtype), "state": state}


def _plain_mix_grad(s):
    case, g, scale = s["case"], s["log_decay"], s["scale"]
    heads, t, kind = case["heads"], case["length"], s["q"].dtype
    q, do = s["q"].float(), s["do"].float()
    k, v = _shared(s["k"], heads), _shared(s["v"], heads)
    at = torch.arange(t, device=q.device)
    dq = scale * _core(do, v, k, g)
    rq, rk, rv, rdo = (x.flip(1) for x in (q, k, v, do))
    dk, dv = scale * _core(rv, rdo, rq, g), scale * _core(rk, rq, rdo, g)
    out = {}
    if case["state"]:
        fade = torch.exp((at[:, None] + 1) * g)[None, :, :, None]
        dq = dq + scale * fade * torch.einsum("bthv,bhkv->bthk", do, s["s0"])
        late = torch.exp(at[:, None] * g)[None, :, :, None]
        dk = dk + late * torch.einsum("bthv,bhkv->bthk", rv, s["ds"])
        dv = dv + late * torch.einsum("bthk,bhkv->bthv", rk, s["ds"])
        out["ds0"] = torch.exp(t * g)[None, :, None, None] * s["ds"] + scale * torch.einsum(
            "bthk,bthv->bhkv", q * fade, do)
    share = heads // case["kv_heads"]
    dk, dv = (x.flip(1).unflatten(2, (case["kv_heads"], share)).sum(3) for x in (dk, dv))
    return {"dq": dq.to(kind), "dk": dk.to(kind), "dv": dv.to(kind), **out}


def _plain_norm(s):
    x = s["x"].float()
    mean = x.mean(-1)
    centred = x - mean[:, None]
    rstd = torch.rsqrt(centred.square().mean(-1) + EPSILON)
    y = centred * rstd[:, None] * s["w"].float() + s["b"].float()
    return {"y": y.to(s["x"].dtype), "mean": mean, "rstd": rstd}


def _plain_norm_grad(s):
    x, dy, kind = s["x"].float(), s["dy"].float(), s["x"].dtype
    xhat = (x - s["mean"][:, None]) * s["rstd"][:, None]
    g = dy * s["w"].float()
    dx = s["rstd"][:, None] * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    return {"dx": dx.to(kind), "dw": (dy * xhat).sum(0).to(kind), "db": dy.sum(0).to(kind)}


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "norm":
        return _plain_norm(state)
    if op == "norm_grad":
        return _plain_norm_grad(state)
    return _plain_mix_grad(state) if op == "mix_grad" else _plain_mix(state)


# ---- 64 bits -----------------------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    if "rows" in case:
        return _exact_norm(s)
    return _exact_mix_grad(s) if case["op"] == "mix_grad" else _exact_mix(s)


def _exact_norm(s):
    x = s["x"].double()
    if s["case"]["op"] == "norm":
        var, mean = torch.var_mean(x, -1, correction=0)
        rstd = (var + EPSILON) ** -0.5
        return {"y": (x - mean[:, None]) * rstd[:, None] * s["w"].double() + s["b"].double(), "mean": mean, "rstd": rstd}
    dy, n = s["dy"].double(), x.shape[1]
    xhat = (x - s["mean"].double()[:, None]) * s["rstd"].double()[:, None]
    gw = dy * s["w"].double()
    inner = gw.sum(-1, keepdim=True) + xhat * (gw * xhat).sum(-1, keepdim=True)
    return {"dx": (gw - inner / n) * s["rstd"].double()[:, None], "dw": torch.einsum("rf,rf->f", dy, xhat), "db": dy.sum(0)}


BLOCK = 2048


def _weights(g, rows, cols):
    """l^(row - col) where col <= row, else 0, straight from the definition."""
    gap = (rows[:, None] - cols[None, :]).double()
    return torch.exp(gap * g).masked_fill_(gap < 0, 0.0)


def _one(q, k, v, g, scale, s0):
    """One head of one sequence: every pair of tokens, by blocks of rows."""
    t = q.shape[0]
    at = torch.arange(t, device=q.device)
    out = q.new_empty(t, v.shape[1])
    for a in range(0, t, BLOCK):
        rows, cols = at[a:a + BLOCK], at[:a + BLOCK]
        out[a:a + BLOCK] = (q[a:a + BLOCK] @ k[:a + BLOCK].T * _weights(g, rows, cols)) @ v[:a + BLOCK]
    if s0 is not None:
        out += torch.exp(g * (at + 1))[:, None] * (q @ s0)
    state = (k * torch.exp(g * (t - 1 - at))[:, None]).T @ v
    if s0 is not None:
        state += torch.exp(g * t) * s0
    return scale * out, state


def _exact_mix(s):
    case, g = s["case"], s["log_decay"].double()
    heads, share = case["heads"], case["heads"] // case["kv_heads"]
    out = torch.empty(*s["q"].shape[:-1], case["value_dim"], dtype=torch.float64, device="cuda")
    state = torch.empty(case["batch"], heads, case["key_dim"], case["value_dim"], dtype=torch.float64, device="cuda")
    start = 0
    for b, n in enumerate(s["lengths"]):
        here = slice(start, start + n) if case["packed"] else b
        start += n
        for h in range(heads):
            s0 = s["s0"][b, h].double() if case["state"] else None
            q, k, v = s["q"][here][:, h].double(), s["k"][here][:, h // share].double(), s["v"][here][:, h // share].double()
            out[here][:, h], state[b, h] = _one(q, k, v, g[h], s["scale"], s0)
    return {"o": out, "state": state}


def _exact_mix_grad(s):
    case, g, scale = s["case"], s["log_decay"].double(), s["scale"]
    heads, share, t = case["heads"], case["heads"] // case["kv_heads"], case["length"]
    got = {"dq": torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"),
           "dk": torch.zeros(s["k"].shape, dtype=torch.float64, device="cuda"),
           "dv": torch.zeros(s["v"].shape, dtype=torch.float64, device="cuda")}
    if case["state"]:
        got["ds0"] = torch.zeros(s["s0"].shape, dtype=torch.float64, device="cuda")
    at = torch.arange(t, device="cuda")
    for b in range(case["batch"]):
        for h in range(heads):
            q, do = s["q"][b, :, h].double(), s["do"][b, :, h].double()
            k, v = s["k"][b, :, h // share].double(), s["v"][b, :, h // share].double()
            for a in range(0, t, BLOCK):
                rows, end = slice(a, a + BLOCK), min(t, a + BLOCK)
                w = scale * _weights(g[h], at[rows], at[:end])
                seen, back = w * (q[rows] @ k[:end].T), w * (do[rows] @ v[:end].T)
                got["dv"][b, :end, h // share] += seen.T @ do[rows]
                got["dq"][b, rows, h] += back @ k[:end]
                got["dk"][b, :end, h // share] += back.T @ q[rows]
            if case["state"]:
                s0, ds = s["s0"][b, h].double(), s["ds"][b, h].double()
                early, late = torch.exp(g[h] * (at + 1))[:, None], torch.exp(g[h] * (t - 1 - at))[:, None]
                got["dq"][b, :, h] += scale * early * (do @ s0.T)
                got["dk"][b, :, h // share] += late * (v @ ds.T)
                got["dv"][b, :, h // share] += late * (k @ ds)
                got["ds0"][b, h] = torch.exp(g[h] * t) * ds + scale * (q * early).T @ do
    return got
