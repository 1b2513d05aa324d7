"""A sequence-mixing block on the engine: a fixed long convolution (FFT), a mixer whose filter depends on the data
(linear attention with a decay per head) and layer normalisation in front of each.

    x <- x + convolve(norm(x))          one filter along the tokens, through the FFT
    x <- x + W_o attend(norm(x))        per head: S <- l S + k v^T, y = S^T q

run() prepares the block and shows its three uses: a prompt in one pass, its continuation token by token from the kept
state (equal to the whole sequence at once), and one training step of the mixer (gradients of the attention and of the
norm in front of it), whose loss falls.

    python examples/sequence_mixing.py
"""
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vkfft-rs_b200"))
import vkfft_rs as V  # noqa: E402


class MixingBlock:
    def __init__(self, ctx, batch, length, heads, head_dim, dtype=torch.bfloat16, seed=0):
        self.ctx, self.device = ctx, ctx.device_profile()
        self.batch, self.heads, self.dim, self.dtype = batch, heads, head_dim, dtype
        self.kind = {torch.float32: V.ElementType.F32, torch.float16: V.ElementType.F16,
                     torch.bfloat16: V.ElementType.BF16}[dtype]
        width = heads * head_dim
        g = torch.Generator(device="cuda").manual_seed(seed)
        weight = lambda *s: (torch.randn(*s, generator=g, device="cuda") / s[0] ** 0.5).to(dtype)  # noqa: E731
        self.w_qkv, self.w_out = weight(width, 3 * width), weight(width, width)
        self.w_qkv[:, width:2 * width] *= 0.1  # a state sums up hundreds of keys
        self.norm_weight = [torch.ones(width, dtype=dtype, device="cuda") for _ in range(2)]
        self.norm_bias = [torch.zeros(width, dtype=dtype, device="cuda") for _ in range(2)]
        # memories of 16 to 1024 tokens
        self.log_decay = torch.log1p(-torch.exp2(-torch.linspace(4, 10, heads, device="cuda")))
        # the fixed filter: a causal kernel of `length` taps, as the spectrum of twice the length
        self.taps = length
        kernel = np.zeros(2 * length, dtype=np.complex64)
        kernel[:length] = np.exp(-0.02 * np.arange(length)) / 50
        forward = V.TransformIr.build(V.FftConfig([2 * length]), V.Direction.FORWARD, self.device)
        self.spectrum = ctx.execute_transform(forward, kernel)
        self._plans = {}

    @staticmethod
    def stream():
        return torch.cuda.current_stream().cuda_stream or 1  # 1: the legacy default stream

    def plan(self, what, *sizes):
        """The handle of an operator at these sizes, built once."""
        key = (what, *sizes)
        if key not in self._plans:
            if what == "norm":
                cfg = V.LayerNormConfig(*sizes).with_element_type(self.kind).with_parameter_type(self.kind)
                ir = V.LayerNormIr.build(cfg, self.device)
            elif what == "attention":
                cfg = V.LinearAttentionConfig(sizes[0], self.heads, self.dim, self.dim).with_batch_count(self.batch)
                # queries, keys and values stand side by side in the rows of one projection
                rows = 3 * self.heads * self.dim
                for s in ("query", "key", "value"):
                    cfg = getattr(cfg, f"with_{s}_strides")(sizes[0] * rows, rows, self.dim)
                ir = V.LinearAttentionIr.build(cfg.with_element_type(self.kind), self.device)
            else:
                cfg = V.FftConfig([2 * self.taps]).with_batch_count(sizes[0]).with_convolution(True)
                ir = V.ConvolutionIr.build_from_spectrum(cfg.with_inverse_normalization(True), self.spectrum, self.device)
            self._plans[key] = ir
        return self._plans[key]

    def norm(self, x, which, keep=False):
        rows = x.numel() // x.shape[-1]
        y = torch.empty_like(x)
        stats = torch.empty(2, rows, device="cuda") if keep else None
        mean, rstd = (stats[0].data_ptr(), stats[1].data_ptr()) if keep else (0, 0)
        self.ctx.execute_layer_norm(self.plan("norm", rows, x.shape[-1]), x.data_ptr(), y.data_ptr(),
                                    self.norm_weight[which].data_ptr(), self.norm_bias[which].data_ptr(), mean, rstd,
                                    stream=self.stream())
        return (y, stats) if keep else y

    def convolve(self, x):
        """The fixed filter along the tokens of [batch, token, channel], zero before the first token."""
        b, t, c = x.shape
        lines = torch.zeros(b * c, 2 * self.taps, dtype=torch.complex64, device="cuda")
        lines.real[:, :t] = x.transpose(1, 2).reshape(b * c, t)
        out = torch.empty_like(lines)
        ir = self.plan("convolution", b * c)
        ws = torch.empty(max(1, ir.workspace_bytes), dtype=torch.uint8, device="cuda")
        self.ctx.execute_nd_real_convolution_resident(ir, lines.data_ptr(), out.data_ptr(), ws.data_ptr(), self.stream())
        return out.real[:, :t].reshape(b, c, t).transpose(1, 2).to(x.dtype)

    def attend(self, qkv, state=None):
        """[batch, token, 3 width] -> [batch, token, width] and the state after the last token."""
        b, t, _ = qkv.shape
        width = self.heads * self.dim
        ir = self.plan("attention", t)
        y = torch.empty(b, t, width, dtype=self.dtype, device="cuda")
        after = torch.empty(b, self.heads, self.dim, self.dim, device="cuda")
        at, size = qkv.data_ptr(), qkv.element_size()
        self.ctx.execute_linear_attention(ir, at, at + width * size, at + 2 * width * size, self.log_decay.data_ptr(),
                                          y.data_ptr(), 0 if state is None else state.data_ptr(), after.data_ptr(),
                                          stream=self.stream())
        return y, after

    def mix(self, x, state=None):
        """The second half of the block, which a single token can continue."""
        y, state = self.attend(self.norm(x, 1) @ self.w_qkv, state)
        return x + y @ self.w_out, state

    def train_step(self, x, target, rate):
        """One step of gradient descent on the mixer's projections and its norm: loss = mean (mix(x) - target)^2."""
        b, t, width = x.shape
        h, stats = self.norm(x, 1, keep=True)
        qkv = h @ self.w_qkv
        y, _ = self.attend(qkv)
        error = (x + y @ self.w_out - target).float()
        d_out = (2 * error / error.numel()).to(self.dtype) * 4096  # a loss scale, taken out again below
        d_y = d_out @ self.w_out.T
        d_qkv = torch.empty_like(qkv)
        at, to, size = qkv.data_ptr(), d_qkv.data_ptr(), qkv.element_size()
        parts = (0, width * size, 2 * width * size)
        self.ctx.execute_linear_attention_backward(
            self.plan("attention", t), *(at + p for p in parts), self.log_decay.data_ptr(), d_y.data_ptr(),
            *(to + p for p in parts), stream=self.stream())
        d_h = d_qkv @ self.w_qkv.T
        d_weight, d_bias = torch.empty_like(self.norm_weight[1]), torch.empty_like(self.norm_bias[1])
        self.ctx.execute_layer_norm_backward(
            self.plan("norm", b * t, width), x.data_ptr(), stats[0].data_ptr(), stats[1].data_ptr(), d_h.data_ptr(),
            self.norm_weight[1].data_ptr(), 0, d_weight.data_ptr(), d_bias.data_ptr(), stream=self.stream())
        flat = lambda v: v.reshape(-1, v.shape[-1])  # noqa: E731
        for p, grad in ((self.w_out, flat(y).T @ flat(d_out)), (self.w_qkv, flat(h).T @ flat(d_qkv)),
                        (self.norm_weight[1], d_weight), (self.norm_bias[1], d_bias)):
            p.sub_((rate / 4096) * grad)
        return float(error.square().mean())


def run(batch=2, length=512, heads=8, head_dim=64, new_tokens=16, rate=0.02, say=print):
    ctx = V.CudaExecutionContext(0)
    try:
        block = MixingBlock(ctx, batch, length, heads, head_dim)
        g = torch.Generator(device="cuda").manual_seed(1)
        x = torch.randn(batch, length, heads * head_dim, generator=g, device="cuda").to(block.dtype)
        x = x + block.convolve(block.norm(x, 0))
        whole, state = block.mix(x)
        # the same as a prompt and its continuation, token by token
        split = length - new_tokens
        parts, kept = [], None
        for a, b in [(0, split)] + [(t, t + 1) for t in range(split, length)]:
            y, kept = block.mix(x[:, a:b].contiguous(), kept)
            parts.append(y)
        away = lambda a, b: float(torch.linalg.vector_norm((a - b).float()) / torch.linalg.vector_norm(b.float()))  # noqa: E731
        tokens_off, state_off = away(torch.cat(parts, 1), whole), away(kept, state)
        say(f"{split} tokens at once and {new_tokens} one by one, against all at once: {tokens_off:.1e} (state {state_off:.1e})")
        target = torch.randn(x.shape, generator=g, device="cuda").to(block.dtype) * 0.1 + x
        losses = [block.train_step(x, target, rate) for _ in range(5)]
        say("loss of five training steps: " + ", ".join(f"{v:.4f}" for v in losses))
        ctx.synchronize(1)
        return tokens_off, state_off, losses
    finally:
        ctx.close()


if __name__ == "__main__":
    run()
