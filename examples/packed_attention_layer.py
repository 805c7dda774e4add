"""One attention layer over packed sequences of different lengths, on the B200
kernels: images of mixed sizes in one batch (training step), and a causal
tower that answers token by token from its cache.

    python examples/packed_attention_layer.py

    h = x + residual,  y = rms_norm(h) · w          rmsnorm
    q, k, v = y · W_qkvᵀ + b                        dinov2.qkv_linear, or an 8-bit product for serving
    q, k turned by their positions                  rotary
    O = softmax(q kᵀ / √d) v within each sequence   packed
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from vision_rs_b200 import dinov2, packed, rmsnorm, rotary  # noqa: E402

E4M3_MAX = 448.0


class PackedAttentionLayer:
    """Weights of the layer: norm ``[hidden]``, QKV ``[3·hidden, hidden]`` bf16 and its f32 bias."""

    def __init__(self, hidden: int, heads: int, causal: bool = False, base: float = 10000.0, seed: int = 0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.dim, self.causal, self.hidden = heads, hidden // heads, causal, hidden
        self.w_norm = torch.ones(hidden, dtype=torch.bfloat16, device="cuda")
        self.w_qkv = (torch.randn(3 * hidden, hidden, generator=g, device="cuda") * hidden ** -0.5).bfloat16()
        self.b_qkv = torch.zeros(3 * hidden, dtype=torch.float32, device="cuda")
        self.inv_freq = rotary.rotary_frequencies(self.dim, base)
        self._w8 = None

    def plan(self, lengths, training=False):
        cu = packed.cu_seqlens(lengths)
        total = sum(lengths)
        return packed.PackedPlan(cu, cu, total, total, self.heads, self.heads, self.dim, self.causal, training)

    def _split(self, qkv):
        return qkv.view(-1, 3 * self.heads, self.dim).split(self.heads, dim=1)

    def _qkv(self, x, residual, eight_bits):
        if not eight_bits:
            y, h = rmsnorm.rms_norm_forward(x, self.w_norm, residual)
            return dinov2.qkv_linear(y, self.w_qkv, self.b_qkv), y, h
        if self._w8 is None:  # the weights' rows in 8 bits, laid out once
            scale = self.w_qkv.float().abs().amax(1, keepdim=True) / E4M3_MAX
            self._w8 = ((self.w_qkv.float() / scale).to(torch.float8_e4m3fn).t(), scale.t().contiguous())
        y8, scale, h = rmsnorm.rms_norm_forward_f8(x, self.w_norm, residual)
        qkv = torch._scaled_mm(y8, self._w8[0], scale_a=scale, scale_b=self._w8[1], out_dtype=torch.bfloat16)
        return qkv + self.b_qkv.bfloat16(), None, h

    def forward(self, x, residual, positions, plan, eight_bits=False):
        """``(O, h, saved)`` for packed tokens ``x [tokens, hidden]``."""
        qkv, y, h = self._qkv(x, residual, eight_bits)
        q, k, v = self._split(qkv)
        rotary.rotary_forward(q, k, positions, self.inv_freq, out=(q, k))  # in place
        out, lse = packed.packed_attention_forward(q, k, v, plan)
        return out.view(-1, self.hidden), h, (y, h, qkv, out, lse, positions, plan)

    def backward(self, grad_out, grad_h, saved):
        """``(grad of x and residual, grad w_norm, grad w_qkv, grad b_qkv)``."""
        y, h, qkv, out, lse, positions, plan = saved
        grad = torch.empty_like(qkv)
        gq, gk, gv = self._split(grad)
        packed.packed_attention_backward(grad_out.view_as(out), *self._split(qkv), out, lse, plan, grads=(gq, gk, gv))
        rotary.rotary_backward(gq, gk, positions, self.inv_freq, out=(gq, gk))
        grad_y = grad @ self.w_qkv
        gx, gw = rmsnorm.rms_norm_backward(grad_y, h, self.w_norm, grad_h=grad_h)
        return gx, gw, grad.t() @ y, grad.float().sum(0)


class Cache:
    """Keys and values of ``n`` sequences with room for ``room`` tokens each."""

    def __init__(self, layer: PackedAttentionLayer, n: int, room: int):
        self.k = torch.empty(n * room, layer.heads, layer.dim, dtype=torch.bfloat16, device="cuda")
        self.v = torch.empty_like(self.k)
        self.first = room * torch.arange(n + 1, dtype=torch.int32, device="cuda")
        self.one = torch.arange(n + 1, dtype=torch.int32, device="cuda")
        self.used = torch.zeros(n, dtype=torch.int32, device="cuda")
        self.room, self.length = room, 0  # the host counts along: every sequence grows by one a step

    def token(self, layer: PackedAttentionLayer, x, residual, eight_bits=False):
        """One new token of every sequence: ``x [n, hidden]`` → ``(O, h)``."""
        n = x.shape[0]
        if self.length == self.room:  # the next row is another sequence's, or none
            raise ValueError(f"the cache holds {self.room} tokens a sequence")
        self.length += 1
        q, k, v = layer._split(layer._qkv(x, residual, eight_bits)[0])
        h = x + residual
        q, k = rotary.rotary_forward(q, k, self.used, layer.inv_freq)  # the position is the number of tokens so far
        at = (self.first[:-1] + self.used).long()
        self.k[at], self.v[at] = k, v
        self.used += 1
        plan = packed.PackedPlan(self.one, self.first, n, self.k.shape[0], layer.heads, layer.heads, layer.dim,
                                 causal=True, used_k=self.used)
        return packed.packed_attention_forward(q, self.k, self.v, plan)[0].view(n, -1), h


def main():
    def timed(f, n=20):
        f()
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(n):
            f()
        b.record()
        torch.cuda.synchronize()
        return a.elapsed_time(b) / n * 1e3

    # images from 16x16 to 40x40 patches with their class tokens, one training step
    lengths = [1 + s * s for s in (40, 16, 32, 24, 37, 28, 20, 40)]
    layer = PackedAttentionLayer(384, 6)
    T = sum(lengths)
    x, r, g = (torch.randn(T, 384, device="cuda").bfloat16() for _ in range(3))
    pos = torch.cat([torch.arange(n) for n in lengths]).cuda()
    plan = layer.plan(lengths, training=True)
    out, h, saved = layer.forward(x, r, pos, plan)
    layer.backward(g, g, saved)
    print(f"images of {min(lengths)} to {max(lengths)} tokens ({T} in all): "
          f"forward {timed(lambda: layer.forward(x, r, pos, plan)):.0f} us, "
          f"backward {timed(lambda: layer.backward(g, g, saved)):.0f} us")

    # a causal tower, token by token
    tower, n = PackedAttentionLayer(768, 12, causal=True), 32
    for eight_bits in (False, True):
        cache = Cache(tower, n, 512)
        tokens = [torch.randn(n, 768, device="cuda").bfloat16() for _ in range(2)]
        us = timed(lambda: cache.token(tower, *tokens, eight_bits=eight_bits), 100)
        print(f"{n} sequences, one token each, {'8-bit' if eight_bits else 'bf16'} product: {us:.0f} us a step")


if __name__ == "__main__":
    main()
