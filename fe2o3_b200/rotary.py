"""Rotary positions: frequencies, also for contexts longer than a model was trained on, and the operator over them.

    rotary = Rotary(ctx, stream, 128, base=500000.0, scaling="yarn", factor=4.0, trained=8192)
    rotary.apply(q, k, positions, heads=32, kv_heads=8, dim=128)          # in place; rows [tokens][heads][dim]
    step = DecodeStep(cache, q, k, v, out, heads=32, rotary=rotary)       # inside a decode step (fe2o3_b200/kv_cache.py)
"""
import math

import numpy as np

from . import ROTARY_HALF, DeviceBuffer, prepare
from .kv_cache import _contiguous, _float_dtype, _numbers


def rotary_frequencies(rotary_dim, base=10000.0, scaling=None, factor=1.0, trained=None, fast=32.0, slow=1.0):
    """Radians a position of every pair, f32 [rotary_dim / 2], and the factor that sine and cosine are multiplied by.

    base ** (-2 i / rotary_dim), and with `scaling` for contexts `factor` times as long as the `trained` one:
      "linear"  positions are squeezed: every frequency by factor;
      "ntk"     the base grows so that the slowest pair turns factor times slower and the fastest as before;
      "yarn"    pairs that turn more than `fast` times in the trained context stay, those that turn less than `slow` times are squeezed by
                factor, those between in proportion to their number; sine and cosine times 0.1 ln(factor) + 1 (Peng, Quesnelle, Fan and Shippole, YaRN:
                Efficient Context Window Extension of Large Language Models, 2023, whose bounds of the ramp and smallest width of it are kept, since
                models were trained with them)."""
    if rotary_dim < 0 or rotary_dim % 2 or base <= 0 or factor < 1:
        raise ValueError("rotary_dim is even, base above 0 and factor at least 1")
    pairs = np.arange(0, rotary_dim, 2, dtype=np.float64)
    f = base ** (-pairs / max(rotary_dim, 1))
    if scaling in (None, "linear"):
        return (f / (factor if scaling else 1.0)).astype(np.float32), 1.0
    if scaling == "ntk":
        if rotary_dim < 4:
            raise ValueError("ntk needs two pairs")
        return ((base * factor ** (rotary_dim / (rotary_dim - 2))) ** (-pairs / rotary_dim)).astype(np.float32), 1.0
    if scaling == "yarn":
        if trained is None or trained < 1:
            raise ValueError("yarn needs the length of the trained context")

        def pair_that_turns(n):   # so many times in the trained context
            return rotary_dim * math.log(trained / (n * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(pair_that_turns(fast)), 0), min(math.ceil(pair_that_turns(slow)), rotary_dim - 1)
        ramp = np.clip((np.arange(len(pairs)) - low) / max(high - low, 0.001), 0, 1)
        return (f * (1 - ramp) + f / factor * ramp).astype(np.float32), 0.1 * math.log(factor) + 1
    raise ValueError(f"scaling is None, linear, ntk or yarn, not {scaling!r}")


class Rotary:
    """Frequencies on the device, and launches of `rotary_v1` with them."""

    def __init__(self, ctx, stream, rotary_dim, layout=ROTARY_HALF, **frequencies):
        self.ctx, self.stream, self.rotary_dim, self.layout = ctx, stream, rotary_dim, layout
        host, self.scale = rotary_frequencies(rotary_dim, **frequencies)
        self.frequencies = DeviceBuffer.from_host(stream, host) if rotary_dim else None

    def args(self):
        """The rotation's own arguments of `rotary_v1` and `kv_cache_rotary_append_v1`."""
        return dict(frequencies=self.frequencies, rotary_dim=self.rotary_dim, layout=self.layout, scale=self.scale)

    def prepare(self, q, k, positions, heads, kv_heads, dim, tokens, q_out=None, k_out=None, backward=False, dtype=None, strides=None, out_strides=None):
        """A prepared launch over rows [tokens][heads][dim] of q and [tokens][kv_heads][dim] of k (None: q alone), in place where no outputs are
        given; with strides ((q token, q head), (k token, k head)) in elements the rows are slices (address, elements)."""
        if k is None:
            kv_heads = 0
        _contiguous(q, k, q_out, k_out)
        _numbers(positions=positions)
        one = _float_dtype(q, dtype)
        for x in (k, q_out, k_out):
            if hasattr(x, "dtype") and _float_dtype(x, dtype) != one:
                raise TypeError(f"q, k and their outputs are of one type, got {q.dtype} and {x.dtype}")
        packed = ((heads * dim, dim), (kv_heads * dim, dim))
        (qt, qh), (kt, kh) = strides or packed
        (qot, qoh), (kot, koh) = out_strides or (packed if q_out is not None else strides or packed)
        return prepare(self.ctx, "rotary_v1", q=q, k=k, positions=positions, q_output=q if q_out is None else q_out, k_output=k if k_out is None else k_out,
                       tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, dtype=one, backward=int(backward), q_token_stride=qt, q_head_stride=qh,
                       k_token_stride=kt, k_head_stride=kh, q_output_token_stride=qot, q_output_head_stride=qoh, k_output_token_stride=kot,
                       k_output_head_stride=koh, **self.args())

    def apply(self, q, k, positions, heads, kv_heads, dim, tokens=None, **kw):
        """The same, launched once on the stream.  tokens: by the size of q, where its rows are packed."""
        if tokens is None:
            if isinstance(q, tuple) or kw.get("strides"):
                raise ValueError("rows inside wider storage need tokens=")
            size = q.numel() if hasattr(q, "numel") else len(q)
            tokens = size // (heads * dim)
        p = self.prepare(q, k, positions, heads, kv_heads, dim, tokens, **kw)
        try:
            p.launch(self.stream)
        finally:
            p.destroy()

    def free(self):
        if self.frequencies is not None:
            self.frequencies.free()
