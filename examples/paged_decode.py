"""Decoding with a paged key-value cache: one attention block, prompts and then token by token.

For every sequence: the prompt's rows go through one fused projection (`tiled_gemm_v1`: x [tokens][d] times W [d][3 d], f32
out), their keys and values into the cache straight from the fused rows (`kv_cache_append_v1` with strides), and the
prompt's own outputs come from `flash_attention_v1`, causal, over the cached rows read back (`kv_cache_read_v1`).  Then each
step projects one token a sequence, appends it and attends (`paged_attention_v1`); the attended row, as bf16, is the next
step's input.  At the end the last step's outputs are compared with attention over all rows in f64.

With --rotary the book of pages lies on the device (`kv_pages_v1`), queries and keys are turned by their positions on the way into the cache
(`kv_cache_rotary_append_v1`), and a whole step, the projection in front of it too, is one CUDA graph.

    python examples/paged_decode.py --sequences 16 --prompt 500 --steps 64 --heads 16 --dim 64 --format e4m3
"""
import argparse
import os
import sys
import time

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def main(argv=None):
    import torch
    import fe2o3_b200 as fe
    from fe2o3_b200.kv_cache import DecodeStep, PagedKvCache
    from fe2o3_b200.rotary import Rotary
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--sequences", type=int, default=16, help="a multiple of 16 (rows of a tiled GEMM)")
    ap.add_argument("--prompt", type=int, default=500)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--heads", type=int, default=16)
    ap.add_argument("--dim", type=int, default=64)
    ap.add_argument("--page-size", type=int, default=16)
    ap.add_argument("--format", choices=("bf16", "e4m3", "i8", "e2m1"), default="bf16")
    ap.add_argument("--rotary", type=int, default=0, help="columns of a head that positions turn; 0: none")
    a = ap.parse_args(argv)
    ctx = fe.GpuContext(0)
    stream = ctx.default_stream()   # torch's default stream too: its copies and these launches are in order
    B, T, H, D = a.sequences, a.prompt, a.heads, a.dim
    d = H * D
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    w = (torch.randn(d, 3 * d, generator=g, device="cuda") * d ** -0.5).bfloat16()
    x = torch.randn(B * T, d, generator=g, device="cuda").bfloat16()

    def projection(rows, fused):   # fused [rows][3][heads][dim] f32: queries, keys, values
        return fe.prepare(ctx, "tiled_gemm_v1", a=rows, b=w, c=fused, m=rows.shape[0], n=3 * d, k=d)

    def part(fused, i):            # rows of one of the three inside the fused ones: address, elements
        return (fused.data_ptr() + 4 * i * d, (fused.shape[0] - 1) * 3 * d + d)

    cache = PagedKvCache(ctx, stream, B, T + a.steps, H, D, a.page_size, format={"bf16": fe.KV_BF16, "e4m3": fe.KV_E4M3, "i8": fe.KV_I8, "e2m1": fe.KV_E2M1}[a.format],
                         tokens=B * T if a.rotary else None)
    rotary = Rotary(ctx, stream, a.rotary) if a.rotary else None
    strides = ((3 * d, D), (3 * d, D))

    # prompts
    fused = torch.zeros(B * T, 3 * d, device="cuda")
    projection(x, fused).launch(stream)
    cache.extend([T] * B)
    q = torch.zeros(B, T, H, D, device="cuda")
    cache.append(part(fused, 1), part(fused, 2), dtype=fe.DTYPE_F32, strides=strides, **(dict(q=part(fused, 0), q_out=q, heads=H, rotary=rotary, q_strides=(3 * d, D)) if rotary else {}))
    if not rotary:
        q = fused.view(B, T, 3, H, D)[:, :, 0]
    k, v = (torch.zeros(B, T, H, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    cache.read(k, v, [T] * B)
    k, v = (t.transpose(1, 2).contiguous() for t in (k, v))
    q = q.bfloat16().transpose(1, 2).contiguous()
    prompt_out = torch.zeros(B, H, T, D, device="cuda")
    fe.prepare(ctx, "flash_attention_v1", q=q, k=k, v=v, output=prompt_out, batch=B, heads=H, seq=T, dim=D, scale=D ** -0.5, causal=1,
               input_dtype=fe.DTYPE_BF16).launch(stream)

    # steps
    row, new, out = torch.zeros(B, d, dtype=torch.bfloat16, device="cuda"), torch.zeros(B, 3 * d, device="cuda"), torch.zeros(B, H, D, dtype=torch.bfloat16, device="cuda")
    row.copy_(prompt_out[:, :, -1].reshape(B, d))
    project = projection(row, new)
    step = DecodeStep(cache, part(new, 0), part(new, 1), part(new, 2), out, heads=H, dtype=fe.DTYPE_F32, out_dtype=fe.DTYPE_BF16,
                      strides=strides, q_strides=(3 * d, D), rotary=rotary)
    graph = torch.cuda.CUDAGraph()
    stream.synchronize()
    if rotary:
        with torch.cuda.graph(graph):
            on = ctx.wrap_stream(torch.cuda.current_stream().cuda_stream)
            project.launch(on)
            step.run(on)
            row.copy_(out.view(B, d))
    torch.cuda.synchronize()
    began = time.perf_counter()
    for _ in range(a.steps):
        if rotary:
            graph.replay()
            continue
        project.launch(stream)
        step.run()
        row.copy_(out.view(B, d))
    stream.synchronize()
    took = time.perf_counter() - began
    status = ctx.take_kernel_status(stream)
    assert status == 0, status

    # the last step again, from the rows that the cache holds
    n = T + a.steps
    k, v = (torch.zeros(B, n, H, D, device="cuda") for _ in range(2))
    cache.read(k, v, [n] * B)
    q = torch.as_tensor(step.turned, device="cuda").view(B, H, D) if rotary else new.view(B, 3, H, D)[:, 0]
    s = torch.einsum("bhd,bnhd->bhn", q.double(), k.double()) * D ** -0.5
    want = torch.einsum("bhn,bnhd->bhd", torch.softmax(s, -1), v.double())
    off = float((out.double() - want).abs().max() / want.abs().max())
    per_token = cache.k_cache.dtype.itemsize * 2 * H * (D * 9 // 16 if a.format == "e2m1" else D) + (8 * H if a.format != "bf16" else 0)
    print(f"{B} sequences, prompts of {T}, {a.steps} steps: {took / a.steps * 1e6:.1f} us a step (host included); cache {a.format}, "
          f"{per_token} bytes a token; last step off by {off:.1e} of its largest value")
    step.destroy()
    project.destroy()
    cache.free()
    return off


if __name__ == "__main__":
    main()
