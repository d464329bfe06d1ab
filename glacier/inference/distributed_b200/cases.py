"""Small single-kernel workloads of the hot path, for kernel profiles.

    python -m glacier.inference.distributed_b200.cases <case> [--reps N]

Each case builds its inputs on cuda:0 (weights by the library's seeded
synthetic generator, the shapes of the Mixtral-8x7B, Qwen2-57B-A14B,
Qwen2.5-14B and Mixtral-8x22B layers), runs three warm-up calls and then ``reps`` calls of the
one kernel family it names, and exits 0.  Inputs that a kernel streams are
larger than the 126 MB L2 (rotating copies where one copy is smaller), so the
DRAM counters of a capture describe HBM traffic.  A capture names the kernel
with ``-k`` and skips the warm-up launches with ``-s``; the launches each case
makes per call are listed in CASES.
"""
from __future__ import annotations

import argparse
import sys

import numpy as np

MIXTRAL = dict(D=4096, F=14336, E=8, k=2, seed=20241201)
QWEN = dict(D=3584, F=2560, E=64, k=8, Fs=20480, seed=20241202)
QWEN14B = dict(D=5120, FF=13824, Hq=40, Hkv=8, max_len=2048, seed=20241203)
MIXTRAL22B = dict(D=6144, F=16384, E=8, k=2, Hq=48, Hkv=8, max_len=4096, seed=20241204)

# case -> (kernels launched per call, one line of what it runs)
CASES = {
    "gemv_k4096": ("q4k_gemv_kernel x1", "y = W x, K=4096, N=28672 (gate+up rows of one expert pair), 4 rotating 66 MB copies"),
    "gemv_k14336": ("q4k_gemv_kernel x1", "y = W x, K=14336, N=8192 (down rows of two experts), 4 rotating 66 MB copies"),
    "gemv_chain": ("q4k_gemv_chain_kernel x1",
                   "64 GEMVs K=4096, N=28672 in one launch, each behind a grid-wide wait, 4 rotating 66 MB copies"),
    "router": ("router_kernel x1", "Mixtral router: T=64, D=4096, E=8, top-2 renormalised, RMSNorm"),
    "router_wide": ("router_wide_kernel x1", "Qwen2-57B router: T=16, D=3584, E=64, top-8, RMSNorm"),
    "wire": ("wire_quantize_kernel x1 + wire_dequantize_kernel x1",
             "symmetric INT8 per token, T=4096, D=4096 (64 MB fp32 in)"),
    "dispatch": ("dispatch_plan_kernel x1", "histogram / scan / stable permute of P=8192 slot ids over E=64"),
    "attention": ("attn_decode_kernel x1 (a 16- or 8-CTA cluster per KV head)",
                  "40 query / 8 KV heads x 128, position 2047 of a 2048-row fp16 cache, 16 rotating layer caches"),
    "kv_plan": ("kv_plan_flat_kernel x1", "page plan of 2048 requests over 16-row pages, a tenth of them chunks of prompts"),
    "rope_append": ("rope_append_kernel x1",
                    "RoPE and store of 8192 rows, 48 query / 8 KV heads x 128, fp16 queries out, 16-row pages"),
    "attn_prompt": ("attn_tiles_kernel x1", "one prompt of 8192 tokens, 48 query / 8 KV heads x 128, fp16 queries"),
    "attn_prompt_f32": ("attn_tiles_kernel x1", "one prompt of 4096 tokens, 40 query / 8 KV heads x 128, fp32 queries"),
    "attn_chunk": ("attn_tiles_kernel x1 + attn_tiles_join_kernel x1",
                   "512 new tokens of a 16384-row sequence, 40 query / 8 KV heads x 128, fp32 queries, 64-row pages"),
    "attn_paged": ("attn_rows_kernel x1",
                   "decode tokens of 64 sequences of 128 to 8192 rows, 48 query / 8 KV heads x 128, fp16 queries, 16-row pages"),
    "decode_fused": ("moe_decode_fused_kernel x1", "Mixtral-8x7B layer decode, T=1 (one launch)"),
    "decode_wide": ("moe_decode_wide_kernel x1", "Qwen2-57B-A14B layer decode with its shared expert, T=1 (one launch)"),
    "stage": ("per layer: attn_decode_kernel x1, q4k_gemv_chain_kernel x1",
              "Qwen2.5-14B dense stage of 2 layers, one token at position 2040"),
    "moe_stage": ("per layer: attn_decode_kernel x1, q4k_gemv_chain_kernel x2, moe_decode_fused_kernel x1",
                  "Mixtral-8x22B mixture-of-experts stage of 2 layers, one token at position 4090"),
}


def _stream(torch):
    from .api import torch_stream_handle
    s = torch.cuda.Stream()
    return s, torch_stream_handle(s)


def case_gemv(torch, glc, K, N, reps):
    w = MIXTRAL
    worker = glc.GpuExpertStageWorker(w["D"], w["F"], w["E"], w["k"], max_tokens=1)
    worker.synth_layer(0, w["seed"])
    g, _u, d, _r = worker.layer_device_ptrs(0)
    base, step = (g, 2 * w["F"] * glc.q4k_row_bytes(w["D"])) if K == w["D"] else \
        (d, 2 * w["D"] * glc.q4k_row_bytes(w["F"]))
    x = torch.from_numpy(np.random.default_rng(7).standard_normal(K).astype(np.float32)).cuda()
    y = torch.empty(N, device="cuda")
    st, s = _stream(torch)
    with torch.cuda.stream(st):
        for i in range(3 + reps):
            glc.gemv_q4k_dev(base + (i % 4) * step, x.data_ptr(), y.data_ptr(), K, N, s)
    torch.cuda.synchronize()
    worker.dispose()


def case_gemv_chain(torch, glc, reps):
    w = MIXTRAL
    K, N = w["D"], 2 * w["F"]
    worker = glc.GpuExpertStageWorker(w["D"], w["F"], w["E"], w["k"], max_tokens=1)
    worker.synth_layer(0, w["seed"])
    g = worker.layer_device_ptrs(0)[0]
    step = N * glc.q4k_row_bytes(K)
    x = torch.from_numpy(np.random.default_rng(7).standard_normal(K).astype(np.float32)).cuda()
    y = torch.empty(N, device="cuda")
    jobs = [dict(W=g + (i % 4) * step, x=x.data_ptr(), y=y.data_ptr(), K=K, N=N, after_previous=i > 0)
            for i in range(64)]
    st, s = _stream(torch)
    with torch.cuda.stream(st):
        for _ in range(3 + reps):
            glc.gemv_q4k_chain_dev(jobs, s)
    torch.cuda.synchronize()
    glc.gemv_poll_error()
    worker.dispose()


def case_router(torch, glc, wide, reps):
    w = QWEN if wide else MIXTRAL
    T = 16 if wide else 64
    D, E, k = w["D"], w["E"], w["k"]
    rng = np.random.default_rng(3)
    x = torch.from_numpy(rng.standard_normal((T, D)).astype(np.float32)).cuda()
    r = torch.from_numpy((rng.standard_normal((D, E)) * 0.02).astype(np.float32)).cuda()
    xin = torch.empty(T, D, device="cuda")
    lg = torch.empty(T, E, device="cuda")
    ids = torch.empty(T, k, dtype=torch.int32, device="cuda")
    wt = torch.empty(T, k, device="cuda")
    st, s = _stream(torch)
    with torch.cuda.stream(st):
        for _ in range(3 + reps):
            glc.router_topk_dev(x.data_ptr(), r.data_ptr(), T, D, E, k, not wide, True, xin.data_ptr(),
                                lg.data_ptr(), ids.data_ptr(), wt.data_ptr(), s)
    torch.cuda.synchronize()


def case_wire(torch, glc, reps):
    T, D, mode = 4096, 4096, 2  # INT8
    x = torch.randn(T, D, device="cuda")
    nb = glc.QuantizationKernels.GetPackedBatchBytes(mode, D, T)
    buf = torch.empty(nb, dtype=torch.uint8, device="cuda")
    y = torch.empty(T, D, device="cuda")
    st, s = _stream(torch)
    with torch.cuda.stream(st):
        for _ in range(3 + reps):
            glc.QuantizationKernels.quantize_dev(mode, x.data_ptr(), T, D, buf.data_ptr(), s)
            glc.QuantizationKernels.dequantize_dev(mode, buf.data_ptr(), T, D, y.data_ptr(), s)
    torch.cuda.synchronize()


def case_dispatch(torch, glc, reps):
    P, E = 8192, 64
    ids = torch.from_numpy(np.random.default_rng(5).integers(0, E, P).astype(np.int32)).cuda()
    counts = torch.empty(E, dtype=torch.int32, device="cuda")
    offs = torch.empty(E + 1, dtype=torch.int32, device="cuda")
    perm = torch.empty(P, dtype=torch.int32, device="cuda")
    inv = torch.empty(P, dtype=torch.int32, device="cuda")
    st, s = _stream(torch)
    with torch.cuda.stream(st):
        for _ in range(3 + reps):
            glc.dispatch_plan_dev(ids.data_ptr(), P, E, counts.data_ptr(), offs.data_ptr(), perm.data_ptr(),
                                  inv.data_ptr(), s)
    torch.cuda.synchronize()


def case_attention(torch, glc, reps):
    q = QWEN14B
    Hq, Hkv, L = q["Hq"], q["Hkv"], q["max_len"]
    ncache = 16  # 16 x 2 x 4 MB: the caches of 16 layers, more than L2
    kc = [(torch.randn(Hkv, L, 128, device="cuda") * 0.5).half() for _ in range(ncache)]
    vc = [(torch.randn(Hkv, L, 128, device="cuda") * 0.5).half() for _ in range(ncache)]
    qv = torch.randn(Hq * 128, device="cuda")
    kn = torch.randn(Hkv * 128, device="cuda")
    vn = torch.randn(Hkv * 128, device="cuda")
    out = torch.empty(Hq * 128, device="cuda")
    wb = glc.attn_workspace_bytes(Hq, Hkv, L)
    work = torch.empty(wb // 4 + 1, device="cuda")
    st, s = _stream(torch)
    with torch.cuda.stream(st):
        for i in range(3 + reps):
            c = i % ncache
            glc.attn_decode_dev(qv.data_ptr(), kn.data_ptr(), vn.data_ptr(), kc[c].data_ptr(), vc[c].data_ptr(),
                                Hq, Hkv, L, L - 1, 1e6, out.data_ptr(), work.data_ptr(), wb, stream=s)
    torch.cuda.synchronize()


def case_kv_plan(torch, glc, reps):
    B, ps, width, rng = 2048, 16, 544, np.random.default_rng(11)
    ctx = rng.integers(0, 8193, B)
    new = np.where(rng.random(B) < 0.1, rng.integers(1, 513, B), 1)
    held, T = -(-ctx // ps), int(new.sum())
    ids = rng.permutation(int(held.sum()) + T).astype(np.int32)
    table = np.zeros((B, width), np.int32)
    at = np.concatenate([[0], np.cumsum(held)])
    for b in range(B):
        table[b, :held[b]] = ids[at[b]:at[b + 1]]
    pool = ids[at[-1]:]
    d = [torch.from_numpy(a.astype(np.int32)).cuda() for a in (ctx, new, table, pool, np.array([len(pool)]))]
    o = [torch.empty(n, dtype=torch.int32, device="cuda") for n in (1, B + 1, B, T, 1)]
    slots = torch.empty(T, dtype=torch.int64, device="cuda")
    st, s = _stream(torch)
    with torch.cuda.stream(st):
        for _ in range(3 + reps):
            glc.kv_plan_dev(d[0].data_ptr(), d[1].data_ptr(), B, ps, d[2].data_ptr(), width, d[3].data_ptr(), len(pool),
                            d[4].data_ptr(), o[0].data_ptr(), T, o[1].data_ptr(), o[2].data_ptr(), o[3].data_ptr(),
                            slots.data_ptr(), o[4].data_ptr(), stream=s)
    torch.cuda.synchronize()


def _pages(torch, glc, lens, Hkv, ps):
    """A cache of random rows in shuffled pages, and the sequences' page table."""
    held = [-(-n // ps) for n in lens]
    n_pages, width = sum(held), max(held)
    kv = [torch.randn(n_pages, Hkv, ps, 128, device="cuda", dtype=torch.float16) for _ in range(2)]
    ids = np.random.default_rng(12).permutation(n_pages).astype(np.int32)
    table, at = np.zeros((len(lens), width), np.int32), 0
    for b, n in enumerate(held):
        table[b, :n] = ids[at:at + n]
        at += n
    return kv, glc.KvPages(kv[0].data_ptr(), kv[1].data_ptr(), n_pages, ps, Hkv), torch.from_numpy(table).cuda()


def case_rope_append(torch, glc, reps):
    T, Hq, Hkv, row = 8192, 48, 8, 64 * 128
    x = torch.randn(T, row, device="cuda")                  # fused q, k, v rows: 268 MB
    keep, cache, _ = _pages(torch, glc, [T], Hkv, 16)
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    slots = torch.randperm(T, device="cuda")
    q = torch.empty(T, Hq * 128, device="cuda", dtype=torch.float16)
    p = x.data_ptr()
    st, s = _stream(torch)
    with torch.cuda.stream(st):
        for _ in range(3 + reps):
            glc.rope_append_dev(p, row, p + Hq * 512, p + (Hq + Hkv) * 512, row, T, Hq, Hkv, pos.data_ptr(),
                                slots.data_ptr(), 1e6, cache, q.data_ptr(), glc.GGUF_F16, stream=s)
    torch.cuda.synchronize()
    glc.paged_poll_error()


def case_attn_prompt(torch, glc, T, Hq, f32, reps):
    Hkv = 8
    q = torch.randn(T, Hq * 128, device="cuda", dtype=torch.float32 if f32 else torch.float16)
    k, v = (torch.randn(T, Hkv * 128, device="cuda", dtype=torch.float16) for _ in range(2))
    out = torch.empty_like(q)
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    st, s = _stream(torch)
    with torch.cuda.stream(st):
        for _ in range(3 + reps):
            glc.attn_prompt_dev(q.data_ptr(), glc.GGUF_F32 if f32 else glc.GGUF_F16, Hq * 128, k.data_ptr(), v.data_ptr(),
                                Hkv * 128, cu.data_ptr(), 1, T, Hq, Hkv, out.data_ptr(), Hq * 128, stream=s)
    torch.cuda.synchronize()
    glc.paged_poll_error()


def case_attn_paged(torch, glc, new, lens, Hq, ps, f32, reps):
    Hkv, B, T = 8, len(lens), sum(new)
    keep, cache, table = _pages(torch, glc, lens, Hkv, ps)
    q = torch.randn(T, Hq * 128, device="cuda", dtype=torch.float32 if f32 else torch.float16)
    out = torch.empty_like(q)
    cu = torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).cuda()
    kv = torch.tensor(lens, dtype=torch.int32, device="cuda")
    wb = glc.attn_paged_workspace_bytes(Hq, Hkv, B, T, max(new))
    work = torch.empty(wb, dtype=torch.uint8, device="cuda")
    st, s = _stream(torch)
    with torch.cuda.stream(st):
        for _ in range(3 + reps):
            glc.attn_paged_dev(q.data_ptr(), glc.GGUF_F32 if f32 else glc.GGUF_F16, Hq * 128, cache, table.data_ptr(),
                               table.shape[1], cu.data_ptr(), kv.data_ptr(), B, T, max(new), Hq, out.data_ptr(), Hq * 128,
                               work.data_ptr(), wb, stream=s)
    torch.cuda.synchronize()
    glc.paged_poll_error()


def case_decode(torch, glc, wide, reps):
    w = QWEN if wide else MIXTRAL
    worker = glc.GpuExpertStageWorker(w["D"], w["F"], w["E"], w["k"], shared_ffn_dim=w.get("Fs", 0),
                                      renormalize=not wide, max_tokens=1)
    worker.synth_layer(0, w["seed"])
    xs = [torch.randn(1, w["D"], device="cuda") for _ in range(4)]
    out = torch.empty(1, w["D"], device="cuda")
    st, s = _stream(torch)
    with torch.cuda.stream(st):
        for i in range(3 + reps):
            worker.forward_dev(0, xs[i % 4].data_ptr(), 1, 3, out.data_ptr(), stream=s)  # RMSNorm | residual
    torch.cuda.synchronize()
    worker.poll_error()
    worker.dispose()


def case_stage(torch, glc, reps):
    q = QWEN14B
    st_ = glc.DenseStage(q["D"], q["FF"], q["Hq"], q["Hkv"], 0, 2, q["max_len"], 1e6, 1e-6)
    for l in range(2):
        st_.synth_layer(l, q["seed"])
    x = torch.randn(q["D"], device="cuda")
    y = torch.empty(q["D"], device="cuda")
    st, s = _stream(torch)
    with torch.cuda.stream(st):
        for i in range(3 + reps):
            st_.forward_dev(2040 + i % 4, x_in_ptr=x.data_ptr(), x_out_ptr=y.data_ptr(), stream=s)
    torch.cuda.synchronize()
    st_.poll_error()
    st_.dispose()


def case_moe_stage(torch, glc, reps):
    q = MIXTRAL22B
    st_ = glc.DenseStage(q["D"], 0, q["Hq"], q["Hkv"], 0, 2, q["max_len"], 1e6, 1e-5, num_experts=q["E"],
                         top_k=q["k"], expert_ffn_dim=q["F"], moe_renormalize=True)
    for l in range(2):
        st_.synth_layer(l, q["seed"])
    x = torch.randn(q["D"], device="cuda")
    y = torch.empty(q["D"], device="cuda")
    st, s = _stream(torch)
    with torch.cuda.stream(st):
        for i in range(3 + reps):
            st_.forward_dev(4090 + i % 4, x_in_ptr=x.data_ptr(), x_out_ptr=y.data_ptr(), stream=s)
    torch.cuda.synchronize()
    st_.poll_error()
    st_.dispose()


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("case", choices=sorted(CASES))
    ap.add_argument("--reps", type=int, default=3)
    a = ap.parse_args(argv)
    import torch

    from . import api as glc
    if not torch.cuda.is_available():
        print("a CUDA device is required", file=sys.stderr)
        return 2
    torch.cuda.set_device(0)
    c, n = a.case, a.reps
    if c == "gemv_k4096":
        case_gemv(torch, glc, 4096, 28672, n)
    elif c == "gemv_k14336":
        case_gemv(torch, glc, 14336, 8192, n)
    elif c == "gemv_chain":
        case_gemv_chain(torch, glc, n)
    elif c in ("router", "router_wide"):
        case_router(torch, glc, c == "router_wide", n)
    elif c == "wire":
        case_wire(torch, glc, n)
    elif c == "dispatch":
        case_dispatch(torch, glc, n)
    elif c == "attention":
        case_attention(torch, glc, n)
    elif c == "kv_plan":
        case_kv_plan(torch, glc, n)
    elif c == "rope_append":
        case_rope_append(torch, glc, n)
    elif c == "attn_prompt":
        case_attn_prompt(torch, glc, 8192, 48, False, n)
    elif c == "attn_prompt_f32":
        case_attn_prompt(torch, glc, 4096, 40, True, n)
    elif c == "attn_chunk":
        case_attn_paged(torch, glc, [512], [16384], 40, 64, True, n)
    elif c == "attn_paged":
        case_attn_paged(torch, glc, [1] * 64, [128 * (1 + 13 * i % 64) for i in range(64)], 48, 16, False, n)
    elif c in ("decode_fused", "decode_wide"):
        case_decode(torch, glc, c == "decode_wide", n)
    elif c == "stage":
        case_stage(torch, glc, n)
    elif c == "moe_stage":
        case_moe_stage(torch, glc, n)
    print(f"{c}: {CASES[c][0]} per call, {3 + n} calls: ok")
    return 0


if __name__ == "__main__":
    sys.exit(main())
