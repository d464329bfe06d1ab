"""CPU restatement of the paged-cache operators (float64 numpy, plain loops).

TEST INFRASTRUCTURE ONLY: imported by tests/ as the CPU reference for
glc_kv_plan_dev, glc_rope_append_dev, glc_attn_prompt_dev and
glc_attn_paged_dev; the product package never imports it.

Parity unpinned: the reference has no paged cache and runs one sequence one
token at a time (DistributedPipelineCoordinator.cs:72-137), so this module
states the semantics the kernels implement.
"""
from __future__ import annotations

import numpy as np

from .attention import rope


def plan(ctx, new, page_size, table, free_list, free_count, T):
    """Returns (table, free_list, left, cu, kv_lens, positions, slots, status)."""
    table, pool = np.array(table, copy=True), np.array(free_list, copy=True)
    B, width = table.shape
    need_pages = lambda x: -(-x // page_size)  # noqa: E731
    stack = list(pool[:free_count])
    for i in range(B):
        if new[i] < 0:
            stack += list(table[i, :need_pages(int(ctx[i]))])
    pool[free_count:len(stack)] = stack[free_count:]
    avail, wanted, status = len(stack), 0, 0
    cu, kv = [0], []
    pos, slots = np.zeros(T, np.int32), np.full(T, -1, np.int64)
    for i in range(B):
        c, a = int(ctx[i]), max(int(new[i]), 0)
        t0 = cu[-1]
        cu.append(t0 + a)
        have, want = need_pages(c), need_pages(c + a)
        served = new[i] >= 0 and t0 + a <= T and want <= width
        if served:
            wanted += want - have
            served = want == have or wanted <= avail
        if not served:
            kv.append(0)
            status += int(new[i] >= 0)
            continue
        for col in range(have, want):
            table[i, col] = stack.pop()
        kv.append(c + a)
        for j in range(a):
            pos[t0 + j] = c + j
            slots[t0 + j] = int(table[i, (c + j) // page_size]) * page_size + (c + j) % page_size
    return (table, pool, len(stack), np.minimum(cu, T).astype(np.int32), np.array(kv, np.int32), pos, slots, status)


def rotate(x, positions, theta):
    """Rotate-half RoPE of x [T][heads][d] at positions [T], float64."""
    out = np.empty(x.shape, np.float64)
    for t in range(x.shape[0]):
        out[t] = rope(x[t], int(positions[t]), theta)
    return out


def attend(q, k, v, first, scale):
    """q [n][Hq][d], k / v [L][Hkv][d]: query i sees keys j <= first + i.  Returns
    (out, bound parts): out float64, and per output |w| @ |v|, the largest
    weight times sum |v|, and the largest scale * sum |q||k| of a seen key."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    n, Hq, d = q.shape
    G = Hq // k.shape[1]
    out, wv, peak = np.zeros((n, Hq, d)), np.zeros((n, Hq, d)), np.zeros((n, Hq, d))
    mag = np.zeros((n, Hq, 1))
    for h in range(Hq):
        kh, vh = k[:, h // G], v[:, h // G]
        for i in range(n):
            see = min(first + i + 1, k.shape[0])
            if see <= 0:
                continue
            s = scale * (kh[:see] @ q[i, h])
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i, h] = w @ vh[:see]
            wv[i, h] = w @ np.abs(vh[:see])
            peak[i, h] = w.max() * np.abs(vh[:see]).sum(0)
            mag[i, h] = scale * (np.abs(kh[:see]) @ np.abs(q[i, h])).max()
    return out, wv, peak, mag


def attend_tolerance(out, wv, peak, mag, L, f32):
    """Elementwise error bound of the kernels' arithmetic against attend().

    A score carries 8 tensor-core steps of 16 products in fp32 (at most 24
    roundings of 2^-23 of sum |q||k|), the row factor and the difference to the
    maximum (3 more), and for fp32 queries the two halves' 2^-22; numerator and
    denominator both feel it.  The exponential is good to 2^-21.  A weight is
    rounded to fp16 (2^-11) or kept as two halves (2^-21), with an absolute
    floor: fp16's half step below its normal range is 2^-25, and weights are
    kept as 2^4 p (fp16 queries on tiles) or 2^10 p, p relative to a value not
    above the row's largest: 2^-29 (fp16) or 2^-35 of the largest, doubled
    for the sum's share.  The sum over keys takes L / 16 steps
    of at most 32 roundings, and rescaling and merging at most 32 more.  The
    output is rounded once to its type."""
    score = mag * (27 * 2.0 ** -23 + (2.0 ** -21 if f32 else 0.0))
    weight = 2 * score + 2.0 ** -20 + (2.0 ** -21 if f32 else 2.0 ** -11)
    total = weight + (L / 16 + 64) * 2.0 ** -23
    final = 2.0 ** -24 if f32 else 2.0 ** -11
    return wv * total + np.abs(out) * final + peak * (2.0 ** -34 if f32 else 2.0 ** -28) + (1e-30 if f32 else 2.0 ** -25)
