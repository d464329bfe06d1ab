"""The paged-cache serving operators, as one list of cases to time and compare.

Four operators that a serving step calls one after another: the page plan (block
tables and slot maps from request lengths), rotary positions with the store of
the new keys and values into the paged cache, causal attention over packed
prompts, and attention of new tokens over the paged cache (chunks of a prompt
and single decode tokens alike).

``run`` computes an operator in elementary torch operations where ``own`` is
false and calls the library where it is true; ``exact`` states each definition
once more in 64 bits.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

HD = 128        # head dimension of the library's caches
THETA = 1e6     # rotary base
DEV = "cuda"


# ------------------------------------------------------------------ the cases
def _text(values) -> str:
    return ",".join(str(int(v)) for v in values)


def _ints(text: str) -> list[int]:
    return [int(t) for t in text.split(",")]


def _ragged(n: int, lo: int, hi: int, salt: int) -> str:
    """n lengths spread over [lo, hi] on a logarithmic scale, fixed by salt."""
    r = np.random.default_rng(salt)
    v = np.exp(r.uniform(math.log(lo), math.log(hi + 1), size=n)).astype(np.int64)
    return _text(np.clip(v, lo, hi))


def listed() -> list[dict]:
    return [
        # one decode step of 64 running requests: one new token each, a page now and then
        {"name": "plan_decode_64", "op": "plan", "requests": 64, "page_size": 16, "max_ctx": 8192, "max_new": 1,
         "prompts": 0.0, "done": 0.0, "rows": 64},
        # a large server's step: 2048 requests, a tenth of them chunks of prompts, some finished ones giving pages back
        {"name": "plan_mixed_2048", "op": "plan", "requests": 2048, "page_size": 16, "max_ctx": 8192, "max_new": 512,
         "prompts": 0.1, "done": 0.05, "rows": 40000},
        # the single new token of one request (Qwen2.5-14B heads)
        {"name": "append_one", "op": "append", "rows": 1, "heads": 40, "kv_heads": 8, "page_size": 16, "q_type": "f32",
         "packed": False, "pad": 0},
        # a step's chunk of prompts (Mixtral-8x22B heads), keys and values kept in packed form too
        {"name": "append_8192", "op": "append", "rows": 8192, "heads": 48, "kv_heads": 8, "page_size": 64,
         "q_type": "f16", "packed": True, "pad": 37},
        # one short question
        {"name": "prompt_short", "op": "prompt", "lens": "33", "heads": 40, "kv_heads": 8, "q_type": "f32", "pad": 0},
        # a ragged batch of prompts packed back to back, an empty one among them
        {"name": "prompt_packed", "op": "prompt", "lens": "517,1,2048,130,0,63,999,1300,257,64,801,333", "heads": 48,
         "kv_heads": 8, "q_type": "f16", "pad": 19},
        # documents in full-precision activations (Qwen2.5-14B heads)
        {"name": "prompt_docs_f32", "op": "prompt", "lens": "2048,1777,4099", "heads": 40, "kv_heads": 8,
         "q_type": "f32", "pad": 0},
        # one long document (Mixtral-8x22B heads)
        {"name": "prompt_16k", "op": "prompt", "lens": "16384", "heads": 48, "kv_heads": 8, "q_type": "f16", "pad": 0},
        # one request's decode token at a 2048-row cache (Qwen2.5-14B heads)
        {"name": "decode_one", "op": "paged", "new": "1", "ctx": "2047", "heads": 40, "kv_heads": 8, "page_size": 16,
         "q_type": "f32", "pad": 0},
        # a decode batch of 64 requests of very different lengths (Mixtral-8x22B heads)
        {"name": "decode_64", "op": "paged", "new": _text([1] * 64), "ctx": _ragged(64, 100, 16000, 5), "heads": 48,
         "kv_heads": 8, "page_size": 16, "q_type": "f16", "pad": 0},
        # the next chunk of a long document
        {"name": "chunk_512_of_32k", "op": "paged", "new": "512", "ctx": "32001", "heads": 40, "kv_heads": 8,
         "page_size": 64, "q_type": "f32", "pad": 0},
        # a mixed step: two chunks of prompts next to 48 decoding requests (28 query heads over 4)
        {"name": "mixed_50", "op": "paged", "new": "1000,300," + _text([1] * 48),
         "ctx": "0,5000," + _ragged(48, 50, 8000, 9), "heads": 28, "kv_heads": 4, "page_size": 32, "q_type": "f16",
         "pad": 11},
    ]


_HEADS = [(40, 8), (48, 8), (32, 8), (28, 4), (64, 8), (5, 1), (8, 8), (6, 2)]


def _log(rng, lo, hi) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    op = rng.choice(["plan", "append", "prompt", "prompt", "paged", "paged", "paged"])
    heads, kv_heads = rng.choice(_HEADS)
    page = rng.choice([16, 32, 64, 128, 256])
    kind = rng.choice(["f32", "f16"])
    pad = rng.choice([0, 0, 1, 29])
    if op == "plan":
        n = _log(rng, 1, 2048)
        new = _log(rng, 1, 512)
        return {"op": op, "requests": n, "page_size": page, "max_ctx": _log(rng, 16, 8192), "max_new": new,
                "prompts": rng.choice([0.0, 0.1, 1.0]) if n * new < 40000 else 0.05,
                "done": rng.choice([0.0, 0.1]), "rows": max(n, min(40000, n * new))}
    if op == "append":
        return {"op": op, "rows": _log(rng, 1, 8000), "heads": heads, "kv_heads": kv_heads, "page_size": page,
                "q_type": kind, "packed": rng.random() < 0.5, "pad": pad}
    if op == "prompt":
        n = _log(rng, 1, 40)
        top = max(1, min(6000, 12000 // n))
        lens = [0 if rng.random() < 0.05 else _log(rng, 1, top) for _ in range(n)]
        return {"op": op, "lens": _text(lens), "heads": heads, "kv_heads": kv_heads, "q_type": kind, "pad": pad}
    n = _log(rng, 1, 64)
    if rng.random() < 0.5:
        new = [1] * n
    else:
        new = [_log(rng, 1, max(1, min(700, 3000 // n))) for _ in range(n)]
    ctx = [0 if rng.random() < 0.1 else _log(rng, 1, 300000 // n if n > 9 else 32000) for _ in range(n)]
    return {"op": "paged", "new": _text(new), "ctx": _text(ctx), "heads": heads, "kv_heads": kv_heads,
            "page_size": page, "q_type": kind, "pad": pad}


# ----------------------------------------------------------------- the inputs
def _dtype(case):
    return torch.float32 if case["q_type"] == "f32" else torch.float16


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32)


def _channel_scale(gen):
    """Keys and queries have a few strong channels; the others are ordinary."""
    return torch.exp(0.5 * torch.randn(HD, generator=gen, device=DEV))


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    rng = np.random.default_rng(seed)
    st = {"case": case}
    if own:
        from glacier.inference import distributed_b200 as glc
        st["glc"] = glc
    {"plan": _prepare_plan, "append": _prepare_append, "prompt": _prepare_prompt,
     "paged": _prepare_paged}[case["op"]](case, gen, rng, st)
    return st


def _prepare_plan(case, gen, rng, st):
    n, ps = case["requests"], case["page_size"]
    ctx = rng.integers(0, case["max_ctx"] + 1, size=n)
    new = np.ones(n, np.int64)
    chunk = rng.random(n) < case["prompts"]
    new[chunk] = rng.integers(1, case["max_new"] + 1, size=int(chunk.sum()))
    done = rng.random(n) < case["done"]
    new[done] = -1
    width = -(-(case["max_ctx"] + case["max_new"]) // ps)
    held = -(-ctx // ps)
    need = int((-(-(ctx + np.maximum(new, 0)) // ps) - held).sum())
    free = need + int(rng.integers(0, 64)) if rng.random() < 0.75 else max(0, need - int(rng.integers(0, need + 1)))
    total = n * width + 64                               # pages of the cache; some belong to requests that wait
    ids = rng.permutation(total).astype(np.int32)
    table = np.full((n, width), -1, np.int32)
    at = 0
    for i in range(n):
        table[i, :held[i]] = ids[at:at + held[i]]
        at += int(held[i])
    pool = np.full(total, -1, np.int32)
    pool[:free] = ids[at:at + free]
    st.update(n=n, ps=ps, width=width, rows=case["rows"], pages=total,
              ctx=torch.from_numpy(ctx.astype(np.int32)).to(DEV), new=torch.from_numpy(new.astype(np.int32)).to(DEV),
              table=torch.from_numpy(table).to(DEV), pool=torch.from_numpy(pool).to(DEV),
              free=torch.tensor([free], dtype=torch.int32, device=DEV))
    if own:
        e = lambda *s, t=torch.int32: torch.empty(*s, dtype=t, device=DEV)  # noqa: E731
        st.update(cu=e(n + 1), kv=e(n), pos=e(case["rows"]), slots=e(case["rows"], t=torch.int64), left=e(1), status=e(1))


def _prepare_append(case, gen, rng, st):
    rows, pad, hq, hk, ps = case["rows"], case["pad"], case["heads"], case["kv_heads"], case["page_size"]
    all_rows = rows + pad
    qkv = _normal(gen, all_rows, (hq + 2 * hk) * HD)     # the projection's rows: q, k, v side by side
    pages = 2 * (-(-rows // ps)) + 3
    slots = np.full(all_rows, -1, np.int64)              # rows behind the last token have no slot
    order = rng.permutation(pages)[:-(-rows // ps)]
    r = np.arange(rows)
    slots[:rows] = order[r // ps] * ps + r % ps
    pos = np.zeros(all_rows, np.int32)
    pos[:rows] = int(rng.integers(0, 32768)) + r
    st.update(rows=all_rows, hq=hq, hk=hk, ps=ps, pages=pages, qkv=qkv, qt=_dtype(case), packed=case["packed"],
              slots=torch.from_numpy(slots).to(DEV), pos=torch.from_numpy(pos).to(DEV),
              kc=torch.zeros(pages, hk, ps, HD, dtype=torch.float16, device=DEV),
              vc=torch.zeros(pages, hk, ps, HD, dtype=torch.float16, device=DEV))
    if own:
        glc = st["glc"]
        st["cache"] = glc.KvPages(st["kc"].data_ptr(), st["vc"].data_ptr(), pages, ps, hk)
        st["q_out"] = torch.empty(all_rows, hq, HD, dtype=st["qt"], device=DEV)
        if case["packed"]:
            st["k_out"] = torch.empty(all_rows, hk, HD, dtype=torch.float16, device=DEV)
            st["v_out"] = torch.empty(all_rows, hk, HD, dtype=torch.float16, device=DEV)


def _prepare_prompt(case, gen, rng, st):
    lens = _ints(case["lens"])
    hq, hk = case["heads"], case["kv_heads"]
    rows = sum(lens) + case["pad"]
    scale = _channel_scale(gen)
    q = (_normal(gen, rows, hq, HD) * scale).to(_dtype(case))
    k = (_normal(gen, rows, hk, HD) * scale).to(torch.float16)
    v = _normal(gen, rows, hk, HD).to(torch.float16)
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    st.update(lens=lens, rows=rows, hq=hq, hk=hk, q=q, k=k, v=v, cu=torch.from_numpy(cu).to(DEV), qt=_dtype(case),
              out=torch.zeros(rows, hq, HD, dtype=_dtype(case), device=DEV))


def _prepare_paged(case, gen, rng, st):
    new, ctx = _ints(case["new"]), _ints(case["ctx"])
    hq, hk, ps = case["heads"], case["kv_heads"], case["page_size"]
    n, rows = len(new), sum(new) + case["pad"]
    kv = [a + b for a, b in zip(new, ctx)]
    held = [-(-a // ps) for a in kv]
    width = max(held) + 3                                # a table is as wide as the longest request may get
    pages = sum(held) + 5
    ids = rng.permutation(pages).astype(np.int32)
    table = np.full((n, width), -1, np.int32)
    at = 0
    for i in range(n):
        table[i, :held[i]] = ids[at:at + held[i]]
        at += held[i]
    scale = _channel_scale(gen)
    q = (_normal(gen, rows, hq, HD) * scale).to(_dtype(case))
    kc = torch.empty(pages, hk, ps, HD, dtype=torch.float16, device=DEV)
    vc = torch.empty(pages, hk, ps, HD, dtype=torch.float16, device=DEV)
    step = max(1, (1 << 27) // (hk * ps * HD))
    for p0 in range(0, pages, step):
        m = min(pages, p0 + step) - p0
        kc[p0:p0 + m] = (_normal(gen, m, hk, ps, HD) * scale).to(torch.float16)
        vc[p0:p0 + m] = _normal(gen, m, hk, ps, HD).to(torch.float16)
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    st.update(new=new, kv=kv, n=n, rows=rows, hq=hq, hk=hk, ps=ps, pages=pages, width=width, q=q, kc=kc, vc=vc,
              qt=_dtype(case), table=torch.from_numpy(table).to(DEV), cu=torch.from_numpy(cu).to(DEV),
              kv_dev=torch.tensor(kv, dtype=torch.int32, device=DEV),
              out=torch.zeros(rows, hq, HD, dtype=_dtype(case), device=DEV))
    if own:
        glc = st["glc"]
        st["cache"] = glc.KvPages(kc.data_ptr(), vc.data_ptr(), pages, ps, hk)
        nb = glc.attn_paged_workspace_bytes(hq, hk, n, rows, max(new))
        st["ws"], st["ws_bytes"] = torch.empty(nb, dtype=torch.uint8, device=DEV), nb


# --------------------------------------------------------------------- a pass
def run(st: dict):
    op = st["case"]["op"]
    if own:
        return {"plan": _own_plan, "append": _own_append, "prompt": _own_prompt, "paged": _own_paged}[op](st)
    return {"plan": _plain_plan, "append": _plain_append, "prompt": _plain_prompt, "paged": _plain_paged}[op](st)


def _own_plan(st):
    glc = st["glc"]
    glc.kv_plan_dev(st["ctx"].data_ptr(), st["new"].data_ptr(), st["n"], st["ps"], st["table"].data_ptr(), st["width"],
                    st["pool"].data_ptr(), st["pages"], st["free"].data_ptr(), st["left"].data_ptr(), st["rows"],
                    st["cu"].data_ptr(), st["kv"].data_ptr(), st["pos"].data_ptr(), st["slots"].data_ptr(),
                    st["status"].data_ptr(), stream=glc.torch_stream_handle())
    return {k: st[k] for k in ("table", "pool", "left", "cu", "kv", "pos", "slots", "status")}


def _own_append(st):
    glc, hq, hk, qkv = st["glc"], st["hq"], st["hk"], st["qkv"]
    p, row = qkv.data_ptr(), (hq + 2 * hk) * HD
    ko, vo = (st["k_out"], st["v_out"]) if st["packed"] else (None, None)
    glc.rope_append_dev(p, row, p + 4 * hq * HD, p + 4 * (hq + hk) * HD, row, st["rows"], hq, hk,
                        st["pos"].data_ptr(), st["slots"].data_ptr(), THETA, st["cache"], st["q_out"].data_ptr(),
                        glc.GGUF_F32 if st["qt"] == torch.float32 else glc.GGUF_F16,
                        ko.data_ptr() if st["packed"] else None, vo.data_ptr() if st["packed"] else None,
                        stream=glc.torch_stream_handle())
    out = [st["q_out"], st["kc"], st["vc"]]
    return out + [ko, vo] if st["packed"] else out


def _own_prompt(st):
    glc, hq, hk = st["glc"], st["hq"], st["hk"]
    glc.attn_prompt_dev(st["q"].data_ptr(), glc.GGUF_F32 if st["qt"] == torch.float32 else glc.GGUF_F16, hq * HD,
                        st["k"].data_ptr(), st["v"].data_ptr(), hk * HD, st["cu"].data_ptr(), len(st["lens"]),
                        st["rows"], hq, hk, st["out"].data_ptr(), hq * HD, stream=glc.torch_stream_handle())
    return st["out"]


def _own_paged(st):
    glc, hq = st["glc"], st["hq"]
    glc.attn_paged_dev(st["q"].data_ptr(), glc.GGUF_F32 if st["qt"] == torch.float32 else glc.GGUF_F16, hq * HD,
                       st["cache"], st["table"].data_ptr(), st["width"], st["cu"].data_ptr(), st["kv_dev"].data_ptr(),
                       st["n"], st["rows"], max(st["new"]), hq, st["out"].data_ptr(), hq * HD, st["ws"].data_ptr(),
                       st["ws_bytes"], stream=glc.torch_stream_handle())
    return st["out"]


def _plain_plan(st):
    n, ps, width, rows, cap = st["n"], st["ps"], st["width"], st["rows"], st["pages"]
    ctx, new = st["ctx"].long(), st["new"].long()
    table, pool = st["table"].clone(), st["pool"].clone()
    free = st["free"].long()[0]
    gone = new < 0
    add = new.clamp(min=0)
    held = (ctx + ps - 1) // ps
    cu = torch.cat([add.new_zeros(1), add.cumsum(0)])
    # finished requests give their pages back, in request order, on top of the free list
    back = torch.where(gone, held, held.new_zeros(()))
    back_end = back.cumsum(0)
    col = torch.arange(width, device=DEV)
    row = torch.arange(n, device=DEV)
    stack = torch.cat([pool, pool.new_full((1,), -1)]).long()
    m = gone[:, None] & (col < held[:, None])
    where = torch.where(m, free + (back_end - back)[:, None] + col, cap)
    stack.scatter_(0, where.clamp(max=cap).reshape(-1), table.long().reshape(-1))
    avail = free + back_end[-1]
    # a request is served when its rows, its table row and every page up to its own fit
    fits = (cu[1:] <= rows) & ((ctx + add + ps - 1) // ps <= width) & ~gone
    need = torch.where(fits, (ctx + add + ps - 1) // ps - held, held.new_zeros(()))
    end = need.cumsum(0)
    ok = fits & ((need == 0) | (end <= avail))
    took = torch.where(ok, need, need.new_zeros(()))
    used = took.sum()
    left = avail - used
    start = took.cumsum(0) - took
    m = ok[:, None] & (col >= held[:, None]) & (col < (held + took)[:, None])
    rank = start[:, None] + col - held[:, None]
    table = torch.where(m, stack[(avail - 1 - rank).clamp(0, cap)].to(torch.int32), table)
    at = torch.arange(cap, device=DEV)
    pool = torch.where((at >= free) & (at < avail), stack[:cap].to(torch.int32), pool)
    kv = torch.where(ok, ctx + add, ctx.new_zeros(()))
    # the rows of the step: position and slot of every new token
    t = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=n - 1)
    live = (t < cu[-1]) & ok[seq]
    pos = torch.where(live, ctx[seq] + t - cu[seq], t.new_zeros(()))
    slots = torch.where(live, table[seq, (pos // ps).clamp(max=width - 1)].long() * ps + pos % ps, t.new_full((), -1))
    bad = ((~ok) & ~gone).sum()
    i32 = torch.int32
    return {"table": table, "pool": pool, "left": left.to(i32).reshape(1), "cu": cu.clamp(max=rows).to(i32),
            "kv": kv.to(i32), "pos": pos.to(i32), "slots": slots, "status": bad.to(i32).reshape(1)}


def _angles(pos):
    i = torch.arange(HD // 2, device=DEV, dtype=torch.float64)
    ang = pos.double()[:, None] * torch.exp(-(2.0 * i / HD) * math.log(THETA))
    return torch.cos(ang), torch.sin(ang)


def _rotate(x, c, s):
    a, b = x[..., :HD // 2], x[..., HD // 2:]
    c, s = c[:, None].to(x.dtype), s[:, None].to(x.dtype)
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def _plain_append(st):
    rows, hq, hk, ps = st["rows"], st["hq"], st["hk"], st["ps"]
    qkv = st["qkv"]
    q = qkv[:, :hq * HD].reshape(rows, hq, HD)
    k = qkv[:, hq * HD:(hq + hk) * HD].reshape(rows, hk, HD)
    v = qkv[:, (hq + hk) * HD:].reshape(rows, hk, HD)
    c, s = _angles(st["pos"])
    qr, kr, vr = _rotate(q, c, s).to(st["qt"]), _rotate(k, c, s).half(), v.half()
    kc, vc, slots = st["kc"].clone(), st["vc"].clone(), st["slots"]
    live = slots >= 0
    page, off = slots[live] // ps, slots[live] % ps
    kc[page, :, off] = kr[live]
    vc[page, :, off] = vr[live]
    return [qr, kc, vc, kr, vr] if st["packed"] else [qr, kc, vc]


def _attend(q, k, v, first, out, wide):
    """out[i, h] = softmax over j <= first + i of q[i, h] . k[j, g] / sqrt(d), times v; one
    KV head's queries and a block of rows at a time, in the type of ``wide``."""
    n, hq, _ = q.shape
    kl, hk = k.shape[0], k.shape[1]
    if n == 0 or kl == 0:
        return
    group = hq // hk
    block = max(1, (1 << 27) // (group * kl))
    j = torch.arange(kl, device=DEV)
    for g in range(hk):
        kg, vg = k[:, g].to(wide), v[:, g].to(wide)
        for r0 in range(0, n, block):
            r1 = min(n, r0 + block)
            qg = q[r0:r1, g * group:(g + 1) * group].to(wide).reshape(-1, HD)
            s = (qg @ kg.T) * (1.0 / math.sqrt(HD))
            last = first + torch.arange(r0, r1, device=DEV).repeat_interleave(group)
            dead = j[None, :] > last[:, None]
            s = s.masked_fill_(dead, -math.inf)
            m = s.amax(dim=1, keepdim=True)
            m = torch.where(m == -math.inf, torch.zeros_like(m), m)
            p = s.sub_(m).exp_()
            o = (p @ vg) / p.sum(dim=1, keepdim=True)
            o = torch.where((last < 0)[:, None], torch.zeros_like(o), o)
            out[r0:r1, g * group:(g + 1) * group] = o.reshape(r1 - r0, group, HD).to(out.dtype)


def _prompt(st, wide, out):
    at = 0
    for n in st["lens"]:
        sl = slice(at, at + n)
        _attend(st["q"][sl], st["k"][sl], st["v"][sl], 0, out[sl], wide)
        at += n
    return out


def _plain_prompt(st):
    return _prompt(st, torch.float32, torch.zeros_like(st["out"]))


def _plain_paged(st):
    out = torch.zeros_like(st["out"])
    ps, hk, at = st["ps"], st["hk"], 0
    for i in range(st["n"]):
        kl, n = st["kv"][i], st["new"][i]
        page = st["table"][i, :-(-kl // ps)].long()
        k = st["kc"][page].transpose(1, 2).reshape(-1, hk, HD)[:kl]
        v = st["vc"][page].transpose(1, 2).reshape(-1, hk, HD)[:kl]
        _attend(st["q"][at:at + n], k, v, kl - n, out[at:at + n], torch.float32)
        at += n
    return out


# ----------------------------------------------------------- what has to move
def work(case: dict) -> dict:
    op = case["op"]
    if op == "plan":
        n = case["requests"]
        tokens = min(case["rows"], int(n * (1 - case["done"]) * (1 + case["prompts"] * case["max_new"] / 2)))
        moved = 8 * (tokens // case["page_size"] + int(case["done"] * n * case["max_ctx"] / 2 / case["page_size"]))
        return {"bytes": 8 * n + 8 * n + moved + 12 * case["rows"] + 16, "flops": 0}
    hq, hk = case["heads"], case["kv_heads"]
    qb = 4 if case["q_type"] == "f32" else 2
    if op == "append":
        live = case["rows"]
        rows = live + case["pad"]
        kv_out = 2 * live * hk * HD * 2 + (2 * rows * hk * HD * 2 if case["packed"] else 0)
        return {"bytes": rows * (hq + 2 * hk) * HD * 4 + rows * hq * HD * qb + kv_out + 12 * rows,
                "flops": 3 * rows * (hq + hk) * HD}
    if op == "prompt":
        lens = _ints(case["lens"])
        rows = sum(lens)
        pairs = sum(n * (n + 1) // 2 for n in lens)
        return {"bytes": rows * (2 * hq * HD * qb + 2 * hk * HD * 2) + 4 * len(lens), "flops": 4 * HD * hq * pairs}
    new, ctx = _ints(case["new"]), _ints(case["ctx"])
    pairs = sum(n * c + n * (n + 1) // 2 for n, c in zip(new, ctx))
    held = sum(n + c for n, c in zip(new, ctx))
    return {"bytes": sum(new) * 2 * hq * HD * qb + held * 2 * hk * HD * 2 + 8 * len(new) +
            4 * sum(-(-(n + c) // case["page_size"]) for n, c in zip(new, ctx)),
            "flops": 4 * HD * hq * pairs}


# -------------------------------------------------- the definitions in 64 bits
def exact(case: dict, seed: int):
    """The outputs of ``run`` from the definitions, row by row, in 64 bits."""
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    return {"plan": _exact_plan, "append": _exact_append, "prompt": _exact_prompt, "paged": _exact_paged}[case["op"]](st)


def _exact_plan(st):
    """One request after another, the way a scheduler would write it down."""
    n, ps, width, rows = st["n"], st["ps"], st["width"], st["rows"]
    ctx, new = st["ctx"].tolist(), st["new"].tolist()
    table, pool = st["table"].cpu().numpy().copy(), st["pool"].cpu().numpy().copy()
    free = int(st["free"][0])
    stack = pool[:free].tolist()
    pages_of = lambda x: (x + ps - 1) // ps  # noqa: E731
    for i in range(n):
        if new[i] < 0:
            stack += table[i, :pages_of(ctx[i])].tolist()
    cu, kv = [0], []
    pos, slots = np.zeros(rows, np.int32), np.full(rows, -1, np.int64)
    bad, wanted, avail = 0, 0, len(stack)
    pool[free:avail] = stack[free:]                       # given back, whether or not this step takes them again
    for i in range(n):
        a = max(new[i], 0)
        t0 = cu[-1]
        cu.append(t0 + a)
        if new[i] < 0:
            kv.append(0)
            continue
        have, want = pages_of(ctx[i]), pages_of(ctx[i] + a)
        if t0 + a > rows or want > width:
            kv.append(0)
            bad += 1
            continue
        wanted += want - have
        if want > have and wanted > avail:
            kv.append(0)
            bad += 1
            continue
        for c in range(have, want):
            table[i, c] = stack.pop()
        kv.append(ctx[i] + a)
        p = np.arange(ctx[i], ctx[i] + a)
        pos[t0:t0 + a] = p
        slots[t0:t0 + a] = table[i, p // ps].astype(np.int64) * ps + p % ps
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    return {"table": torch.from_numpy(table).to(DEV), "pool": torch.from_numpy(pool).to(DEV), "left": i32([len(stack)]),
            "cu": i32([min(c, rows) for c in cu]), "kv": i32(kv), "pos": torch.from_numpy(pos).to(DEV),
            "slots": torch.from_numpy(slots).to(DEV), "status": i32([bad])}


def _exact_append(st):
    """Rotation of each pair as a product of complex numbers."""
    rows, hq, hk, ps = st["rows"], st["hq"], st["hk"], st["ps"]
    x = st["qkv"].double().reshape(rows, hq + 2 * hk, HD)
    i = torch.arange(HD // 2, device=DEV, dtype=torch.float64)
    turn = torch.polar(torch.ones((), device=DEV, dtype=torch.float64),
                       st["pos"].double()[:, None] * THETA ** (-i / (HD // 2)))
    z = torch.complex(x[:, :hq + hk, :HD // 2].contiguous(), x[:, :hq + hk, HD // 2:].contiguous()) * turn[:, None]
    qk = torch.cat([z.real, z.imag], dim=-1)
    q, k, v = qk[:, :hq], qk[:, hq:], x[:, hq + hk:]
    kc, vc = st["kc"].double(), st["vc"].double()
    for r in (st["slots"] >= 0).nonzero()[:, 0].split(4096):
        s = st["slots"][r]
        kc[s // ps, :, s % ps] = k[r]
        vc[s // ps, :, s % ps] = v[r]
    return [q, kc, vc, k, v] if st["packed"] else [q, kc, vc]


def _exact_rows(q, k, v, first, out):
    """The definition per query head, a block of queries against the keys they may see."""
    n, hq, _ = q.shape
    group = hq // k.shape[1]
    for h in range(hq):
        kh, vh = k[:, h // group].double(), v[:, h // group].double()
        step = max(1, (1 << 26) // max(1, k.shape[0]))
        for r0 in range(max(0, -first), n, step):
            r1 = min(n, r0 + step)
            see = first + r1
            if see <= 0:
                continue
            s = torch.einsum("id,jd->ij", q[r0:r1, h].double(), kh[:see]) / math.sqrt(HD)
            late = torch.arange(see, device=DEV)[None] > (first + torch.arange(r0, r1, device=DEV))[:, None]
            w = torch.softmax(s.masked_fill(late, -math.inf), dim=1)
            out[r0:r1, h] = torch.einsum("ij,jd->id", w, vh[:see])


def _exact_prompt(st):
    out = torch.zeros(st["rows"], st["hq"], HD, dtype=torch.float64, device=DEV)
    at = 0
    for n in st["lens"]:
        sl = slice(at, at + n)
        _exact_rows(st["q"][sl], st["k"][sl], st["v"][sl], 0, out[sl])
        at += n
    return out


def _exact_paged(st):
    out = torch.zeros(st["rows"], st["hq"], HD, dtype=torch.float64, device=DEV)
    ps, at = st["ps"], 0
    for i in range(st["n"]):
        kl, n = st["kv"][i], st["new"][i]
        j = torch.arange(kl, device=DEV)
        page = st["table"][i].long()[j // ps]
        _exact_rows(st["q"][at:at + n], st["kc"][page, :, j % ps], st["vc"][page, :, j % ps], kl - n, out[at:at + n])
        at += n
    return out
