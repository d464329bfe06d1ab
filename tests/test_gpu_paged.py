"""The paged-cache operators on the GPU against the float64 oracle
(oracle/paged.py): page plan (bit-exact), rotary store, attention over packed
prompts and over pages.

Tolerances: attention elementwise within oracle.paged.attend_tolerance, which
derives the bound from the kernels' arithmetic.  Rotary outputs: the reduced
angle is rounded to fp32 (pi * 2^-24), sincosf adds 2 ulp and the rotation
three roundings, so |error| <= 2^-20 (|a| + |b|) of the pair, plus the output
rounding (fp16: 2^-11 relative, 2^-25 absolute); stored values are one
rounding, bit-exact.
"""
import numpy as np
import pytest

from oracle import paged as ref

pytestmark = pytest.mark.gpu

THETA = 1e6
F32, F16 = 0, 1
NP = {F32: np.float32, F16: np.float16}
SCALE = 1 / np.sqrt(128)


def dev(torch, a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


# ------------------------------------------------------------------ page plan
def plan_case(rng, B, ps, max_ctx, max_new, done=0.1, short=0, width=None, ctx=None, new=None):
    ctx = rng.integers(0, max_ctx + 1, B) if ctx is None else np.asarray(ctx)
    new = rng.integers(0, max_new + 1, B) if new is None else np.asarray(new)
    new = np.where(rng.random(B) < done, -1, new)
    held = -(-ctx // ps)
    need = int((-(-(ctx + np.maximum(new, 0)) // ps) - held).sum())
    width = width or int(-(-(max_ctx + max_new) // ps) + 1)
    free = max(0, need + 3 - short)
    ids = rng.permutation(int(held.sum()) + free + 7).astype(np.int32)
    table, at = np.full((B, width), -1, np.int32), 0
    for i in range(B):
        table[i, :min(held[i], width)] = ids[at:at + min(held[i], width)]
        at += held[i]
    pool = np.full(len(ids), -1, np.int32)
    pool[:free] = ids[at:at + free]
    return ctx.astype(np.int32), new.astype(np.int32), table, pool, free


def run_plan(torch, glc, ctx, new, ps, table, pool, free, T, times=1):
    B, width = table.shape
    d = {k: dev(torch, v) for k, v in dict(ctx=ctx, new=new, table=table, pool=pool, free=np.array([free], np.int32)).items()}
    o = {k: torch.full((n,), 77, dtype=torch.int32, device="cuda") for k, n in dict(left=1, cu=B + 1, kv=B, pos=T, bad=1).items()}
    slots = torch.full((T,), 77, dtype=torch.int64, device="cuda")
    for _ in range(times):
        glc.kv_plan_dev(d["ctx"].data_ptr() or 1, d["new"].data_ptr() or 1, B, ps, d["table"].data_ptr() or 1, width,
                        d["pool"].data_ptr(), len(pool), d["free"].data_ptr(), o["left"].data_ptr(), T,
                        o["cu"].data_ptr(), o["kv"].data_ptr() or 2, o["pos"].data_ptr(), slots.data_ptr(),
                        o["bad"].data_ptr(), stream=glc.torch_stream_handle())
    torch.cuda.synchronize()
    return (d["table"], d["pool"], int(o["left"]), o["cu"], o["kv"], o["pos"], slots, int(o["bad"]))


def same_plan(got, want):
    for name, g, w in zip(("table", "free list", "left", "cu", "kv_lens", "positions", "slots", "status"), got, want):
        g = g if isinstance(g, int) else g.cpu().numpy()
        assert np.array_equal(g, w), name


@pytest.mark.parametrize("B,ps,max_ctx,max_new,T,short", [
    (1, 16, 100, 1, 1, 0), (1, 256, 0, 700, 800, 0), (5, 16, 40, 3, 16, 0), (64, 16, 5000, 1, 64, 0),
    (33, 32, 300, 200, 4000, 0), (1024, 16, 200, 4, 4096, 0), (1025, 16, 200, 4, 4096, 0), (3000, 64, 500, 30, 60000, 0),
    (257, 16, 60, 60, 9000, 40), (1500, 16, 60, 60, 50000, 900), (40, 128, 300, 300, 2000, 0), (9, 16, 50, 50, 0, 0),
    (4096, 16, 90, 3, 9000, 100), (4097, 16, 90, 3, 9000, 0), (9000, 32, 90, 3, 18000, 300)])
def test_plan_matches_oracle(cuda, glc, B, ps, max_ctx, max_new, T, short):
    rng = np.random.default_rng(B * 7 + ps + T)
    ctx, new, table, pool, free = plan_case(rng, B, ps, max_ctx, max_new, short=short)
    want = ref.plan(ctx, new, ps, table, pool, free, T)
    same_plan(run_plan(cuda, glc, ctx, new, ps, table, pool, free, T), want)
    same_plan(run_plan(cuda, glc, ctx, new, ps, table, pool, free, T, times=3), want)  # the same inputs again


def test_plan_narrow_table_and_all_finished(cuda, glc):
    rng = np.random.default_rng(1)
    a = plan_case(rng, 20, 16, 60, 60, width=5)
    same_plan(run_plan(cuda, glc, *a[:2], 16, *a[2:], 2000), ref.plan(*a[:2], 16, *a[2:], 2000))
    a = plan_case(rng, 300, 16, 300, 0, done=2.0)
    same_plan(run_plan(cuda, glc, *a[:2], 16, *a[2:], 8), ref.plan(*a[:2], 16, *a[2:], 8))


def test_plan_without_requests(cuda, glc):
    torch = cuda
    got = run_plan(torch, glc, np.zeros(0, np.int32), np.zeros(0, np.int32), 16, np.zeros((0, 4), np.int32),
                   np.arange(6, dtype=np.int32), 4, 3)
    assert got[2] == 4 and list(got[3].cpu()) == [0] and list(got[6].cpu()) == [-1] * 3 and got[7] == 0


def test_plan_holds_on_bad_lengths(cuda, glc):
    """Negative and absurd lengths are not served and touch nothing out of bounds."""
    torch = cuda
    big = 2**31 - 1
    ctx = np.array([-5, 10, big, 10, -7], np.int32)
    new = np.array([3, 2, big, big, -1], np.int32)
    table = np.zeros((5, 4), np.int32)
    pool = np.arange(10, dtype=np.int32)
    got = run_plan(torch, glc, ctx, new, 16, table, pool, 10, 8)
    assert list(got[4].cpu()) == [0, 12, 0, 0, 0] and got[7] == 3 and got[2] == 10
    assert list(got[3].cpu()) == [0, 3, 5, 8, 8, 8]
    got = run_plan(torch, glc, ctx[1:2], new[1:2], 16, table[:1], pool, 2**30, 8)  # a count past the list's room
    assert got[2] == 10


# --------------------------------------------------------------- rotary store
def make_pages(torch, n_pages, ps, Hkv, layout, fill=0.0):
    if layout == "head":      # [page][head][row][128]
        a = [torch.full((n_pages, Hkv, ps, 128), fill, dtype=torch.float16, device="cuda") for _ in range(2)]
        return a[0], a[1], {}, lambda t: t
    if layout == "row":       # [page][row][head][128]
        a = [torch.full((n_pages, ps, Hkv, 128), fill, dtype=torch.float16, device="cuda") for _ in range(2)]
        return a[0], a[1], dict(page_stride=ps * Hkv * 128, head_stride=128, row_stride=Hkv * 128), \
            lambda t: t.transpose(1, 2)
    # keys and values of a page side by side: [page][2][head][row][128]
    both = torch.full((n_pages, 2, Hkv, ps, 128), fill, dtype=torch.float16, device="cuda")
    return both[:, 0], both[:, 1], dict(page_stride=2 * Hkv * ps * 128), lambda t: t


def rot_bound(x, ref64, t):
    a, b = np.abs(x[..., :64]), np.abs(x[..., 64:])
    e = np.concatenate([a + b, a + b], -1) * 2.0 ** -20
    return e + (np.abs(ref64) * 2.0 ** -11 + 2.0 ** -25 if t == F16 else 1e-30)


@pytest.mark.parametrize("T,Hq,Hkv,ps,layout,qt,packed,fused", [
    (1, 40, 8, 16, "head", F32, False, True), (1, 5, 1, 256, "row", F16, True, False),
    (7, 6, 2, 16, "both", F32, True, True), (300, 28, 4, 64, "row", F16, False, True),
    (129, 48, 8, 32, "head", F32, True, False), (65, 0, 2, 128, "head", F32, False, False),
    (33, 3, 3, 16, "head", F16, True, True)])
def test_append_matches_oracle(cuda, glc, T, Hq, Hkv, ps, layout, qt, packed, fused):
    torch = cuda
    rng = np.random.default_rng(T + Hq)
    row = (Hq + 2 * Hkv) * 128 + (4 if fused else 0)
    x = rng.standard_normal((T, row)).astype(np.float32)
    q, k, v = (x[:, a * 128:b * 128].reshape(T, -1, 128) for a, b in
               ((0, Hq), (Hq, Hq + Hkv), (Hq + Hkv, Hq + 2 * Hkv)))
    n_pages = 2 * (-(-T // ps)) + 2
    slots = rng.permutation(n_pages * ps)[:T].astype(np.int64)
    if T > 4:
        slots[[1, T - 1]] = -1
    pos = rng.integers(0, 100000, T).astype(np.int32)
    pos[0] = 0
    kc, vc, strides, view = make_pages(torch, n_pages, ps, Hkv, layout, fill=3.0)
    before = [view(t).cpu().numpy().copy() for t in (kc, vc)]
    cache = glc.KvPages(kc.data_ptr(), vc.data_ptr(), n_pages, ps, Hkv, **strides)
    if fused:
        d = dev(torch, x)
        qp, kp, vp, qs, ks = d.data_ptr(), d.data_ptr() + 4 * Hq * 128, d.data_ptr() + 4 * (Hq + Hkv) * 128, row, row
    else:
        dq, dk, dv = dev(torch, q), dev(torch, k), dev(torch, v)
        qp, kp, vp, qs, ks = dq.data_ptr() or None, dk.data_ptr(), dv.data_ptr(), Hq * 128, Hkv * 128
    qo = torch.full((T, max(Hq, 1), 128), 9.0, dtype=torch.float32 if qt == F32 else torch.float16, device="cuda")
    ko, vo = (torch.empty(T, Hkv, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    ds, dp = dev(torch, slots), dev(torch, pos)
    glc.rope_append_dev(qp, qs, kp, vp, ks, T, Hq, Hkv, dp.data_ptr(), ds.data_ptr(), THETA, cache,
                        qo.data_ptr() if Hq else None, qt, ko.data_ptr() if packed else None,
                        vo.data_ptr() if packed else None, stream=glc.torch_stream_handle())
    glc.paged_poll_error()
    rq, rk = ref.rotate(q, pos, THETA), ref.rotate(k, pos, THETA)
    if Hq:
        assert np.all(np.abs(qo.cpu().numpy() - rq) <= rot_bound(q, rq, qt))
    gk, gv = (view(t).cpu().numpy() for t in (kc, vc))
    kb = rot_bound(k, rk, F16)
    touched = np.zeros((n_pages, ps), bool)
    for t in range(T):
        if slots[t] < 0:
            continue
        p, r = divmod(int(slots[t]), ps)
        touched[p, r] = True
        assert np.all(np.abs(gk[p, :, r] - rk[t]) <= kb[t])
        assert np.array_equal(gv[p, :, r], v[t].astype(np.float16))
    for g, b in zip((gk, gv), before):
        assert np.array_equal(g.transpose(0, 2, 1, 3)[~touched], b.transpose(0, 2, 1, 3)[~touched])
    if packed:
        assert np.all(np.abs(ko.cpu().numpy() - rk) <= kb)
        assert np.array_equal(vo.cpu().numpy(), v.astype(np.float16))


def test_append_in_place_without_cache(cuda, glc):
    torch = cuda
    rng = np.random.default_rng(2)
    q, k = rng.standard_normal((9, 4, 128)).astype(np.float32), rng.standard_normal((9, 2, 128)).astype(np.float32)
    pos = np.arange(9, dtype=np.int32) * 1000 + 7
    dq, dk, dp = dev(torch, q), dev(torch, k), dev(torch, pos)
    glc.rope_append_dev(dq.data_ptr(), 512, dk.data_ptr(), dk.data_ptr(), 256, 9, 4, 2, dp.data_ptr(), None, THETA, None,
                        dq.data_ptr(), F32, stream=glc.torch_stream_handle())
    rq = ref.rotate(q, pos, THETA)
    assert np.all(np.abs(dq.cpu().numpy() - rq) <= rot_bound(q, rq, F32))


def test_append_slot_past_the_cache(cuda, glc):
    torch = cuda
    k = torch.ones(3, 1, 128, device="cuda")
    kc, vc, _, _ = make_pages(torch, 2, 16, 1, "head")
    slots = torch.tensor([5, 32, 2**40], dtype=torch.int64, device="cuda")
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")
    glc.rope_append_dev(None, 0, k.data_ptr(), k.data_ptr(), 128, 3, 0, 1, pos.data_ptr(), slots.data_ptr(), THETA,
                        glc.KvPages(kc.data_ptr(), vc.data_ptr(), 2, 16, 1), None, F32, stream=glc.torch_stream_handle())
    with pytest.raises(glc.GlcError, match="out of range") as e:
        glc.paged_poll_error()
    assert e.value.status == -1
    glc.paged_poll_error()  # read and cleared
    assert float(vc.sum()) == 128 and float(vc[0, 0, 5].sum()) == 128


# ------------------------------------------------------------------ attention
def check_attention(got, q, k, v, first, f32, scale=SCALE):
    out, wv, peak, mag = ref.attend(q, k, v, first, scale)
    tol = ref.attend_tolerance(out, wv, peak, mag, k.shape[0], f32)
    err = np.abs(got.astype(np.float64) - out)
    assert np.all(err <= tol), f"largest error / bound {np.nanmax(err / tol)}"


def run_prompt(torch, glc, q, k, v, cu, qt, pad_cols=0, scale=0.0, out=None):
    """q [T][Hq][128] etc. as numpy; rows with pad_cols extra elements between tokens."""
    T, Hq, Hkv = q.shape[0], q.shape[1], k.shape[1]

    def rows(a):
        w = np.full((T, a.shape[1] * 128 + pad_cols), np.nan, a.dtype)
        w[:, :a.shape[1] * 128] = a.reshape(T, -1)
        return dev(torch, w)
    dq, dk, dv, dc = rows(q.astype(NP[qt])), rows(k), rows(v), dev(torch, np.asarray(cu, np.int32))
    if out is None:
        out = torch.full((T, Hq * 128 + pad_cols), 7.0, dtype=dq.dtype, device="cuda")
    glc.attn_prompt_dev(dq.data_ptr(), qt, Hq * 128 + pad_cols, dk.data_ptr(), dv.data_ptr(), Hkv * 128 + pad_cols,
                        dc.data_ptr(), len(cu) - 1, T, Hq, Hkv, out.data_ptr(), Hq * 128 + pad_cols, scale=scale,
                        stream=glc.torch_stream_handle())
    glc.paged_poll_error()
    return out.cpu().numpy()


@pytest.mark.parametrize("qt", [F32, F16])
@pytest.mark.parametrize("lens,Hq,Hkv,pad", [
    ([1], 5, 1, 0), ([33], 40, 8, 0), ([2, 0, 1, 0], 8, 8, 3), ([127, 128, 129], 6, 2, 5), ([300], 16, 1, 0),
    ([17, 260, 64], 28, 4, 1), ([515], 3, 3, 0), ([1] * 70, 12, 1, 0), ([400, 31], 13, 1, 2), ([600, 1, 40], 48, 8, 0)])
def test_prompt_matches_oracle(cuda, glc, lens, Hq, Hkv, pad, qt):
    rng = np.random.default_rng(sum(lens) + Hq)
    T = sum(lens) + pad
    q = rng.standard_normal((T, Hq, 128)).astype(NP[qt])
    k, v = (rng.standard_normal((T, Hkv, 128)).astype(np.float16) for _ in range(2))
    live = sum(lens)
    k[live:], v[live:], q[live:] = np.nan, np.inf, np.nan      # rows behind the last sequence
    cu = np.concatenate([[0], np.cumsum(lens)])
    got = run_prompt(cuda, glc, q, k, v, cu, qt, pad_cols=8 if pad else 0)
    w = got[:, :Hq * 128].reshape(T, Hq, 128)
    for b in range(len(lens)):
        s = slice(cu[b], cu[b + 1])
        check_attention(w[s], q[s], k[s], v[s], 0, qt == F32)
    assert np.all(w[live:] == 7) and np.all(got[:, Hq * 128:] == 7)


@pytest.mark.parametrize("qt", [F32, F16])
@pytest.mark.parametrize("lens,Hq,Hkv", [
    ([517, 1, 700, 130, 0, 63, 199, 300, 257, 64, 301, 333], 48, 8), ([3, 140, 1, 90, 250] * 9, 32, 8),
    ([1] * 170 + [40] * 30, 8, 8), ([30, 3] * 100, 16, 4), ([129, 1, 260] * 12, 8, 8)])
def test_prompt_many_items(cuda, glc, lens, Hq, Hkv, qt):
    """More items than SMs, with and without a second row tile: one CTA works
    through several.  Sequences are checked one in five (the oracle is slow), and
    all of them against themselves alone, bit for bit."""
    torch = cuda
    rng = np.random.default_rng(len(lens))
    T, cu = sum(lens), np.concatenate([[0], np.cumsum(lens)])
    q = rng.standard_normal((T, Hq, 128)).astype(NP[qt])
    k, v = (rng.standard_normal((T, Hkv, 128)).astype(np.float16) for _ in range(2))
    got = run_prompt(torch, glc, q, k, v, cu, qt).reshape(T, Hq, 128)
    for b in range(len(lens)):
        s = slice(cu[b], cu[b + 1])
        if not lens[b]:
            continue
        if b % 5 == 0 and lens[b] < 600:
            h = slice(0, 2 * Hq // Hkv)          # two KV heads
            check_attention(got[s][:, h], q[s][:, h], k[s][:, :2], v[s][:, :2], 0, qt == F32)
        if lens[b] * Hq // Hkv > 16:             # the tile kernel by itself
            alone = run_prompt(torch, glc, q[s], k[s], v[s], [0, lens[b]], qt).reshape(lens[b], Hq, 128)
            assert np.array_equal(alone, got[s]), b


@pytest.mark.parametrize("qt", [F32, F16])
def test_prompt_neighbours_do_not_leak(cuda, glc, qt):
    """A sequence of NaN and infinities between two others changes neither."""
    rng = np.random.default_rng(4)
    lens = [70, 45, 90]
    T, cu = sum(lens), np.concatenate([[0], np.cumsum(lens)])
    q, k, v = (rng.standard_normal((T, 4, 128)).astype(np.float16) for _ in range(3))
    k, v = k[:, :2], v[:, :2].copy()
    v[70:115], k[70:100] = np.inf, np.nan
    got = run_prompt(cuda, glc, q, k, v, cu, qt).reshape(T, 4, 128)
    for s in (slice(0, 70), slice(115, 205)):
        check_attention(got[s], q[s], k[s], v[s], 0, qt == F32)


@pytest.mark.parametrize("qt,qmag,kmag,scale", [(F32, 1e5, 1.0, 1e-6), (F32, 1e-20, 1.0, 1e18), (F32, 3.0, 30.0, 0.0),
                                                (F16, 6e4, 1.0, 1e-5), (F16, 3.0, 30.0, 0.0), (F32, 1.0, 1.0, 0.5)])
def test_prompt_extreme_scores(cuda, glc, qt, qmag, kmag, scale):
    """Large and tiny queries, peaked softmax rows, a scale of the caller's."""
    rng = np.random.default_rng(6)
    T, Hq, Hkv = 150, 4, 2
    q = (rng.uniform(-1, 1, (T, Hq, 128)) * qmag).astype(NP[qt])
    k = (rng.uniform(-1, 1, (T, Hkv, 128)) * kmag).astype(np.float16)
    v = rng.standard_normal((T, Hkv, 128)).astype(np.float16)
    got = run_prompt(cuda, glc, q, k, v, [0, T], qt, scale=scale).reshape(T, Hq, 128)
    check_attention(got, q, k, v, 0, qt == F32, scale or SCALE)


class Paged:
    """A batch over a paged cache whose unused rows and pages hold NaN."""

    def __init__(self, torch, glc, rng, new, kv, Hq, Hkv, ps, qt, layout="head", pad=0, page_scale=1):
        self.torch, self.glc, self.new, self.kv, self.qt = torch, glc, list(new), list(kv), qt
        self.Hq, self.Hkv, self.ps = Hq, Hkv, ps
        B, self.T = len(new), sum(new) + pad
        held = [-(-max(a, 0) // ps) for a in kv]
        self.width, self.n_pages = max(held + [1]) + 2, sum(held) + 3
        ids = rng.permutation(self.n_pages)
        self.table = np.full((B, self.width), -1, np.int32)
        self.kc, self.vc, strides, view = make_pages(torch, self.n_pages, ps, Hkv, layout, fill=float("nan"))
        self.k, self.v, at = [], [], 0
        for b in range(B):
            n = max(kv[b], 0)
            self.table[b, :held[b]] = ids[at:at + held[b]]
            at += held[b]
            k, v = (rng.standard_normal((n, Hkv, 128)).astype(np.float16) for _ in range(2))
            self.k.append(k)
            self.v.append(v)
            for src, dst in ((k, view(self.kc)), (v, view(self.vc))):
                for i in range(held[b]):
                    part = dev(torch, src[i * ps:(i + 1) * ps])
                    dst[int(self.table[b, i]), :, :part.shape[0]] = part.transpose(0, 1)
        self.q = rng.standard_normal((self.T, Hq, 128)).astype(NP[qt])
        self.cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.cache = glc.KvPages(self.kc.data_ptr(), self.vc.data_ptr(), self.n_pages, ps, Hkv, **strides)
        self.dq, self.dc, self.dt = dev(torch, self.q), dev(torch, self.cu), dev(torch, self.table)
        self.dkv = dev(torch, np.array(kv, np.int32))
        self.out = torch.full((self.T, Hq, 128), 7.0, dtype=self.dq.dtype, device="cuda")
        self.max_new = max(self.new)
        nb = glc.attn_paged_workspace_bytes(Hq, Hkv, B, self.T, self.max_new)
        self.ws = torch.full((nb,), 255, dtype=torch.uint8, device="cuda")

    def call(self, stream=None):
        glc = self.glc
        glc.attn_paged_dev(self.dq.data_ptr(), self.qt, self.Hq * 128, self.cache, self.dt.data_ptr(), self.width,
                           self.dc.data_ptr(), self.dkv.data_ptr(), len(self.new), self.T, self.max_new, self.Hq,
                           self.out.data_ptr(), self.Hq * 128, self.ws.data_ptr(), self.ws.numel(),
                           stream=stream or glc.torch_stream_handle())

    def check(self, skip=()):
        got = self.out.cpu().numpy()
        for b, n in enumerate(self.new):
            if b in skip:
                continue
            s = slice(self.cu[b], self.cu[b + 1])
            check_attention(got[s], self.q[s], self.k[b], self.v[b], self.kv[b] - n, self.qt == F32)
        assert np.all(got[self.cu[-1]:] == 7)


PAGED = [  # new, kv_lens, Hq, Hkv, page size, layout, pad rows
    ([1], [1], 40, 8, 16, "head", 0), ([1], [2048], 40, 8, 16, "head", 0), ([1], [700], 5, 1, 256, "row", 0),
    ([1, 1, 1, 1], [5, 0, 129, 1000], 48, 8, 16, "both", 3), ([3, 1, 2], [3, 64, 65], 8, 8, 64, "head", 0),
    ([16], [300], 3, 3, 32, "row", 1), ([17], [300], 4, 4, 32, "head", 0), ([40], [40], 28, 4, 16, "head", 0),
    ([64], [1500], 40, 8, 64, "head", 0), ([130, 1, 7, 1], [131, 900, 7, 1], 6, 2, 128, "row", 5),
    ([5, 0, 9], [2, 30, 0], 16, 1, 16, "head", 0), ([300], [301], 12, 2, 256, "both", 0),
    ([1] * 40, list(range(1, 800, 20)), 28, 4, 32, "row", 0), ([2], [5000], 64, 8, 16, "head", 0),
    ([200, 3], [1000, 257], 13, 1, 16, "head", 2)]


@pytest.mark.parametrize("qt", [F32, F16])
@pytest.mark.parametrize("case", PAGED, ids=lambda c: f"{len(c[0])}x{c[0][0]}of{c[1][0]}-{c[2]}h{c[3]}p{c[4]}{c[5]}")
def test_paged_matches_oracle(cuda, glc, case, qt):
    new, kv, Hq, Hkv, ps, layout, pad = case
    p = Paged(cuda, glc, np.random.default_rng(sum(kv) + Hq), new, kv, Hq, Hkv, ps, qt, layout, pad)
    p.call()
    glc.paged_poll_error()
    p.check()
    first = p.out.clone()
    p.call()                                                   # the same again, bit for bit
    glc.paged_poll_error()
    assert cuda.equal(first, p.out)


@pytest.mark.parametrize("qt", [F32, F16])
def test_paged_equals_packed(cuda, glc, qt):
    """A whole prompt over pages and packed: one definition, two bounds."""
    torch = cuda
    p = Paged(torch, glc, np.random.default_rng(8), [333], [333], 12, 4, 32, qt)
    p.call()
    p.check()
    got = run_prompt(torch, glc, p.q, p.k[0], p.v[0], [0, 333], qt).reshape(333, 12, 128)
    check_attention(got, p.q, p.k[0], p.v[0], 0, qt == F32)


@pytest.mark.parametrize("new", [1, 50])
def test_paged_bad_page_and_length(cuda, glc, new):
    torch = cuda
    p = Paged(torch, glc, np.random.default_rng(9), [new, new, new], [200, 333, 400], 8, 2, 16, F32)
    p.dt[1, 3], p.dt[1, 4] = 10**6, -4
    p.call()
    with pytest.raises(glc.GlcError, match="out of range"):
        glc.paged_poll_error()
    p.check(skip=(1,))
    p.dt[1] = dev(torch, p.table[1])
    p.dkv[2] = 10**6                                           # more rows than the table has
    p.call()
    with pytest.raises(glc.GlcError, match="out of range"):
        glc.paged_poll_error()
    p.check(skip=(2,))
    p.dkv[2] = 400
    p.dkv[0] = -3
    p.call()
    with pytest.raises(glc.GlcError, match="out of range"):
        glc.paged_poll_error()
    p.check(skip=(0,))


def test_paged_longer_than_max_new_is_recorded(cuda, glc):
    p = Paged(cuda, glc, np.random.default_rng(10), [1, 30], [100, 200], 8, 2, 16, F16)
    p.max_new = 1
    p.call()
    with pytest.raises(glc.GlcError, match="out of range"):
        glc.paged_poll_error()
    p.check(skip=(1,))


def test_paged_rows_outside_are_not_read(cuda, glc):
    """First rows that leave [0, T] are held inside it."""
    torch = cuda
    p = Paged(torch, glc, np.random.default_rng(11), [4, 4], [50, 60], 8, 2, 16, F32)
    p.dc.copy_(dev(torch, np.array([-10, 4, 10**9], np.int32)))
    p.call()
    torch.cuda.synchronize()
    try:
        glc.paged_poll_error()
    except glc.GlcError:
        pass
    assert torch.isfinite(p.out).all()


def test_paged_first_rows_that_do_not_ascend(cuda, glc):
    """Sequences that name the same rows over and over: recorded, and nothing
    outside the outputs' rows is written; the workspace serves the next call."""
    torch = cuda
    p = Paged(torch, glc, np.random.default_rng(15), [150] * 4, [3000, 2000, 1500, 1200], 16, 2, 16, F16, pad=5)
    guard = torch.full((64 + p.out.numel() + 64,), 7.0, dtype=p.out.dtype, device="cuda")
    p.out = guard[64:-64].view(p.out.shape)
    p.dc.copy_(dev(torch, np.array([0, 600, 0, 600, 0], np.int32)))
    p.max_new = 600
    p.ws = torch.full((glc.attn_paged_workspace_bytes(16, 2, 4, p.T, 600),), 255, dtype=torch.uint8, device="cuda")
    p.call()
    with pytest.raises(glc.GlcError, match="out of range"):
        glc.paged_poll_error()
    assert torch.all(guard[:64] == 7) and torch.all(guard[-64:] == 7) and torch.all(p.out[600:] == 7)
    p.dc.copy_(dev(torch, p.cu))
    p.call()
    glc.paged_poll_error()
    p.check()


@pytest.mark.parametrize("new,kv", [([1, 1, 1], [100, 600, 33]), ([100, 5], [400, 700])])
def test_paged_captured_and_replayed(cuda, glc, new, kv):
    """A captured call follows the device's lengths: replays with other ones."""
    torch = cuda
    p = Paged(torch, glc, np.random.default_rng(12), new, kv, 12, 2, 16, F16)
    p.call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        p.call(stream=torch.cuda.current_stream().cuda_stream)
    for cut in (0, 30, 1):
        kv2 = [a - cut for a in kv]
        p.dkv.copy_(dev(torch, np.array(kv2, np.int32)))
        p.out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        p2_k, p2_v, p.k, p.v, old = p.k, p.v, [a[:n] for a, n in zip(p.k, kv2)], [a[:n] for a, n in zip(p.v, kv2)], p.kv
        p.kv = kv2
        p.check()
        p.k, p.v, p.kv = p2_k, p2_v, old
    glc.paged_poll_error()


def test_two_calls_at_once(cuda, glc):
    """Two streams, two workspaces, many calls in flight."""
    torch = cuda
    rng = np.random.default_rng(13)
    ps = [Paged(torch, glc, rng, [1] * 6, [900, 3, 44, 1200, 17, 600], 40, 8, 16, F32),
          Paged(torch, glc, rng, [70, 3], [500, 90], 28, 4, 32, F16)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ps]
    for _ in range(20):
        for p, s in zip(ps, streams):
            p.call(stream=s.cuda_stream)
    glc.paged_poll_error()
    for p in ps:
        p.check()


@pytest.mark.parametrize("qt", [F32, F16])
@pytest.mark.parametrize("B,Hq,Hkv,ps", [(7, 28, 4, 32), (50, 8, 8, 16), (300, 6, 2, 16), (560, 16, 1, 64)])
def test_paged_mixed_batches(cuda, glc, B, Hq, Hkv, ps, qt):
    """Chunks next to decode tokens, idle sequences and sequences without keys:
    both kernels in one call, also with more sequences than a CTA keeps lengths of."""
    rng = np.random.default_rng(B)
    new, kv = [], []
    for b in range(B):
        n = (1, 1, 2, 0, 1, 1)[b % 6] if b % 23 else int(rng.integers(17, 60))
        new.append(n)
        kv.append(0 if b % 29 == 5 else n + int(rng.integers(0, 700 if b % 50 else 2600)))
    p = Paged(cuda, glc, rng, new, kv, Hq, Hkv, ps, qt, pad=3)
    p.call()
    glc.paged_poll_error()
    skip = [b for b in range(B) if B > 60 and b % 7 and b % 23 and b % 29 != 5]   # the oracle is slow
    p.check(skip=skip)
    first = p.out.clone()
    p.call()
    glc.paged_poll_error()
    assert cuda.equal(first, p.out)


@pytest.mark.parametrize("qt", [F32, F16])
@pytest.mark.parametrize("new", [1, 3, 40])
def test_paged_all_without_keys(cuda, glc, new, qt):
    p = Paged(cuda, glc, np.random.default_rng(16), [new] * 3, [0] * 3, 8, 2, 16, qt, pad=2)
    p.call()
    glc.paged_poll_error()
    assert cuda.all(p.out[:3 * new] == 0) and cuda.all(p.out[3 * new:] == 7)


@pytest.mark.parametrize("qt", [F32, F16])
def test_prompt_of_single_rows(cuda, glc, qt):
    """Few rows in all: sequences of one or two tokens among empty ones."""
    rng = np.random.default_rng(17)
    lens = [0, 1, 0, 2, 1, 0, 0, 3] + [0] * 300 + [1]
    T, cu = sum(lens), np.concatenate([[0], np.cumsum(lens)])
    q = rng.standard_normal((T, 4, 128)).astype(NP[qt])
    k, v = (rng.standard_normal((T, 2, 128)).astype(np.float16) for _ in range(2))
    got = run_prompt(cuda, glc, q, k, v, cu, qt).reshape(T, 4, 128)
    for b in range(len(lens)):
        s = slice(cu[b], cu[b + 1])
        if lens[b]:
            check_attention(got[s], q[s], k[s], v[s], 0, qt == F32)


@pytest.mark.parametrize("new,kv", [([1, 1, 2], [5000, 40, 3100]), ([70, 90], [3500, 1800])])
def test_graphs_that_share_a_workspace(cuda, glc, new, kv):
    """Two captured calls on one workspace, replayed in turn with keys split over
    CTAs and lengths that change between replays."""
    torch = cuda
    rng = np.random.default_rng(18)
    ps = [Paged(torch, glc, rng, new, kv, 12, 2, 16, F16), Paged(torch, glc, rng, new[::-1], kv[::-1], 12, 2, 16, F32)]
    ps[1].ws = ps[0].ws
    graphs = []
    for p in ps:
        p.call()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            p.call(stream=torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    full = [(p.k, p.v, p.kv) for p in ps]
    for cut in (0, 129, 1300):
        for p, (k, v, kv0) in zip(ps, full):
            p.kv = [max(a - cut, n) for a, n in zip(kv0, p.new)]
            p.k, p.v = [a[:n] for a, n in zip(k, p.kv)], [a[:n] for a, n in zip(v, p.kv)]
            p.dkv.copy_(dev(torch, np.array(p.kv, np.int32)))
            p.out.fill_(7.0)
        for _ in range(3):
            for g in graphs:
                g.replay()
        glc.paged_poll_error()
        for p in ps:
            p.check()


def test_mixed_call_is_done_when_the_next_starts(cuda, glc):
    """A copy right behind a call of both kernels sees all of its rows, live and
    captured, while the queries and the outputs change between calls."""
    torch = cuda
    rng = np.random.default_rng(19)
    p = Paged(torch, glc, rng, [1, 1, 40, 2, 1, 1, 1, 150], [900, 5000, 700, 64, 0, 3, 1700, 2000], 12, 2, 16, F16)
    flip = -p.dq
    p.call()
    glc.paged_poll_error()
    p.check()
    want = p.out.clone()
    p.dq.copy_(flip)
    p.call()
    want2 = p.out.clone()
    glc.paged_poll_error()
    assert not torch.equal(want, want2)
    stream = torch.cuda.Stream()
    copies = torch.empty(12, *p.out.shape, dtype=p.out.dtype, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for i in range(12):
            p.dq.neg_()
            p.out.fill_(7.0)
            p.call(stream=stream.cuda_stream)
            copies[i].copy_(p.out)
    glc.paged_poll_error()
    assert all(torch.equal(copies[i], want2 if i % 2 else want) for i in range(12))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for i in range(4):
            p.dq.neg_()
            p.out.fill_(7.0)
            p.call(stream=torch.cuda.current_stream().cuda_stream)
            copies[i].copy_(p.out)
    for _ in range(3):
        copies.zero_()
        g.replay()
        glc.paged_poll_error()
        assert all(torch.equal(copies[i], want2 if i % 2 else want) for i in range(4))


def test_host_memory_is_refused(cuda, glc):
    torch = cuda
    a = np.zeros(1 << 16, np.uint8)
    p = (a.ctypes.data + 15) & ~15
    with pytest.raises(glc.GlcError, match="device memory|known to CUDA"):
        glc.attn_prompt_dev(p, F32, 128, p, p, 128, p, 1, 1, 1, 1, p, 128, stream=glc.torch_stream_handle())


def test_offsets_past_32_bits(cuda, glc):
    """Pages far apart: a page stride that takes the offsets past 2^32 elements."""
    torch = cuda
    rng = np.random.default_rng(14)
    ps, Hkv, n_pages, stride = 16, 1, 9, (1 << 29) + 2048     # 4.8e9 elements in all
    buf = torch.empty(8 * stride + ps * 128 * 2, dtype=torch.float16, device="cuda")
    cache = glc.KvPages(buf.data_ptr(), buf.data_ptr() + ps * 128 * 2, n_pages, ps, Hkv, page_stride=stride)
    n = 40
    x = rng.standard_normal((n, 6, 128)).astype(np.float32)
    d = dev(torch, x)
    table = np.array([[8, 0, 7, -1]], np.int32)
    pos = np.arange(n, dtype=np.int32)
    slots = table[0, pos // ps].astype(np.int64) * ps + pos % ps
    qo = torch.empty(n, 4, 128, device="cuda")
    ds, dp, dt = dev(torch, slots), dev(torch, pos), dev(torch, table)
    p0, row = d.data_ptr(), 6 * 128
    glc.rope_append_dev(p0, row, p0 + 4 * 512, p0 + 4 * 640, row, n, 4, 1, dp.data_ptr(), ds.data_ptr(), THETA, cache,
                        qo.data_ptr(), F32, stream=glc.torch_stream_handle())
    cu, kv = dev(torch, np.array([0, n], np.int32)), dev(torch, np.array([n], np.int32))
    nb = glc.attn_paged_workspace_bytes(4, 1, 1, n, n)
    ws, out = torch.empty(nb, dtype=torch.uint8, device="cuda"), torch.empty(n, 4, 128, device="cuda")
    glc.attn_paged_dev(qo.data_ptr(), F32, 512, cache, dt.data_ptr(), 4, cu.data_ptr(), kv.data_ptr(), 1, n, n, 4,
                       out.data_ptr(), 512, ws.data_ptr(), nb, stream=glc.torch_stream_handle())
    glc.paged_poll_error()
    rows = torch.stack([buf[int(s // ps) * stride + int(s % ps) * 128:][:128] for s in slots]).cpu().numpy()
    vals = torch.stack([buf[int(s // ps) * stride + ps * 128 + int(s % ps) * 128:][:128] for s in slots]).cpu().numpy()
    rk = ref.rotate(x[:, 4:5], pos, THETA)
    assert np.all(np.abs(rows[:, None] - rk) <= rot_bound(x[:, 4:5], rk, F16))
    assert np.array_equal(vals, x[:, 5].astype(np.float16))
    check_attention(out.cpu().numpy(), qo.cpu().numpy(), rows[:, None], vals[:, None], 0, True)


# ------------------------------------------------------- the steps of a server
def test_serving_steps(cuda, glc):
    """Plan, rotate and store, attend, over several steps of a changing batch:
    prompts, chunks, decode tokens, requests that finish and come.  Every step's
    attention is checked on the keys and values as stored, and a decode step
    against the single-sequence decode attention on a contiguous cache."""
    torch = cuda
    rng = np.random.default_rng(20)
    Hq, Hkv, ps, B, width, n_pages, T = 10, 2, 16, 4, 12, 26, 96
    kc, vc, _, _ = make_pages(torch, n_pages, ps, Hkv, "head", fill=float("nan"))
    cache = glc.KvPages(kc.data_ptr(), vc.data_ptr(), n_pages, ps, Hkv)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    table, cu, kv, pos, bad = i32(B, width), i32(B + 1), i32(B), i32(T), i32(1)
    slots = torch.zeros(T, dtype=torch.int64, device="cuda")
    pool = dev(torch, rng.permutation(n_pages).astype(np.int32))
    counts = [dev(torch, np.array([n_pages], np.int32)), i32(1)]
    nb = glc.attn_paged_workspace_bytes(Hq, Hkv, B, T, T)
    ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
    qo, out = torch.empty(T, Hq, 128, device="cuda"), torch.empty(T, Hq, 128, device="cuda")
    held = np.zeros(B, np.int32)
    steps = [[40, 7, 0, 1], [1, 50, 20, 1], [1, 1, 1, 1], [-1, 1, 33, 30], [25, 1, 1, -1], [1, 1, -1, 60], [1, 1, 0, 1]]
    stream = glc.torch_stream_handle()
    hist = [[] for _ in range(B)]
    for n, new in enumerate(steps):
        x = rng.standard_normal((T, (Hq + 2 * Hkv) * 128)).astype(np.float32)
        d, dctx, dnew = dev(torch, x), dev(torch, held), dev(torch, np.array(new, np.int32))
        glc.kv_plan_dev(dctx.data_ptr(), dnew.data_ptr(), B, ps, table.data_ptr(), width, pool.data_ptr(), n_pages,
                        counts[n % 2].data_ptr(), counts[1 - n % 2].data_ptr(), T, cu.data_ptr(), kv.data_ptr(),
                        pos.data_ptr(), slots.data_ptr(), bad.data_ptr(), stream=stream)
        p0, row = d.data_ptr(), (Hq + 2 * Hkv) * 128
        glc.rope_append_dev(p0, row, p0 + 4 * Hq * 128, p0 + 4 * (Hq + Hkv) * 128, row, T, Hq, Hkv, pos.data_ptr(),
                            slots.data_ptr(), THETA, cache, qo.data_ptr(), F32, stream=stream)
        glc.attn_paged_dev(qo.data_ptr(), F32, Hq * 128, cache, table.data_ptr(), width, cu.data_ptr(), kv.data_ptr(),
                           B, T, max(max(new), 1), Hq, out.data_ptr(), Hq * 128, ws.data_ptr(), nb, stream=stream)
        glc.paged_poll_error()
        assert int(bad) == 0, n
        held = np.where(np.array(new) < 0, 0, held + np.maximum(new, 0)).astype(np.int32)
        assert list(kv.cpu()) == list(held)
        gk, gv, tb, c = kc.cpu().numpy(), vc.cpu().numpy(), table.cpu().numpy(), cu.cpu().numpy()
        assert int(counts[1 - n % 2]) == n_pages - int((-(-held // ps)).sum())
        used = np.concatenate([tb[b, :-(-held[b] // ps)] for b in range(B)])
        assert len(set(used.tolist())) == len(used)                       # no page twice
        for b in range(B):
            if new[b] < 0:
                hist[b] = []
                continue
            xs = x[c[b]:c[b + 1]].reshape(new[b], Hq + 2 * Hkv, 128)
            hist[b].extend(xs[:, Hq + Hkv:].astype(np.float16))
            j = np.arange(held[b])
            k, v = (a[tb[b, j // ps], :, j % ps] for a in (gk, gv))
            assert np.array_equal(v, np.array(hist[b], np.float16).reshape(-1, Hkv, 128))
            if new[b]:
                check_attention(out[c[b]:c[b + 1]].cpu().numpy(), qo[c[b]:c[b + 1]].cpu().numpy(), k, v, held[b] - new[b],
                                True)
            if new[b] == 1:   # the single-sequence decode attention on the same rows
                L = 256
                kk, vv = (torch.zeros(Hkv, L, 128, dtype=torch.float16, device="cuda") for _ in range(2))
                kk[:, :held[b]], vv[:, :held[b]] = dev(torch, k).transpose(0, 1), dev(torch, v).transpose(0, 1)
                o1 = torch.empty(Hq, 128, device="cuda")
                w1 = torch.zeros(glc.attn_workspace_bytes(Hq, Hkv, L), dtype=torch.uint8, device="cuda")
                t0 = int(c[b])
                dq, dk, dv = (dev(torch, xs[0, a:e]) for a, e in ((0, Hq), (Hq, Hq + Hkv), (Hq + Hkv, Hq + 2 * Hkv)))
                glc.attn_decode_dev(dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), kk.data_ptr(), vv.data_ptr(), Hq, Hkv,
                                    L, int(held[b]) - 1, THETA, o1.data_ptr(), w1.data_ptr(), w1.numel(), stream=stream)
                torch.cuda.synchronize()
                a, e = o1.cpu().numpy(), out[t0].cpu().numpy()
                assert np.linalg.norm(a - e) <= 1e-3 * np.linalg.norm(a)
