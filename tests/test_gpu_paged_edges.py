"""Calls of the paged-cache operators next to a limit."""
import os
import subprocess
import sys
import threading

import numpy as np
import pytest

from oracle import paged as ref
from test_gpu_paged import Paged, dev, plan_case, run_plan, same_plan

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)
LIBDIR = os.path.join(REPO, "glacier", "inference", "distributed_b200")


def plans_ascending(torch, glc):
    """Every request count around the one where static and dynamic shared memory
    together pass 48 KB, ascending, so that no larger call came before."""
    for B in range(2440, 2461):
        ctx, new, table, pool, free = plan_case(np.random.default_rng(B), B, 16, 90, 3)
        want = ref.plan(ctx, new, 16, table, pool, free, 6000)
        same_plan(run_plan(torch, glc, ctx, new, 16, table, pool, free, 6000), want)


def test_plan_of_every_size_in_a_fresh_process(cuda):
    code = ("import torch\nfrom glacier.inference import distributed_b200 as glc\n"
            "from test_gpu_paged_edges import plans_ascending\nplans_ascending(torch, glc)\n")
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([REPO, HERE, os.environ.get("PYTHONPATH", "")]))
    out = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout[-2000:] + out.stderr[-2000:]


def test_plans_from_two_host_threads(cuda, glc):
    """Calls of 2,500 and of 4,096 requests at once: neither changes what the other
    may launch."""
    torch = cuda
    cases = [plan_case(np.random.default_rng(B), B, 16, 90, 3) for B in (2500, 4096)]
    for c in cases:
        run_plan(torch, glc, c[0], c[1], 16, *c[2:], 9000)
    errors, stop = [], threading.Event()

    def many(c, n):
        ctx, new, table, pool, free = c
        B, width = table.shape
        s = torch.cuda.Stream()
        d = [torch.from_numpy(a).cuda() for a in (ctx, new, table, pool, np.array([free], np.int32))]
        o = [torch.zeros(k, dtype=torch.int32, device="cuda") for k in (1, B + 1, B, 9000, 1)]
        slots = torch.zeros(9000, dtype=torch.int64, device="cuda")
        torch.cuda.synchronize()
        a = [t.data_ptr() for t in d + o + [slots]]
        try:
            for i in range(n):
                if stop.is_set():
                    break
                glc.kv_plan_dev(a[0], a[1], B, 16, a[2], width, a[3], len(pool), a[4], a[5], 9000, a[6], a[7], a[8], a[10],
                                a[9], stream=s.cuda_stream)
                if i % 100 == 99:
                    s.synchronize()
        except glc.GlcError as e:
            errors.append(e)
            stop.set()
        s.synchronize()

    threads = [threading.Thread(target=many, args=(c, 6000)) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors


@pytest.mark.parametrize("T,Hq,Hkv", [(1, 40, 8), (700, 48, 8), (3000, 13, 1)])
def test_rotary_store_in_place_gives_the_same_bits(cuda, glc, T, Hq, Hkv):
    """Queries rotated where they lie, by warps that take one and several heads."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(T)
    q, k, v = (torch.randn(T, h, 128, generator=g, device="cuda") for h in (Hq, Hkv, Hkv))
    pos = torch.arange(T, dtype=torch.int32, device="cuda") * 11
    out = [torch.empty_like(q), torch.empty_like(q), q.clone()]
    packed = [torch.zeros(2, T, Hkv, 128, dtype=torch.float16, device="cuda") for _ in range(3)]
    for o, p in zip(out, packed):
        src = o if o is out[2] else q
        glc.rope_append_dev(src.data_ptr(), Hq * 128, k.data_ptr(), v.data_ptr(), Hkv * 128, T, Hq, Hkv, pos.data_ptr(), None,
                            1e6, None, o.data_ptr(), glc.GGUF_F32, p[0].data_ptr(), p[1].data_ptr(),
                            stream=glc.torch_stream_handle())
    glc.paged_poll_error()
    for o, p in zip(out[1:], packed[1:]):
        assert torch.equal(o, out[0]) and torch.equal(p, packed[0])


def built(tmp_path, name):
    exe = str(tmp_path / name)
    subprocess.check_call(["/usr/local/cuda/bin/nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O2",
                           "--expt-relaxed-constexpr", "-I", os.path.join(REPO, "include"), "-I", os.path.join(LIBDIR, "csrc"),
                           os.path.join(HERE, "cpp", name + ".cu"), "-o", exe, "-L", LIBDIR, "-lglacier_b200",
                           "-Xlinker", f"-rpath={LIBDIR}"])
    return exe


def test_bad_argument_does_not_hide_a_timeout(cuda, tmp_path):
    out = subprocess.run([built(tmp_path, "paged_error_check"), "order"], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout + out.stderr


def test_no_error_is_lost_to_a_poll(cuda, tmp_path):
    out = subprocess.run([built(tmp_path, "paged_error_check"), "lost"], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout + out.stderr


def test_places_of_the_join_are_written_after_a_timeout(cuda, tmp_path):
    out = subprocess.run([built(tmp_path, "tiles_scheduler_check")], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout + out.stderr


def test_every_array_in_host_memory_is_refused(cuda, glc):
    """Each device array of each call, replaced by ordinary host memory."""
    torch = cuda
    Hq, Hkv, T, B, ps = 4, 2, 20, 2, 16
    g = lambda *s, t=torch.int32: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
    host = np.zeros(1 << 16, np.uint8)
    bad = (host.ctypes.data + 63) & ~63
    f16, f32, i64 = torch.float16, torch.float32, torch.int64
    kc, vc = g(4, Hkv, ps, 128, t=f16), g(4, Hkv, ps, 128, t=f16)
    q, k, v, o = g(T, Hq, 128, t=f32), g(T, Hkv, 128, t=f32), g(T, Hkv, 128, t=f32), g(T, Hq, 128, t=f32)
    ko, vo = g(T, Hkv, 128, t=f16), g(T, Hkv, 128, t=f16)
    cu = torch.tensor([0, 10, 20], dtype=torch.int32, device="cuda")
    kv = torch.tensor([10, 10], dtype=torch.int32, device="cuda")
    slots = torch.arange(T, device="cuda")
    ws = g(glc.attn_paged_workspace_bytes(Hq, Hkv, B, T, T), t=torch.uint8)
    held = []                                     # arrays whose pointers are in use

    def p(t):
        held.append(t)
        return t.data_ptr()

    def pages(k_ptr, v_ptr):
        return glc.KvPages(k_ptr, v_ptr, 4, ps, Hkv)
    st = glc.torch_stream_handle()
    plan = dict(ctx_lens_ptr=p(g(B)), new_lens_ptr=p(g(B)), block_table_ptr=p(g(B, 4)), free_list_ptr=p(g(8)),
                free_count_ptr=p(g(1)), free_count_out_ptr=p(g(1)), cu_new_ptr=p(g(B + 1)), kv_lens_ptr=p(g(B)),
                positions_ptr=p(g(T)), slots_ptr=p(g(T, t=i64)), status_ptr=p(g(1)))
    append = dict(q_ptr=p(q), k_ptr=p(k), v_ptr=p(v), positions_ptr=p(g(T)), slots_ptr=p(slots), q_out_ptr=p(o),
                  k_out_ptr=p(ko), v_out_ptr=p(vo), cache_k=p(kc), cache_v=p(vc))
    prompt = dict(q_ptr=p(q), k_ptr=p(ko), v_ptr=p(vo), cu_seqlens_ptr=p(cu), out_ptr=p(o))
    paged = dict(q_ptr=p(q), block_table_ptr=p(g(B, 4)), cu_new_ptr=p(cu), kv_lens_ptr=p(kv), out_ptr=p(o), work_ptr=p(ws),
                 cache_k=p(kc), cache_v=p(vc))

    def call_append(a):
        a = dict(a)
        cache = pages(a.pop("cache_k"), a.pop("cache_v"))
        glc.rope_append_dev(**a, cache=cache, q_stride=Hq * 128, kv_stride=Hkv * 128, T=T, n_heads=Hq, n_kv_heads=Hkv,
                            rope_theta=1e6, stream=st)

    def call_paged(a):
        a = dict(a)
        cache = pages(a.pop("cache_k"), a.pop("cache_v"))
        glc.attn_paged_dev(**a, cache=cache, q_type=glc.GGUF_F32, q_stride=Hq * 128, max_pages=4, B=B, T=T, max_new=10,
                           n_heads=Hq, out_stride=Hq * 128, work_bytes=ws.numel(), stream=st)
    calls = [(plan, lambda a: glc.kv_plan_dev(**a, B=B, page_size=ps, max_pages=4, capacity=8, T=T, stream=st)),
             (append, call_append),
             (prompt, lambda a: glc.attn_prompt_dev(**a, q_type=glc.GGUF_F32, q_stride=Hq * 128, kv_stride=Hkv * 128, B=B, T=T,
                                                    n_heads=Hq, n_kv_heads=Hkv, out_stride=Hq * 128, stream=st)),
             (paged, call_paged)]
    for args, call in calls:
        call(args)
        for name in args:
            with pytest.raises(glc.GlcError, match="device memory|known to CUDA") as e:
                call({**args, name: bad})
            assert e.value.status == -1 and name.replace("_ptr", "").split("_")[-1][:3] in str(e.value), name
    glc.paged_poll_error()


@pytest.mark.parametrize("qt", [0, 1])
def test_decode_of_the_longest_tables(cuda, glc, qt):
    """Two sequences of 2^31 - 128 rows, the most a table may name, over two pages: one
    that is repeated, with keys of zero, and one behind it whose 64 keys score 20.  The
    sums of the weights are exact (multiples of 2^12, at most 2^18 of them); what rounds
    is the exponential (2^-20) and the join of 148 parts, in fp32, of numerator and
    denominator: 2 x 150 x 2^-24 < 2^-15 of the weighted values.  fp32 queries add their
    16-key products up exactly too (multiples of 2^11 below 2^35).  fp16 queries leave
    them in the tensor core's accumulator, which may cut a unit of the last place, 2^-23
    of the running sum, at each of a CTA's n tiles: equal products, so the sum after i
    tiles is i / n of the last, and the cuts together at most (n + 1) / 2 x 2^-23 of the
    repeated page's share; n is 2 (2^24 - 1 + 2) / 148 + 1."""
    torch = cuda
    ps, kv = 64, 2**31 - 128
    width = kv // ps
    rng = np.random.default_rng(21)
    val = rng.integers(-32, 33, (2, 128)) / 8
    kc, vc = (torch.zeros(2, 1, ps, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    kc[1, 0, :, 0] = 20
    vc[:, 0] = torch.from_numpy(val).cuda()[:, None, :]
    table = torch.zeros(2, width, dtype=torch.int32, device="cuda")
    table[:, -1] = 1
    dt = torch.float32 if qt == 0 else torch.float16
    q, out = torch.zeros(2, 1, 128, dtype=dt, device="cuda"), torch.zeros(2, 1, 128, dtype=dt, device="cuda")
    q[:, 0, 0] = 1
    cu = torch.arange(3, dtype=torch.int32, device="cuda")
    lens = torch.tensor([kv, kv - 64], dtype=torch.int32, device="cuda")     # the second ends before the last page
    ws = torch.empty(glc.attn_paged_workspace_bytes(1, 1, 2, 2, 1), dtype=torch.uint8, device="cuda")
    glc.attn_paged_dev(q.data_ptr(), qt, 128, glc.KvPages(kc.data_ptr(), vc.data_ptr(), 2, ps, 1), table.data_ptr(), width,
                       cu.data_ptr(), lens.data_ptr(), 2, 2, 1, 1, out.data_ptr(), 128, ws.data_ptr(), ws.numel(), scale=1.0,
                       stream=glc.torch_stream_handle())
    glc.paged_poll_error()
    w = np.array([kv - 64, 64 * np.exp(20.0)])
    w /= w.sum()
    got = out[:, 0].double().cpu().numpy()
    final = 2.0**-24 if qt == 0 else 2.0**-11
    cut = 0.0 if qt == 0 else (2 * (2**24 + 1) / 148 + 2) / 2 * 2.0**-23
    for g, wt in zip(got, (w, np.array([1.0, 0.0]))):
        want = wt @ val
        tol = (wt @ np.abs(val)) * 2.0**-15 + wt[0] * np.abs(val[0]) * cut + np.abs(want) * final + 1e-30
        assert (np.abs(g - want) <= tol).all()


@pytest.mark.parametrize("qt", [0, 1])
@pytest.mark.parametrize("new,kv", [([4, 4], [50, 60]), ([30, 50], [900, 60]), ([4, 40, 1, 2, 1, 3], [50, 600, 9, 70, 1, 400])])
def test_first_rows_outside_are_held_inside(cuda, glc, new, kv, qt):
    """A first row below 0 counts as 0, a last one past T as T: the rows that are left
    are right, nothing is recorded and nothing beside the outputs is written."""
    torch = cuda
    p = Paged(torch, glc, np.random.default_rng(22), new, kv, 8, 2, 16, qt)
    guard = torch.full((p.out.numel() + 4096,), 7.0, dtype=p.out.dtype, device="cuda")
    p.out = guard[2048:-2048].view(p.out.shape)
    around = torch.full((p.dq.numel() + 4096,), float("nan"), dtype=p.dq.dtype, device="cuda")
    around[2048:-2048] = p.dq.flatten()
    p.dq = around[2048:-2048].view(p.dq.shape)
    cu = p.cu.copy()
    cu[0], cu[-1] = -10, 10**9
    p.dc.copy_(dev(torch, cu))
    p.call()
    glc.paged_poll_error()
    p.check()
    assert torch.all(guard[:2048] == 7) and torch.all(guard[-2048:] == 7)


@pytest.mark.parametrize("new", [[1, 0, 2], [1, 0, 2, 0, 1, 1], [40, 0, 2], [40, 0, 2, 0, 1, 1]])
def test_idle_sequences_may_have_any_length(cuda, glc, new):
    """A padded batch: what stands in kv_lens for a sequence without new tokens is not
    used and not an error, whichever kernels run."""
    torch = cuda
    kv = [n + 30 * b for b, n in enumerate(new)]
    p = Paged(torch, glc, np.random.default_rng(23), new, kv, 8, 2, 16, 1)
    for garbage in (-1, 10**9, 2**31 - 1):
        p.dkv[1] = garbage
        p.out.fill_(7.0)
        p.call()
        glc.paged_poll_error()
        p.check()
