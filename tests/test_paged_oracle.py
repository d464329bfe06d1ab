"""Closed-form cases of the paged-cache oracle, and the refusals of the paged
entry points that are decided on the host (no GPU is touched)."""
import numpy as np
import pytest

from oracle import paged
from oracle.attention import attn_decode, rope

F32, F16 = 0, 1
P = 0x10000  # a pointer that no call below may follow


def test_plan_by_hand():
    table = np.array([[7, 3, -1, -1], [5, -1, -1, -1], [2, 9, -1, -1]], np.int32)
    pool = np.array([1, 4, 6, 0, 0, 0], np.int32)
    # request 0: 17 cached + 20 new -> pages 2 -> 3; request 1 finished (10 cached); request 2: 32 + 1 -> a new page
    t, f, left, cu, kv, pos, slots, bad = paged.plan([17, 10, 32], [20, -1, 1], 16, table, pool, 3, 24)
    assert list(f[:4]) == [1, 4, 6, 5]           # page 5 came back on top
    assert list(t[0]) == [7, 3, 5, -1] and list(t[2]) == [2, 9, 6, -1]
    assert left == 2 and list(cu) == [0, 20, 20, 21] and list(kv) == [37, 0, 33] and bad == 0
    assert pos[0] == 17 and slots[0] == 3 * 16 + 1 and slots[15] == 5 * 16 and slots[20] == 6 * 16
    assert list(slots[21:]) == [-1, -1, -1]


def test_plan_out_of_pages_and_rows():
    table = np.full((3, 2), -1, np.int32)
    out = paged.plan([0, 0, 0], [16, 17, 1], 16, table, np.array([8, 9], np.int32), 2, 40)
    assert list(out[4]) == [16, 0, 0] and out[7] == 2   # 1 + 2 pages wanted of 2; the third wants a fourth
    out = paged.plan([0, 0], [30, 30], 16, table[:2], np.arange(8, dtype=np.int32), 8, 40)
    assert list(out[4]) == [30, 0] and list(out[3]) == [0, 30, 40] and out[7] == 1


def test_attend_against_decode_oracle():
    rng = np.random.default_rng(3)
    Hq, Hkv, L, pos = 6, 2, 20, 13
    q, kn, vn = (rng.standard_normal((h, 128)).astype(np.float32) for h in (Hq, Hkv, Hkv))
    kc, vc = (rng.standard_normal((Hkv, L, 128)).astype(np.float16) for _ in range(2))
    ref, kc2, vc2 = attn_decode(q, kn, vn, kc, vc, pos, 1e6)
    out, *_ = paged.attend(rope(q, pos, 1e6)[None], kc2.transpose(1, 0, 2)[:pos + 1], vc2.transpose(1, 0, 2)[:pos + 1],
                           pos, 1 / np.sqrt(128))
    assert np.allclose(out[0], ref, rtol=1e-12, atol=1e-12)


def test_attend_without_keys_is_zero():
    q = np.ones((3, 2, 128))
    out, *_ = paged.attend(q, np.ones((1, 1, 128)), np.full((1, 1, 128), 5.0), -2, 1.0)
    assert np.all(out[:2] == 0) and np.all(out[2] == 5)


def plan_args(**kw):
    a = dict(ctx_lens_ptr=P, new_lens_ptr=2 * P, B=1, page_size=16, block_table_ptr=P, max_pages=4, free_list_ptr=P,
             capacity=4, free_count_ptr=P, free_count_out_ptr=2 * P, T=1, cu_new_ptr=P, kv_lens_ptr=3 * P,
             positions_ptr=P, slots_ptr=P, status_ptr=P, stream=1)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,status,text", [
    ({"ctx_lens_ptr": None}, -1, "null"), ({"status_ptr": None}, -1, "null"), ({"slots_ptr": None}, -1, "null"),
    ({"B": -1}, -1, "requests"), ({"T": -1}, -1, "rows"), ({"max_pages": 0}, -1, "pages"),
    ({"capacity": -1}, -1, "pages"), ({"page_size": 24}, -4, "page_size"), ({"page_size": 512}, -4, "page_size"),
    ({"kv_lens_ptr": P}, -1, "alias"), ({"kv_lens_ptr": 2 * P}, -1, "alias"),
    ({"free_count_out_ptr": P}, -1, "alias")])
def test_plan_refuses(glc, kw, status, text):
    with pytest.raises(glc.GlcError, match=text) as e:
        glc.kv_plan_dev(**plan_args(**kw))
    assert e.value.status == status


def pages(glc, **kw):
    a = dict(k_ptr=P, v_ptr=P, n_pages=4, page_size=16, n_kv_heads=2)
    a.update(kw)
    return glc.KvPages(**a)


BAD_PAGES = [({"k_ptr": None}, -1, "null"), ({"k_ptr": P + 8}, -1, "aligned"), ({"page_size": 48}, -4, "page_size"),
             ({"page_size": 8}, -4, "page_size"), ({"head_dim": 64}, -4, "head_dim"), ({"n_pages": 0}, -1, "pages"),
             ({"row_stride": 64}, -1, "strides"), ({"row_stride": 132}, -1, "strides"),
             ({"head_stride": 0}, -1, "strides"), ({"page_stride": -8}, -1, "strides"),
             ({"page_stride": 1 << 38}, -1, "strides")]


def append_args(glc, **kw):
    a = dict(q_ptr=P, q_stride=512, k_ptr=P, v_ptr=P, kv_stride=256, T=1, n_heads=4, n_kv_heads=2, positions_ptr=P,
             slots_ptr=P, rope_theta=1e6, cache=pages(glc), q_out_ptr=2 * P, q_out_type=F32, stream=1)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,status,text", [
    ({"T": -1}, -1, "rows"), ({"n_kv_heads": 0}, -1, "KV heads"), ({"k_ptr": None}, -1, "null"),
    ({"q_out_ptr": None}, -1, "null"), ({"slots_ptr": None}, -1, "null"), ({"k_out_ptr": P}, -1, "null"),
    ({"q_out_type": 2}, -4, "type"), ({"rope_theta": 0.0}, -1, "rope_theta"),
    ({"rope_theta": float("nan")}, -1, "rope_theta"), ({"rope_theta": float("inf")}, -1, "rope_theta"),
    ({"q_ptr": P + 4}, -1, "aligned"), ({"q_stride": 514}, -1, "aligned"), ({"q_stride": 508}, -1, "shorter"),
    ({"kv_stride": 252}, -1, "shorter"), ({"q_out_ptr": P, "q_out_type": F16}, -1, "in place"),
    ({"q_out_ptr": P, "q_stride": 1024}, -1, "in place"), ({"n_kv_heads": 1}, -1, "cache of 2")])
def test_append_refuses(glc, kw, status, text):
    with pytest.raises(glc.GlcError, match=text) as e:
        glc.rope_append_dev(**append_args(glc, **kw))
    assert e.value.status == status


@pytest.mark.parametrize("kw,status,text", BAD_PAGES)
def test_page_sets_refused(glc, kw, status, text):
    for call in (lambda c: glc.rope_append_dev(**append_args(glc, cache=c)),
                 lambda c: glc.attn_paged_dev(**paged_args(glc, cache=c))):
        with pytest.raises(glc.GlcError, match=text) as e:
            call(pages(glc, **kw))
        assert e.value.status == status


def prompt_args(**kw):
    a = dict(q_ptr=P, q_type=F32, q_stride=512, k_ptr=P, v_ptr=P, kv_stride=256, cu_seqlens_ptr=P, B=1, T=1,
             n_heads=4, n_kv_heads=2, out_ptr=P, out_stride=512, stream=1)
    a.update(kw)
    return a


def paged_args(glc, **kw):
    a = dict(q_ptr=P, q_type=F32, q_stride=512, cache=pages(glc), block_table_ptr=P, max_pages=4, cu_new_ptr=P,
             kv_lens_ptr=P, B=1, T=1, max_new=1, n_heads=4, out_ptr=P, out_stride=512, work_ptr=P,
             work_bytes=1 << 40, stream=1)
    a.update(kw)
    return a


ROWS = [({"q_ptr": None}, -1, "null"), ({"out_ptr": None}, -1, "null"), ({"q_type": 30}, -4, "type"),
        ({"n_heads": 5}, -4, "heads"), ({"n_heads": 34}, -4, "heads"), ({"B": -1}, -1, "sequences"),
        ({"T": -1}, -1, "sequences"), ({"q_stride": 510}, -1, "aligned"), ({"q_stride": 508}, -1, "shorter"),
        ({"out_stride": 508}, -1, "shorter"), ({"q_ptr": P + 4}, -1, "aligned"), ({"scale": -1.0}, -1, "scale"),
        ({"scale": float("nan")}, -1, "scale"), ({"scale": float("inf")}, -1, "scale"),
        ({"q_type": F16, "q_stride": 516}, -1, "aligned")]


@pytest.mark.parametrize("kw,status,text", ROWS + [
    ({"head_dim": 64}, -4, "head_dim"), ({"kv_stride": 248}, -1, "apart"), ({"kv_stride": 260}, -1, "apart"),
    ({"k_ptr": P + 2}, -1, "apart"), ({"cu_seqlens_ptr": None}, -1, "null"), ({"n_kv_heads": 0}, -4, "heads")])
def test_prompt_refuses(glc, kw, status, text):
    with pytest.raises(glc.GlcError, match=text) as e:
        glc.attn_prompt_dev(**prompt_args(**kw))
    assert e.value.status == status


@pytest.mark.parametrize("kw,status,text", ROWS + [
    ({"block_table_ptr": None}, -1, "null"), ({"max_pages": 0}, -1, "tables"), ({"max_new": -1}, -1, "tables"),
    ({"max_pages": 1 << 28}, -1, "tables"), ({"work_bytes": 0}, -1, "workspace"),
    ({"work_ptr": P + 4}, -1, "workspace")])
def test_paged_refuses(glc, kw, status, text):
    with pytest.raises(glc.GlcError, match=text) as e:
        glc.attn_paged_dev(**paged_args(glc, **kw))
    assert e.value.status == status


def test_empty_calls_do_nothing(glc):
    """No rows: nothing is launched, so no device is needed."""
    glc.rope_append_dev(**append_args(glc, T=0))
    glc.attn_prompt_dev(**prompt_args(T=0))
    glc.attn_prompt_dev(**prompt_args(B=0))
    glc.attn_paged_dev(**paged_args(glc, B=0))
    glc.attn_paged_dev(**paged_args(glc, T=0))


def test_workspace_bytes_refuses(glc):
    for bad in ((4, 3, 1, 1, 1), (0, 1, 1, 1, 1), (4, 2, -1, 1, 1), (4, 2, 1, -1, 1), (4, 2, 1, 1, -1), (34, 2, 1, 1, 1)):
        with pytest.raises(glc.GlcError):
            glc.attn_paged_workspace_bytes(*bad)
    assert glc.attn_paged_workspace_bytes(40, 8, 64, 64, 1) > 0


@pytest.mark.parametrize("kw", [dict(max_pages=1 << 27, page_size=16), dict(max_pages=1 << 23, page_size=256),
                                dict(capacity=2**31 - 1)])
def test_plan_refuses_positions_past_32_bits(glc, kw):
    with pytest.raises(glc.GlcError, match="page plan") as e:
        glc.kv_plan_dev(**plan_args(**kw))
    assert e.value.status == -1


@pytest.mark.parametrize("heads,kv", [(40, 8), (28, 4), (16, 1), (8, 8)])
def test_workspace_of_the_largest_call_serves_smaller_ones(glc, heads, kv):
    sizes = [glc.attn_paged_workspace_bytes(heads, kv, B, T, T) for B, T in
             ((1, 1), (2, 17), (2, 64), (9, 300), (9, 4096), (64, 16384), (64, 70000), (500, 1000000))]
    assert sizes == sorted(sizes)
    for T in (1, 40, 5000, 400000):
        by_new = [glc.attn_paged_workspace_bytes(heads, kv, 300, T, n) for n in (0, 1, 2, 16, 17, 500)]
        assert by_new == sorted(by_new)
        by_batch = [glc.attn_paged_workspace_bytes(heads, kv, B, T, 500) for B in (0, 1, 4, 5, 40, 300, 5000)]
        assert by_batch == sorted(by_batch)
