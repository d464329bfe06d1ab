"""Refusals of the paged entry points for memory that a call reads and writes at once
(decided on the host: no GPU is touched)."""
import pytest

from test_paged_oracle import F16, F32, P, append_args, paged_args, pages, plan_args


@pytest.mark.parametrize("kw", [
    dict(q_out_ptr=P + 16), dict(q_out_ptr=P - 16), dict(T=9, q_out_ptr=P + 2048),
    dict(T=9, q_out_ptr=P, q_stride=512, k_ptr=P + 9 * 2048 - 16),         # in place, over the first key
    dict(T=4, q_stride=1024, q_out_ptr=P + 2048, k_ptr=8 * P, v_ptr=8 * P),   # between the rows, but longer than a gap
    dict(q_out_ptr=2 * P, v_ptr=2 * P + 1024), dict(T=3, q_out_ptr=2 * P, q_out_type=F16, k_ptr=2 * P + 3 * 1024 - 16),
    dict(k_out_ptr=P, v_out_ptr=4 * P), dict(k_out_ptr=4 * P, v_out_ptr=P + 512),
    dict(n_heads=0, q_ptr=None, q_stride=0, q_out_ptr=None, k_out_ptr=4 * P, v_out_ptr=P + 1008)])
def test_append_refuses_outputs_over_inputs(glc, kw):
    with pytest.raises(glc.GlcError, match="overlap") as e:
        glc.rope_append_dev(**append_args(glc, **kw))
    assert e.value.status == -1


@pytest.mark.parametrize("kw", [
    dict(), dict(q_out_ptr=P), dict(q_out_ptr=P - 2048), dict(q_out_ptr=P + 2048),
    dict(T=2, q_stride=1024, q_out_ptr=P + 2048, q_out_type=F16, k_ptr=8 * P, v_ptr=8 * P),   # inside a gap
    dict(T=3, q_out_ptr=2 * P, q_out_type=F16, k_ptr=2 * P + 3 * 1024, v_ptr=2 * P + 3 * 1024),
    dict(k_out_ptr=P + 2048, v_out_ptr=P + 4096),
    dict(n_heads=0, q_ptr=None, q_stride=0, q_out_ptr=None, k_out_ptr=P + 1024, v_out_ptr=4 * P)])
def test_append_takes_outputs_beside_inputs(glc, kw):
    """These go on to the check of the memory, which fails for a made-up pointer."""
    a = append_args(glc, **kw)
    if a["q_out_ptr"] == P:
        a.update(k_ptr=8 * P, v_ptr=8 * P, q_out_type=F32)
    with pytest.raises(glc.GlcError, match="device|CUDA"):
        glc.rope_append_dev(**a)


def apart(**kw):
    """A plan of 100 requests and 100 rows whose arrays lie side by side."""
    a = plan_args(B=100, T=100, capacity=40, max_pages=4)
    at = P
    for name, n in (("ctx_lens", 400), ("new_lens", 400), ("free_count", 4), ("free_count_out", 4), ("block_table", 1600),
                    ("free_list", 160), ("cu_new", 404), ("kv_lens", 400), ("positions", 400), ("slots", 800), ("status", 4)):
        a[name + "_ptr"] = at
        at += n
    a.update({k: a[v[0]] + v[1] for k, v in kw.items()})
    return a


@pytest.mark.parametrize("out", ["block_table_ptr", "free_list_ptr", "free_count_out_ptr", "cu_new_ptr", "kv_lens_ptr",
                                 "positions_ptr", "slots_ptr", "status_ptr"])
@pytest.mark.parametrize("over,offset", [("ctx_lens_ptr", 0), ("ctx_lens_ptr", 396), ("new_lens_ptr", 200),
                                         ("free_count_ptr", 0)])
def test_plan_refuses_outputs_over_inputs(glc, out, over, offset):
    with pytest.raises(glc.GlcError, match="alias") as e:
        glc.kv_plan_dev(**apart(**{out: (over, offset)}))
    assert e.value.status == -1


def test_plan_takes_arrays_side_by_side(glc):
    """Goes on to the check of the memory, which fails for a made-up pointer."""
    with pytest.raises(glc.GlcError, match="device|CUDA"):
        glc.kv_plan_dev(**apart())


@pytest.mark.parametrize("ps", [16, 32, 64, 128, 256])
def test_paged_refuses_tables_whose_tiles_pass_31_bits(glc, ps):
    """The kernels round a key count up to tiles of 128 in 32 bits."""
    most = (2**31 - 128) // ps
    for n in (most + 1, (2**31 - 1) // ps + 1):
        with pytest.raises(glc.GlcError, match="tables") as e:
            glc.attn_paged_dev(**paged_args(glc, cache=pages(glc, page_size=ps), max_pages=n))
        assert e.value.status == -1
    with pytest.raises(glc.GlcError, match="device|CUDA"):     # goes on to the check of the memory
        glc.attn_paged_dev(**paged_args(glc, cache=pages(glc, page_size=ps), max_pages=most))
