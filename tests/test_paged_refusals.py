"""Refusals of the paged entry points for memory that a call reads and writes at once
(decided on the host: no GPU is touched)."""
import pytest

from test_paged_oracle import F16, F32, P, append_args


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
