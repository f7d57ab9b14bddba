"""What the rotary / ragged-batch KV-cache calls promise beside their results, without a GPU: refusals of buffers that meet."""
import pytest

from test_rope_kv_host import INVALID_SHAPE, P, bwd_call, eng  # noqa: F401


@pytest.mark.parametrize("override", [dict(dgk=P[9] + 64), dict(dgq=P[10] + 252), dict(dgq=P[8] + 128), dict(dgk=P[8]), dict(dgk=P[8] + 4 * (2 * 8 * 64 - 1))])
def test_norm_gradients_that_overlap_are_refused(eng, override):  # noqa: F811
    assert eng.lib.axb_qkv_norm_rope_bwd(*bwd_call(**override)) == INVALID_SHAPE
    assert "two outputs overlap" in eng.last_error()


@pytest.mark.parametrize("override", [dict(dgk=P[9]), dict(dgk=P[9] + 256), dict(dgq=P[8] + 4 * 2 * 8 * 64), dict(dgq=None), dict(dgk=None)])
def test_norm_gradients_side_by_side_or_in_one_buffer_are_not(eng, override):  # noqa: F811
    """A call that passes every check of its arguments ends at the missing device here (never run with one: the addresses are made up)."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("needs a machine without a GPU")
    assert eng.lib.axb_qkv_norm_rope_bwd(*bwd_call(**override)) != INVALID_SHAPE
    assert "no CUDA device" in eng.last_error()
