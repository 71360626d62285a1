"""CPU-side checks of the attention operators beside test_cpu_attention.py: arguments that are handed on or refused before
anything is launched."""
import pytest
import torch


def test_widths_reach_the_attention_in_front_of_the_volume():
    import raft_stereo_amd as R
    f, w1, w2 = torch.zeros(2, 8, 2, 16), torch.tensor([16, 9]), torch.tensor([7, 16])
    seen = []

    def attention(*args, **kw):
        seen.append((len(args), kw))
        return args[:2]
    for kw in ({}, dict(width1=w1), dict(width2=w2), dict(width1=w1, width2=w2)):
        with pytest.raises(RuntimeError, match="no CPU path"):       # from the block, behind the attention
            R.make_corr_fn("reg_hip", f, f, attention=attention, **kw)
        assert seen.pop() == (2, kw)
    for kw in (dict(width1=w1), dict(width2=w2)):
        with pytest.raises(ValueError, match="need attention"):
            R.make_corr_fn("reg_hip", f, f, **kw)


def test_scales_beyond_fp32_in_log2_are_refused():
    from raft_stereo_amd._lib import lib
    from test_cpu_attention import attn
    assert lib.rc_cross_attn_fwd_work_bytes(attn(scale=2.0 ** 126)) >= 0
    for scale in (2.0 ** 127, 3.0e38):         # finite, but not times log2 e
        a = attn(scale=scale)
        assert lib.rc_cross_attn_fwd_work_bytes(a) == lib.rc_cross_attn_bwd_work_bytes(a) == -1
        assert lib.rc_cross_attn_fwd(a, 16, 16, 16, 16, None, None, 16, None) == -1


def test_row_attention_frequencies_survive_empty_storage():
    """Deferred initialisation: parameters come from a checkpoint, the frequencies do not."""
    import raft_stereo_amd as R
    want = R.RowAttentionHip(32, heads=2).freqs.clone()
    before = torch.are_deterministic_algorithms_enabled()
    torch.use_deterministic_algorithms(True)       # (fills empty storage with NaN)
    try:
        assert torch.equal(R.RowAttentionHip(32, heads=2).to_empty(device="cpu").freqs, want)
        assert torch.equal(R.RowAttentionHip(32, heads=2).to("meta").to_empty(device="cpu").freqs, want)
        with torch.device("meta"):
            m = R.RowAttentionHip(32, heads=2)
        assert torch.equal(m.to_empty(device="cpu").half().freqs, want) and m.q.weight.device.type == "cpu"
        ptr = m.freqs.data_ptr()
        assert m.to("cpu").freqs.data_ptr() == ptr      # nothing to move: a captured graph may read them there
    finally:
        torch.use_deterministic_algorithms(before)
