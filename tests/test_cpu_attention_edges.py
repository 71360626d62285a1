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


@pytest.mark.parametrize("dtype, N, Tq, Tk, Hq, Hk, D, divided", [
    # as many items as the card has room for, or too few keys for what joining them costs
    ("f32", 96, 128, 117, 4, 4, 64, False), ("f16", 96, 312, 312, 1, 1, 256, False), ("bf16", 300, 100, 300, 1, 1, 64, False),
    ("f16", 3, 1157, 1102, 8, 4, 96, False), ("bf16", 33, 1, 1100, 8, 8, 128, False), ("bf16", 4, 1, 1000, 8, 8, 64, False),
    ("f32", 256, 100, 300, 1, 1, 64, False),
    # few items and many keys
    ("bf16", 1, 1, 16384, 8, 1, 128, True), ("f32", 4, 1, 1124, 4, 2, 256, True), ("f16", 1, 4096, 4096, 4, 4, 128, True),
    ("bf16", 20, 100, 1000, 1, 1, 128, True), ("f32", 64, 100, 300, 1, 1, 64, True), ("bf16", 16, 1, 8192, 32, 8, 128, True),
    ("f32", 3, 1000, 2000, 16, 16, 64, True)])
def test_keys_are_divided_where_it_pays(dtype, N, Tq, Tk, Hq, Hk, D, divided):
    """Scratch without a mask is the parts of divided keys."""
    from raft_stereo_amd import _lib
    from test_cpu_attention import attn
    a = attn(N=N, Tq=Tq, Tk=Tk, Hq=Hq, Hk=Hk, D=D, dtype={"f32": _lib.RC_F32, "f16": _lib.RC_F16, "bf16": _lib.RC_BF16}[dtype])
    assert (_lib.lib.rc_cross_attn_fwd_work_bytes(a) > 0) == divided
