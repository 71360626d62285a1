"""CPU-side checks of the attention operators: refusals at the C entry points (before anything is launched), and the
oracle's gradients against differences of its own forward forms."""
import numpy as np
import pytest

from oracle import attention_oracle as A


def attn(**kw):
    from raft_stereo_amd._lib import Attn, RC_F16
    a = Attn()
    a.N, a.Tq, a.Tk, a.Hq, a.Hk, a.D, a.dtype, a.scale = 2, 8, 9, 4, 2, 64, RC_F16, 0.125
    for name, H in (("q_stride", 4), ("k_stride", 2), ("v_stride", 2)):
        st = getattr(a, name)
        st[0], st[1], st[2] = 9 * H * 64, H * 64, 64
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(a, k)[v[0]] = v[1]
        else:
            setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,rc", [
    (dict(D=12), -2), (dict(D=264), -2), (dict(D=0), -2), (dict(dtype=3), -2), (dict(N=-1), -1), (dict(Tq=-1), -1),
    (dict(Hk=3), -1), (dict(Hk=0), -1), (dict(Hq=0), -1), (dict(scale=0.0), -1), (dict(scale=float("nan")), -1),
    (dict(scale=float("inf")), -1), (dict(q_stride=(1, 4)), -1), (dict(k_stride=(0, -64)), -1),
    (dict(v_stride=(1, 1 << 24)), -1), (dict(v_stride=(1, 1 << 22)), -1), (dict(k_stride=(2, 1 << 22)), -1),
    (dict(Tk=1 << 31), -1), (dict(N=1 << 30, Tk=1 << 20), -1),
    (dict(key_mask=16, mask_stride=-1), -1)])
def test_attention_descriptions_are_checked(kw, rc):
    from raft_stereo_amd._lib import lib
    a = attn(**kw)
    assert lib.rc_cross_attn_fwd_work_bytes(a) == rc and lib.rc_cross_attn_bwd_work_bytes(a) == rc
    assert lib.rc_cross_attn_fwd(a, 16, 16, 16, 16, None, None, 16, None) == rc
    assert lib.rc_cross_attn_bwd(a, 16, 16, 16, 16, None, 16, 16, 16, 16, 16, 16, None) == rc
    assert lib.rc_last_error_string()


def test_attention_operands_are_checked():
    from raft_stereo_amd._lib import lib
    a = attn()
    assert lib.rc_cross_attn_fwd_work_bytes(a) >= 0 and lib.rc_cross_attn_bwd_work_bytes(a) > 0
    for i in range(4):
        for bad in (None, 8):
            p = [16] * 4
            p[i] = bad
            assert lib.rc_cross_attn_fwd(a, *p, None, None, 16, None) == -1
    assert lib.rc_cross_attn_fwd(a, 16, 16, 16, 16, 24, None, 16, None) == -1        # misaligned rest
    for i in (0, 1, 2, 3, 5, 6, 10):                  # (4, the rest, may be left out)
        p = [16] * 11
        p[i] = None
        assert lib.rc_cross_attn_bwd(a, *p, None) == -1
    p = [16] * 11
    p[8] = None                                       # dk without dv
    assert lib.rc_cross_attn_bwd(a, *p, None) == -1
    for i in (4, 8):
        p = [16] * 11
        p[i] = 24                                     # misaligned
        assert lib.rc_cross_attn_bwd(a, *p, None) == -1
    assert lib.rc_cross_attn_fwd(None, 16, 16, 16, 16, None, None, 16, None) == -1
    assert lib.rc_cross_attn_fwd(attn(N=0), None, None, None, None, None, None, None, None) == 0      # nothing to do
    assert lib.rc_cross_attn_fwd(attn(Tq=0), None, 16, 16, None, None, None, None, None) == 0


def heads(**kw):
    from raft_stereo_amd._lib import Heads
    h = Heads()
    h.x, h.T, h.H = 16, 5, 2
    h.stride[0], h.stride[1], h.stride[2] = 640, 128, 64
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(h, k)[v[0]] = v[1]
        else:
            setattr(h, k, v)
    return h


@pytest.mark.parametrize("q,rest,rc", [
    (dict(), dict(D=12), -2), (dict(), dict(D=264), -2), (dict(), dict(dtype=5), -2), (dict(), dict(n=6), -2),
    (dict(), dict(n=36), -2), (dict(), dict(n=-4), -2), (dict(), dict(freqs=None), -1), (dict(), dict(y=None), -1),
    (dict(), dict(y=8), -1), (dict(x=None), {}, -1), (dict(x=8), {}, -1), (dict(stride=(1, -64)), {}, -1),
    (dict(stride=(2, 4)), {}, -1), (dict(T=-1), {}, -1), (dict(T=1 << 31), {}, -1),
    (dict(weight=16, weight_dtype=9), {}, -2), (dict(pos=16, pos_dtype=9), {}, -2)])
def test_norm_rotate_arguments_are_checked(q, rest, rc):
    from raft_stereo_amd._lib import lib, RC_F16
    a = dict(D=64, dtype=RC_F16, n=32, freqs=16, y=16, N=2)
    a.update(rest)
    for side in range(2):
        ok, bad = heads(), heads(**q)
        qs, ks = (bad, ok) if side == 0 else (ok, bad)
        ys = (a["y"], 16) if side == 0 else (16, a["y"])
        assert lib.rc_qk_norm_rotate_fwd(qs, ks, *ys, a["N"], a["D"], a["dtype"], a["freqs"], 0, a["n"], 0, 1e-6, None) == rc
        assert lib.rc_qk_norm_rotate_bwd(qs, ks, 16, 16, *ys, 16, 16, 16, a["N"], a["D"], a["dtype"], a["freqs"], 0,
                                         a["n"], 0, 1e-6, None) == rc
        assert lib.rc_last_error_string()


def test_norm_rotate_backward_operands_are_checked():
    from raft_stereo_amd._lib import lib, RC_F16
    call = lambda k, gq, gk, dk, dwk, work: lib.rc_qk_norm_rotate_bwd(heads(), k, gq, gk, 16, dk, 16, dwk, work, 2, 64, RC_F16,
                                                                      16, 0, 32, 0, 1e-6, None)
    assert call(None, None, None, None, None, 16) == -1          # no gradient
    assert call(None, 8, None, None, None, 16) == -1             # misaligned
    assert call(heads(), 16, None, 16, 16, 16) == -1
    assert call(heads(), 16, 16, 16, 16, None) == -1             # no scratch for the weight gradients
    assert call(None, 16, None, None, 16, 16) == -1              # a key weight's gradient without keys
    assert lib.rc_qk_norm_rotate_bwd_work_bytes(12) < 0 and lib.rc_qk_norm_rotate_bwd_work_bytes(64) > 0
    assert lib.rc_qk_norm_rotate_fwd(None, None, 16, None, 2, 64, RC_F16, 16, 0, 32, 0, 1e-6, None) == -1
    assert lib.rc_qk_norm_rotate_fwd(heads(T=0, x=None), None, None, None, 2, 64, RC_F16, 16, 0, 32, 0, 1e-6, None) == 0


def test_operators_refuse_cpu_tensors():
    import torch
    import raft_stereo_amd as R
    x = torch.randn(1, 4, 2, 32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        R.cross_attention_hip(x, x, x)
    with pytest.raises(RuntimeError, match="no CPU path"):
        R.qk_norm_rotate_hip(x, x)
    with pytest.raises(RuntimeError, match="no CPU path"):
        R.RowAttentionHip(32, heads=1)(torch.randn(1, 32, 2, 8), torch.randn(1, 32, 2, 9))
    for kw in (dict(heads=0), dict(heads=4, kv_heads=3), dict(heads=3), dict(head_dim=264)):
        with pytest.raises(ValueError):
            R.RowAttentionHip(32, **kw)


def test_row_attention_frequencies_survive_a_cast():
    import torch
    import raft_stereo_amd as R
    m = R.RowAttentionHip(32, heads=2)
    want = m.freqs.clone()
    assert want.dtype is torch.float64 and torch.equal(m.half().freqs, want) and m.q.weight.dtype is torch.float16
    assert list(m.state_dict()) == ["q_weight", "k_weight", "q.weight", "k.weight", "v.weight", "out.weight", "out.bias"]


def test_oracle_gradients_against_differences():
    rng = np.random.default_rng(0)
    N, Tq, Tk, Hq, Hk, D, h = 2, 5, 7, 4, 2, 8, 1e-6
    x = [rng.standard_normal(s) for s in ((N, Tq, Hq, D), (N, Tk, Hk, D), (N, Tk, Hk, D))]
    g = rng.standard_normal((N, Tq, Hq, D))
    ok = A.allowed_keys(N, Tk, [5, Tk], rng.random((N, Tk)) < 0.8)
    res = A.attention(*x, g, ok)
    for i, name in enumerate(("dq", "dk", "dv")):
        d = rng.standard_normal(x[i].shape)
        f = lambda s: (A.attention(*[a + s * d if j == i else a for j, a in enumerate(x)], None, ok)["out"][0] * g).sum()
        assert abs((f(h) - f(-h)) / (2 * h) - (res[name][0] * d).sum()) < 1e-6
    y, w, gy = rng.standard_normal((2, 3, 2, 24)), rng.standard_normal(24), rng.standard_normal((2, 3, 2, 24))
    for il in (False, True):
        res = A.norm_rotate(y, w, [0.3, 0.7, 1.1, 2.0], None, 1e-3, il, gy)
        d, dw = rng.standard_normal(y.shape), rng.standard_normal(24)
        f = lambda s, t: (A.norm_rotate(y + s * d, w + t * dw, [0.3, 0.7, 1.1, 2.0], None, 1e-3, il)["y"][0] * gy).sum()
        assert abs((f(h, 0) - f(-h, 0)) / (2 * h) - (res["dx"][0] * d).sum()) < 1e-6
        assert abs((f(0, h) - f(0, -h)) / (2 * h) - (res["dw"][0] * dw).sum()) < 1e-6


def test_oracle_of_an_empty_sequence():
    x = np.random.default_rng(1).standard_normal((2, 3, 1, 8))
    res = A.attention(x, x, x, x, A.allowed_keys(2, 3, [0, 2]))
    assert not res["out"][0][0].any() and not res["dq"][0][0].any() and not res["dk"][0][0].any()
    assert not res["dv"][0][1, 2].any() and res["dv"][0][1, 1].any()
