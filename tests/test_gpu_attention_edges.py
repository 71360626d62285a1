"""GPU tests of the attention operators where the way that the library takes decides: infinite scores in parts of divided
keys, many parts, rows that end inside a tile, long rows in fp16, norms of more tokens than one block's share.  Expected
values and bounds are the oracle's (64-bit formulas; element by element the roundings that the operators document)."""
import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from oracle import attention_oracle as A
from test_gpu_attention import DT, assert_within, host, norm_inputs, rand, run_attention

pytestmark = pytest.mark.gpu
INF = float("inf")


@pytest.fixture(scope="module")
def R():
    import raft_stereo_amd
    assert torch.cuda.is_available(), "these tests need a GPU"
    return raft_stereo_amd


# ---------------------------------------------------------------------------------- allowed keys with infinite scores
def with_bias_column(rng, shape, dtype, out):
    """Operands whose last key element is a bias (the queries have a one there), -inf for the keys in `out`."""
    N, Tq, Tk, Hq, Hk, D = shape
    q, k, v = rand(rng, (N, Tq, Hq, D), dtype), rand(rng, (N, Tk, Hk, D), dtype), rand(rng, (N, Tk, Hk, D), dtype)
    g = rand(rng, (N, Tq, Hq, D), dtype)
    q[..., -1] = 1.0
    k[..., -1] = torch.where(torch.from_numpy(out)[:, :, None], -INF, k[..., -1])
    return q, k, v, g


DIVIDED = [(1, 1, 3000, 4, 2, 64), (2, 3, 1500, 4, 1, 128), (1, 2, 1500, 2, 1, 256), (2, 70, 1500, 2, 1, 64),
           (1, 40, 700, 1, 1, 256), (1, 5, 2600, 2, 1, 24)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", DIVIDED, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("where", ["first", "middle", "all but the last"])
def test_minus_infinity_in_a_part_of_divided_keys(R, shape, dtype, where):
    """A score of -inf is a probability of zero, wherever the keys are cut."""
    N, Tk = shape[0], shape[2]
    out = np.zeros((N, Tk), bool)
    out[:, {"first": slice(0, 513), "middle": slice(Tk // 3, Tk - 64), "all but the last": slice(0, Tk - 1)}[where]] = True
    q, k, v, g = with_bias_column(np.random.default_rng(len(where)), shape, dtype, out)
    want = A.attention(host(q), np.nan_to_num(host(k), neginf=0.0), host(v), host(g), ~out, dtype=dtype)
    got = run_attention(R, q, k, v, g, None, None, dtype)
    assert_within(got["out"], want["out"], "out")
    assert_within(run_attention(R, q, k, v, None, None, None, dtype)["out"], want["out"], "out (inference)")
    # (the last element of dq is 0 times -inf)
    assert_within(got["dq"][..., :-1], [x[..., :-1] for x in want["dq"]], "dq")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(3, 1, 3000, 4, 2, 64), (3, 70, 1500, 2, 1, 64), (3, 1, 40, 4, 2, 64)],
                         ids=lambda s: "x".join(map(str, s)))
def test_rows_without_a_finite_score(R, shape, dtype):
    """Keys, but every score -inf: NaN, as 0 / 0 is.  No key: zeros.  A value that is not finite shows, however small its
    probability.  The same where the keys are divided and where they are not."""
    N, Tk = shape[0], shape[2]
    out = np.zeros((N, Tk), bool)
    out[0] = True
    out[2, Tk // 2:] = True
    q, k, v, _ = with_bias_column(np.random.default_rng(1), shape, dtype, out)
    v[2, -1, :, 5] = INF
    got = run_attention(R, q, k, v, None, [Tk, 0, Tk], None, dtype)["out"]
    assert got[0].isnan().all() and not got[1].any()
    assert got[2, ..., 5].isnan().all() and got[2, ..., :5].isfinite().all() and got[2, ..., 6:].isfinite().all()
    k[2, 7] = float("nan")
    assert run_attention(R, q, k, v, None, [Tk, 0, Tk], None, dtype)["out"][2].isnan().all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(260, 20, 33, 1, 1, 32), (130, 37, 100, 4, 2, 64), (64, 100, 380, 4, 4, 24), (2, 70, 150, 2, 1, 64),
                                   (1, 90, 300, 4, 2, 96), (2, 130, 129, 2, 2, 128), (1, 33, 70, 2, 1, 160), (1, 65, 90, 1, 1, 256)],
                         ids=lambda s: "x".join(map(str, s)))
def test_infinite_keys_beside_query_rows_that_end_inside_a_tile(R, shape, dtype):
    """Keys with scores of -inf have gradients of zero; the places behind the last query row add nothing to them."""
    N, Tq, Tk = shape[:3]
    rng = np.random.default_rng(2)
    out = rng.random((N, Tk)) < 0.3
    out[:, 0] = False
    q, k, v, g = with_bias_column(rng, shape, dtype, out)
    want = A.attention(host(q), np.nan_to_num(host(k), neginf=0.0), host(v), host(g), ~out, dtype=dtype)
    got = run_attention(R, q, k, v, g, None, None, dtype)
    for name in ("out", "dk", "dv"):
        assert_within(got[name], want[name], name)
    assert not got["dk"].cpu()[torch.from_numpy(out)].any() and not got["dv"].cpu()[torch.from_numpy(out)].any()


# --------------------------------------------------------------------------------------------- long rows and many parts
@pytest.mark.parametrize("D, Tq", [(64, 1), (64, 40), (32, 40), (128, 40), (128, 1), (256, 40)])
def test_fp16_keeps_the_tail_of_a_long_row(R, D, Tq):
    """One dominant key and thousands whose probabilities lie below fp16's smallest number: together they count.  (Enough
    sequences that the keys are not divided; they share the operands.)"""
    N, Tk = 512, 8192
    q, k, v = torch.zeros(1, Tq, 1, D), torch.zeros(1, Tk, 1, D), torch.ones(1, Tk, 1, D)
    q[..., 0] = 4.0
    k[0, 0, 0, 0], v[0, 0] = 4.5, 0.0         # scores of 18 and 0: 2^-25.97
    v[..., D // 2:] = 0.0
    q, k, v = q.half(), k.half(), v.half()
    g = rand(np.random.default_rng(0), (1, Tq, 1, D), "f16")
    want = A.attention(*(host(x) for x in (q, k, v, g)), None, scale=1.0, dtype="f16")
    t = [x.cuda().expand(N, -1, -1, -1).detach().requires_grad_() for x in (q, k, v)]
    out = R.cross_attention_hip(*t, scale=1.0)
    assert torch.equal(out, out[:1].expand_as(out))
    assert_within(out[:1], want["out"], "out")
    if D == 64:
        grads = torch.autograd.grad(out, t, g.cuda().expand(N, -1, -1, -1))
        for name, d in zip(("dq", "dk", "dv"), grads):
            assert_within(d[:1], want[name], name)


# -------------------------------------------------------------------------------------------------- forward mode
def test_forward_mode_is_refused(R):
    """There is no forward-mode derivative: a dual operand raises, it does not lose its tangent."""
    x, w = torch.randn(1, 6, 2, 32, device="cuda"), torch.ones(32, device="cuda")
    freqs = torch.ones(16, device="cuda")
    plain = R.cross_attention_hip(x, x, x), R.qk_norm_rotate_hip(x, x, w, w, freqs)
    with forward_ad.dual_level():
        for i in range(3):
            args = [x, x, x]
            args[i] = forward_ad.make_dual(x, torch.ones_like(x))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                R.cross_attention_hip(*args)
        for i in range(4):
            args = [x, x, w, w]
            args[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                R.qk_norm_rotate_hip(*args, freqs)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            R.qk_norm_rotate_hip(x, x, w, w, forward_ad.make_dual(freqs, freqs))
        assert torch.equal(R.cross_attention_hip(x, x, x), plain[0])     # no dual operand: nothing to refuse
        assert torch.equal(R.qk_norm_rotate_hip(x, x, w, w, freqs)[0], plain[1][0])


# ------------------------------------------------------------------------------------------------ widths on the way
@pytest.mark.parametrize("impl", ["reg_hip", "alt_hip"])
def test_padded_batches_in_front_of_the_volume(R, impl):
    """What lies behind an image's columns has no influence on the other image's features."""
    torch.manual_seed(3)
    m = R.RowAttentionHip(32, heads=2).cuda()
    f1, f2 = torch.randn(2, 32, 4, 48, device="cuda"), torch.randn(2, 32, 4, 48, device="cuda")
    w1, w2 = torch.tensor([48, 30], device="cuda"), torch.tensor([41, 48], device="cuda")
    coords = torch.rand(2, 2, 4, 48, device="cuda") * 48
    with torch.no_grad():
        got = R.make_corr_fn(impl, f1, f2, attention=m, width1=w1, width2=w2)(coords)
        assert torch.equal(got, R.make_corr_fn(impl, *m(f1, f2, w1, w2))(coords))
        one = R.make_corr_fn(impl, f1, f2, attention=m, width2=w2)(coords)
        assert torch.equal(one, R.make_corr_fn(impl, *m(f1, f2, None, w2))(coords)) and not torch.equal(one, got)
