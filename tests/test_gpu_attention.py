"""GPU parity tests of the attention operators (cross_attention_hip, qk_norm_rotate_hip) and of the module built from
them, against plain 64-bit forms.  Tolerances are the oracle's bounds: element by element, the sum of the roundings
that the operators document (half a step of the operand type each) and of fp32 arithmetic."""
import itertools

import numpy as np
import pytest
import torch

from oracle import attention_oracle as A

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def R():
    import raft_stereo_amd
    assert torch.cuda.is_available(), "these tests need a GPU"
    return raft_stereo_amd


def rand(rng, shape, dtype, scale=1.0):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32) * scale).to(DT[dtype])


def host(t):
    return t.detach().cpu().double().numpy()


def assert_within(got, want, name):
    value, bound = want
    got = host(got)
    assert got.shape == value.shape, (name, got.shape, value.shape)
    assert np.isfinite(got).all(), name
    over = np.abs(got - value) > bound
    if over.any():
        i = np.unravel_index(np.argmax(np.abs(got - value) - bound), got.shape)
        raise AssertionError(f"{name}: {over.mean():.2%} beyond the bound, worst at {i}: {got[i]} vs {value[i]} +- {bound[i]}")


# ------------------------------------------------------------------------------------------------- attention
SHAPES = [  # N, Tq, Tk, Hq, Hk, D
    (1, 1, 1, 1, 1, 8),
    (2, 1, 65, 4, 2, 64),
    (3, 5, 63, 6, 2, 40),
    (2, 33, 64, 2, 1, 32),
    (2, 64, 33, 2, 2, 128),
    (1, 130, 129, 3, 3, 96),
    (2, 17, 257, 8, 1, 256),
    (1, 200, 1, 2, 2, 64),
    (1, 1, 700, 16, 2, 128),
    (5, 80, 80, 4, 4, 64),
    (1, 7, 2100, 4, 1, 64),
    (2, 150, 75, 1, 1, 192),
    (3, 129, 200, 2, 2, 24),
]

# enough sequences of few keys for the backward pass to take a workgroup for each (the rows of an image): every number
# of waves, keys that end inside a wave's block, query tiles that end inside, heads that share
SHAPES += [
    (260, 20, 33, 1, 1, 32),
    (130, 37, 100, 4, 2, 64),
    (90, 70, 129, 6, 3, 40),
    (128, 33, 190, 2, 2, 32),
    (70, 5, 250, 4, 4, 64),
    (64, 100, 380, 4, 4, 24),
    (256, 1, 1, 2, 1, 8),
]

# lengths that are divided: keys over workgroups with rows that fill a tile and more, query rows in the backward pass,
# an even and an odd count of key tiles for the heads whose loads run ahead, more sequences than the card has dies
SHAPES += [
    (2, 70, 1500, 2, 1, 64),
    (1, 600, 300, 2, 1, 128),
    (1, 520, 70, 2, 1, 256),
    (1, 300, 1100, 1, 1, 96),
    (2, 40, 577, 3, 3, 128),
    (20, 40, 70, 2, 2, 64),
    (1, 90, 600, 1, 1, 160),
    (4, 1, 1124, 4, 2, 256),
    (2, 3, 515, 2, 1, 32),
]


def masks(kind, N, Tk, rng):
    """(lengths, mask): lengths of nothing, one, more than there are and less than nothing; a mask that leaves a
    sequence empty."""
    lengths = mask = None
    if kind in ("lengths", "both"):
        lengths = [int(rng.integers(1, Tk + 1)) for _ in range(N)]
        for i, l in zip(range(N), (Tk // 2 + 1, 0, 1) if N > 1 else (max(1, Tk - 1),)):
            lengths[i] = l
        if N > 3:
            lengths[3], lengths[4 % N] = Tk + 1000, -5
    if kind in ("holes", "both"):
        mask = rng.random((N, Tk)) < 0.7
        mask[0, 0] = True
        if N > 1:
            mask[N - 1] = False
    return lengths, mask


def run_attention(R, q, k, v, g, lengths, mask, dtype, lengths_dtype=torch.int32, **kw):
    t = [x.cuda().requires_grad_(g is not None) for x in (q, k, v)]
    lt = None if lengths is None else torch.tensor(lengths, dtype=lengths_dtype, device="cuda")
    mt = None if mask is None else torch.from_numpy(mask).cuda()
    out = R.cross_attention_hip(*t, key_mask=mt, key_lengths=lt, **kw)
    assert out.dtype == DT[dtype] and out.is_contiguous() and out.shape == q.shape
    if g is None:
        return {"out": out}
    return dict(zip(("out", "dq", "dk", "dv"), (out,) + torch.autograd.grad(out, t, g.cuda())))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", ["none", "lengths", "holes", "both"])
def test_attention_matches_the_formula(R, shape, dtype, kind):
    N, Tq, Tk, Hq, Hk, D = shape
    rng = np.random.default_rng(sum(shape) * 7 + len(kind))
    q, k, v = rand(rng, (N, Tq, Hq, D), dtype, 1.5), rand(rng, (N, Tk, Hk, D), dtype), rand(rng, (N, Tk, Hk, D), dtype)
    g = rand(rng, (N, Tq, Hq, D), dtype)
    lengths, mask = masks(kind, N, Tk, rng)
    ok = A.allowed_keys(N, Tk, lengths, mask)
    want = A.attention(*(host(x) for x in (q, k, v, g)), ok, dtype=dtype)
    got = run_attention(R, q, k, v, g, lengths, mask, dtype, torch.int64 if Tq % 2 else torch.int32)
    for name in ("out", "dq", "dk", "dv"):
        assert_within(got[name], want[name], name)
    with torch.no_grad():      # inference takes its own route through the library
        plain = run_attention(R, q, k, v, None, lengths, mask, dtype)["out"]
    assert_within(plain, want["out"], "out (inference)")
    empty = ~ok.any(axis=1)
    for n in np.flatnonzero(empty):
        assert not got["out"][n].any() and not got["dq"][n].any() and not plain[n].any()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(2, 40, 100, 4, 2, 64), (3, 1, 300, 8, 2, 128), (2, 70, 70, 1, 1, 256)],
                         ids=lambda s: "x".join(map(str, s)))
def test_masked_places_may_hold_anything(R, shape, dtype):
    N, Tq, Tk, Hq, Hk, D = shape
    rng = np.random.default_rng(5)
    q, k, v = rand(rng, (N, Tq, Hq, D), dtype), rand(rng, (N, Tk, Hk, D), dtype), rand(rng, (N, Tk, Hk, D), dtype)
    g = rand(rng, (N, Tq, Hq, D), dtype)
    lengths, mask = [Tk - 7] + [Tk // 2] * (N - 1), rng.random((N, Tk)) < 0.6
    ok = torch.from_numpy(A.allowed_keys(N, Tk, lengths, mask))
    clean = run_attention(R, q, k, v, g, lengths, mask, dtype)
    worst = torch.finfo(DT[dtype])
    for bad in (float("nan"), float("inf"), float("-inf"), worst.max, worst.min):
        kb, vb = k.clone(), v.clone()
        kb[~ok], vb[~ok] = bad, bad
        dirty = run_attention(R, q, kb, vb, g, lengths, mask, dtype)
        for name in clean:
            assert torch.equal(clean[name], dirty[name]), (name, bad)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D, Tq, Hq", [(64, 200, 1), (128, 150, 2), (256, 140, 1), (64, 1, 4)])
def test_the_widest_strides(R, dtype, D, Tq, Hq):
    """Tokens 16 bytes short of 8 MiB apart: every tile's rows stay in reach, and the rows behind the last give nothing."""
    Tk, wide = 141, ((8 << 20) - 16) // DT[dtype].itemsize
    rng = np.random.default_rng(D + Tq)
    q, k, v, g = (rand(rng, (1, T, H, D), dtype) for T, H in ((Tq, Hq), (Tk, 1), (Tk, 1), (Tq, Hq)))
    ok = A.allowed_keys(1, Tk, None, None)
    want = A.attention(*(host(x) for x in (q, k, v, g)), ok, dtype=dtype)

    def spread(x):
        T, H = x.shape[1:3]
        base = torch.empty(T * wide + H * D, dtype=x.dtype, device="cuda")
        y = base.as_strided((1, T, H, D), (T * wide, wide, D, 1))
        y.copy_(x)
        return y.detach().requires_grad_()

    t = [spread(x) for x in (q, k, v)]
    assert all(x.stride(1) * x.element_size() == (8 << 20) - 16 for x in t)
    out = R.cross_attention_hip(*t)
    got = dict(zip(("out", "dq", "dk", "dv"), (out,) + torch.autograd.grad(out, t, g.cuda())))
    for name in want.keys() & got.keys():
        assert_within(got[name], want[name], name)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(2, 40, 100, 4, 2, 64), (3, 1, 300, 8, 2, 128), (2, 70, 1500, 1, 1, 256), (90, 70, 129, 6, 3, 40)],
                         ids=lambda s: "x".join(map(str, s)))
def test_keys_that_take_no_part_get_nothing_from_bad_queries(R, shape, dtype):
    """NaN and infinities in queries and incoming gradients stay away from the gradients of masked keys, and a sequence
    without a key gives zeros whatever its queries hold."""
    N, Tq, Tk, Hq, Hk, D = shape
    rng = np.random.default_rng(6)
    q, k, v = rand(rng, (N, Tq, Hq, D), dtype), rand(rng, (N, Tk, Hk, D), dtype), rand(rng, (N, Tk, Hk, D), dtype)
    g = rand(rng, (N, Tq, Hq, D), dtype)
    mask = rng.random((N, Tk)) < 0.6
    mask[N - 1] = False
    off = torch.from_numpy(~mask)
    for bad in (float("nan"), float("inf"), float("-inf")):
        for where in ("q", "g"):
            x = {"q": q.clone(), "g": g.clone()}
            x[where][:, Tq // 2] = bad
            got = run_attention(R, x["q"], k, v, x["g"], None, mask, dtype)
            for name in ("dk", "dv"):
                assert not got[name].cpu()[off].any(), (name, bad, where)
            for name in ("out", "dq"):
                assert not got[name][N - 1].any(), (name, bad, where)
            assert not run_attention(R, x["q"], k, v, None, None, mask, dtype)["out"][N - 1].any()


@pytest.mark.parametrize("D, Tq", [(8, 1), (8, 5), (72, 1)])
def test_more_sequences_than_a_launch_holds_threads(R, D, Tq):
    """2^24 sequences and some: a workgroup for each is 2^32 threads.  The whole agrees with its parts, forward and back."""
    N, Tk = (1 << 24) + 37, 2
    gen = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(1, Tq, 1, D, generator=gen, device="cuda", dtype=torch.bfloat16).expand(N, -1, -1, -1)
    kv = torch.randn(N, Tk, 1, 8, generator=gen, device="cuda", dtype=torch.bfloat16).repeat(1, 1, 1, D // 8)
    mask = torch.rand(N, Tk, generator=gen, device="cuda") < 0.7
    parts = [slice(0, 300), slice((1 << 22) - 9, (1 << 22) + 300), slice((1 << 24) - 270, N)]   # (as many as take the same way)

    def run(n):
        t = [x[n].detach().requires_grad_() for x in (q, kv, kv)]
        out = R.cross_attention_hip(*t, key_mask=mask[n])
        return (out,) + torch.autograd.grad(out, t, out.detach())

    whole = run(slice(None))
    for n in parts:
        for a, b in zip(whole, run(n)):
            assert torch.isfinite(b).all() and b.any() and torch.equal(a[n], b), n


def test_what_is_not_finite_in_allowed_places_shows(R):
    q, k, v = (torch.randn(1, 4, 1, 32, device="cuda") for _ in range(3))
    k[0, 2] = float("nan")
    assert R.cross_attention_hip(q, k, v).isnan().all()
    k[0, 2] = 0
    v[0, 1, 0, 5] = float("inf")
    out = R.cross_attention_hip(q, k, v)
    assert out[..., 5].isinf().all() and out[..., 6].isfinite().all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_scale_and_large_scores(R, dtype):
    """Scores far from zero: the running maximum keeps exp2 in range."""
    rng = np.random.default_rng(2)
    N, Tq, Tk, H, D = 2, 35, 190, 2, 64
    q, k, v, g = (rand(rng, (N, t, H, D), dtype, s) for t, s in ((Tq, 8.0), (Tk, 8.0), (Tk, 1.0), (Tq, 1.0)))
    for scale in (0.01, 1.0):
        want = A.attention(*(host(x) for x in (q, k, v, g)), None, scale=scale, dtype=dtype)
        got = run_attention(R, q, k, v, g, None, None, dtype, scale=scale)
        for name in got:
            assert_within(got[name], want[name], (name, scale))


@pytest.mark.parametrize("size", [1e-6, 1.0, 3e3])
def test_fp16_gradients_of_any_size(R, size):
    """The scores' gradients of a long row are far below fp16's smallest normal number, or (a scaled loss) large."""
    rng = np.random.default_rng(3)
    N, Tq, Tk, Hq, Hk, D = 1, 70, 600, 2, 1, 64
    q, k, v = (rand(rng, (N, t, h, D), "f16") for t, h in ((Tq, Hq), (Tk, Hk), (Tk, Hk)))
    g = torch.from_numpy(rng.standard_normal((N, Tq, Hq, D)) * size).float()
    # (fp16 itself loses what is below its smallest number: the incoming gradient and the results are compared in fp16)
    g = g.half()
    want = A.attention(*(host(x) for x in (q, k, v, g)), None, dtype="f16")
    got = run_attention(R, q, k, v, g, None, None, "f16")
    for name in got:
        assert_within(got[name], want[name], name)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_gradient_against_differences(R, dtype):
    rng = np.random.default_rng(4)
    N, Tq, Tk, Hq, Hk, D = 2, 37, 53, 4, 2, 32
    q, k, v = rand(rng, (N, Tq, Hq, D), dtype), rand(rng, (N, Tk, Hk, D), dtype), rand(rng, (N, Tk, Hk, D), dtype)
    g = rand(rng, (N, Tq, Hq, D), dtype)
    ok = A.allowed_keys(N, Tk, [Tk, 20], None)
    got = run_attention(R, q, k, v, g, [Tk, 20], None, dtype)
    want = A.attention(*(host(x) for x in (q, k, v, g)), ok, dtype=dtype)
    args = [host(x) for x in (q, k, v)]
    h = 1e-5
    for i, name in enumerate(("dq", "dk", "dv")):
        d = rng.standard_normal(args[i].shape)
        at = lambda s: [a + s * d if j == i else a for j, a in enumerate(args)]
        f = lambda s: (A.attention(*at(s), None, ok)["out"][0] * host(g)).sum()
        slope = (f(h) - f(-h)) / (2 * h)
        tol = (want[name][1] * np.abs(d)).sum() + 1e-7 * abs(slope) + 1e-6
        assert abs((host(got[name]) * d).sum() - slope) <= tol, name


def test_attention_takes_slices_and_any_strides(R):
    """Slices of a wider projection are read in place; other layouts give the same bits through a copy."""
    N, T, Tk, H, D = 2, 50, 70, 3, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    wide = torch.randn((N, T, 4 * H, D), generator=g, device="cuda").half()
    kv = torch.randn((N, Tk, 2, H, D), generator=g, device="cuda").half()
    q, k, v = wide[:, :, H:2 * H], kv[:, :, 0], kv[:, :, 1]
    ref = R.cross_attention_hip(q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(R.cross_attention_hip(q, k, v), ref)
    heads_first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    assert torch.equal(R.cross_attention_hip(*heads_first), ref)
    planes = [x.permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2) for x in (q, k, v)]    # D is not the fastest
    assert torch.equal(R.cross_attention_hip(*planes), ref)
    odd = [torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(x.shape).copy_(x) for x in (q, k, v)]
    assert torch.equal(R.cross_attention_hip(*odd), ref)
    one = R.cross_attention_hip(q, k[:1].expand(N, -1, -1, -1), v[:1].expand(N, -1, -1, -1))
    assert torch.equal(one[0], ref[0])
    # the gradient of a shared (expanded) operand is summed over the sequences by torch
    leaves = [x.detach().float().contiguous().requires_grad_(True) for x in (q, k[:1], v[:1])]
    out = R.cross_attention_hip(leaves[0], leaves[1].expand(N, -1, -1, -1), leaves[2].expand(N, -1, -1, -1))
    go = torch.randn(out.shape, generator=g, device="cuda")
    got = torch.autograd.grad(out, leaves, go.transpose(1, 2).contiguous().transpose(1, 2))
    full = [leaves[0].detach().requires_grad_(True)] + [x.detach().expand(N, -1, -1, -1).contiguous().requires_grad_(True) for x in leaves[1:]]
    want = torch.autograd.grad(R.cross_attention_hip(*full), full, go)
    assert torch.equal(got[0], want[0])
    for a, b in zip(got[1:], want[1:]):
        assert torch.equal(a, b.sum(0, keepdim=True))


def test_attention_offsets_beyond_32_bits(R):
    """A long cache whose tokens lie 64 KiB apart: 4.6 GB from the first to the last."""
    T, D = 70000, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    cache = torch.empty((1, T, 512, D), dtype=torch.bfloat16, device="cuda")
    k, v = cache[:, :, 3:4], cache[:, :, 500:501]
    kd, vd = (torch.randn((1, T, 1, D), generator=g, device="cuda").bfloat16() for _ in range(2))
    k.copy_(kd)
    v.copy_(vd)
    for Tq in (1, 40):
        q = torch.randn((1, Tq, 2, D), generator=g, device="cuda").bfloat16()
        assert torch.equal(R.cross_attention_hip(q, k, v), R.cross_attention_hip(q, kd, vd))
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    dense = [x.detach().requires_grad_(True) for x in (q, kd, vd)]
    go = torch.randn(q.shape, generator=g, device="cuda").bfloat16()
    a = torch.autograd.grad(R.cross_attention_hip(*leaves), leaves, go)
    b = torch.autograd.grad(R.cross_attention_hip(*dense), dense, go)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("shape", [(0, 4, 5), (2, 0, 5), (2, 4, 0)])
def test_attention_of_nothing(R, shape):
    N, Tq, Tk = shape
    q, k, v = (torch.randn((N, t, 2, 32), device="cuda", requires_grad=True) for t in (Tq, Tk, Tk))
    out = R.cross_attention_hip(q, k, v)
    assert out.shape == (N, Tq, 2, 32) and not out.any()
    for d, x in zip(torch.autograd.grad(out, (q, k, v), torch.ones_like(out)), (q, k, v)):
        assert d.shape == x.shape and not d.any()


def test_attention_repeats_bit_for_bit_and_skips_unwanted_gradients(R):
    rng = np.random.default_rng(8)
    q, k, v = (rand(rng, s, "bf16").cuda() for s in ((2, 300, 4, 64), (2, 333, 2, 64), (2, 333, 2, 64)))
    g = rand(rng, (2, 300, 4, 64), "bf16").cuda()

    def grads(which):
        t = [x.clone().requires_grad_(w) for x, w in zip((q, k, v), which)]
        out = R.cross_attention_hip(*t)
        return torch.autograd.grad(out, [x for x, w in zip(t, which) if w], g)
    a, b = grads((True, True, True)), grads((True, True, True))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert torch.equal(grads((True, False, False))[0], a[0])
    assert torch.equal(grads((False, False, True))[0], a[2])
    assert torch.equal(grads((False, True, False))[0], a[1])
    t = q.clone().requires_grad_(True)
    out = R.cross_attention_hip(t, k, v)
    d, = torch.autograd.grad(out, t, g, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), t)


def test_gradients_where_saved_tensors_were_moved(R):
    """Saved tensors that a hook has put elsewhere, with other strides, give the same gradients."""
    g = torch.Generator(device="cuda").manual_seed(2)
    wide = torch.randn((2, 40, 12, 64), generator=g, device="cuda").half()
    pos = torch.randint(0, 1000, (2, 80), generator=g, device="cuda")[:, ::2]
    mask = torch.rand((40, 2), generator=g, device="cuda").t() > 0.3
    freqs, w = torch.linspace(0.01, 1.0, 32, device="cuda"), torch.ones(128, device="cuda")[::2]
    go = torch.randn((2, 40, 4, 64), generator=g, device="cuda").half()

    def grads(hooks):
        leaf, wl = wide.clone().requires_grad_(True), w.clone().requires_grad_(True)
        with hooks:
            q, k = R.qk_norm_rotate_hip(leaf[:, :, :4], leaf[:, :, 4:8], wl, wl, freqs, pos, pos)
            out = R.cross_attention_hip(q, k, leaf[:, :, 8:], key_mask=mask)
        junk = torch.full((64 << 20,), 7, dtype=torch.uint8, device="cuda")   # takes what the hooks have freed
        res = torch.autograd.grad(out, (leaf, wl), go)
        del junk
        return res
    import contextlib
    for a, b in zip(grads(contextlib.nullcontext()), grads(torch.autograd.graph.save_on_cpu())):
        assert torch.equal(a, b)


def test_attention_refuses(R):
    x = torch.randn(2, 8, 4, 32, device="cuda")
    f = R.cross_attention_hip
    for exc, args, kw in [
        (RuntimeError, (x.cpu(), x, x), {}), (RuntimeError, (x, x.cpu(), x.cpu()), {}),
        (TypeError, (x.double(),) * 3, {}), (TypeError, (x, x.half(), x.half()), {}),
        (ValueError, (x[0], x, x), {}), (ValueError, (x, x, x[:, :4]), {}), (ValueError, (x, x[:1], x[:1]), {}),
        (ValueError, (x[..., :12],) * 3, {}), (ValueError, (x, x[..., :16], x[..., :16]), {}),
        (ValueError, (x, x[:, :, :3], x[:, :, :3]), {}), (ValueError, (x, x[:, :, :0], x[:, :, :0]), {}),
        (ValueError, (torch.randn(1, 2, 1, 264, device="cuda"),) * 3, {}),
        (TypeError, (x, x, x), dict(key_mask=torch.zeros(2, 8, device="cuda"))),
        (ValueError, (x, x, x), dict(key_mask=torch.ones(2, 7, device="cuda", dtype=torch.bool))),
        (RuntimeError, (x, x, x), dict(key_mask=torch.ones(2, 8, dtype=torch.bool))),
        (TypeError, (x, x, x), dict(key_lengths=torch.ones(2, device="cuda"))),
        (ValueError, (x, x, x), dict(key_lengths=torch.ones(3, device="cuda", dtype=torch.int32))),
        (RuntimeError, (x, x, x), dict(key_lengths=torch.ones(2, dtype=torch.int32))),
        (ValueError, (x, x, x), dict(scale=0.0)), (ValueError, (x, x, x), dict(scale=float("nan"))),
        (ValueError, (x, x, x), dict(scale=-1.0)), (ValueError, (x, x, x), dict(scale=float("inf"))),
    ]:
        with pytest.raises(exc):
            f(*args, **kw)


# --------------------------------------------------------------------------------------------- norm and rotation
NORM_SHAPES = [  # N, Tq, Tk, Hq, Hk, D, rotated
    (1, 1, 1, 1, 1, 8, 8),
    (3, 1, 0, 5, 0, 128, 128),
    (2, 7, 9, 4, 1, 64, 64),
    (2, 33, 5, 3, 3, 40, 16),
    (1, 130, 77, 2, 2, 32, 32),
    (2, 19, 21, 9, 3, 256, 128),
    (4, 60, 3, 1, 1, 96, 0),
    (2, 5, 5, 6, 2, 16, 8),
    (1, 2500, 10, 1, 1, 80, 80),
]


def norm_inputs(shape, dtype, rng, pos):
    N, Tq, Tk, Hq, Hk, D, rot = shape
    freqs = 10000.0 ** (-2.0 * np.arange(rot // 2) / max(rot, 1)) if rot else None
    sides = []
    for T, H in ((Tq, Hq), (Tk, Hk)):
        if H == 0:
            sides.append(None)
            continue
        x, g = rand(rng, (N, T, H, D), dtype, 2.0), rand(rng, (N, T, H, D), dtype)
        w = torch.from_numpy(1.0 + 0.3 * rng.standard_normal(D)).float()
        p = None
        if rot and pos == "far":
            p = torch.from_numpy(rng.integers(0, 2 ** 31 - T, (N, 1)) + np.arange(T))
        elif rot and pos == "shared":
            p = torch.from_numpy(rng.integers(-50, 4000, T).astype(np.int32))
        elif rot and pos == "float":
            p = torch.from_numpy((rng.random((N, T)) * 700).astype(np.float32))
        sides.append((x, g, w, p))
    return freqs, sides


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", NORM_SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("pos,interleaved", [("index", False), ("far", False), ("shared", True), ("float", True)])
def test_norm_rotate_matches_the_formula(R, shape, dtype, pos, interleaved):
    rng = np.random.default_rng(sum(shape) * 3 + len(pos))
    freqs, sides = norm_inputs(shape, dtype, rng, pos)
    N, D, eps = shape[0], shape[5], 1e-5
    dev = lambda t: None if t is None else t.cuda()
    xs = [None if s is None else s[0].cuda().requires_grad_(True) for s in sides]
    ws = [None if s is None else s[2].cuda().requires_grad_(True) for s in sides]
    ps = [None if s is None else dev(s[3]) for s in sides]
    ft = None if freqs is None else torch.from_numpy(freqs).cuda()
    out = R.qk_norm_rotate_hip(xs[0], xs[1], ws[0], ws[1], ft, ps[0], ps[1], eps=eps, interleaved=interleaved)
    outs = (out,) if sides[1] is None else out
    used = [i for i in (0, 1) if sides[i] is not None]
    leaves = [t for i in used for t in (xs[i], ws[i])]
    grads = torch.autograd.grad(outs, leaves, [sides[i][1].cuda() for i in used])
    with torch.no_grad():
        again = R.qk_norm_rotate_hip(xs[0], xs[1], ws[0], ws[1], ft, ps[0], ps[1], eps=eps, interleaved=interleaved)
        again = (again,) if sides[1] is None else again
    for j, i in enumerate(used):
        x, g, w, p = sides[i]
        want = A.norm_rotate(host(x), host(w), freqs, None if p is None else p.numpy(), eps, interleaved, host(g), dtype,
                             sums=x.shape[0] * x.shape[1] * x.shape[2])
        assert outs[j].is_contiguous() and torch.equal(outs[j], again[j])
        assert_within(outs[j], want["y"], ("y", i))
        assert_within(grads[2 * j], want["dx"], ("dx", i))
        assert_within(grads[2 * j + 1], want["dw"], ("dw", i))


def test_norm_rotate_gradient_against_differences(R):
    rng = np.random.default_rng(6)
    N, T, H, D, n, h = 2, 9, 3, 32, 12, 1e-5
    x, g, w = rand(rng, (N, T, H, D), "f32"), rand(rng, (N, T, H, D), "f32"), torch.randn(D)
    freqs = np.linspace(0.1, 1.0, n)
    xt, wt = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    dx, dw = torch.autograd.grad(R.qk_norm_rotate_hip(xt, None, wt, freqs=torch.from_numpy(freqs).cuda()), (xt, wt), g.cuda())
    f = lambda a, b: (A.norm_rotate(a, b, freqs)["y"][0] * host(g)).sum()
    want = A.norm_rotate(host(x), host(w), freqs, g=host(g), sums=N * T * H)
    for got, name, at in ((dx, "dx", lambda s, d: f(host(x) + s * d, host(w))), (dw, "dw", lambda s, d: f(host(x), host(w) + s * d))):
        d = rng.standard_normal(got.shape)
        slope = (at(h, d) - at(-h, d)) / (2 * h)
        tol = (want[name][1] * np.abs(d)).sum() + 1e-7 * abs(slope) + 1e-6
        assert abs((host(got) * d).sum() - slope) <= tol, name


@pytest.mark.parametrize("wdtype", ["f16", "bf16", None])
def test_norm_rotate_weights_of_other_types_and_slices(R, wdtype):
    rng = np.random.default_rng(7)
    N, T, H, D = 3, 11, 4, 64
    wide = rand(rng, (N, T, 3 * H, D), "bf16").cuda()
    w = None if wdtype is None else rand(rng, (D,), wdtype).cuda().requires_grad_(True)
    freqs = torch.linspace(0.01, 1.0, D // 2, device="cuda")       # float32 frequencies
    q, k = wide[:, :, :H], wide[:, :, H:2 * H]
    a = R.qk_norm_rotate_hip(q.clone().requires_grad_(True), k.clone(), w, w, freqs)
    b = R.qk_norm_rotate_hip(q, k, w, w, freqs)
    planes = q.permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2)
    c = R.qk_norm_rotate_hip(planes, k, w, w, freqs)
    assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(a, b, c))
    want = A.norm_rotate(host(q), None if w is None else host(w), freqs.cpu().double().numpy(), dtype="bf16")
    assert_within(a[0], want["y"], "y")
    if w is not None:
        assert torch.autograd.grad(sum(t.float().sum() for t in a), w)[0].dtype == w.dtype
    # one of the two results alone is used
    qt = q.detach().clone().requires_grad_(True)
    y, _ = R.qk_norm_rotate_hip(qt, k, None, None, freqs)
    y.float().sum().backward()
    y2 = R.qk_norm_rotate_hip(qt, None, None, None, freqs)
    assert torch.equal(y2, y)
    d2, = torch.autograd.grad(y2.float().sum(), qt)
    assert torch.equal(d2, qt.grad)


def test_norm_rotate_of_more_tokens_than_a_launch_holds_threads(R):
    T, D = (1 << 27) + 11, 256       # 32 lanes each
    x = torch.randn(1, 1, 1, D, device="cuda", dtype=torch.bfloat16)
    freqs = 1e4 ** (-torch.arange(4, device="cuda", dtype=torch.float64) / 4)
    y = R.qk_norm_rotate_hip(x.expand(1, T, 1, D), freqs=freqs)
    for t in (0, 1, (1 << 25) - 1, 1 << 25, (1 << 27) - 1, 1 << 27, T - 1):
        pos = torch.tensor([t], device="cuda")
        assert torch.equal(y[:, t:t + 1], R.qk_norm_rotate_hip(x, freqs=freqs, q_pos=pos)), t
    y = y.view(-1, D)
    for t in range(0, T, 1 << 25):      # no token was left out: the rest of the head is the same in all of them
        assert (y[t:t + (1 << 25), 8:] == y[0, 8:]).all()


@pytest.mark.parametrize("shape", [(0, 3, 2), (2, 0, 2), (2, 3, 0)])
def test_norm_rotate_of_nothing(R, shape):
    N, T, H = shape
    x = torch.randn((N, T, H, 64), device="cuda", requires_grad=True)
    k = torch.randn((N, 4, 2, 64), device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    y, yk = R.qk_norm_rotate_hip(x, k, w, w, torch.ones(32, device="cuda"))
    assert y.shape == x.shape
    d = torch.autograd.grad(y.sum(), (x, w))
    assert d[0].shape == x.shape and not d[1].any()


def test_norm_rotate_refuses(R):
    x, w, f = torch.randn(2, 8, 4, 32, device="cuda"), torch.ones(32, device="cuda"), torch.ones(16, device="cuda")
    for exc, args, kw in [
        (RuntimeError, (x.cpu(),), {}), (RuntimeError, (x, x.cpu()), {}), (TypeError, (x.double(),), {}),
        (TypeError, (x, x.half()), {}), (ValueError, (x[0],), {}), (ValueError, (x[..., :12],), {}),
        (ValueError, (x, x[:1]), {}), (ValueError, (x, x[..., :16]), {}),
        (ValueError, (x, None, w[:16]), {}), (TypeError, (x, None, w.double()), {}), (RuntimeError, (x, None, w.cpu()), {}),
        (ValueError, (x,), dict(k_weight=w)), (ValueError, (x,), dict(k_pos=torch.zeros(8, device="cuda", dtype=torch.int32), freqs=f)),
        (ValueError, (x,), dict(freqs=torch.ones(6, device="cuda"))), (ValueError, (x,), dict(freqs=torch.ones(20, device="cuda"))),
        (TypeError, (x,), dict(freqs=f.half())), (RuntimeError, (x,), dict(freqs=f.cpu())),
        (ValueError, (x,), dict(q_pos=torch.zeros(8, device="cuda", dtype=torch.int32))),
        (TypeError, (x,), dict(freqs=f, q_pos=torch.zeros(8, device="cuda", dtype=torch.float64))),
        (ValueError, (x,), dict(freqs=f, q_pos=torch.zeros(7, device="cuda", dtype=torch.int32))),
        (RuntimeError, (x,), dict(freqs=f, q_pos=torch.zeros(8, dtype=torch.int32))),
        (ValueError, (x,), dict(eps=-1.0)), (ValueError, (x,), dict(eps=float("nan"))),
    ]:
        with pytest.raises(exc):
            R.qk_norm_rotate_hip(*args, **kw)


# ------------------------------------------------------------------------------------------- streams and graphs
def test_on_another_stream(R):
    x = torch.randn(4, 200, 2, 64, device="cuda").half()
    ref = R.cross_attention_hip(*R.qk_norm_rotate_hip(x, x), x)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = R.cross_attention_hip(*R.qk_norm_rotate_hip(x, x), x)
    torch.cuda.current_stream().wait_stream(st)
    got.record_stream(torch.cuda.current_stream())
    assert torch.equal(got, ref)


@pytest.mark.parametrize("Tq,Tk,D", [(1, 3000, 128), (70, 900, 64), (5, 1100, 256)])
def test_graphs_with_masks_and_divided_keys(R, Tq, Tk, D):
    """The mask's bits and the splits' parts are scratch of each graph; the mask is read again at every replay."""
    g = torch.Generator(device="cuda").manual_seed(4)
    mk = lambda *s: torch.randn(s, generator=g, device="cuda").half()
    sets = [[mk(2, Tq, 4, D), mk(2, Tk, 2, D), mk(2, Tk, 2, D), torch.rand(2, Tk, generator=g, device="cuda") < 0.5] for _ in range(2)]
    call = lambda x: R.cross_attention_hip(*x[:3], key_mask=x[3])
    call(sets[0])
    torch.cuda.synchronize()
    graphs = []
    for x in sets:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = call(x)
        graphs.append((gr, out))
    for r in range(5):
        for x, (gr, out) in zip(sets, graphs):
            x[0].copy_(mk(*x[0].shape))
            x[3].copy_(torch.rand(x[3].shape, generator=g, device="cuda") < 0.2 * r)     # none at all the first time
            want = call(x)
            gr.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            assert r or not out.any()


def test_two_threads_at_once(R):
    """Each thread on a stream of its own, forward and back, against the same calls one after the other."""
    from concurrent.futures import ThreadPoolExecutor
    shapes = [(3, 1, 3000, 4, 2, 128), (300, 40, 60, 2, 2, 32), (2, 300, 700, 4, 2, 96), (2, 90, 130, 2, 1, 256)]
    sets = []
    for n, (N, Tq, Tk, Hq, Hk, D) in enumerate(shapes):
        g = torch.Generator(device="cuda").manual_seed(n)
        mk = lambda *s: torch.randn(s, generator=g, device="cuda").bfloat16()
        sets.append((mk(N, Tq, Hq, D), mk(N, Tk, Hk, D), mk(N, Tk, Hk, D), torch.rand(N, Tk, generator=g, device="cuda") < 0.7))

    def run(x):
        t = [y.detach().requires_grad_() for y in x[:3]]
        q, k = R.qk_norm_rotate_hip(t[0], t[1])
        out = R.cross_attention_hip(q, k, t[2], key_mask=x[3])
        return (out.detach(),) + torch.autograd.grad(out, t, out.detach())

    want = [run(x) for x in sets]
    torch.cuda.synchronize()

    def worker(order):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            got = [(i, run(sets[i])) for _ in range(4) for i in order]
        st.synchronize()
        return got

    with ThreadPoolExecutor(2) as pool:
        for got in pool.map(worker, ([0, 1, 2, 3], [3, 2, 1, 0])):
            for i, tensors in got:
                assert all(torch.equal(a, b) for a, b in zip(tensors, want[i])), shapes[i]


@pytest.mark.parametrize("Tq,Tk", [(1, 900), (70, 90)])
def test_inference_graphs(R, Tq, Tk):
    """Two graphs captured side by side, replayed in turn with eager calls between them."""
    g = torch.Generator(device="cuda").manual_seed(3)
    mk = lambda *s: torch.randn(s, generator=g, device="cuda").bfloat16()
    freqs = torch.linspace(0.01, 1.0, 32, device="cuda")
    lengths = torch.tensor([Tk, Tk // 2, 0], dtype=torch.int32, device="cuda")
    inputs = [[mk(3, Tq, 8, 64), mk(3, Tk, 2, 64), mk(3, Tk, 2, 64)] for _ in range(2)]

    def step(q, k, v):
        qn, kn = R.qk_norm_rotate_hip(q, k, None, None, freqs)
        return R.cross_attention_hip(qn, kn, v, key_lengths=lengths)
    step(*inputs[0])
    torch.cuda.synchronize()
    graphs = []
    for x in inputs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step(*x)
        graphs.append((gr, out))
    for _ in range(4):
        for x, (gr, out) in zip(inputs, graphs):
            for t in x:
                t.copy_(mk(*t.shape))
            want = step(*x)
            gr.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)


def test_training_graph(R):
    g = torch.Generator(device="cuda").manual_seed(4)
    mk = lambda *s: torch.randn(s, generator=g, device="cuda").half()
    x = [mk(2, 60, 4, 32), mk(2, 75, 2, 32), mk(2, 75, 2, 32)]
    go, w = mk(2, 60, 4, 32), torch.ones(32, device="cuda")
    freqs = torch.linspace(0.01, 1.0, 16, device="cuda")

    def step(q, k, v, w):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, w)]
        qn, kn = R.qk_norm_rotate_hip(leaves[0], leaves[1], leaves[3], leaves[3], freqs)
        out = R.cross_attention_hip(qn, kn, leaves[2])
        return (out.detach(),) + torch.autograd.grad(out, leaves, go)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step(*x, w)
    torch.cuda.current_stream().wait_stream(st)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        outs = step(*x, w)
    for _ in range(4):
        for t in x:
            t.copy_(mk(*t.shape))
        want = step(*x, w)
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


# ---------------------------------------------------------------------------------------- rows of feature maps
def plain_rows(m, f1, f2, w1=None, w2=None):
    """RowAttentionHip.forward in torch's elementary operations, in the maps' type (double on the CPU)."""
    def heads(x, layer, n):
        return (x @ layer.weight.t()).view(*x.shape[:2], n, m.head_dim)

    def norm_rotate(x, w):
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + m.eps) * w
        n = m.freqs.shape[0]
        angle = torch.arange(x.shape[1], dtype=x.dtype)[:, None, None] * m.freqs
        a, b = y[..., :n], y[..., n:2 * n]
        return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin(), y[..., 2 * n:]], -1)

    def attend(q, k, v, lengths):
        G = m.heads // m.kv_heads
        k, v = k.repeat_interleave(G, 2), v.repeat_interleave(G, 2)
        s = torch.einsum("nthd,nshd->nhts", q, k) / m.head_dim ** 0.5
        if lengths is not None:
            s = s.masked_fill(torch.arange(k.shape[1]) >= lengths.repeat_interleave(f1.shape[2])[:, None, None, None], -1e30)
        return torch.einsum("nhts,nshd->nthd", torch.softmax(s, -1), v)
    rows = [f.permute(0, 2, 3, 1).flatten(0, 1) for f in (f1, f2)]
    hs = [(norm_rotate(heads(x, m.q, m.heads), m.q_weight), norm_rotate(heads(x, m.k, m.kv_heads), m.k_weight),
           heads(x, m.v, m.kv_heads)) for x in rows]
    out = []
    for i, (f, lengths) in enumerate(((f1, w2), (f2, w1))):
        a = attend(hs[i][0], hs[1 - i][1], hs[1 - i][2], lengths).flatten(2) @ m.out.weight.t() + m.out.bias
        out.append((rows[i] + a).view(f.shape[0], f.shape[2], f.shape[3], f.shape[1]).permute(0, 3, 1, 2))
    return out


@pytest.mark.parametrize("widths", [False, True])
def test_row_attention_matches_the_plain_module(R, widths):
    """Forward and all gradients.  fp32 throughout; about ten fp32 stages of at most 128 terms each stay under
    10 * 128 * 2^-24 = 8e-5 of the largest value."""
    torch.manual_seed(0)
    m = R.RowAttentionHip(48, heads=4, kv_heads=2, head_dim=24)
    with torch.no_grad():
        m.q_weight.add_(0.2 * torch.randn(24)), m.k_weight.add_(0.2 * torch.randn(24))
    f1, f2 = torch.randn(2, 48, 3, 37), torch.randn(2, 48, 3, 45)
    w1, w2 = (torch.tensor([37, 20]), torch.tensor([45, 31])) if widths else (None, None)
    import copy
    md = copy.deepcopy(m).double()
    d = [f.double().requires_grad_(True) for f in (f1, f2)]
    want = plain_rows(md, *d, w1, w2)
    gs = [torch.randn(o.shape) for o in want]
    want_g = torch.autograd.grad(want, d + list(md.parameters()), [g.double() for g in gs])
    m = m.cuda()
    t = [f.cuda().requires_grad_(True) for f in (f1, f2)]
    got = m(*t, *(None if w is None else w.cuda() for w in (w1, w2)))
    got_g = torch.autograd.grad(got, t + list(m.parameters()), [g.cuda() for g in gs])
    for a, b in itertools.chain(zip(got, want), zip(got_g, want_g)):
        assert a.shape == b.shape
        assert float((a.detach().cpu().double() - b.detach()).abs().max()) <= 8e-5 * float(b.detach().abs().max())


@pytest.mark.parametrize("impl", ["reg_hip", "alt_hip"])
def test_correlation_on_attended_features(R, impl):
    """The whole run: feature maps through the attention, into the volume, looked up, and back to the parameters."""
    torch.manual_seed(1)
    m = R.RowAttentionHip(64, heads=2).cuda()
    f1, f2 = torch.randn(1, 64, 4, 48, device="cuda"), torch.randn(1, 64, 4, 48, device="cuda")
    coords = torch.rand(1, 2, 4, 48, device="cuda") * 48
    corr = R.make_corr_fn(impl, f1, f2, attention=m)(coords)
    with torch.no_grad():
        a1, a2 = m(f1, f2)
        assert torch.equal(corr, R.make_corr_fn(impl, a1, a2)(coords))
        assert not torch.equal(corr, R.make_corr_fn(impl, f1, f2)(coords))
        half = R.make_corr_fn(impl, f1.half(), f2.half(), mixed_precision=True, attention=m)(coords)
        assert half.isfinite().all() and m(f1.half(), f2.half())[0].dtype == torch.float16
        assert float((half - corr).abs().max()) <= 2e-2 * float(corr.abs().max())
    corr.square().mean().backward()
    assert all(p.grad is not None and p.grad.isfinite().all() and p.grad.any() for p in m.parameters())


def test_row_attention_keeps_its_frequencies(R):
    m = R.RowAttentionHip(32, heads=1).cuda()
    before = m.freqs.clone()
    m = m.half()
    assert m.freqs.dtype is torch.float64 and torch.equal(m.freqs, before) and m.freqs.is_cuda
    assert "freqs" not in m.state_dict()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out = R.RowAttentionHip(32, heads=1).cuda()(torch.randn(1, 32, 2, 9, device="cuda"), torch.randn(1, 32, 2, 7, device="cuda"))
    assert out[0].shape == (1, 32, 2, 9) and out[1].shape == (1, 32, 2, 7)
