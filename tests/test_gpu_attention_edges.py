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


LONG = [  # Tq, Tk, Hq, D and keys of a part: the few-row form and the one of many rows, up to 512 parts of one row
    ("bf16", 1, 16385, 2, 64, 256), ("f16", 3, 70000, 1, 64, 256), ("bf16", 1, 131067, 2, 64, 256), ("f16", 1, 131067, 1, 128, 256),
    ("f32", 1, 16385, 2, 64, 64), ("f32", 2, 32760, 1, 64, 64), ("f32", 1, 9000, 2, 256, 64), ("f32", 1, 65500, 1, 32, 128),
    ("bf16", 40, 65500, 1, 64, 128), ("f32", 40, 32760, 1, 40, 64),
]


@pytest.mark.parametrize("dtype, Tq, Tk, Hq, D, part", LONG)
@pytest.mark.parametrize("kind", ["none", "lengths", "parts"])
def test_many_parts_match_the_formula(R, dtype, Tq, Tk, Hq, D, part, kind):
    """Long rows, with parts (and runs of them) that no key is left in, forward and back."""
    rng = np.random.default_rng(Tk + len(kind))
    q, k, v = rand(rng, (1, Tq, Hq, D), dtype, 1.5), rand(rng, (1, Tk, 1, D), dtype), rand(rng, (1, Tk, 1, D), dtype)
    g = rand(rng, (1, Tq, Hq, D), dtype)
    lengths = [Tk - 3 * part - 7] if kind == "lengths" else None
    mask = None
    if kind == "parts":
        mask = np.repeat(rng.random((1, Tk // part + 1)) < 0.5, part, axis=1)[:, :Tk] & (rng.random((1, Tk)) < 0.9)
        mask[:, Tk // 4:Tk // 2] = False
    want = A.attention(*(host(x) for x in (q, k, v, g)), A.allowed_keys(1, Tk, lengths, mask), dtype=dtype)
    got = run_attention(R, q, k, v, g, lengths, mask, dtype)
    for name in ("out", "dq", "dk", "dv"):
        assert_within(got[name], want[name], name)


@pytest.mark.parametrize("dtype, Tq, Tk, Hq, D, part", LONG)
def test_every_part_counts_once(R, dtype, Tq, Tk, Hq, D, part):
    """Equal probabilities, and a one in the first and the last place of each part, the parts' ones dealt to the elements in
    turn: an element sums few parts, so that one lost or doubled is far outside the bound."""
    q, k, v = torch.zeros(1, Tq, Hq, D), rand(np.random.default_rng(3), (1, Tk, 1, D), dtype).float(), torch.zeros(1, Tk, 1, D)
    for s in range((Tk + part - 1) // part):
        for at in (s * part, min(Tk, (s + 1) * part) - 1):
            v[0, at, 0, s % D] += 1.0
    q, k, v = (x.to(DT[dtype]) for x in (q, k, v))
    value, bound = A.attention(host(q), host(k), host(v), None, None, dtype=dtype)["out"]
    assert (bound[value > 0] < 0.5 / Tk).all()                    # a part brings 1 / Tk at least
    assert_within(run_attention(R, q, k, v, None, None, None, dtype)["out"], (value, bound), "out")


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


# ------------------------------------------------------------------------------- norm and rotation of many tokens
def norm_plan(tokens, H, D, most):
    """The launch that the library makes: heads of a group, chunks of a token, blocks, and the longest fp32 chain of a
    weight gradient's sum (what a lane goes through, then the block's groups)."""
    lanes = 1
    while lanes * 8 < D:
        lanes *= 2
    per, hp = 256 // lanes, H
    while hp > 1 and tokens * -(-H // hp) < 2048 * per:
        hp = (hp + 1) // 2
    chunks = -(-H // hp)
    wanted = -(-tokens * chunks // per)
    blocks = min(wanted, most)
    return hp, chunks, blocks, wanted, -(-wanted // blocks) * hp + per


MANY = [  # N, Tq, Tk, Hq, Hk, D, rotated, positions, pairs, slices of a wider projection
    (2, 4100, 4150, 5, 3, 256, 128, "far", False, True),       # several heads a group, the last chunk with fewer
    (1, 8200, 0, 9, 0, 256, 256, "float", True, False),        # five heads: two loads of four
    (1, 16500, 700, 3, 4, 200, 64, "shared", False, True),     # all three heads in one group; the other side a small one
    (3, 470, 0, 5, 0, 256, 64, "far", True, True),             # 512 to 1024 blocks: the weights' sums in two turns
    (1, 33000, 2100, 2, 6, 128, 128, "index", False, False),
    (5, 3300, 3301, 6, 7, 72, 16, "far", True, True),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", MANY, ids=lambda s: "x".join(map(str, s[:7])))
def test_norm_rotate_of_many_tokens_matches_the_formula(R, shape, dtype):
    N, D = shape[0], shape[5]
    pos, interleaved, sliced = shape[7:]
    rng = np.random.default_rng(sum(shape[:7]))
    freqs, sides = norm_inputs(shape[:7], dtype, rng, pos)
    eps = 1e-5
    leaves, xs, ws, ps, plans = [], [], [], [], []
    for s in sides:
        if s is None:
            xs.append(None), ws.append(None), ps.append(None), plans.append(None)
            continue
        x, g, w, p = s
        H = x.shape[2]
        leaf = x.cuda()
        if sliced:
            wide = torch.full((N, x.shape[1], 2 * H + 1, D), 7.0, dtype=x.dtype, device="cuda")
            wide[:, :, 1:H + 1] = leaf
            leaf = wide[:, :, 1:H + 1]
        leaf = leaf.detach().requires_grad_()
        w = w.to(x.dtype)      # weights in the operands' type
        s[2].copy_(w)
        xs.append(leaf), ws.append(w.cuda().requires_grad_()), ps.append(None if p is None else p.cuda())
        leaves += [leaf, ws[-1]]
        plans.append(norm_plan(N * x.shape[1], H, D, 1024 if sides[1] is None else 512))
    # the ways that small calls do not take
    hp, chunks, blocks, wanted, _ = plans[0]
    assert blocks > 512 or wanted > blocks
    assert hp > 1 or wanted > 512
    out = R.qk_norm_rotate_hip(xs[0], xs[1], ws[0], ws[1], torch.from_numpy(freqs).cuda(), ps[0], ps[1], eps=eps, interleaved=interleaved)
    outs = (out,) if sides[1] is None else out
    used = [i for i in (0, 1) if sides[i] is not None]
    grads = torch.autograd.grad(outs, leaves, [sides[i][1].cuda() for i in used])
    for j, i in enumerate(used):
        x, g, w, p = sides[i]
        want = A.norm_rotate(host(x), host(w), freqs, None if p is None else p.numpy(), eps, interleaved, host(g), dtype, sums=plans[i][4])
        assert_within(outs[j], want["y"], ("y", i))
        assert_within(grads[2 * j], want["dx"], ("dx", i))
        dw, bound = want["dw"]
        assert grads[2 * j + 1].dtype == x.dtype
        assert_within(grads[2 * j + 1], (dw, bound + A.HALF_STEP[dtype] * (np.abs(dw) + bound)), ("dw", i))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", MANY, ids=lambda s: "x".join(map(str, s[:6])))
def test_every_head_counts_once_in_the_weights_gradient(R, shape, dtype):
    """Heads of ones and minus ones have the norm 1, so the gradients of the weights are sums of small whole numbers, exact
    in fp32 in any order where r is: a head that is lost or counted twice changes some of them by one or more."""
    N, Tq, Tk, Hq, Hk, D = shape[:6]
    gen = torch.Generator(device="cuda").manual_seed(5)
    xs, gs = [], []
    for T, H in ((Tq, Hq), (Tk, Hk)):
        if H:
            xs.append((torch.randint(0, 2, (N, T, H, D), generator=gen, device="cuda") * 2 - 1).to(DT[dtype]))
            gs.append((torch.randint(1, 3, (N, T, H, 1), generator=gen, device="cuda") * xs[-1]).to(DT[dtype]))
    ws = [torch.ones(D, device="cuda", requires_grad=True) for _ in xs]
    out = R.qk_norm_rotate_hip(xs[0], xs[1] if len(xs) > 1 else None, *ws, eps=0.0)
    dws = torch.autograd.grad(out, ws, gs)
    for x, g, dw in zip(xs, gs, dws):
        want = (x.double() * g.double()).sum(dim=(0, 1, 2))
        chain = norm_plan(N * x.shape[1], x.shape[2], D, 1024 if len(xs) == 1 else 512)[4]
        # r may be off by 2 * 2^-24 (the mean's rounding, the root's), and the sums are rounded then
        assert (dw.double() - want).abs().max() <= (3 + chain) * 2.0 ** -24 * want.max() < 0.5


# ------------------------------------------------------------------------------------------- saved tensors and graphs
def test_saved_tensors_come_back_with_other_strides(R):
    """A hook may hand saved tensors back in another layout and off 16-byte boundaries: the values count."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    mk = lambda *s: torch.randn(s, generator=gen, device="cuda")
    q, k, v, go, w = mk(2, 40, 4, 64), mk(2, 50, 2, 64), mk(2, 50, 2, 64), mk(2, 40, 4, 64), 1 + 0.1 * mk(64)
    mask, lengths = torch.rand(2, 50, generator=gen, device="cuda") < 0.7, torch.tensor([50, 30], device="cuda")
    freqs, pos = torch.linspace(0.01, 1.0, 32, device="cuda"), torch.randint(0, 900, (2, 40), generator=gen, device="cuda")

    def turned(t):
        """The same values, the first dimension the fastest, from an odd place on."""
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:]
        back = flat.view(tuple(t.shape[1:]) + (t.shape[0],)).movedim(-1, 0) if t.dim() > 1 else \
            torch.empty(2 * t.numel() + 1, dtype=t.dtype, device=t.device)[1::2]
        return back.copy_(t)

    def grads(dtype, unpack):
        leaves = [x.to(dtype).requires_grad_() for x in (q, k, v)] + [w.clone().requires_grad_()]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            a, b = R.qk_norm_rotate_hip(leaves[0], leaves[1], leaves[3], leaves[3], freqs, pos)
            out = R.cross_attention_hip(a, b, leaves[2], key_mask=mask, key_lengths=lengths)
        return torch.autograd.grad(out, leaves, go.to(dtype))
    for dtype in (torch.float32, torch.float16):
        for a, b in zip(grads(dtype, lambda t: t), grads(dtype, lambda t: turned(t.detach()))):
            assert torch.equal(a, b)


def test_row_attention_with_widths_in_a_graph(R):
    """Forward and gradients of padded batches, captured and replayed with other widths."""
    torch.manual_seed(4)
    m = R.RowAttentionHip(32, heads=2).cuda()
    f = [torch.randn(2, 32, 3, 40, device="cuda") for _ in range(2)]
    w = [torch.tensor([40, 17], device="cuda"), torch.tensor([25, 40], device="cuda")]
    go = [torch.randn_like(x) for x in f]

    def step():
        t = [x.detach().requires_grad_() for x in f]
        params = [p.detach().requires_grad_() for p in m.parameters()]
        out = torch.func.functional_call(m, dict(zip((n for n, _ in m.named_parameters()), params)), (*t, *w))
        return tuple(o.detach() for o in out) + torch.autograd.grad(out, t + params, go)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step()
    torch.cuda.current_stream().wait_stream(st)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        outs = step()
    for r in range(4):
        for x in f:
            x.copy_(torch.randn_like(x))
        w[0].copy_(torch.tensor([40 - r, 3 * r])), w[1].copy_(torch.tensor([7 * r, 40]))
        want = step()
        gr.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(130, 37, 100, 4, 2, 64), (300, 20, 50, 1, 1, 32), (1, 70, 1500, 2, 1, 96), (2, 150, 700, 2, 2, 128), (1, 600, 90, 2, 1, 256)],
                         ids=lambda s: "x".join(map(str, s)))
def test_gradients_of_some_operands(R, shape, dtype):
    """What is not wanted changes nothing about what is."""
    N, Tq, Tk, Hq, Hk, D = shape
    rng = np.random.default_rng(8)
    x = [rand(rng, s, dtype) for s in ((N, Tq, Hq, D), (N, Tk, Hk, D), (N, Tk, Hk, D))]
    g, mask = rand(rng, (N, Tq, Hq, D), dtype), rng.random((N, Tk)) < 0.8
    want = A.attention(*(host(t) for t in x), host(g), A.allowed_keys(N, Tk, None, mask), dtype=dtype)
    for which in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 0, 1)):
        t = [a.cuda().requires_grad_(bool(w)) for a, w in zip(x, which)]
        out = R.cross_attention_hip(*t, key_mask=torch.from_numpy(mask).cuda())
        got = torch.autograd.grad(out, [a for a, w in zip(t, which) if w], g.cuda())
        for name, d in zip([n for n, w in zip(("dq", "dk", "dv"), which) if w], got):
            assert_within(d, want[name], (name, which))
