"""The attention operators as workloads: what is run, on what inputs, and what it has to return.

Two operators, each in inference and in training:

    attend        cross_attention_hip   attention of query tokens over the tokens of another sequence (the pixels of the
                                        other image's row; an encoder's states), grouped heads, masked keys
    norm_rotate   qk_norm_rotate_hip    RMS norm of every query and key head and its rotation by position, in one pass

A case is a dict of plain values: `op`, `train` (forward and backward), `dtype`, `n` sequences, `tq` / `tk` tokens,
`hq` / `hk` heads, `dim` elements per head; `mask` for attend ("none", "lengths": sequences of different lengths,
"holes": a boolean mask); `rot` rotated elements, `pos` ("index", "far") and `interleaved` for norm_rotate, whose
`tk` = 0 means that only queries are given.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
BASE = 10000.0


def _attend(name, dtype, n, tq, tk, hq, hk, dim, mask="none", train=False):
    return {"name": name, "op": "attend", "train": train, "dtype": dtype, "n": n, "tq": tq, "tk": tk, "hq": hq, "hk": hk,
            "dim": dim, "mask": mask}


def _rotate(name, dtype, n, tq, tk, hq, hk, dim, rot, pos="index", interleaved=False, train=False):
    return {"name": name, "op": "norm_rotate", "train": train, "dtype": dtype, "n": n, "tq": tq, "tk": tk, "hq": hq,
            "hk": hk, "dim": dim, "rot": rot, "pos": pos, "interleaved": interleaved}


def listed():
    return [
        # one new token in each of four sequences over a short encoder's states: the smallest call, latency counts
        _attend("step_short", "bf16", 4, 1, 1000, 8, 8, 64),
        # one new token in each of sixteen sequences over long states of different lengths, shared heads: serving
        _attend("step_long", "bf16", 16, 1, 8192, 32, 8, 128, "lengths"),
        # the realtime configuration's rows (one 480x640 pair at 1/8), four heads: a small ordinary call
        _attend("rows_realtime", "f16", 60, 80, 80, 4, 4, 64),
        # KITTI, 8 pairs at 1/4: every row's pixels over the other row's, all 256 feature channels in one head
        _attend("rows_kitti", "f16", 768, 312, 312, 1, 1, 256),
        # a batch of long queries over long states with holes in the padding mask: the largest call
        _attend("long_holes", "bf16", 8, 2047, 4095, 16, 4, 128, "holes"),
        # SceneFlow training crops, 8 pairs at 1/4, eight heads of 32
        _attend("rows_sceneflow_train", "bf16", 640, 180, 180, 8, 8, 32, "none", True),
        # training on long ragged sequences with shared heads
        _attend("long_train", "bf16", 2, 2048, 4096, 16, 4, 128, "lengths", True),
        # fp32 training on rows of two different odd widths
        _attend("rows_f32_train", "f32", 96, 128, 117, 4, 4, 64, "none", True),
        # KITTI, 8 pairs: both images' tokens before their attention
        _rotate("norm_kitti", "f16", 768, 312, 312, 4, 4, 64, 64),
        # the query of one new token in each of sixteen sequences, far along
        _rotate("norm_step", "bf16", 16, 1, 0, 32, 0, 128, 128, "far"),
        # training on long sequences, half of every head rotated
        _rotate("norm_long_train", "bf16", 8, 2047, 4095, 16, 4, 128, 64, "far", False, True),
        # SceneFlow training in fp32, neighbouring elements paired
        _rotate("norm_sceneflow_train", "f32", 640, 180, 180, 8, 8, 32, 32, "index", True, True),
    ]


def _cost(case):
    w = work(case)
    return max(w["flops"] / 1.0e15, w["bytes"] / 5.0e12)


def draw(rng):
    """One case of the ranges that the listed ones stand for."""
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    most = max(_cost(c) for c in listed())
    while True:
        dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
        dim = rng.choice([32, 32, 40, 64, 64, 80, 96, 128, 128, 192, 256])
        hk = rng.choice([1, 2, 3, 4, 8])
        hq = hk * rng.choice([1, 1, 1, 2, 3, 4, 8])
        train = rng.random() < 0.5
        if rng.random() < 0.6:
            kind = rng.choice(["step", "rows", "long"])
            if kind == "step":
                n, tq, tk, train = spread(1, 64), rng.choice([1, 1, 1, 2, 5]), spread(64, 16384), False
            elif kind == "rows":
                n, tq = spread(16, 1024), spread(16, 800)
                tk = max(1, int(tq * rng.uniform(0.5, 1.5)))
            else:
                n, tq, tk = spread(1, 8), spread(256, 4096), spread(256, 8192)
            case = _attend("", dtype, n, tq, tk, hq, hk, dim, rng.choice(["none", "lengths", "holes"]), train)
        else:
            rot = rng.choice([dim, dim, dim // 16 * 8])
            n, tq, tk = spread(1, 1024), spread(1, 4096), spread(1, 4096)
            if rng.random() < 0.3:
                tk = hk = 0
            case = _rotate("", dtype, n, tq, tk, hq, hk, dim, rot, rng.choice(["index", "far"]), rng.random() < 0.4, train)
        del case["name"]
        # the plain form's score matrices and their gradients have to fit the card several times over as well
        if _cost(case) <= most and case["n"] * case["hq"] * case["tq"] * case["tk"] <= 2 ** 30 and _elements(case) <= 2 ** 28:
            return case


def _elements(case):
    return case["n"] * case["dim"] * (case["tq"] * case["hq"] + case["tk"] * case["hk"])


def _lengths(case):
    """Lengths of the sequences of the other side, spread from a quarter to all of `tk`; of eight or more one is empty."""
    n, tk = case["n"], case["tk"]
    out = [max(1, round(tk * (0.25 + 0.75 * (i + 1) / n))) for i in range(n)]
    if n >= 8:
        out[0] = 0
    return out


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    n, tq, tk, hq, hk, dim = (case[k] for k in ("n", "tq", "tk", "hq", "hk", "dim"))
    if case["op"] == "attend":
        keys = sum(_lengths(case)) if case["mask"] == "lengths" else n * tk
        q, kv = n * tq * hq * dim * es, keys * hk * dim * es
        fwd = 4 * tq * keys * hq * dim
        extra = {"none": 0, "lengths": 4 * n, "holes": n * tk}[case["mask"]]
        if not case["train"]:
            return {"bytes": 2 * q + 2 * kv + extra, "flops": fwd}
        # q, k, v, the output's gradient in; the output and three gradients (whole, masked places too) out; the
        # backward pass needs four products of the size of each of the forward pass's two
        return {"bytes": 4 * q + 2 * kv + 2 * n * tk * hk * dim * es + extra, "flops": 3 * fwd}
    x = _elements(case)
    extra = 8 * n * (tq + tk) + 4 * 2 * dim + 8 * (case["rot"] // 2)
    if not case["train"]:
        return {"bytes": 2 * x * es + extra, "flops": 8 * x}
    return {"bytes": 4 * x * es + extra + 4 * 2 * dim, "flops": 28 * x}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    n, tq, tk, hq, hk, dim = (case[k] for k in ("n", "tq", "tk", "hq", "hk", "dim"))

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    st = {"case": case}
    if case["op"] == "attend":
        # normalised queries and keys; a query resembles the key at its own place (the pixel it matches)
        k = randn(n, tk, hk, dim)
        at = torch.arange(tq, device="cuda") * tk // tq
        like = k[:, at].unsqueeze(3).expand(n, tq, hk, hq // hk, dim).reshape(n, tq, hq, dim)
        st["q"] = (randn(n, tq, hq, dim) + 0.4 * like).to(dt)
        st["k"], st["v"] = k.to(dt), randn(n, tk, hk, dim).to(dt)
        st["key_lengths"] = st["key_mask"] = None
        if case["mask"] == "lengths":
            order = torch.randperm(n, generator=g, device="cuda")
            st["key_lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")[order]
        elif case["mask"] == "holes":
            st["key_mask"] = torch.rand((n, tk), generator=g, device="cuda") >= 0.25
        if case["train"]:
            st["g"] = randn(n, tq, hq, dim).to(dt)
            st["leaves"] = [st[key].requires_grad_(True) for key in ("q", "k", "v")]
        return st
    # what a projection hands over: heads of different sizes
    st["q"] = (randn(n, tq, hq, dim) * (0.5 + torch.rand((hq, 1), generator=g, device="cuda"))).to(dt)
    st["q_weight"] = 1.0 + 0.2 * randn(dim)
    st["k"] = st["k_weight"] = st["k_pos"] = None
    if tk:
        st["k"] = (randn(n, tk, hk, dim) * (0.5 + torch.rand((hk, 1), generator=g, device="cuda"))).to(dt)
        st["k_weight"] = 1.0 + 0.2 * randn(dim)
    rot = case["rot"]
    st["freqs"] = BASE ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64, device="cuda") / rot)

    def positions(t):
        if case["pos"] == "index":
            return torch.arange(t, device="cuda")
        start = torch.randint(0, 1 << 20, (n, 1), generator=g, device="cuda")
        return start + torch.arange(t, device="cuda")

    st["q_pos"] = positions(tq)
    if tk:
        st["k_pos"] = positions(tk)
    if case["train"]:
        st["gq"] = randn(n, tq, hq, dim).to(dt)
        st["leaves"] = [st[key].requires_grad_(True) for key in ("q", "q_weight")]
        if tk:
            st["gk"] = randn(n, tk, hk, dim).to(dt)
            st["leaves"] += [st[key].requires_grad_(True) for key in ("k", "k_weight")]
    return st


# ---------------------------------------------------------------------------------------------- the plain forms
def _allowed(st):
    """[n, tk] truth values: keys that may be attended to, or None for all."""
    if st["key_mask"] is not None:
        return st["key_mask"]
    if st["key_lengths"] is not None:
        return torch.arange(st["k"].shape[1], device="cuda")[None] < st["key_lengths"][:, None]
    return None


def _plain_attend(q, k, v, allowed):
    n, tq, hq, dim = q.shape
    tk, hk = k.shape[1], k.shape[2]
    group = hq // hk
    # the heads that share a key head become more rows of its matrix product
    rows = q.float().reshape(n, tq, hk, group, dim).permute(0, 2, 3, 1, 4).reshape(n, hk, group * tq, dim)
    keys, values = k.float().permute(0, 2, 3, 1), v.float().permute(0, 2, 1, 3)
    if allowed is not None:
        values = torch.where(allowed[:, None, :, None], values, 0.0)
    s = torch.matmul(rows, keys) * (1.0 / math.sqrt(dim))
    if allowed is not None:
        s = torch.where(allowed[:, None, None, :], s, float("-inf"))
    top = s.detach().amax(dim=-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0.0, top)
    e = torch.exp(s - top)
    total = e.sum(dim=-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    out = torch.matmul(p, values)
    return out.reshape(n, hk, group, tq, dim).permute(0, 3, 1, 2, 4).reshape(n, tq, hq, dim).to(q.dtype)


def _plain_norm_rotate(x, weight, freqs, pos, interleaved):
    x32 = x.float()
    y = x32 * torch.rsqrt((x32 * x32).mean(dim=-1, keepdim=True) + EPS) * weight
    angle = pos.double()[..., None] * freqs
    cos, sin = angle.cos().float().unsqueeze(-2), angle.sin().float().unsqueeze(-2)
    half = freqs.numel()
    turned, rest = y[..., :2 * half], y[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).reshape(turned.shape)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, rest], dim=-1).to(x.dtype)


def run(state):
    case = state["case"]
    if case["op"] == "attend":
        if own:
            from raft_stereo_amd import cross_attention_hip
            outs = (cross_attention_hip(state["q"], state["k"], state["v"], key_mask=state["key_mask"],
                                        key_lengths=state["key_lengths"]),)
        else:
            outs = (_plain_attend(state["q"], state["k"], state["v"], _allowed(state)),)
        grads = (state["g"],) if case["train"] else ()
    else:
        if own:
            from raft_stereo_amd import qk_norm_rotate_hip
            outs = qk_norm_rotate_hip(state["q"], state["k"], state["q_weight"], state["k_weight"], state["freqs"],
                                      state["q_pos"], state["k_pos"], eps=EPS, interleaved=case["interleaved"])
            outs = outs if isinstance(outs, tuple) else (outs,)
        else:
            outs = tuple(_plain_norm_rotate(state[x], state[x + "_weight"], state["freqs"], state[x + "_pos"],
                                            case["interleaved"]) for x in ("q", "k") if state[x] is not None)
        grads = tuple(state[key] for key in ("gq", "gk") if key in state) if case["train"] else ()
    if not case["train"]:
        return outs
    return tuple(o.detach() for o in outs) + torch.autograd.grad(outs, state["leaves"], grads)


# ------------------------------------------------------------------------------------- the definitions in 64 bits
def _exact_attend(st, case):
    n, tq, tk, hq, hk, dim = (case[k] for k in ("n", "tq", "tk", "hq", "hk", "dim"))
    group, scale = hq // hk, dim ** -0.5
    results = [torch.empty((n, tq, hq, dim), dtype=torch.float64, device="cuda")]
    if case["train"]:
        results += [torch.empty_like(results[0])] + [torch.zeros((n, tk, hk, dim), dtype=torch.float64, device="cuda")
                                                     for _ in range(2)]
    allowed = _allowed(st)
    per = max(1, int(2 ** 27 // max(1, hq * tq * tk)))
    for lo in range(0, n, per):
        part = slice(lo, min(n, lo + per))
        # [sequence, head, token, element], every query head beside its own copy of the keys
        q = st["q"].detach()[part].double().transpose(1, 2)
        k, v = (st[key].detach()[part].double().transpose(1, 2).repeat_interleave(group, dim=1) for key in ("k", "v"))
        s = q @ k.transpose(2, 3) * scale
        if allowed is not None:
            ok = allowed[part][:, None, None, :]
            s = s.masked_fill(~ok, -math.inf)
            v = v.masked_fill(~allowed[part][:, None, :, None], 0.0)
            k = k.masked_fill(~allowed[part][:, None, :, None], 0.0)
        p = torch.exp(s - torch.logsumexp(s, dim=-1, keepdim=True)).nan_to_num(nan=0.0)
        del s
        results[0][part] = (p @ v).transpose(1, 2)
        if not case["train"]:
            continue
        g = st["g"][part].double().transpose(1, 2)
        dv = p.transpose(2, 3) @ g
        dp = g @ v.transpose(2, 3)
        ds = p * (dp - (p * dp).sum(dim=-1, keepdim=True))
        del dp, p
        dk = ds.transpose(2, 3) @ q * scale
        results[1][part] = (ds @ k * scale).transpose(1, 2)
        for r, d in ((results[2], dk), (results[3], dv)):
            r[part] = d.reshape(d.shape[0], hk, group, tk, dim).sum(dim=2).transpose(1, 2)
    return tuple(results)


def _exact_norm_rotate(st, case):
    outs, dxs = [], []
    for key in ("q", "k"):
        if st[key] is None:
            continue
        x, w = st[key].detach().double(), st[key + "_weight"].detach().double()
        half = case["rot"] // 2
        first = torch.arange(half, device="cuda") * (2 if case["interleaved"] else 1)
        second = first + (1 if case["interleaved"] else half)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                           st[key + "_pos"].double().unsqueeze(-1) * st["freqs"]).unsqueeze(-2)

        def rotated(y, by):
            z = torch.complex(y[..., first], y[..., second]) * by
            y = y.clone()
            y[..., first], y[..., second] = z.real, z.imag
            return y

        r = 1.0 / torch.sqrt(x.square().sum(dim=-1, keepdim=True) / case["dim"] + EPS)
        outs.append(rotated(x * r * w, turn))
        if case["train"]:
            u = rotated(st["g" + key].double(), turn.conj())
            wu = w * u
            dxs += [r * (wu - x * (r * r) * (wu * x).sum(dim=-1, keepdim=True) / case["dim"]),
                    (u * x * r).sum(dim=(0, 1, 2))]
    return tuple(outs + dxs)


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return _exact_attend(st, case) if case["op"] == "attend" else _exact_norm_rotate(st, case)
