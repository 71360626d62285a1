"""Attention along a row, backed by libraftcorr_hip.so: what feature maps go through before they are correlated.

    qk_norm_rotate_hip(q, k, q_weight, k_weight, freqs, ...)   RMS norm and position rotation of query and key heads
    cross_attention_hip(q, k, v, ...)                          attention over the tokens of another sequence
    RowAttentionHip(dim, heads)                                both, between the rows of two feature maps

The correlation volume is the score half of an attention between the pixels of two image rows (core/corr.py:148-156 of
the reference: f1^T f2 / sqrt(D), the rows of one image wider than the other's allowed); these operators add the other
half.  The reference has no counterpart.  Operands are sequences of heads [N, T, H, D]; the projections around them are
torch's, like the convolutions of the update block.  There is no CPU or eager fallback: tensors must live on a GPU.
"""
import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from raft_stereo_amd import _lib
from raft_stereo_amd._lib import lib, check, Attn, Heads
from raft_stereo_amd.corr import _DT, _stream, _on_device

_POS = {torch.int32: _lib.RC_POS_I32, torch.int64: _lib.RC_POS_I64, torch.float32: _lib.RC_POS_F32}
_MAX_STRIDE_BYTES = 1 << 23     # between tokens or heads: a tile's rows are addressed with 32 bits
_MAX_SPAN_BYTES = 1 << 30       # from a token's first head to its last


def _check_heads(t, what):
    if not torch.is_tensor(t) or not t.is_cuda:
        raise RuntimeError(f"raft_stereo_amd attention kernels need GPU tensors (there is no CPU path): {what}")
    if t.dtype not in _DT:
        raise TypeError(f"unsupported dtype {t.dtype} for {what}")
    if t.dim() != 4:
        raise ValueError(f"{what} must be [N, T, heads, D], got {tuple(t.shape)}")
    if t.shape[3] % 8 or not 8 <= t.shape[3] <= _lib.RC_HEAD_DIM_MAX:
        raise ValueError(f"the head dimension of {what} must be a multiple of 8 in 8..{_lib.RC_HEAD_DIM_MAX}, "
                         f"got {t.shape[3]}")


def _check_same(t, like, what, of):
    if t.dtype != like.dtype:
        raise TypeError(f"{what} is {t.dtype}, {of} {like.dtype}")
    if t.device != like.device:
        raise RuntimeError(f"{what} and {of} live on different devices")


def _refuse_duals(what, *tensors):
    """There is no forward-mode derivative, and the kernels would drop a dual tensor's tangent without a word."""
    if getattr(forward_ad, "_current_level", 0) < 0:      # (outside every dual_level: nothing to look for)
        return
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what} has no forward-mode derivative: its operands must not be dual tensors")


def _heads_view(t):
    """`t` as (tensor, strides of sequence, token and head) the kernels can address: dense heads, everything on 16-byte
    boundaries (slices of a wider projection qualify, and expanded dimensions).  Anything else is copied."""
    es = t.element_size()
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        _, T, H, D = t.shape
        if H * D * es < _MAX_STRIDE_BYTES:
            return t, (T * H * D, H * D, D)
    st = [s if n > 1 else 0 for n, s in zip(t.shape[:3], t.stride()[:3])]
    if t.stride(3) != 1 or t.data_ptr() % 16 or any(s * es % 16 for s in st) or max(st[1:]) * es >= _MAX_STRIDE_BYTES \
            or t.shape[2] * st[2] * es >= _MAX_SPAN_BYTES:
        t = t.clone(memory_format=torch.contiguous_format)
        st = list(t.stride()[:3])
        if max(s if n > 1 else 0 for n, s in zip(t.shape[1:3], st[1:])) * es >= _MAX_STRIDE_BYTES:
            raise ValueError(f"heads of {tuple(t.shape)} are too wide: a token has to stay under 8 MiB")
    return t, st


def _unit_stride(t):
    """Positions or a mask, None or with the tokens side by side."""
    return t if t is None or t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _dense(t):
    """`t` contiguous and on a 16-byte boundary."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


# --------------------------------------------------------------------------------------------- norm and rotation
def _check_weight(w, x, what):
    if w is None:
        return
    if w.dim() != 1 or w.shape[0] != x.shape[3]:
        raise ValueError(f"{what} must be [{x.shape[3]}], got {tuple(w.shape)}")
    if w.dtype not in _DT:
        raise TypeError(f"unsupported dtype {w.dtype} for {what}")
    if w.device != x.device:
        raise RuntimeError(f"{what} lives on a different device than the heads")


def _check_pos(pos, x, what):
    """Positions whose tokens lie side by side."""
    if pos is None:
        return None
    if pos.dtype not in _POS:
        raise TypeError(f"{what} must be int32, int64 or float32, got {pos.dtype}")
    if pos.device != x.device:
        raise RuntimeError(f"{what} lives on a different device than the heads")
    N, T = x.shape[:2]
    if tuple(pos.shape) not in ((T,), (N, T)):
        raise ValueError(f"{what} must be [{T}] or [{N}, {T}], got {tuple(pos.shape)}")
    return _unit_stride(pos)


def _heads_desc(x, st, weight, pos):
    d = Heads()
    d.x = x.data_ptr()
    d.T, d.H = x.shape[1], x.shape[2]
    d.stride[0], d.stride[1], d.stride[2] = st
    if weight is not None:
        d.weight, d.weight_dtype = weight.data_ptr(), _DT[weight.dtype]
    if pos is not None:
        d.pos, d.pos_dtype = pos.data_ptr(), _POS[pos.dtype]
        d.pos_stride = pos.stride(0) if pos.dim() == 2 and x.shape[0] > 1 else 0
    return d


def _norm_rotate_desc(q, k, q_weight, k_weight, freqs, q_pos, k_pos, rest):
    """The operands as the library takes them, and q and k as they are described (copies, where they have to be)."""
    eps, interleaved = rest
    q, st = _heads_view(q)
    desc_q = _heads_desc(q, st, q_weight, q_pos)
    desc_k = None
    if k is not None:
        k, st = _heads_view(k)
        desc_k = _heads_desc(k, st, k_weight, k_pos)
    tail = (_DT[q.dtype], None if freqs is None else freqs.data_ptr(), int(freqs is not None and freqs.dtype is torch.float64),
            0 if freqs is None else freqs.shape[0], interleaved, eps)
    return q, k, desc_q, desc_k, tail


def _norm_rotate_raw(q, k, desc_q, desc_k, tail):
    dev = q.device
    with _on_device(dev):
        yq = torch.empty_like(q, memory_format=torch.contiguous_format)
        yk = None if k is None else torch.empty_like(k, memory_format=torch.contiguous_format)
        rc = lib.rc_qk_norm_rotate_fwd(desc_q, desc_k, yq.data_ptr(), None if yk is None else yk.data_ptr(), q.shape[0],
                                       q.shape[3], *tail, _stream(dev))
        if rc:
            check(rc, "rc_qk_norm_rotate_fwd")
    return yq, yk


class _NormRotateFn(torch.autograd.Function):
    """Keeps its inputs for the backward pass, which works the norm out again.  (They are laid out and described again
    there: a hook on saved tensors may have moved them.)"""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, freqs, q_pos, k_pos, rest):
        ctx.save_for_backward(q, k, q_weight, k_weight, freqs, q_pos, k_pos)
        ctx.rest = rest
        ctx.set_materialize_grads(False)
        return _norm_rotate_raw(*_norm_rotate_desc(q, k, q_weight, k_weight, freqs, q_pos, k_pos, rest))

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        if gq is None and gk is None:
            return (None,) * 8
        q, k, qw, kw, freqs, q_pos, k_pos = ctx.saved_tensors
        qw, kw, freqs = (None if t is None else t.contiguous() for t in (qw, kw, freqs))
        q_pos, k_pos = _unit_stride(q_pos), _unit_stride(k_pos)      # (by name: they have to outlive the call)
        q, k, desc_q, desc_k, tail = _norm_rotate_desc(q, k, qw, kw, freqs, q_pos, k_pos, ctx.rest)
        dev, D = q.device, q.shape[3]
        want = ctx.needs_input_grad
        with _on_device(dev):
            gq = torch.zeros(q.shape, dtype=q.dtype, device=dev) if gq is None else _dense(gq)
            dq = torch.empty_like(gq)
            gk_ptr = dk = dk_ptr = dwq = dwk = dwq_ptr = dwk_ptr = work_ptr = None
            if k is not None:
                gk = torch.zeros(k.shape, dtype=k.dtype, device=dev) if gk is None else _dense(gk)
                dk = torch.empty_like(gk)
                gk_ptr, dk_ptr = gk.data_ptr(), dk.data_ptr()
            if qw is not None and want[2]:
                dwq = torch.empty(D, dtype=torch.float32, device=dev)
                dwq_ptr = dwq.data_ptr()
            if kw is not None and want[3]:
                dwk = torch.empty(D, dtype=torch.float32, device=dev)
                dwk_ptr = dwk.data_ptr()
            if dwq is not None or dwk is not None:
                work = torch.empty(int(lib.rc_qk_norm_rotate_bwd_work_bytes(D)), dtype=torch.uint8, device=dev)
                work_ptr = work.data_ptr()
            check(lib.rc_qk_norm_rotate_bwd(desc_q, desc_k, gq.data_ptr(), gk_ptr, dq.data_ptr(), dk_ptr, dwq_ptr, dwk_ptr,
                                            work_ptr, q.shape[0], D, *tail, _stream(dev)), "rc_qk_norm_rotate_bwd")
        return (dq, dk, None if dwq is None else dwq.to(qw.dtype), None if dwk is None else dwk.to(kw.dtype),
                None, None, None, None)


def qk_norm_rotate_hip(q, k=None, q_weight=None, k_weight=None, freqs=None, q_pos=None, k_pos=None, eps=1e-6,
                       interleaved=False):
    """RMS norm of every query and key head and its rotation by position, in one pass.

    q `[N, Tq, Hq, D]` and k `[N, Tk, Hk, D]` (its own length and number of heads; None: queries alone, where the keys
    were made by an earlier call).  `y = x / sqrt(mean(x^2) + eps) * weight` over D, weights `[D]` (None: ones); then
    pair i is turned by the angle `pos * freqs[i]`: elements `(i, i + n)`, or `(2i, 2i + 1)` if `interleaved`, of the
    first `2 n` for the n frequencies in `freqs` (float32 or float64, radians per position; None: the norm alone).
    Positions are `[T]` or `[N, T]`, int32, int64 or float32 (None: 0, 1, ...); angles are reduced to one turn in
    64 bits, so positions far along lose nothing.  Everything else is fp32 and rounded once.  n must be a multiple of 4.
    Returns `(q', k')`, contiguous, or `q'` alone if k is None.  Differentiable w.r.t. q, k and the weights, once, in
    reverse mode (dual tensors are refused)."""
    _check_heads(q, "q")
    _check_weight(q_weight, q, "q_weight")
    if k is not None:
        _check_heads(k, "k")
        _check_same(k, q, "k", "q")
        if k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
            raise ValueError(f"q and k must agree in sequences and head dimension: {tuple(q.shape)} vs {tuple(k.shape)}")
        _check_weight(k_weight, k, "k_weight")
    elif k_weight is not None or k_pos is not None:
        raise ValueError("k_weight and k_pos need k")
    _refuse_duals("qk_norm_rotate_hip", q, k, q_weight, k_weight, freqs, q_pos, k_pos)
    if freqs is not None:
        if freqs.dim() != 1 or freqs.shape[0] % 4 or 2 * freqs.shape[0] > q.shape[3]:
            raise ValueError(f"freqs must be [n] with n a multiple of 4 and at most {q.shape[3] // 2}, "
                             f"got {tuple(freqs.shape)}")
        if freqs.dtype not in (torch.float32, torch.float64):
            raise TypeError(f"freqs must be float32 or float64, got {freqs.dtype}")
        if freqs.device != q.device:
            raise RuntimeError("freqs lives on a different device than the heads")
        freqs = freqs.detach().contiguous() if freqs.shape[0] else None
    elif q_pos is not None or k_pos is not None:
        raise ValueError("positions need freqs")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    q_pos = _check_pos(q_pos, q, "q_pos")
    k_pos = None if k is None else _check_pos(k_pos, k, "k_pos")
    q_weight = None if q_weight is None else q_weight.contiguous()
    k_weight = None if k_weight is None else k_weight.contiguous()
    args = (q, k, q_weight, k_weight, freqs, q_pos, k_pos, (float(eps), int(bool(interleaved))))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args[:4]):
        yq, yk = _NormRotateFn.apply(*args)
    else:
        yq, yk = _norm_rotate_raw(*_norm_rotate_desc(*args))
    return yq if k is None else (yq, yk)


# ------------------------------------------------------------------------------------------------ cross attention
def _attn_desc(q, k, v, key_mask, key_lengths, scale):
    """The operands as the library takes them, and q, k and v as they are described (copies, where they have to be)."""
    (q, qs), (k, ks), (v, vs) = _heads_view(q), _heads_view(k), _heads_view(v)
    a = Attn()
    N, a.Tq, a.Hq, a.D = q.shape
    a.N, a.Tk, a.Hk = N, k.shape[1], k.shape[2]
    a.dtype, a.scale = _DT[q.dtype], scale
    for dst, st in ((a.q_stride, qs), (a.k_stride, ks), (a.v_stride, vs)):
        dst[0], dst[1], dst[2] = st
    if key_mask is not None:
        a.key_mask, a.mask_stride = key_mask.data_ptr(), key_mask.stride(0) if N > 1 else 0
    if key_lengths is not None:
        a.key_lengths, a.lengths_i64 = key_lengths.data_ptr(), int(key_lengths.dtype is torch.int64)
    return a, q, k, v


def _work(nbytes, what, dev):
    if nbytes < 0:
        check(int(nbytes), what)
    return torch.empty(int(nbytes), dtype=torch.uint8, device=dev) if nbytes else None


def _attention_raw(a, q, k, v, train):
    dev = q.device
    N, Tq, Hq, _ = q.shape
    with _on_device(dev):
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        lse = torch.empty((N, Hq, Tq), dtype=torch.float32, device=dev) if train else None
        rest = torch.empty_like(out) if train and out.dtype is not torch.float32 else None
        work = _work(lib.rc_cross_attn_fwd_work_bytes(a), "rc_cross_attn_fwd_work_bytes", dev)
        rc = lib.rc_cross_attn_fwd(a, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                   None if rest is None else rest.data_ptr(), None if lse is None else lse.data_ptr(), None if work is None else work.data_ptr(),
                                   _stream(dev))
        if rc:
            check(rc, "rc_cross_attn_fwd")
    return out, rest, lse


class _CrossAttentionFn(torch.autograd.Function):
    """Keeps the operands, the result (16-bit: with what rounding took from it) and each row's log-sum-exp; the backward
    pass works the scores out again.  (All of them are laid out and described again there: a hook on saved tensors may have
    moved them.)"""

    @staticmethod
    def forward(ctx, q, k, v, key_mask, key_lengths, scale):
        out, rest, lse = _attention_raw(*_attn_desc(q, k, v, key_mask, key_lengths, scale), True)
        ctx.save_for_backward(q, k, v, out, rest, lse, key_mask, key_lengths)
        ctx.scale = scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        q, k, v, out, rest, lse, key_mask, key_lengths = ctx.saved_tensors
        out, lse, rest = _dense(out), _dense(lse), None if rest is None else _dense(rest)
        key_mask, key_lengths = _unit_stride(key_mask), None if key_lengths is None else key_lengths.contiguous()
        a, q, k, v = _attn_desc(q, k, v, key_mask, key_lengths, ctx.scale)
        dev = q.device
        g = _dense(grad_out)
        want_q, want_kv = ctx.needs_input_grad[0], ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        with _on_device(dev):
            dq = torch.empty_like(g) if want_q else None
            dk = torch.empty_like(k, memory_format=torch.contiguous_format) if want_kv else None
            dv = torch.empty_like(v, memory_format=torch.contiguous_format) if want_kv else None
            work = _work(lib.rc_cross_attn_bwd_work_bytes(a), "rc_cross_attn_bwd_work_bytes", dev)
            ptr = lambda t: None if t is None else t.data_ptr()
            check(lib.rc_cross_attn_bwd(a, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), ptr(rest),
                                        lse.data_ptr(), g.data_ptr(), ptr(dq), ptr(dk), ptr(dv), ptr(work), _stream(dev)),
                  "rc_cross_attn_bwd")
        return dq, dk, dv, None, None, None


def cross_attention_hip(q, k, v, key_mask=None, key_lengths=None, scale=None):
    """Attention of query tokens over the tokens of another sequence: `softmax(scale q k^T) v` for each head.

    q `[N, Tq, Hq, D]`, k and v `[N, Tk, Hk, D]`, Hq a multiple of Hk (the Hq / Hk query heads in a row share a key and
    value head), any lengths from 0 on; scale defaults to `1 / sqrt(D)`.  A key takes part if its index is below
    `key_lengths[n]` (int32 or int64 `[N]`; beyond Tk counts as Tk, negative as 0) and `key_mask[n, t]` is True (bool
    `[N, Tk]`); what the others hold, infinities and NaN included, has no influence.  A sequence without any key gives
    zeros, and zero gradients; a row whose keys all score -inf gives NaN.  Lengths save the work of the keys behind them,
    a mask does not: padding is better given as lengths.  Scores, the softmax's maximum and sum, and all products' sums
    are fp32; 16-bit operands have their probabilities (and in the backward pass their scores' gradients) rounded to 16
    bits for the second product.  Returns `[N, Tq, Hq, D]` contiguous.  Differentiable w.r.t. q, k and v, once, in reverse mode (dual tensors
    are refused); the same bits on every run."""
    for t, what in ((q, "q"), (k, "k"), (v, "v")):
        _check_heads(t, what)
    for t, what in ((k, "k"), (v, "v")):
        _check_same(t, q, what, "q")
    N, Tq, Hq, D = q.shape
    if k.shape != v.shape or k.shape[0] != N or k.shape[3] != D:
        raise ValueError(f"k and v must be [{N}, Tk, heads, {D}], got {tuple(k.shape)} and {tuple(v.shape)}")
    Tk, Hk = k.shape[1], k.shape[2]
    if Hk < 1 or Hq < 1 or Hq % Hk:
        raise ValueError(f"{Hq} query heads are no multiple of {Hk} key heads")
    if key_mask is not None:
        if key_mask.dtype is not torch.bool:
            raise TypeError(f"key_mask must be bool (True: the key takes part), got {key_mask.dtype}")
        if tuple(key_mask.shape) != (N, Tk):
            raise ValueError(f"key_mask must be [{N}, {Tk}], got {tuple(key_mask.shape)}")
        if key_mask.device != q.device:
            raise RuntimeError("key_mask lives on a different device than q")
        key_mask = _unit_stride(key_mask)
    if key_lengths is not None:
        if key_lengths.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"key_lengths must be int32 or int64, got {key_lengths.dtype}")
        if tuple(key_lengths.shape) != (N,):
            raise ValueError(f"key_lengths must be [{N}], got {tuple(key_lengths.shape)}")
        if key_lengths.device != q.device:
            raise RuntimeError("key_lengths lives on a different device than q")
        key_lengths = key_lengths.contiguous()
    _refuse_duals("cross_attention_hip", q, k, v)
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < 2.0 ** 127:       # (times log2 e, it has to be an fp32 number)
        raise ValueError(f"scale must be positive and below 2^127, got {scale}")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _CrossAttentionFn.apply(q, k, v, key_mask, key_lengths, scale)
    return _attention_raw(*_attn_desc(q, k, v, key_mask, key_lengths, scale), False)[0]


# ------------------------------------------------------------------------------------------- rows of feature maps
class RowAttentionHip(nn.Module):
    """Lets two feature maps attend to each other along their rows before they are correlated.

    `forward(fmap1, fmap2, width1=None, width2=None)` takes `[B, dim, H, W1]` and `[B, dim, H, W2]` and returns both
    maps with the attention's result added: every pixel of a row looks at all pixels of the same row of the other map
    (rectified stereo: its match lies there, which is also why the correlation is one-dimensional, core/corr.py:148-156).
    Queries and keys are normalised per head and rotated by their column.  `width1` / `width2` (int32 or int64 `[B]`):
    columns of each image that hold data; the padding behind them is not attended to.  Handed to
    `make_corr_fn(..., attention=module)`, which takes the widths too, it runs in front of the volume."""

    def __init__(self, dim, heads=4, kv_heads=None, head_dim=None, base=10000.0, eps=1e-6):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if heads < 1 or kv_heads < 1 or heads % kv_heads:
            raise ValueError(f"{heads} query heads are no multiple of {kv_heads} key heads")
        head_dim = dim // heads if head_dim is None else head_dim
        if head_dim % 8 or not 8 <= head_dim <= _lib.RC_HEAD_DIM_MAX:
            raise ValueError(f"head_dim must be a multiple of 8 in 8..{_lib.RC_HEAD_DIM_MAX}, got {head_dim}")
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.base, self.eps = base, eps
        self.q = nn.Linear(dim, heads * head_dim, bias=False)
        self.k = nn.Linear(dim, kv_heads * head_dim, bias=False)
        self.v = nn.Linear(dim, kv_heads * head_dim, bias=False)
        self.out = nn.Linear(heads * head_dim, dim)
        self.q_weight = nn.Parameter(torch.ones(head_dim))
        self.k_weight = nn.Parameter(torch.ones(head_dim))
        self.register_buffer("freqs", self._make_freqs("cpu"), persistent=False)

    def _make_freqs(self, device):
        n = self.head_dim // 8 * 4
        return (self.base ** (-torch.arange(n, dtype=torch.float64, device="cpu") / n)).to(device)   # the same bits on any device

    def _apply(self, *args, **kwargs):
        """The frequencies are moved with the module, but neither rounded (`.half()`) nor left as empty storage is
        (`.to_empty()`): wherever they are replaced, they are made again."""
        before = self.freqs
        super()._apply(*args, **kwargs)
        if self.freqs is not before:        # (a captured graph reads them where they are)
            self.freqs = self._make_freqs(self.freqs.device)
        return self

    def _project(self, rows, layer, heads):
        y = F.linear(rows, layer.weight.to(rows.dtype))
        return y.view(*y.shape[:2], heads, self.head_dim)

    def _onto(self, fmap, rows, q, k, v, lengths):
        a = cross_attention_hip(q, k, v, key_lengths=lengths)
        y = F.linear(a.flatten(2), self.out.weight.to(a.dtype), self.out.bias.to(a.dtype))
        B, C, H, W = fmap.shape
        return (rows + y).view(B, H, W, C).permute(0, 3, 1, 2).contiguous()

    def forward(self, fmap1, fmap2, width1=None, width2=None):
        if fmap1.dim() != 4 or fmap2.dim() != 4 or fmap1.shape[:3] != fmap2.shape[:3]:
            raise ValueError(f"fmap shapes disagree: {tuple(fmap1.shape)} vs {tuple(fmap2.shape)}")
        if fmap1.dtype != fmap2.dtype:
            raise TypeError(f"unsupported feature dtypes {fmap1.dtype}/{fmap2.dtype}")
        H = fmap1.shape[2]
        rows, heads, lengths = [], [], []
        for fmap, width in ((fmap1, width1), (fmap2, width2)):
            x = fmap.permute(0, 2, 3, 1).flatten(0, 1).contiguous()                       # [B*H, W, dim]
            rows.append(x)
            q, k = qk_norm_rotate_hip(self._project(x, self.q, self.heads), self._project(x, self.k, self.kv_heads),
                                      self.q_weight, self.k_weight, self.freqs, eps=self.eps)
            heads.append((q, k, self._project(x, self.v, self.kv_heads)))
            if width is not None and tuple(width.shape) != (fmap.shape[0],):
                raise ValueError(f"widths must be [{fmap.shape[0]}], got {tuple(width.shape)}")
            lengths.append(None if width is None else width.repeat_interleave(H))
        (q1, k1, v1), (q2, k2, v2) = heads
        return (self._onto(fmap1, rows[0], q1, k2, v2, lengths[1]),
                self._onto(fmap2, rows[1], q2, k1, v1, lengths[0]))
