"""Plaintext operators around an encrypted prefill, on libb200fhe's kernels.

What runs in the clear beside the encrypted graph: rotary positions for the
plain twin of a decoder layer (the reference's approx/attention.py:23-59), the
client's head on the decrypted hidden state (final_logits, the reference's
application/client.py:60-100) with 4-bit weights, and the score of decrypted
hidden states against tokens with its gradient.

Every call is asynchronous on the current stream of its tensors' device and
can be captured into a CUDA graph; scratch and outputs come from torch's
allocator on that stream.  Tensors used on a stream other than the one they
were made on are the caller's to order, as with any torch operation.  Gradients
are explicit calls: nothing here records an autograd graph or carries tangents,
and tensors that require a gradient are refused unless gradients are switched
off, dual tensors of forward-mode differentiation always.  Arguments
are checked before anything launches: ValueError for shapes, types, strides
and devices (there is no CPU fallback).
"""

from __future__ import annotations

import math
import struct

import torch
from torch.autograd import forward_ad

from ._native import call, check, lib

_DTYPES = {torch.float64: 0, torch.float32: 1, torch.float16: 2, torch.bfloat16: 3}
_HEADS = struct.Struct("PP6qi4x")  # b2f_rope_heads

_current_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream


def _dual(t) -> bool:
    """A tensor with a tangent; there are none outside forward_ad.dual_level()."""

    return forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None


def _plain_tensor(t, index: int) -> bool:
    """A strided CUDA tensor on device `index` that asks for no gradient."""

    return isinstance(t, torch.Tensor) and t.get_device() == index and not t.is_neg() \
        and not (t.requires_grad and torch.is_grad_enabled()) and t.layout is torch.strided \
        and not _dual(t)


def _refuse(what: str, index: int | None, **tensors) -> None:
    """Raise for the first tensor that _plain_tensor turns down."""

    for name, t in tensors.items():
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"{what}: {name} is a {type(t).__name__}, not a tensor")
        if not t.is_cuda:
            raise ValueError(f"{what}: {name} is on {t.device}, not on a CUDA device")
        if index is not None and t.get_device() != index:
            raise ValueError(f"{what}: {name} is on {t.device}, expected cuda:{index}")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{what}: {name} requires a gradient, which this call does not "
                             "record (use the explicit gradient call under torch.no_grad())")
        if _dual(t):
            raise ValueError(f"{what}: {name} is a dual tensor, whose tangent this call does "
                             "not carry (take forward_ad.unpack_dual(...).primal)")
        if not _plain_tensor(t, t.get_device()):
            raise ValueError(f"{what}: {name} is not a plain strided tensor")


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------


def rope_frequencies(rotary_dim: int, theta: float = 500000.0,
                     scaling: dict | None = None) -> tuple[list[float], float]:
    """Angle per position (radians) of each pair, and the factor on cos and sin.

    theta^(-2i/rotary_dim), with one of the usual scalings for long contexts:

    * ``{"type": "linear", "factor"}``: every frequency divided by factor;
    * ``{"type": "bands", "factor", "low", "high", "original"}``: frequencies that
      turn more than `high` times within the original context stay, those below
      `low` turns are divided, those between are mixed linearly in the turns;
    * ``{"type": "yarn", "factor", "original", "fast", "slow"}``: a ramp over the
      pair index between the pairs that turn `fast` and `slow` times, and cos
      and sin times 0.1 ln(factor) + 1 (or ``"attention_factor"``)."""

    r = int(rotary_dim)
    if r < 2 or r % 2:
        raise ValueError(f"rope: {r} rotated elements (an even number)")
    if not theta > 0 or not math.isfinite(theta):
        raise ValueError(f"rope: theta {theta}")
    freqs = [float(theta) ** (-2.0 * i / r) for i in range(r // 2)]
    if scaling is None:
        return freqs, 1.0
    kind = scaling.get("type")
    keys = {"linear": ("factor",), "bands": ("factor", "low", "high", "original"),
            "yarn": ("factor", "original", "fast", "slow")}.get(kind)
    if keys is None:
        raise ValueError(f"rope: scaling {kind!r} not in ['bands', 'linear', 'yarn']")
    missing = [k for k in keys if k not in scaling]
    if missing:
        raise ValueError(f"rope: {kind} scaling without {missing}")
    sc = {k: float(scaling[k]) for k in keys}
    if any(not v > 0 or not math.isfinite(v) for v in sc.values()):
        raise ValueError(f"rope: {kind} scaling {sc}")
    factor = sc["factor"]
    if kind == "linear":
        return [f / factor for f in freqs], 1.0
    if kind == "bands":
        if not sc["high"] > sc["low"]:
            raise ValueError(f"rope: bands from {sc['low']} to {sc['high']} turns")
        out = []
        for f in freqs:
            turns = sc["original"] * f / (2 * math.pi)
            keep = min(max((turns - sc["low"]) / (sc["high"] - sc["low"]), 0.0), 1.0)
            out.append((1 - keep) * f / factor + keep * f)
        return out, 1.0
    if not theta > 1:
        raise ValueError(f"rope: yarn scaling with theta {theta}")

    def pair(turns: float) -> float:
        return r * math.log(sc["original"] / (turns * 2 * math.pi)) / (2 * math.log(theta))

    low = max(math.floor(pair(sc["fast"])), 0)
    high = min(math.ceil(pair(sc["slow"])), r - 1)
    out = []
    for i, f in enumerate(freqs):
        ramp = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
        out.append(ramp * f / factor + (1 - ramp) * f)
    return out, float(scaling.get("attention_factor", 0.1 * math.log(factor) + 1.0))


class RopePlan:
    """Head geometry and frequencies of rotary positions, kept on one device.

    ``layout``: "half" pairs element i with i + rotary_dim / 2, "interleaved"
    2i with 2i + 1.  Elements from rotary_dim on pass through."""

    def __init__(self, head_dim: int, *, rotary_dim: int | None = None, theta: float = 500000.0,
                 layout: str = "half", scaling: dict | None = None,
                 device: str | torch.device = "cuda"):
        self.head_dim = int(head_dim)
        self.rotary_dim = self.head_dim if rotary_dim is None else int(rotary_dim)
        if not 2 <= self.head_dim <= 1024 or not 2 <= self.rotary_dim <= self.head_dim:
            raise ValueError(f"rope: {self.rotary_dim} rotated of {self.head_dim} elements "
                             "(2 up to the head's, heads of up to 1024)")
        if layout not in ("half", "interleaved"):
            raise ValueError(f"rope: layout {layout!r} not in ['half', 'interleaved']")
        self.layout, self.interleaved = layout, int(layout == "interleaved")
        freqs, self.factor = rope_frequencies(self.rotary_dim, theta, scaling)
        dev = torch.device(device)
        if dev.type != "cuda":
            raise ValueError("rope: libb200fhe runs on CUDA devices only (no CPU fallback)")
        self.freqs = torch.tensor(freqs, dtype=torch.float64, device=dev)
        self.device, self.index = self.freqs.device, self.freqs.get_device()


def _rope_refuse(what, q, k, positions, plan):
    if not isinstance(plan, RopePlan):
        raise ValueError(f"{what}: plan is a {type(plan).__name__}")
    _refuse(what, plan.index, q=q, k=k, positions=positions)
    for name, t in (("q", q),) if k is None else (("q", q), ("k", k)):
        if t.dim() not in (3, 4) or t.shape[-1] != plan.head_dim:
            raise ValueError(f"{what}: {name} of shape {tuple(t.shape)}, expected [(batch,) seq, "
                             f"heads, {plan.head_dim}]")
        if t.dtype not in _DTYPES or t.dtype != q.dtype:
            raise ValueError(f"{what}: {name} is {t.dtype}")
        if t.shape[:-2] != q.shape[:-2]:
            raise ValueError(f"{what}: {name} of shape {tuple(t.shape)} beside q of "
                             f"{tuple(q.shape)}")
        if not 1 <= t.shape[-2] <= 4096:
            raise ValueError(f"{what}: {name} has {t.shape[-2]} heads (1 to 4096)")
    if positions.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{what}: positions are {positions.dtype} (int64 or int32)")
    raise ValueError(f"{what}: positions of shape {tuple(positions.shape)} for tokens of "
                     f"{tuple(q.shape[:-2])}")


def _rope_part(t, shape):
    """(packed b2f_rope_heads, output, input kept alive) of one tensor."""

    st = t.stride()
    if st[-1] != 1:
        t = t.contiguous()
        st = t.stride()
    out = torch.empty_like(t, memory_format=torch.contiguous_format)
    heads, dim = shape[-2], shape[-1]
    row = heads * dim
    return _HEADS.pack(t.data_ptr(), out.data_ptr(), st[0] if len(shape) == 4 else 0, st[-3],
                       st[-2], row * shape[-3], row, dim, heads), out, t


def _rope(what, q, k, positions, plan, gradient):
    if not (type(plan) is RopePlan and _plain_tensor(q, plan.index)
            and _plain_tensor(positions, plan.index)
            and (k is None or _plain_tensor(k, plan.index) and k.dtype is q.dtype)
            and 3 <= q.dim() <= 4 and q.dtype in _DTYPES):
        _rope_refuse(what, q, k, positions, plan)
    if _current_device() != plan.index:
        with torch.cuda.device(plan.index):
            return _rope(what, q, k, positions, plan, gradient)
    shape = tuple(q.shape)
    outer = shape[:-2]
    batch, seq = outer if len(outer) == 2 else (1, outer[0])
    pos = positions.stride()
    wide = positions.dtype is torch.int64
    kshape = shape if k is None else tuple(k.shape)
    if not (wide or positions.dtype is torch.int32) \
            or tuple(positions.shape) not in ((seq,), (batch, seq)) \
            or shape[-1] != plan.head_dim or kshape[-1] != plan.head_dim \
            or kshape[:-2] != outer or not 1 <= shape[-2] <= 4096 or not 1 <= kshape[-2] <= 4096:
        _rope_refuse(what, q, k, positions, plan)
    a = _rope_part(q, shape)
    b = None if k is None else _rope_part(k, kshape)
    if batch and seq:
        rc = lib.b2f_rope(a[0] if b is None else a[0] + b[0], 1 if b is None else 2,
                          _DTYPES[q.dtype], batch, seq, plan.head_dim, plan.rotary_dim,
                          plan.interleaved, positions.data_ptr(), wide,
                          pos[0] if len(pos) == 2 else 0, pos[-1], plan.freqs.data_ptr(),
                          plan.factor, gradient, _raw_stream(plan.index))
        if rc:
            check(rc, what)
    return a[1] if b is None else (a[1], b[1])


def rope(q: torch.Tensor, k: torch.Tensor | None = None, *, positions: torch.Tensor,
         plan: RopePlan):
    """Rotary positions of q, or of q and k in one launch.

    q, k: [seq, heads, head_dim] or [batch, seq, heads, head_dim] (f64, f32, f16
    or bf16; strides free, a last one other than 1 costs a copy), positions
    [seq] or [batch, seq] (int64 or int32).  Returns contiguous tensors.  Angles
    are taken in binary64, products in binary32 (binary64 for f64)."""

    return _rope("rope", q, k, positions, plan, 0)


def rope_grad(grad_q: torch.Tensor, grad_k: torch.Tensor | None = None, *,
              positions: torch.Tensor, plan: RopePlan):
    """The gradient of `rope`: the rotation by the negative angle."""

    return _rope("rope_grad", grad_q, grad_k, positions, plan, 1)


# ---------------------------------------------------------------------------
# matrix-vector products with 4-bit weights
# ---------------------------------------------------------------------------


class Q4Weight:
    """A 4-bit weight [rows, cols] laid out for `q4_matvec` (`pack_q4`,
    `quantize_q4`): scale * (code - zero) per group of columns."""

    def __init__(self, shape, group, packed, scale_dtype, zeros):
        self.shape = (int(shape[0]), int(shape[1]))
        self.group = int(group)
        self.packed = packed  # codes, scales and zero points in records of 16 x 64
        self.scale_dtype = scale_dtype
        self.zeros = bool(zeros)
        self.device, self.index = packed.device, packed.get_device()
        self._args = (_DTYPES[scale_dtype], int(self.zeros), *self.shape, self.group)

    def nbytes(self) -> int:
        return self.packed.numel()


def _group(what: str, group: int, cols: int) -> int:
    group = int(group)
    if group != 32 and (group < 64 or group % 64):
        raise ValueError(f"{what}: groups of {group} columns (32 or a multiple of 64)")
    return -(-cols // group)


def pack_q4(codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None, *,
            group: int = 128) -> Q4Weight:
    """Lay out codes [rows, cols] (uint8, 0..15) with scales and zero points
    (uint8, 0..15; none: 8) [rows, ceil(cols / group)] for `q4_matvec`.  Done
    once per weight: it waits for the device to check the codes."""

    _refuse("pack_q4", None, codes=codes)
    _refuse("pack_q4", codes.get_device(), scales=scales, zeros=zeros)
    if _current_device() != codes.get_device():
        with torch.cuda.device(codes.get_device()):
            return pack_q4(codes, scales, zeros, group=group)
    if codes.dim() != 2 or codes.dtype != torch.uint8 or not codes.numel():
        raise ValueError(f"pack_q4: codes of shape {tuple(codes.shape)}, {codes.dtype}")
    n, k = codes.shape
    groups = _group("pack_q4", group, k)
    if tuple(scales.shape) != (n, groups) or scales.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"pack_q4: scales of shape {tuple(scales.shape)}, {scales.dtype}, "
                         f"expected [{n}, {groups}] in float16 or bfloat16")
    if zeros is not None and (tuple(zeros.shape) != (n, groups) or zeros.dtype != torch.uint8):
        raise ValueError(f"pack_q4: zeros of shape {tuple(zeros.shape)}, {zeros.dtype}")
    for name, t in (("codes", codes), ("zeros", zeros)):
        if t is not None and int(t.max()) > 15:
            raise ValueError(f"pack_q4: {name} above 15")
    codes, scales = codes.contiguous(), scales.contiguous()
    zeros = None if zeros is None else zeros.contiguous()
    packed = torch.empty(lib.b2f_q4_packed_bytes(n, k, int(group), int(zeros is not None)),
                         dtype=torch.uint8, device=codes.device)
    call("b2f_q4_pack", codes.data_ptr(), scales.data_ptr(),
         None if zeros is None else zeros.data_ptr(), n, k, int(group), packed.data_ptr(),
         _raw_stream(codes.get_device()))
    return Q4Weight((n, k), group, packed, scales.dtype, zeros is not None)


def q4_codes(weight: torch.Tensor, *, group: int = 128, symmetric: bool = True,
             scale_dtype: torch.dtype = torch.bfloat16):
    """Codes, scales and zero points (None when symmetric) of a finite weight
    [rows, cols] (f32, f16 or bf16): round to nearest against the stored scale,
    max|w| / 7 of a group, or its range in 15 steps with an integer zero."""

    _refuse("q4_codes", None, weight=weight)
    if _current_device() != weight.get_device():
        with torch.cuda.device(weight.get_device()):
            return q4_codes(weight, group=group, symmetric=symmetric, scale_dtype=scale_dtype)
    dev = weight.device
    if weight.dim() != 2 or not weight.numel() or _DTYPES.get(weight.dtype, 0) == 0:
        raise ValueError(f"q4_codes: weight of shape {tuple(weight.shape)}, {weight.dtype}")
    if scale_dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"q4_codes: scales in {scale_dtype} (float16 or bfloat16)")
    n, k = weight.shape
    groups = _group("q4_codes", group, k)
    w = weight if weight.stride(1) == 1 and weight.stride(0) >= k else weight.contiguous()
    codes = torch.empty((n, k), dtype=torch.uint8, device=dev)
    scales = torch.empty((n, groups), dtype=scale_dtype, device=dev)
    zeros = None if symmetric else torch.empty((n, groups), dtype=torch.uint8, device=dev)
    call("b2f_q4_quantize", w.data_ptr(), _DTYPES[w.dtype], max(w.stride(0), k), n, k,
         int(group), int(bool(symmetric)), _DTYPES[scale_dtype], codes.data_ptr(),
         scales.data_ptr(), None if zeros is None else zeros.data_ptr(),
         _raw_stream(weight.get_device()))
    return codes, scales, zeros


def quantize_q4(weight: torch.Tensor, *, group: int = 128, symmetric: bool = True,
                scale_dtype: torch.dtype = torch.bfloat16) -> Q4Weight:
    """A weight in 4 bits, laid out for `q4_matvec` (`q4_codes` + `pack_q4`)."""

    codes, scales, zeros = q4_codes(weight, group=group, symmetric=symmetric,
                                    scale_dtype=scale_dtype)
    return pack_q4(codes, scales, zeros, group=group)


def q4_matvec(x: torch.Tensor, weight: Q4Weight, *,
              out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """x [..., cols] times the weight's transpose: [..., rows], up to 1024 rows
    of x (f32, f16 or bf16), summed in binary32.  f32 rows, and one or two rows
    of a 16-bit type, may be taken as fixed-point numbers, off by at most 2^-30
    of the largest of their 64 columns.  Returns x's type, or float32 with
    ``out_dtype=torch.float32``."""

    if type(weight) is not Q4Weight:
        raise ValueError(f"q4_matvec: weight is a {type(weight).__name__}")
    if not _plain_tensor(x, weight.index):
        _refuse("q4_matvec", weight.index, x=x)
    if _current_device() != weight.index:
        with torch.cuda.device(weight.index):
            return q4_matvec(x, weight, out_dtype=out_dtype)
    n, k = weight.shape
    shape, dtype = x.shape, x.dtype
    code = _DTYPES.get(dtype, 0)
    if not shape or shape[-1] != k or code == 0:
        raise ValueError(f"q4_matvec: x of shape {tuple(shape)}, {dtype}, for {k} columns")
    if out_dtype is None:
        out_dtype = dtype
    elif out_dtype is not dtype and out_dtype is not torch.float32:
        raise ValueError(f"q4_matvec: output in {out_dtype} for x in {dtype}")
    rows = x.numel() // k
    if rows > 1024:
        raise ValueError(f"q4_matvec: {rows} rows (up to 1024)")
    ld = k
    if not x.is_contiguous():
        x = x if x.dim() == 2 else x.reshape(rows, k)
        if x.stride(1) != 1 and k > 1 or rows > 1 and x.stride(0) < k:
            x = x.contiguous()
        ld = x.stride(0) if rows > 1 else k
    y = x.new_empty((*shape[:-1], n), dtype=out_dtype)
    if rows:
        rc = lib.b2f_q4_matvec(x.data_ptr(), code, ld, rows, weight.packed.data_ptr(),
                               *weight._args, y.data_ptr(),
                               out_dtype is torch.float32, _raw_stream(weight.index))
        if rc:
            check(rc, "q4_matvec")
    return y


# ---------------------------------------------------------------------------
# cross entropy over the vocabulary
# ---------------------------------------------------------------------------


def _rows16(m: torch.Tensor, d: int) -> torch.Tensor:
    """m with rows as the TMA loads read them: contiguous, 16-byte aligned."""

    s0, s1 = m.stride()
    if s1 == 1 and s0 >= d and s0 % 8 == 0 and m.data_ptr() % 16 == 0:
        return m
    return m.clone(memory_format=torch.contiguous_format)


def _loss_args(what, hidden, weight, labels, **more):
    index = hidden.get_device() if isinstance(hidden, torch.Tensor) else -1
    if index < 0 or not (_plain_tensor(hidden, index) and _plain_tensor(weight, index)
                         and _plain_tensor(labels, index)
                         and all(_plain_tensor(t, index) for t in more.values())):
        _refuse(what, None, hidden=hidden)
        _refuse(what, index, weight=weight, labels=labels, **more)
    if hidden.dim() != 2 or weight.dim() != 2 or hidden.shape[1] != weight.shape[1]:
        raise ValueError(f"{what}: hidden of shape {tuple(hidden.shape)}, weight of "
                         f"{tuple(weight.shape)}")
    dtype = hidden.dtype
    if not (dtype is torch.float16 or dtype is torch.bfloat16) or weight.dtype is not dtype:
        raise ValueError(f"{what}: hidden is {dtype}, weight {weight.dtype} (both float16 or "
                         "both bfloat16)")
    t, d = hidden.shape
    v = weight.shape[0]
    if d % 8 or not d or not v:
        raise ValueError(f"{what}: weight of shape {tuple(weight.shape)} (a hidden size that is "
                         "a multiple of 8, at least one word)")
    if labels.dtype is not torch.int64 or labels.dim() != 1 or labels.shape[0] != t:
        raise ValueError(f"{what}: labels of shape {tuple(labels.shape)}, {labels.dtype}, for "
                         f"{t} tokens (int64)")
    for name, x in more.items():
        if x.dtype is not torch.float32 or x.dim() != 1 or x.shape[0] != t:
            raise ValueError(f"{what}: {name} of shape {tuple(x.shape)}, {x.dtype}, for {t} "
                             "tokens (float32)")
    return index, t, v, d


def vocab_loss(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, *,
               ignore_index: int = -100) -> tuple[torch.Tensor, torch.Tensor]:
    """Cross entropy of softmax(hidden @ weight.T) against labels, per token,
    without the logits: (loss [tokens], lse [tokens]) in float32.

    hidden [tokens, D], weight [words, D] (both f16 or both bf16, D a multiple
    of 8; rows off 16-byte boundaries cost a copy), labels int64.  A label of
    ignore_index gives 0 for both; any other label outside the vocabulary gives a
    loss of NaN, as do logits that overflow (and sums that the device did not
    deliver, which `wait_errors` counts)."""

    index, t, v, d = _loss_args("vocab_loss", hidden, weight, labels)
    if _current_device() != index:
        with torch.cuda.device(index):
            return vocab_loss(hidden, weight, labels, ignore_index=ignore_index)
    h, w, lab = _rows16(hidden, d), _rows16(weight, d), labels.contiguous()
    loss = h.new_empty((t,), dtype=torch.float32)
    lse = torch.empty_like(loss)
    if t:
        ws = h.new_empty((lib.b2f_vocab_loss_workspace(t, v, d),), dtype=torch.uint8)
        rc = lib.b2f_vocab_loss(h.data_ptr(), h.stride(0), w.data_ptr(), w.stride(0),
                                _DTYPES[h.dtype], t, v, d, lab.data_ptr(), int(ignore_index),
                                loss.data_ptr(), lse.data_ptr(), ws.data_ptr(), ws.numel(),
                                _raw_stream(index))
        if rc:
            check(rc, "vocab_loss")
    return loss, lse


def vocab_loss_grad(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor,
                    lse: torch.Tensor, grad_loss: torch.Tensor, *, ignore_index: int = -100,
                    need_hidden: bool = True, need_weight: bool = True):
    """The gradient of `vocab_loss` for grad_loss [tokens] (float32), from the
    lse it returned for the same inputs: (grad_hidden, grad_weight) in the
    operands' type, None for one that is not needed.

    The logits are computed again in pieces of the vocabulary, and the softmax's
    gradient is rounded to the operands' type (f16: to no less than 2^-38 of the
    largest |grad_loss|), up to 64 tokens in two parts; from 65 tokens on
    what that leaves at the label still joins both gradients.  Rows of ignored tokens
    contribute nothing and get zero, whatever they hold; so do tokens under a
    grad_loss of zero whose hidden state is finite."""

    index, t, v, d = _loss_args("vocab_loss_grad", hidden, weight, labels, lse=lse,
                                grad_loss=grad_loss)
    if not (need_hidden or need_weight):
        raise ValueError("vocab_loss_grad: no gradient asked for")
    if _current_device() != index:
        with torch.cuda.device(index):
            return vocab_loss_grad(hidden, weight, labels, lse, grad_loss,
                                   ignore_index=ignore_index, need_hidden=need_hidden,
                                   need_weight=need_weight)
    h, w, lab = _rows16(hidden, d), _rows16(weight, d), labels.contiguous()
    lse, g = lse.contiguous(), grad_loss.contiguous()
    like = torch.contiguous_format
    dh = torch.empty_like(h, memory_format=like) if need_hidden else None
    dw = torch.empty_like(w, memory_format=like) if need_weight else None
    ws = h.new_empty((max(lib.b2f_vocab_loss_grad_workspace(t, v, d, bool(need_hidden)), 16),),
                     dtype=torch.uint8)
    rc = lib.b2f_vocab_loss_grad(h.data_ptr(), h.stride(0), w.data_ptr(), w.stride(0),
                                 _DTYPES[h.dtype], t, v, d, lab.data_ptr(), int(ignore_index),
                                 lse.data_ptr(), g.data_ptr(),
                                 None if dh is None else dh.data_ptr(),
                                 None if dw is None else dw.data_ptr(), ws.data_ptr(),
                                 ws.numel(), _raw_stream(index))
    if rc:
        check(rc, "vocab_loss_grad")
    return dh, dw


def wait_errors(device: str | torch.device | None = None) -> int:
    """How many waits inside `vocab_loss` and `vocab_loss_grad` ran out on a device
    (the current one) since the library was loaded: 0 on a healthy device.  What was
    waited for is NaN in their results.  Waits for the device."""

    with torch.cuda.device(device):
        torch.cuda.synchronize()
        count = lib.b2f_vocab_loss_wait_errors()
    if count < 0:
        raise RuntimeError("wait_errors: the device's counter cannot be read")
    return count
