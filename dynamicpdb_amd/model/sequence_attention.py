"""Operators of sequence tracks: attention of one sequence over another (or itself) with grouped heads, masked keys and a learned
bucketed relative position bias; that bias as a matrix; and the norm of query / key heads with the position rotation in the same
pass.  Each has its backward pass; attention has a form for few queries over many keys (the key axis cut over workgroups).  The
arithmetic runs in libdfold_hip.so (csrc/seq_attn_fwd.hip, seq_attn_bwd.hip, seq_relpos.hip, seq_norm_rope.hip): bf16 / fp16 operands
on the matrix pipes with fp32 softmax statistics and accumulators, results independent of the order of workgroups.

    q, k = qk_norm_rope(q, k, w_q, w_k, q_positions, k_positions)
    o = cross_attention(q, k, v, kv_lens=lens, rel_table=table)
    bias = relative_position_bias(table, n_queries, n_keys)

Device tensors only (no CPU fallback).  Nothing is kept between calls; workspaces come from torch's allocator, so the calls may be
recorded into a graph and run on any stream or device (the device of the tensors, its current stream)."""
import ctypes
import functools
import math
import struct
from ctypes import c_double, c_float, c_int16, c_int32, c_int64, c_void_p

import torch
import torch.nn as nn
from torch.autograd import Function, forward_ad
from torch.autograd.function import once_differentiable

from .. import _lib, ops
from .._lib import check
from ..ops import BF16
from .functional import linear

F16, F32 = torch.float16, torch.float32
DTYPES = {BF16: 0, F16: 1, F32: 2}                                    # DFOLD_DT_*
REL_FAR, REL_MAX_DISTANCE = 256, 1024                                 # DFOLD_REL_*
MAX_OFFSET, MAX_LEN, MAX_ROW = 1 << 29, 1 << 30, 1 << 24
MIN_SCALE = 2.0 ** -120                                               # what the kernels form of a scale stays a normal fp32 number
MAX_EPS = torch.finfo(F32).max
ROWS, TILE = 128, 64                                                  # softmax rows / keys of a workgroup, rows of an LDS tile

# The C ABI's descriptors as struct formats: one pack per call (filling ctypes structures field by field costs as much host time as the
# launch).  The classes give names to the same layouts.


class RelBias(ctypes.Structure):
    _fields_ = [("table", c_void_p), ("q_offsets", c_void_p), ("q_offset", c_int32), ("num_buckets", c_int32), ("bidirectional", c_int32),
                ("reserved", c_int32), ("far_border", c_int16 * REL_FAR)]


class AttnDesc(ctypes.Structure):
    _fields_ = ([(n, c_void_p) for n in ("q", "k", "v", "o", "lse", "ws", "key_mask", "kv_lens")] +
                [(n, c_int64) for n in ("q_sb", "q_sl", "q_sh", "k_sb", "k_sl", "k_sh", "v_sb", "v_sl", "v_sh", "o_sb", "o_sl", "o_sh", "mask_sb")] +
                [(n, c_int32) for n in ("dtype", "B", "Lq", "Lk", "H", "Hkv", "D", "splits", "pack", "pair")] + [("scale", c_float), ("rel", RelBias)])


class AttnGrad(ctypes.Structure):
    _fields_ = [("d_o", c_void_p), ("do_sb", c_int64), ("do_sl", c_int64), ("do_sh", c_int64), ("dq", c_void_p), ("dk", c_void_p),
                ("dv", c_void_p), ("delta", c_void_p), ("dtable", c_void_p), ("ws", c_void_p), ("splits_q", c_int32), ("splits_k", c_int32), ("pair_q", c_int32), ("pair_k", c_int32)]


class RopePart(ctypes.Structure):
    _fields_ = ([(n, c_void_p) for n in ("x", "y", "g", "w", "dw", "pos")] +
                [(n, c_int64) for n in ("x_sb", "x_sl", "x_sh", "g_sb", "g_sl", "g_sh", "pos_sb")] + [("L", c_int32), ("H", c_int32)])


class RopeDesc(ctypes.Structure):
    _fields_ = [("part", RopePart * 2), ("ws", c_void_p), ("base", c_double), ("eps", c_float), ("dtype", c_int32), ("B", c_int32),
                ("D", c_int32), ("rotary_dim", c_int32), ("interleaved", c_int32)]


_REL = struct.Struct(f"@2P4i{2 * REL_FAR}s")
_ATTN = struct.Struct("@8P13q10if4x")
_GRAD = struct.Struct("@P3q6P4i")
_PART = struct.Struct("@6P7q2i")
_ROPE = struct.Struct("@Pdf5i")
_NO_REL = bytes(_REL.size)
_NO_PART = bytes(_PART.size)


# ------------------------------------------------------------------------------------------------
# argument helpers
# ------------------------------------------------------------------------------------------------

def _call(name, *args, t):
    """one C ABI call on the current stream of t's device.  Arguments: a descriptor's bytes, pointers as c_void_p, whole numbers."""
    dev = t.get_device()
    fn = getattr(_lib.lib(), name)
    if dev == torch._C._cuda_getDevice():
        check(fn(*args, c_void_p(torch._C._cuda_getCurrentRawStream(dev))), name)
    else:                                       # (launches go to the current device)
        with torch.cuda.device(dev):
            check(fn(*args, c_void_p(torch._C._cuda_getCurrentRawStream(dev))), name)


def _require_cuda(t):
    if not t.is_cuda:
        raise RuntimeError("dynamicpdb_amd sequence operators need an MI355X device tensor (no CPU fallback)")


def _same_device(dev, name, t):
    """dev: the device's number (-1: the CPU)"""
    if t.get_device() != dev:
        raise ValueError(f"{name} is on {t.device}, expected {'cpu' if dev < 0 else f'cuda:{dev}'}")


def _rows16(t):
    """t itself if the kernels can read it as it lies -- dense last axis, every other stride a multiple of 16 bytes, rows less than
    2^24 elements apart, aligned base -- else a dense copy"""
    aligned = t.data_ptr() % 16 == 0
    if aligned and t.is_contiguous():           # (a multiple of 16 bytes per row: the head size is checked)
        return t
    v = 16 // t.element_size()
    if t.numel() == 0 or (aligned and t.stride(-1) == 1 and all(s % v == 0 for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1) and
                          (t.shape[1] == 1 or t.stride(1) < MAX_ROW)):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _strides(t):
    """strides of the three leading axes, 0 for axes of one entry (theirs may be anything, also in a tensor that is dense for torch)"""
    a, b, c, _ = t.stride()
    n0, n1, n2, _ = t.shape
    if n0 > 1 and n1 > 1 and n2 > 1:
        return a, b, c
    if n1 == 0:
        return 0, 0, 0
    return a if n0 > 1 else 0, b if n1 > 1 else 0, c if n2 > 1 else 0


def _dense_like(t):
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _addr(t):
    return 0 if t is None else t.data_ptr()


def _mask_bytes(mask):
    """[B, Lk] mask as bytes that are 0 where a key is masked; dense rows"""
    if mask.dtype == torch.bool:
        mask = mask.view(torch.uint8)
    elif mask.dtype != torch.uint8:
        mask = (mask != 0).view(torch.uint8)
    return mask if mask.stride(-1) == 1 or mask.shape[-1] == 1 else mask.contiguous()


@functools.lru_cache(maxsize=None)
def far_borders(num_buckets, max_distance, bidirectional):
    """First distance of each bucket beyond the ones of a single distance.  With half buckets per side, e = half // 2 and m = half - e,
    bucket e + k starts at the first whole n with log(n / e) / log(max_distance / e) * m >= k, i.e. n^m e^k >= e^m max_distance^k:
    decided in whole numbers, so that a distance that lies exactly on a border falls into its bucket whatever a logarithm rounds to."""
    half = num_buckets // 2 if bidirectional else num_buckets
    e = half // 2
    m = half - e
    out, n = [], e
    for k in range(1, m):
        rhs = e ** m * max_distance ** k
        while n ** m * e ** k < rhs:
            n += 1
        out.append(n)
    return tuple(out)


@functools.lru_cache(maxsize=None)
def _border_bytes(num_buckets, max_distance, bidirectional):
    far = far_borders(num_buckets, max_distance, bidirectional)
    return struct.pack(f"@{REL_FAR}h", *far, *([0] * (REL_FAR - len(far))))


def _reach(num_buckets, max_distance, bidirectional):
    """distance from which on a side's last bucket holds everything"""
    far = far_borders(num_buckets, max_distance, bidirectional)
    return far[-1] if far else (num_buckets // 2 if bidirectional else num_buckets) // 2


def _check_rel(table, max_distance, bidirectional):
    if table.dim() != 2 or table.dtype != F32:
        raise ValueError("the bias table must be fp32 [num_buckets, heads]")
    nb = table.shape[0]
    half = nb // 2 if bidirectional else nb
    if bidirectional and nb % 2:
        raise ValueError("num_buckets must be even for a bidirectional bias")
    if not 2 <= half <= REL_FAR:
        raise ValueError(f"num_buckets must be between 2 and {REL_FAR} per direction")
    if not isinstance(max_distance, int) or not half // 2 < max_distance <= REL_MAX_DISTANCE:
        raise ValueError(f"max_distance must be a whole number above num_buckets' single distances ({half // 2}) and at most {REL_MAX_DISTANCE}")


def _rel_desc(table, num_buckets, max_distance, bidirectional, q_offset, q_offsets=None):
    return _REL.pack(table.data_ptr(), _addr(q_offsets), q_offset, num_buckets, bidirectional, 0, _border_bytes(num_buckets, max_distance, bidirectional))


def _once(fn):
    """once_differentiable, whose bookkeeping only a pass that builds a graph of the gradients needs"""
    guarded = once_differentiable(fn)
    return lambda ctx, *g: guarded(ctx, *g) if torch.is_grad_enabled() else fn(ctx, *g)


def _needs_node(grad):
    """whether a call goes through its autograd node: an input takes a gradient (grad), or may carry a forward-mode tangent (the node has
    no derivative for that and raises), or the call is traced (the node is recorded).  The bare call would give, or record, a result
    without its derivative or its launch."""
    return (grad and torch.is_grad_enabled()) or forward_ad._current_level >= 0 or torch._C._get_tracing_state() is not None


# ------------------------------------------------------------------------------------------------
# relative position bias as a matrix
# ------------------------------------------------------------------------------------------------

def _bias_forward(table, q_len, k_len, max_distance, bidirectional, q_offset, dtype):
    t = table if table.is_contiguous() else table.contiguous()
    nb, H = t.shape
    out = torch.empty((H, q_len, k_len), dtype=dtype, device=t.device)
    if q_len and k_len:
        _call("dfold_relpos_fwd", _rel_desc(t, nb, max_distance, bidirectional, q_offset), c_void_p(out.data_ptr()), DTYPES[dtype], H, q_len, k_len, t=t)
    return out


class RelativeBiasFn(Function):
    @staticmethod
    def forward(ctx, table, *args):
        ctx.args, ctx.table_shape = args, table.shape
        return _bias_forward(table, *args)

    @staticmethod
    @_once
    def backward(ctx, g):
        q_len, k_len, max_distance, bidirectional, q_offset, dtype = ctx.args
        nb, H = ctx.table_shape
        dev = g.device
        if g.numel() == 0:
            return (torch.zeros((nb, H), dtype=F32, device=dev),) + (None,) * 6
        if not g.is_contiguous() or g.data_ptr() % 16:
            g = g.clone(memory_format=torch.contiguous_format)
        dtable = torch.empty((nb, H), dtype=F32, device=dev)
        n = _lib.lib().dfold_relpos_ws(H, q_len, nb)
        if n <= 0:
            raise ValueError("relative_position_bias: too many heads x buckets")
        ws = torch.empty(n, dtype=F32, device=dev)
        # (the backward reads the borders, not the entries)
        _call("dfold_relpos_bwd", _rel_desc(dtable, nb, max_distance, bidirectional, q_offset), c_void_p(g.data_ptr()), DTYPES[dtype], H, q_len, k_len,
              c_void_p(dtable.data_ptr()), c_void_p(ws.data_ptr()), t=g)
        return (dtable,) + (None,) * 6


def relative_position_bias(table, q_len, k_len, *, max_distance=128, bidirectional=True, q_offset=0, dtype=torch.float32):
    """[heads, q_len, k_len] bias of query i and key j: table[bucket(j - i - q_offset), head], differentiable in the table.

    table fp32 [num_buckets, heads].  Of the half = num_buckets / 2 buckets per direction (bidirectional; distances > 0 use the second
    half; else half = num_buckets and keys behind the query count as distance 0) the first half // 2 hold one distance each, the others
    grow logarithmically up to max_distance, beyond which everything shares the last.  dtype: fp32, bf16 or fp16 of the result."""
    _check_rel(table, max_distance, bidirectional)
    if not (isinstance(q_len, int) and isinstance(k_len, int) and 0 <= q_len <= MAX_LEN and 0 <= k_len <= 1 << 28):
        raise ValueError("q_len, k_len must be whole numbers >= 0, k_len at most 2^28")
    if not isinstance(q_offset, int) or abs(q_offset) > MAX_OFFSET:
        raise ValueError(f"q_offset must be a whole number, at most {MAX_OFFSET}")
    if dtype not in DTYPES:
        raise ValueError("dtype must be float32, bfloat16 or float16")
    if not 1 <= table.shape[1] <= 65535:
        raise ValueError("the table needs between 1 and 65535 heads")
    _require_cuda(table)
    args = (table, q_len, k_len, max_distance, bool(bidirectional), q_offset, dtype)
    if _needs_node(table.requires_grad):
        return RelativeBiasFn.apply(*args)
    return _bias_forward(*args)


class RelativePositionBias(nn.Module):
    """Learned bias table [num_buckets, no_heads]; forward(q_len, k_len, q_offset) gives the matrix, `table` goes into
    cross_attention(rel_table=...), which never forms it."""

    def __init__(self, num_buckets, no_heads, max_distance=128, bidirectional=True):
        super().__init__()
        self.max_distance, self.bidirectional = max_distance, bidirectional
        self.table = nn.Parameter(torch.zeros(num_buckets, no_heads))
        _check_rel(self.table, max_distance, bidirectional)

    def forward(self, q_len, k_len, q_offset=0, dtype=torch.float32):
        return relative_position_bias(self.table, q_len, k_len, max_distance=self.max_distance, bidirectional=self.bidirectional,
                                      q_offset=q_offset, dtype=dtype)


# ------------------------------------------------------------------------------------------------
# norm + rotation of query and key heads
# ------------------------------------------------------------------------------------------------

def _rope_part(x, y, w, pos, g=None, dw=None):
    if x is None or x.numel() == 0:
        return _NO_PART
    _, L, H, _ = x.shape
    pos_sb = 0 if pos is None or pos.shape[0] == 1 else pos.stride(0)
    return _PART.pack(x.data_ptr(), y.data_ptr(), _addr(g), _addr(w), _addr(dw), _addr(pos), *_strides(x), *(_strides(g) if g is not None else (0, 0, 0)),
                      pos_sb, L, H)


def _rope_desc(parts, ref, opts, ws=None):
    rotary_dim, base, interleaved, eps = opts
    return parts[0] + parts[1] + _ROPE.pack(_addr(ws), base, eps, DTYPES[ref.dtype], ref.shape[0], ref.shape[3], rotary_dim, interleaved)


def _rope_forward(q, k, w_q, w_k, q_pos, k_pos, *opts):
    """results and the (readable) inputs they were computed from"""
    oq = ok = None
    part_q = part_k = _NO_PART
    if q is not None:
        q = _rows16(q)
        oq = _dense_like(q)
        part_q = _rope_part(q, oq, w_q, q_pos)
    if k is not None:
        k = _rows16(k)
        ok = _dense_like(k)
        part_k = _rope_part(k, ok, w_k, k_pos)
    if part_q is not _NO_PART or part_k is not _NO_PART:
        ref = q if q is not None else k
        _call("dfold_qk_norm_rope_fwd", _rope_desc((part_q, part_k), ref, opts), t=ref)
    return oq, ok, (q, k, w_q, w_k, q_pos, k_pos)


class QKNormRopeFn(Function):
    @staticmethod
    def forward(ctx, *args):
        oq, ok, saved = _rope_forward(*args)
        ctx.opts = args[6:]
        ctx.save_for_backward(*saved)
        return oq, ok

    @staticmethod
    @_once
    def backward(ctx, gq, gk):
        q, k, w_q, w_k, q_pos, k_pos = ctx.saved_tensors
        ref = q if q is not None else k
        grads, parts, ws = [None] * 4, [], None
        gq, gk = (None if x is None else _rows16(g) for x, g in ((q, gq), (k, gk)))      # (copies live until the launch)
        for i, (x, w, pos, g) in enumerate(((q, w_q, q_pos, gq), (k, w_k, k_pos, gk))):
            if x is None:
                parts.append(_NO_PART)
                continue
            dx = grads[i] = _dense_like(x)
            dw = None
            if w is not None and ctx.needs_input_grad[2 + i]:
                dw = grads[2 + i] = torch.empty_like(w) if x.numel() else torch.zeros_like(w)
                if ws is None:
                    ws = torch.empty(_lib.lib().dfold_qk_norm_rope_ws(), dtype=F32, device=ref.device)
            parts.append(_rope_part(x, dx, w, pos, g, dw))
        if parts != [_NO_PART, _NO_PART]:
            _call("dfold_qk_norm_rope_bwd", _rope_desc(parts, ref, ctx.opts, ws), t=ref)
        return (*grads, None, None, None, None, None, None)


def _positions(pos, x, dev, name):
    if pos is None or x is None:
        return None
    _same_device(dev, name, pos)
    if pos.dtype != torch.int64:
        if pos.dtype != torch.int32:
            raise ValueError(f"{name} must be int64 or int32")
        pos = pos.long()
    if pos.dim() == 1:
        pos = pos[None]
    B, L = x.shape[:2]
    if pos.dim() != 2 or pos.shape[0] not in (1, B) or pos.shape[1] != L:
        raise ValueError(f"{name} must be [{L}] or [{B}, {L}]")
    return pos if L <= 1 or pos.stride(1) == 1 else pos.contiguous()


def _heads(t, dt, name):
    if t.dim() != 4 or t.dtype is not dt:
        raise ValueError(f"{name} must be [B, L, heads, D], q and k of one type")


def _head_weight(w, D, dev, name):
    _same_device(dev, name, w)
    if w.dtype is not F32 or w.dim() != 1 or w.shape[0] != D:
        raise ValueError(f"{name} must be fp32 [{D}]")
    return w if w.is_contiguous() else w.contiguous()


def qk_norm_rope(q, k, w_q=None, w_k=None, q_positions=None, k_positions=None, *, rotary_dim=None, base=10000.0, interleaved=False, eps=1e-6):
    """Every head of q [B, Lq, H, D] and k [B, Lk, Hkv, D] divided by its root mean square, times w (fp32 [D] or None), then its first
    rotary_dim dimensions (default: all; a multiple of 16; 0: none) rotated by position * base^(-2 i / rotary_dim): pairs
    (i, i + rotary_dim / 2), or (2 i, 2 i + 1) if interleaved.  k may be None (keys that are rotated already).  Positions: int64 / int32
    [L] or [B, L], default 0, 1, ...; angles are reduced in fp64 (right to fp32 rounding up to positions of 2^28).  bf16, fp16 or fp32;
    one launch for q and k; differentiable (once) in q, k, w_q, w_k."""
    ref = q if q is not None else k
    if ref is None:
        raise ValueError("qk_norm_rope needs q or k")
    dt, dev = ref.dtype, ref.get_device()
    if dt not in DTYPES:
        raise ValueError("q, k must be bfloat16, float16 or float32")
    _heads(ref, dt, "q" if q is not None else "k")
    B, _, _, D = ref.shape
    if k is not None and k is not ref:
        _heads(k, dt, "k")
        _same_device(dev, "k", k)
        if k.shape[0] != B or k.shape[3] != D:
            raise ValueError("q and k differ in batch or head size")
    if D % 8 or not 8 <= D <= 256:
        raise ValueError("the head size must be a multiple of 8, at most 256")
    if rotary_dim is None:
        if D % 16:
            raise ValueError("this head size is not a multiple of 16: give rotary_dim")
        rotary_dim = D
    if not isinstance(rotary_dim, int) or not 0 <= rotary_dim <= D or rotary_dim % 16:
        raise ValueError("rotary_dim must be a multiple of 16, at most the head size")
    if not (0 < base < math.inf and 0 <= eps <= MAX_EPS):
        raise ValueError("base must be positive and finite, eps not negative and within fp32")
    grad = ref.requires_grad or (k is not None and k.requires_grad)
    if w_q is not None:
        w_q = _head_weight(w_q, D, dev, "w_q")
        grad = grad or w_q.requires_grad
    if w_k is not None:
        w_k = _head_weight(w_k, D, dev, "w_k")
        grad = grad or w_k.requires_grad
    q_positions, k_positions = _positions(q_positions, q, dev, "q_positions"), _positions(k_positions, k, dev, "k_positions")
    _require_cuda(ref)
    args = (q, k, w_q, w_k, q_positions, k_positions, rotary_dim, float(base), bool(interleaved), float(eps))
    if _needs_node(grad):
        return QKNormRopeFn.apply(*args)
    return _rope_forward(*args)[:2]


# ------------------------------------------------------------------------------------------------
# attention of one sequence over another
# ------------------------------------------------------------------------------------------------

_PARTS = (1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, 128, 192, 256, 384, 512, 768, 1024)


def _parts(groups, units, n_cu, join, alone=False):
    """Cut factor of a launch of `groups` workgroups that each walk `units` tiles.  Estimated in tile times: the longest part, times the
    rounds that w = workgroups per CU make (two share a CU, each at two thirds of its speed; `alone`: a workgroup fills its CU), plus
    `join` for writing and adding the parts.  Measured against it, us: 94 tiles of 8 groups: 102 whole, 14.4 in 24 parts, 13.9 in 32,
    15.4 in 47; 16 tiles of 256 groups: 24 whole, 28 in 2; 256 tiles of 128 groups, ragged: 161 in 4, 178 in 6."""
    best, best_cost = 1, None
    for parts in _PARTS:
        if parts > max(units, 1):
            break
        w = groups * parts / n_cu
        rounds = math.ceil(w) if alone else 1.5 * (w // 2) + (0.0 if w % 2 == 0 else 1.0 if w % 2 <= 1 else 1.5)
        cost = -(-units // parts) * max(rounds, 1.0) + (join if parts > 1 else 0)
        if best_cost is None or cost * 1.05 < best_cost:
            best, best_cost = parts, cost
    return best


def _pair(workgroups, tiles, n_cu):
    """Two waves per 32 rows (keys) where a launch would otherwise leave SIMDs with a single wave and a workgroup walks enough tiles to pay
    for the join.  One against two, us: D = 64, 64 workgroups of 64 tiles 67 / 52 (forward), 76 / 60 (dQ); 256 of 16 tiles 23.5 / 20.8,
    29.0 / 26.2; D = 32, 256 of 8 tiles 10.1 / 10.2, 12.7 / 12.2; a token, 3 tiles 10.3 / 10.8."""
    return int(workgroups <= n_cu and tiles >= 12)


@functools.lru_cache(maxsize=4096)
def _attn_plan(B, Lq, Lk, H, Hkv, rel_width, n_cu):
    """(pack, splits, pair) of the forward.  pack: the query heads of a group share tiles if that at least halves the number of row blocks
    (their bias rows have to fit 32 KB of LDS); K and V are then read once per group."""
    G = H // Hkv
    blocks, packed = -(-Lq // ROWS) * G, -(-(Lq * G) // ROWS)
    pack = G if 2 * packed <= blocks and G * rel_width * 4 <= 32768 else 1
    groups = B * (H // pack) * -(-(Lq * pack) // ROWS)
    parts = _parts(groups, -(-Lk // TILE), n_cu, 5)
    return pack, parts, _pair(groups * parts, -(-Lk // TILE) // parts, n_cu)


@functools.lru_cache(maxsize=4096)
def _grad_plan(B, Lq, Lk, H, Hkv, D, num_buckets, n_cu):
    """(splits_q, splits_k, pair_q, pair_k, floats of delta, floats of delta and workspace) of the backward"""
    nrb, nkb = -(-Lq // ROWS), -(-Lk // ROWS)
    splits_q = _parts(B * H * nrb, -(-Lk // TILE), n_cu, 6)
    splits_k = _parts(B * Hkv * nkb, (H // Hkv) * -(-Lq // TILE), n_cu, 6, alone=D > 64)
    delta = (B * H * Lq * (1 + splits_q if splits_q > 1 else 1) + 3) // 4 * 4
    ws = (splits_q * B * Lq * H * D if splits_q > 1 else 0) + (2 * splits_k * B * Lk * Hkv * D if splits_k > 1 else 0)
    return (splits_q, splits_k, _pair(B * H * nrb * splits_q, -(-Lk // TILE) // splits_q, n_cu),
            _pair(B * Hkv * nkb * splits_k, (H // Hkv) * -(-Lq // TILE) // splits_k, n_cu), delta,
            delta + ws + splits_k * B * H * nkb * num_buckets)


def _attn_desc(q, k, v, o, lse, ws, key_mask, kv_lens, rel, scale, pack=1, splits=1, pair=0):
    B, Lq, H, D = q.shape
    mask_sb = 0 if key_mask is None or B == 1 else key_mask.stride(0)
    return _ATTN.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), _addr(lse), _addr(ws), _addr(key_mask), _addr(kv_lens), *_strides(q),
                      *_strides(k), *_strides(v), *_strides(o), mask_sb, DTYPES[q.dtype], B, Lq, k.shape[1], H, k.shape[2], D, splits, pack, pair, scale) + rel


def _attn_forward(train, q, k, v, table, key_mask, kv_lens, q_offsets, q_offset, max_distance, bidirectional, scale):
    """the result and what a backward pass needs"""
    q, k, v = _rows16(q), _rows16(k), _rows16(v)
    B, Lq, H, D = q.shape
    Lk, Hkv = k.shape[1], k.shape[2]
    dev = q.device
    o = _dense_like(q)
    lse = torch.empty((2, B, H, Lq), dtype=F32, device=dev) if train else None
    if table is not None and not table.is_contiguous():
        table = table.contiguous()
    if B and Lq:
        rel, width = _NO_REL, 0
        if table is not None:
            nb = table.shape[0]
            rel = _rel_desc(table, nb, max_distance, bidirectional, q_offset, q_offsets)
            width = 2 * _reach(nb, max_distance, bidirectional) + 1
        pack, splits, pair = _attn_plan(B, Lq, Lk, H, Hkv, width, ops.cu_count(dev))
        ws = torch.empty(splits * B * H * Lq * (D + 2), dtype=F32, device=dev) if splits > 1 else None
        _call("dfold_seq_attn_fwd", _attn_desc(q, k, v, o, lse, ws, key_mask, kv_lens, rel, scale, pack, splits, pair), t=q)
    return o, (q, k, v, table, key_mask, kv_lens, q_offsets, o, lse)


class CrossAttentionFn(Function):
    @staticmethod
    def forward(ctx, *args):
        o, saved = _attn_forward(True, *args)
        ctx.opts = args[7:]
        ctx.save_for_backward(*saved)
        return o

    @staticmethod
    @_once
    def backward(ctx, g):
        q, k, v, table, key_mask, kv_lens, q_offsets, o, lse = ctx.saved_tensors
        q_offset, max_distance, bidirectional, scale = ctx.opts
        B, Lq, H, D = q.shape
        Lk, Hkv = k.shape[1], k.shape[2]
        dtable = None
        if o.numel() == 0 or k.numel() == 0:
            dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
            if table is not None:
                dtable = torch.zeros_like(table)
        else:
            g = _rows16(g)
            dq, dk, dv = _dense_like(q), _dense_like(k), _dense_like(v)
            rel, nb = _NO_REL, 0
            if table is not None:
                dtable, nb = torch.empty_like(table), table.shape[0]
                rel = _rel_desc(table, nb, max_distance, bidirectional, q_offset, q_offsets)
            splits_q, splits_k, pair_q, pair_k, n_delta, n = _grad_plan(B, Lq, Lk, H, Hkv, D, nb, ops.cu_count(q.device))
            ws = torch.empty(n, dtype=F32, device=q.device)          # delta, then the workspace
            delta = ws.data_ptr()
            grad = _GRAD.pack(g.data_ptr(), *_strides(g), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), delta, _addr(dtable), delta + 4 * n_delta,
                              splits_q, splits_k, pair_q, pair_k)
            _call("dfold_seq_attn_bwd", _attn_desc(q, k, v, o, lse, None, key_mask, kv_lens, rel, scale), grad, t=q)
        need = ctx.needs_input_grad
        return (dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, dtable if need[3] else None) + (None,) * 7


def cross_attention(q, k, v, *, key_mask=None, kv_lens=None, rel_table=None, max_distance=128, bidirectional=True, q_offset=0, scale=None):
    """softmax(scale q k^T + bias) v of q [B, Lq, H, D] over k, v [B, Lk, Hkv, D] (H a multiple of Hkv: query head h reads key head
    h // (H / Hkv)), bf16 or fp16, D a multiple of 8 up to 128; any strides (a copy is made where rows are not 16-byte aligned).

    key_mask [B, Lk] (bool, or 0 / 1 in any type) and kv_lens [B] (int32 / int64: keys j < kv_lens[b] exist) remove keys: what K and V
    hold there is never used, gradients there are zero.  A query without any key gives zeros and takes no gradient.  rel_table fp32
    [num_buckets, H] adds the bias of relative_position_bias without forming it; q_offset: position of query 0 minus position of key 0, a
    whole number or an int32 / int64 tensor [B] (one token at its own position per sequence).  scale defaults to D^-1/2 (2^-120 to 2^120
    in magnitude, either sign).
    Differentiable (once) in q, k, v and rel_table; repeated calls give the same bits.  P and dS are rounded to the operand type between
    the products (an fp16 dS beyond 65504 in units of a power of two that holds it; one below 2^-25 is 0: scale an fp16 loss)."""
    dt, dev = q.dtype, q.get_device()
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError("q must be [B, Lq, H, D], k and v [B, Lk, Hkv, D]")
    if (dt is not BF16 and dt is not F16) or k.dtype is not dt or v.dtype is not dt:
        raise ValueError("q, k, v must all be bfloat16 or all float16")
    B, Lq, H, D = q.shape
    Bk, Lk, Hkv, Dk = k.shape
    if k.shape != v.shape or Bk != B or Dk != D:
        raise ValueError("k and v must be [B, Lk, Hkv, D] with q's B and D")
    if not (H > 0 and Hkv > 0) or H % Hkv:
        raise ValueError("the query heads must be a multiple of the key heads")
    if D % 8 or not 8 <= D <= 128:
        raise ValueError("the head size must be a multiple of 8, at most 128")
    if Lq > MAX_LEN or Lk > MAX_LEN or H * D >= MAX_ROW:
        raise ValueError("sequences are at most 2^30 long, rows (heads x head size) below 2^24")
    _same_device(dev, "k", k)
    _same_device(dev, "v", v)
    if key_mask is not None:
        _same_device(dev, "key_mask", key_mask)
        if key_mask.shape != (B, Lk):
            raise ValueError(f"key_mask must be [{B}, {Lk}]")
        key_mask = _mask_bytes(key_mask)
    if kv_lens is not None:
        _same_device(dev, "kv_lens", kv_lens)
        if kv_lens.dim() != 1 or kv_lens.shape[0] != B or (kv_lens.dtype is not torch.int32 and kv_lens.dtype is not torch.int64):
            raise ValueError(f"kv_lens must be int32 or int64 [{B}]")
        if kv_lens.dtype is torch.int64:
            kv_lens = kv_lens.clamp(0, Lk).int()
        kv_lens = kv_lens.contiguous()
    q_offsets = None
    if rel_table is not None:
        _same_device(dev, "rel_table", rel_table)
        _check_rel(rel_table, max_distance, bidirectional)
        if rel_table.shape[1] != H:
            raise ValueError(f"rel_table must have {H} columns, one per query head")
        if torch.is_tensor(q_offset):
            _same_device(dev, "q_offset", q_offset)
            if q_offset.shape != (B,) or q_offset.dtype not in (torch.int32, torch.int64):
                raise ValueError(f"q_offset must be a whole number or int32 / int64 [{B}]")
            q_offsets = (q_offset.clamp(-MAX_OFFSET, MAX_OFFSET).int() if q_offset.dtype == torch.int64 else q_offset).contiguous()
            q_offset = 0
        elif not isinstance(q_offset, int) or abs(q_offset) > MAX_OFFSET:
            raise ValueError(f"q_offset must be a whole number, at most {MAX_OFFSET}")
    else:
        q_offset = 0
    scale = D ** -0.5 if scale is None else float(scale)
    if not MIN_SCALE <= abs(scale) <= 1 / MIN_SCALE:
        raise ValueError("scale must be between 2^-120 and 2^120 in magnitude")
    _require_cuda(q)
    args = (q, k, v, rel_table, key_mask, kv_lens, q_offsets, q_offset, max_distance, bool(bidirectional), scale)
    if _needs_node(q.requires_grad or k.requires_grad or v.requires_grad or (rel_table is not None and rel_table.requires_grad)):
        return CrossAttentionFn.apply(*args)
    return _attn_forward(False, *args)[0]


class CrossAttention(nn.Module):
    """Multi-head attention of x [B, Lq, c_q] over context [B, Lk, c_kv] (or of x over itself): projections on the MFMA engine, optional
    norm of the heads, rotation and relative position bias, output projection.  Weights fp32, arithmetic bf16 like the other modules;
    the result has x's type."""

    def __init__(self, c_q, c_kv, c_hidden, no_heads, no_kv_heads=None, qk_norm=True, rotary_dim=0, rotary_base=10000.0, num_buckets=0,
                 max_distance=128, bidirectional=True):
        super().__init__()
        no_kv_heads = no_kv_heads or no_heads
        if c_q % 8 or c_kv % 8 or c_hidden % 8 or c_hidden > 128 or no_heads % no_kv_heads:
            raise ValueError("c_q, c_kv, c_hidden must be multiples of 8 (c_hidden <= 128), no_heads a multiple of no_kv_heads")
        if rotary_dim and not qk_norm:
            raise ValueError("the rotation comes with the norm of the heads: rotary_dim needs qk_norm")
        self.c_hidden, self.no_heads, self.no_kv_heads = c_hidden, no_heads, no_kv_heads
        self.qk_norm, self.rotary_dim, self.rotary_base = qk_norm, rotary_dim, rotary_base
        self.linear_q = nn.Linear(c_q, no_heads * c_hidden, bias=False)
        self.linear_kv = nn.Linear(c_kv, 2 * no_kv_heads * c_hidden, bias=False)
        self.linear_o = nn.Linear(no_heads * c_hidden, c_q)
        if qk_norm:
            self.q_norm = nn.Parameter(torch.ones(c_hidden))
            self.k_norm = nn.Parameter(torch.ones(c_hidden))
        self.rel_bias = RelativePositionBias(num_buckets, no_heads, max_distance, bidirectional) if num_buckets else None

    def forward(self, x, context=None, mask=None, kv_lens=None, q_positions=None, k_positions=None, q_offset=0):
        """mask [B, Lk] (1: key exists), kv_lens [B]; positions of the rotation (default 0, 1, ...), q_offset of the bias."""
        _require_cuda(x)
        with torch.cuda.device(x.device):            # (the projections launch on the current device)
            return self._attend(x, context, mask, kv_lens, q_positions, k_positions, q_offset)

    def _attend(self, x, context, mask, kv_lens, q_positions, k_positions, q_offset):
        context = x if context is None else context
        B, Lq, Lk, D = x.shape[0], x.shape[1], context.shape[1], self.c_hidden
        q = linear(x.to(BF16), self.linear_q.weight).view(B, Lq, self.no_heads, D)
        kv = linear(context.to(BF16), self.linear_kv.weight).view(B, Lk, 2 * self.no_kv_heads, D)
        k, v = kv[:, :, :self.no_kv_heads], kv[:, :, self.no_kv_heads:]
        if self.qk_norm:
            q, k = qk_norm_rope(q, k, self.q_norm, self.k_norm, q_positions, k_positions, rotary_dim=self.rotary_dim, base=self.rotary_base)
        rel = {} if self.rel_bias is None else dict(rel_table=self.rel_bias.table, max_distance=self.rel_bias.max_distance,
                                                    bidirectional=self.rel_bias.bidirectional, q_offset=q_offset)
        o = cross_attention(q, k, v, key_mask=mask, kv_lens=kv_lens, **rel)
        return linear(o.reshape(B, Lq, self.no_heads * D), self.linear_o.weight, self.linear_o.bias, out_fp32=x.dtype == torch.float32).to(x.dtype)
