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
import contextlib
import ctypes
import functools
import math
from ctypes import Structure, byref, c_double, c_float, c_int16, c_int32, c_int64, c_void_p

import torch
import torch.nn as nn
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from .. import _lib, ops
from .._lib import check, stream
from ..ops import BF16
from .functional import linear

DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}      # DFOLD_DT_*
REL_FAR, REL_MAX_DISTANCE = 256, 1024                                 # DFOLD_REL_*
MAX_OFFSET = 1 << 29
ROWS, TILE = 128, 64                                                  # softmax rows / keys of a workgroup, rows of an LDS tile


class _RelBias(Structure):
    _fields_ = [("table", c_void_p), ("q_offsets", c_void_p), ("q_offset", c_int32), ("num_buckets", c_int32), ("bidirectional", c_int32),
                ("reserved", c_int32), ("far_border", c_int16 * REL_FAR)]


class _AttnDesc(Structure):
    _fields_ = ([(n, c_void_p) for n in ("q", "k", "v", "o", "lse", "ws", "key_mask", "kv_lens")] +
                [(n, c_int64) for n in ("q_sb", "q_sl", "q_sh", "k_sb", "k_sl", "k_sh", "v_sb", "v_sl", "v_sh", "o_sb", "o_sl", "o_sh", "mask_sb")] +
                [(n, c_int32) for n in ("dtype", "B", "Lq", "Lk", "H", "Hkv", "D", "splits", "pack")] + [("scale", c_float), ("rel", _RelBias)])


class _AttnGrad(Structure):
    _fields_ = [("d_o", c_void_p), ("do_sb", c_int64), ("do_sl", c_int64), ("do_sh", c_int64), ("dq", c_void_p), ("dk", c_void_p),
                ("dv", c_void_p), ("delta", c_void_p), ("dtable", c_void_p), ("ws", c_void_p), ("splits_q", c_int32), ("splits_k", c_int32)]


class _RopePart(Structure):
    _fields_ = ([(n, c_void_p) for n in ("x", "y", "g", "w", "dw", "pos")] +
                [(n, c_int64) for n in ("x_sb", "x_sl", "x_sh", "g_sb", "g_sl", "g_sh", "pos_sb")] + [("L", c_int32), ("H", c_int32)])


class _RopeDesc(Structure):
    _fields_ = [("part", _RopePart * 2), ("ws", c_void_p), ("base", c_double), ("eps", c_float), ("dtype", c_int32), ("B", c_int32),
                ("D", c_int32), ("rotary_dim", c_int32), ("interleaved", c_int32)]


# ------------------------------------------------------------------------------------------------
# argument helpers
# ------------------------------------------------------------------------------------------------

def _need(cond, msg):
    if not cond:
        raise ValueError(msg)


def _require_cuda(t):
    if not t.is_cuda:
        raise RuntimeError("dynamicpdb_amd sequence operators need an MI355X device tensor (no CPU fallback)")


def _same_device(ref, **others):
    for name, t in others.items():
        _need(t is None or t.device == ref.device, f"{name} is on {t.device if t is not None else None}, expected {ref.device}")


def _on(t):
    """the launches of a call go to the device its tensors live on, whatever the current device is"""
    return contextlib.nullcontext() if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


def _rows16(t):
    """t itself if the kernels can read it as it lies -- dense last axis, every other stride a multiple of 16 bytes, aligned base --
    else a dense copy"""
    v = 16 // t.element_size()
    if t.numel() == 0 or (t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and
                          all(s % v == 0 for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1)):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _strides(t):
    """strides of the leading axes, 0 for axes of one entry (theirs may be anything)"""
    return [s if n > 1 else 0 for s, n in zip(t.stride()[:-1], t.shape[:-1])]


def _addr(t):
    return None if t is None else t.data_ptr()


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
def _border_array(num_buckets, max_distance, bidirectional):
    b = far_borders(num_buckets, max_distance, bidirectional)
    return (c_int16 * REL_FAR)(*b)


def _check_rel(table, max_distance, bidirectional):
    _need(table.dim() == 2 and table.dtype == torch.float32, "the bias table must be fp32 [num_buckets, heads]")
    nb = table.shape[0]
    half = nb // 2 if bidirectional else nb
    _need(not bidirectional or nb % 2 == 0, "num_buckets must be even for a bidirectional bias")
    _need(half >= 2 and half <= REL_FAR, f"num_buckets must be between 2 and {REL_FAR} per direction")
    _need(isinstance(max_distance, int) and half // 2 < max_distance <= REL_MAX_DISTANCE,
          f"max_distance must be a whole number above num_buckets' single distances ({half // 2}) and at most {REL_MAX_DISTANCE}")


def _fill_rel(rel, table, max_distance, bidirectional, q_offset, q_offsets=None):
    rel.table, rel.q_offsets, rel.q_offset = table.data_ptr(), _addr(q_offsets), q_offset
    rel.num_buckets, rel.bidirectional = table.shape[0], int(bidirectional)
    ctypes.memmove(rel.far_border, _border_array(table.shape[0], max_distance, bool(bidirectional)), 2 * REL_FAR)


# ------------------------------------------------------------------------------------------------
# relative position bias as a matrix
# ------------------------------------------------------------------------------------------------

class RelativeBiasFn(Function):
    @staticmethod
    def forward(ctx, table, q_len, k_len, max_distance, bidirectional, q_offset, dtype):
        t = table.detach().contiguous()
        H = t.shape[1]
        ctx.args = (q_len, k_len, max_distance, bidirectional, q_offset, dtype, t.shape)
        out = torch.empty((H, q_len, k_len), dtype=dtype, device=t.device)
        if out.numel():
            rel = _RelBias()
            _fill_rel(rel, t, max_distance, bidirectional, q_offset)
            with _on(t):
                check(_lib.lib().dfold_relpos_fwd(byref(rel), c_void_p(out.data_ptr()), c_int32(DTYPES[dtype]), c_int32(H), c_int32(q_len),
                                                  c_int32(k_len), stream()), "dfold_relpos_fwd")
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        q_len, k_len, max_distance, bidirectional, q_offset, dtype, shape = ctx.args
        nb, H = shape
        if g.numel() == 0:
            return (torch.zeros(shape, dtype=torch.float32, device=g.device),) + (None,) * 6
        if not g.is_contiguous() or g.data_ptr() % 16:
            g = g.clone(memory_format=torch.contiguous_format)
        dtable = torch.empty(shape, dtype=torch.float32, device=g.device)
        with _on(g):
            L = _lib.lib()
            n = L.dfold_relpos_ws(c_int32(H), c_int32(q_len), c_int32(nb))
            _need(n > 0, "relative_position_bias: too many heads x buckets")
            ws = torch.empty(n, dtype=torch.float32, device=g.device)
            rel = _RelBias()
            _fill_rel(rel, dtable, max_distance, bidirectional, q_offset)      # (the backward reads the borders, not the entries)
            check(L.dfold_relpos_bwd(byref(rel), c_void_p(g.data_ptr()), c_int32(DTYPES[dtype]), c_int32(H), c_int32(q_len), c_int32(k_len),
                                     c_void_p(dtable.data_ptr()), c_void_p(ws.data_ptr()), stream()), "dfold_relpos_bwd")
        return (dtable,) + (None,) * 6


def relative_position_bias(table, q_len, k_len, *, max_distance=128, bidirectional=True, q_offset=0, dtype=torch.float32):
    """[heads, q_len, k_len] bias of query i and key j: table[bucket(j - i - q_offset), head], differentiable in the table.

    table fp32 [num_buckets, heads].  Of the half = num_buckets / 2 buckets per direction (bidirectional; distances > 0 use the second
    half; else half = num_buckets and keys behind the query count as distance 0) the first half // 2 hold one distance each, the others
    grow logarithmically up to max_distance, beyond which everything shares the last.  dtype: fp32, bf16 or fp16 of the result."""
    _check_rel(table, max_distance, bidirectional)
    _need(isinstance(q_len, int) and isinstance(k_len, int) and 0 <= q_len <= 1 << 30 and 0 <= k_len <= 1 << 30, "q_len, k_len must be whole numbers >= 0")
    _need(isinstance(q_offset, int) and abs(q_offset) <= MAX_OFFSET, f"q_offset must be a whole number, at most {MAX_OFFSET}")
    _need(dtype in DTYPES, "dtype must be float32, bfloat16 or float16")
    _need(1 <= table.shape[1] <= 65535, "the table needs between 1 and 65535 heads")
    _require_cuda(table)
    return RelativeBiasFn.apply(table, q_len, k_len, max_distance, bool(bidirectional), q_offset, dtype)


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

class QKNormRopeFn(Function):
    @staticmethod
    def forward(ctx, q, k, w_q, w_k, q_pos, k_pos, rotary_dim, base, interleaved, eps):
        q, k = (None if t is None else _rows16(t.detach()) for t in (q, k))
        w_q, w_k = (None if t is None else t.detach().contiguous() for t in (w_q, w_k))
        ctx.opts = (rotary_dim, base, interleaved, eps)
        ctx.save_for_backward(q, k, w_q, w_k, q_pos, k_pos)
        outs = [None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k)]
        d = QKNormRopeFn._desc(ctx.opts, (q, k), outs, (w_q, w_k), (q_pos, k_pos))
        if d is not None:
            with _on(outs[0] if outs[0] is not None else outs[1]):
                check(_lib.lib().dfold_qk_norm_rope_fwd(byref(d), stream()), "dfold_qk_norm_rope_fwd")
        return tuple(outs)

    @staticmethod
    def _desc(opts, xs, ys, ws, poss, gs=(None, None)):
        d = _RopeDesc()
        d.rotary_dim, d.base, d.interleaved, d.eps = opts[0], opts[1], int(opts[2]), opts[3]
        any_part = False
        for part, x, y, w, pos, g in zip(d.part, xs, ys, ws, poss, gs):
            if x is None or x.numel() == 0:
                continue
            any_part = True
            d.dtype, d.B, d.D = DTYPES[x.dtype], x.shape[0], x.shape[3]
            part.x, part.y, part.w, part.pos = _addr(x), _addr(y), _addr(w), _addr(pos)
            part.x_sb, part.x_sl, part.x_sh = _strides(x)
            part.L, part.H = x.shape[1], x.shape[2]
            if pos is not None:
                part.pos_sb = pos.stride(0) if pos.shape[0] > 1 else 0
            if g is not None:
                part.g = _addr(g)
                part.g_sb, part.g_sl, part.g_sh = _strides(g)
        return d if any_part else None

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        q, k, w_q, w_k, q_pos, k_pos = ctx.saved_tensors
        gs = [None if x is None else _rows16(g) for x, g in ((q, gq), (k, gk))]
        dxs = [None if x is None else torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k)]
        ref = q if q is not None else k
        dws = [None, None]
        d = QKNormRopeFn._desc(ctx.opts, (q, k), dxs, (w_q, w_k), (q_pos, k_pos), gs)
        with _on(ref):
            L = _lib.lib()
            for i, (x, w) in enumerate(((q, w_q), (k, w_k))):
                if w is not None and ctx.needs_input_grad[2 + i]:
                    empty = x is None or x.numel() == 0
                    dws[i] = (torch.zeros if empty else torch.empty)(w.shape, dtype=torch.float32, device=w.device)
                    if not empty:
                        d.part[i].dw = dws[i].data_ptr()
            if d is not None:
                if dws[0] is not None or dws[1] is not None:
                    ws = torch.empty(L.dfold_qk_norm_rope_ws(), dtype=torch.float32, device=ref.device)
                    d.ws = ws.data_ptr()
                check(L.dfold_qk_norm_rope_bwd(byref(d), stream()), "dfold_qk_norm_rope_bwd")
        return dxs[0], dxs[1], dws[0], dws[1], None, None, None, None, None, None


def _positions(pos, x, name):
    if pos is None or x is None:
        return None
    _need(pos.dtype in (torch.int64, torch.int32), f"{name} must be int64 or int32")
    if pos.dim() == 1:
        pos = pos[None]
    _need(pos.dim() == 2 and pos.shape[0] in (1, x.shape[0]) and pos.shape[1] == x.shape[1], f"{name} must be [{x.shape[1]}] or [{x.shape[0]}, {x.shape[1]}]")
    pos = pos.long()
    return pos if pos.shape[1] <= 1 or pos.stride(1) == 1 else pos.contiguous()


def qk_norm_rope(q, k, w_q=None, w_k=None, q_positions=None, k_positions=None, *, rotary_dim=None, base=10000.0, interleaved=False, eps=1e-6):
    """Every head of q [B, Lq, H, D] and k [B, Lk, Hkv, D] divided by its root mean square, times w (fp32 [D] or None), then its first
    rotary_dim dimensions (default: all; a multiple of 16; 0: none) rotated by position * base^(-2 i / rotary_dim): pairs
    (i, i + rotary_dim / 2), or (2 i, 2 i + 1) if interleaved.  k may be None (keys that are rotated already).  Positions: int64 / int32
    [L] or [B, L], default 0, 1, ...; any size (angles are reduced in fp64).  bf16, fp16 or fp32; one launch for q and k; differentiable
    in q, k, w_q, w_k."""
    ref = q if q is not None else k
    _need(ref is not None, "qk_norm_rope needs q or k")
    _same_device(ref, q=q, k=k, w_q=w_q, w_k=w_k, q_positions=q_positions, k_positions=k_positions)
    _need(ref.dtype in DTYPES, "q, k must be bfloat16, float16 or float32")
    for name, t in (("q", q), ("k", k)):
        _need(t is None or (t.dim() == 4 and t.dtype == ref.dtype), f"{name} must be [B, L, heads, D], q and k of one type")
    _need(q is None or k is None or (q.shape[0] == k.shape[0] and q.shape[3] == k.shape[3]), "q and k differ in batch or head size")
    D = ref.shape[3]
    _need(D % 8 == 0 and 8 <= D <= 256, "the head size must be a multiple of 8, at most 256")
    rd = (D // 16 * 16 if D % 16 else D) if rotary_dim is None else rotary_dim
    _need(rotary_dim is not None or rd == D, "this head size is not a multiple of 16: give rotary_dim")
    _need(isinstance(rd, int) and 0 <= rd <= D and rd % 16 == 0, "rotary_dim must be a multiple of 16, at most the head size")
    _need(base > 0 and math.isfinite(base) and eps >= 0, "base must be positive and eps not negative")
    for name, w in (("w_q", w_q), ("w_k", w_k)):
        _need(w is None or (w.dtype == torch.float32 and w.shape == (D,)), f"{name} must be fp32 [{D}]")
    q_positions, k_positions = _positions(q_positions, q, "q_positions"), _positions(k_positions, k, "k_positions")
    _require_cuda(ref)
    return QKNormRopeFn.apply(q, k, w_q, w_k, q_positions, k_positions, rd, float(base), bool(interleaved), float(eps))


# ------------------------------------------------------------------------------------------------
# attention of one sequence over another
# ------------------------------------------------------------------------------------------------

def _parts(groups, units, n_cu, least):
    """Cut factor of a launch of `groups` workgroups that each walk `units` tiles: as many parts as bring the launch to two workgroups
    per CU, each of at least `least` tiles (below that, writing and adding the parts costs more than the idle CUs)."""
    return max(1, min(2 * n_cu // max(groups, 1), units // least))


def _attn_plan(B, Lq, Lk, H, Hkv, rel_width, n_cu):
    """(pack, splits) of the forward.  pack: the query heads of a group share tiles if that at least halves the number of row blocks
    (their bias rows have to fit 32 KB of LDS); K and V are then read once per group."""
    G = H // Hkv
    blocks, packed = -(-Lq // ROWS) * G, -(-(Lq * G) // ROWS)
    pack = G if 2 * packed <= blocks and G * rel_width * 4 <= 32768 else 1
    groups = B * (H // pack) * -(-(Lq * pack) // ROWS)
    return pack, _parts(groups, -(-Lk // TILE), n_cu, 2)


class CrossAttentionFn(Function):
    @staticmethod
    def forward(ctx, q, k, v, table, key_mask, kv_lens, q_offsets, q_offset, max_distance, bidirectional, scale, train):
        q, k, v = (_rows16(t.detach()) for t in (q, k, v))
        B, Lq, H, D = q.shape
        Lk, Hkv = k.shape[1], k.shape[2]
        dev = q.device
        if table is not None:
            table = table.detach().contiguous()
        o = torch.empty((B, Lq, H, D), dtype=q.dtype, device=dev)
        lse = torch.empty((B, H, Lq), dtype=torch.float32, device=dev) if train else None
        ctx.opts = (q_offset, max_distance, bidirectional, scale)
        ctx.save_for_backward(q, k, v, table, key_mask, kv_lens, q_offsets, o, lse)
        if o.numel():
            d = CrossAttentionFn._desc(ctx.opts, q, k, v, table, key_mask, kv_lens, q_offsets, o, lse)
            width = 0
            if table is not None:
                nb = table.shape[0]
                far = far_borders(nb, max_distance, bidirectional)
                width = 2 * (far[-1] if far else (nb // 2 if bidirectional else nb) // 2) + 1
            with _on(q):
                d.pack, d.splits = _attn_plan(B, Lq, Lk, H, Hkv, width, ops.cu_count(dev))
                if d.splits > 1:
                    ws = torch.empty(d.splits * B * H * Lq * (D + 1), dtype=torch.float32, device=dev)
                    d.ws = ws.data_ptr()
                check(_lib.lib().dfold_seq_attn_fwd(byref(d), stream()), "dfold_seq_attn_fwd")
        return o

    @staticmethod
    def _desc(opts, q, k, v, table, key_mask, kv_lens, q_offsets, o, lse):
        q_offset, max_distance, bidirectional, scale = opts
        d = _AttnDesc()
        d.q, d.k, d.v, d.o, d.lse = (_addr(t) for t in (q, k, v, o, lse))
        d.key_mask, d.kv_lens = _addr(key_mask), _addr(kv_lens)
        d.q_sb, d.q_sl, d.q_sh = _strides(q)
        d.k_sb, d.k_sl, d.k_sh = _strides(k)
        d.v_sb, d.v_sl, d.v_sh = _strides(v)
        d.o_sb, d.o_sl, d.o_sh = _strides(o)
        if key_mask is not None:
            d.mask_sb = key_mask.stride(0) if key_mask.shape[0] > 1 else 0
        d.dtype, d.scale = DTYPES[q.dtype], scale
        d.B, d.Lq, d.H, d.D = q.shape
        d.Lk, d.Hkv = k.shape[1], k.shape[2]
        if table is not None:
            _fill_rel(d.rel, table, max_distance, bidirectional, q_offset, q_offsets)
        return d

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        q, k, v, table, key_mask, kv_lens, q_offsets, o, lse = ctx.saved_tensors
        B, Lq, H, D = q.shape
        Lk, Hkv = k.shape[1], k.shape[2]
        dev = q.device
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (q, k, v))
        dtable = None
        if o.numel() == 0 or k.numel() == 0:
            for t in (dq, dk, dv):
                t.zero_()
            dtable = None if table is None else torch.zeros_like(table)
        else:
            g = _rows16(g)
            a = CrossAttentionFn._desc(ctx.opts, q, k, v, table, key_mask, kv_lens, q_offsets, o, lse)
            b = _AttnGrad()
            b.d_o, b.dq, b.dk, b.dv = (_addr(t) for t in (g, dq, dk, dv))
            b.do_sb, b.do_sl, b.do_sh = _strides(g)
            with _on(q):
                n_cu = ops.cu_count(dev)
                nrb, nkb = -(-Lq // ROWS), -(-Lk // ROWS)
                b.splits_q = _parts(B * H * nrb, -(-Lk // TILE), n_cu, 4)
                b.splits_k = _parts(B * Hkv * nkb, (H // Hkv) * -(-Lq // TILE), n_cu, 4)
                up4 = lambda x: (x + 3) // 4 * 4
                n = up4(b.splits_q * dq.numel()) if b.splits_q > 1 else 0
                n += up4(2 * b.splits_k * dk.numel()) if b.splits_k > 1 else 0
                if table is not None:
                    dtable = torch.empty_like(table)
                    b.dtable = dtable.data_ptr()
                    n += up4(b.splits_k * B * H * nkb * table.shape[0])
                delta = torch.empty((1 + b.splits_q if b.splits_q > 1 else 1, B, H, Lq), dtype=torch.float32, device=dev)
                b.delta = delta.data_ptr()
                if n:
                    ws = torch.empty(n, dtype=torch.float32, device=dev)
                    b.ws = ws.data_ptr()
                check(_lib.lib().dfold_seq_attn_bwd(byref(a), byref(b), stream()), "dfold_seq_attn_bwd")
        need = ctx.needs_input_grad
        return (dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, dtable if need[3] else None) + (None,) * 8


def cross_attention(q, k, v, *, key_mask=None, kv_lens=None, rel_table=None, max_distance=128, bidirectional=True, q_offset=0, scale=None):
    """softmax(scale q k^T + bias) v of q [B, Lq, H, D] over k, v [B, Lk, Hkv, D] (H a multiple of Hkv: query head h reads key head
    h // (H / Hkv)), bf16 or fp16, D a multiple of 8 up to 128; any strides (a copy is made where rows are not 16-byte aligned).

    key_mask [B, Lk] (bool, or 0 / 1 in any type) and kv_lens [B] (int32 / int64: keys j < kv_lens[b] exist) remove keys: what K and V
    hold there is never used, gradients there are zero.  A query without any key gives zeros and takes no gradient.  rel_table fp32
    [num_buckets, H] adds the bias of relative_position_bias without forming it; q_offset: position of query 0 minus position of key 0, a
    whole number or an int32 / int64 tensor [B] (one token at its own position per sequence).  scale defaults to D^-1/2.
    Differentiable (once) in q, k, v and rel_table; repeated calls give the same bits."""
    _need(q.dim() == 4 and k.dim() == 4 and v.dim() == 4, "q must be [B, Lq, H, D], k and v [B, Lk, Hkv, D]")
    _need(q.dtype in (torch.bfloat16, torch.float16) and k.dtype == q.dtype and v.dtype == q.dtype, "q, k, v must all be bfloat16 or all float16")
    B, Lq, H, D = q.shape
    _need(k.shape == v.shape and k.shape[0] == B and k.shape[3] == D, "k and v must be [B, Lk, Hkv, D] with q's B and D")
    Lk, Hkv = k.shape[1], k.shape[2]
    _need(H > 0 and Hkv > 0 and H % Hkv == 0, "the query heads must be a multiple of the key heads")
    _need(8 <= D <= 128 and D % 8 == 0, "the head size must be a multiple of 8, at most 128")
    _need(Lq <= 1 << 30 and Lk <= 1 << 30, "sequences are at most 2^30 long")
    _same_device(q, k=k, v=v, key_mask=key_mask, kv_lens=kv_lens, rel_table=rel_table)
    if key_mask is not None:
        _need(key_mask.shape == (B, Lk), f"key_mask must be [{B}, {Lk}]")
        key_mask = _mask_bytes(key_mask)
    if kv_lens is not None:
        _need(kv_lens.shape == (B,) and kv_lens.dtype in (torch.int32, torch.int64), f"kv_lens must be int32 or int64 [{B}]")
        kv_lens = kv_lens.clamp(max=Lk).int().contiguous() if kv_lens.dtype == torch.int64 else kv_lens.contiguous()
    q_offsets = None
    if rel_table is not None:
        _check_rel(rel_table, max_distance, bidirectional)
        _need(rel_table.shape[1] == H, f"rel_table must have {H} columns, one per query head")
        if torch.is_tensor(q_offset):
            _same_device(q, q_offset=q_offset)
            _need(q_offset.shape == (B,) and q_offset.dtype in (torch.int32, torch.int64), f"q_offset must be a whole number or int32 / int64 [{B}]")
            q_offsets = (q_offset.clamp(-MAX_OFFSET, MAX_OFFSET).int() if q_offset.dtype == torch.int64 else q_offset).contiguous()
            q_offset = 0
        else:
            _need(isinstance(q_offset, int) and abs(q_offset) <= MAX_OFFSET, f"q_offset must be a whole number, at most {MAX_OFFSET}")
    else:
        q_offset = 0
    scale = D ** -0.5 if scale is None else float(scale)
    _need(math.isfinite(scale), "scale must be finite")
    _require_cuda(q)
    train = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, rel_table))
    return CrossAttentionFn.apply(q, k, v, rel_table, key_mask, kv_lens, q_offsets, q_offset, max_distance, bool(bidirectional), scale, train)


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
