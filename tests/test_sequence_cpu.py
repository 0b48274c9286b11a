"""Sequence-track operators, what needs no GPU: bucket borders against whole-number arithmetic, refusals of the Python entry points and
of the C ABI (argument checks come before any launch), launch plans, no CPU fallback."""
import math
from ctypes import byref, c_int32, c_void_p, sizeof
from fractions import Fraction

import pytest
import torch

from dynamicpdb_amd.model import sequence_attention as S


@pytest.mark.parametrize("nb,dist,both", [(32, 128, True), (32, 128, False), (64, 256, True), (4, 2, True), (4, 1024, True), (16, 5, True), (3, 9, False),
                                          (512, 1024, True), (48, 300, True)])
def test_bucket_borders(nb, dist, both):
    half = nb // 2 if both else nb
    e = half // 2
    m = half - e
    far = S.far_borders(nb, dist, both)
    assert len(far) == m - 1 and all(a <= b for a, b in zip((e,) + far, far)) and (not far or far[-1] <= dist)
    for k, n in enumerate(far, 1):         # first n with (n / e)^m >= (dist / e)^k
        assert Fraction(n, e) ** m >= Fraction(dist, e) ** k
        assert n == e or Fraction(n - 1, e) ** m < Fraction(dist, e) ** k
    if m <= 32:                            # the logarithm's form, away from borders
        for n in range(e, dist + 10):
            x = math.log(n / e) / math.log(dist / e) * m
            if abs(x - round(x)) > 1e-9:
                assert min(int(x), m - 1) == sum(f <= n for f in far)


def _qkv(B=2, Lq=3, Lk=5, H=4, Hkv=2, D=32, dt=torch.bfloat16):
    return torch.zeros(B, Lq, H, D, dtype=dt), torch.zeros(B, Lk, Hkv, D, dtype=dt), torch.zeros(B, Lk, Hkv, D, dtype=dt)


@pytest.mark.parametrize("shape,kw", [
    (dict(dt=torch.float32), {}), (dict(D=12), {}), (dict(D=136), {}), (dict(H=3), {}),
    ({}, dict(key_mask=torch.ones(2, 4))), ({}, dict(kv_lens=torch.ones(3, dtype=torch.int32))), ({}, dict(kv_lens=torch.ones(2))),
    ({}, dict(rel_table=torch.zeros(32, 3))), ({}, dict(rel_table=torch.zeros(31, 4))), ({}, dict(rel_table=torch.zeros(32, 4, dtype=torch.bfloat16))),
    ({}, dict(rel_table=torch.zeros(32, 4), max_distance=8)), ({}, dict(rel_table=torch.zeros(32, 4), max_distance=1025)),
    ({}, dict(rel_table=torch.zeros(514, 4), max_distance=900)), ({}, dict(rel_table=torch.zeros(2, 4))),
    ({}, dict(rel_table=torch.zeros(32, 4), q_offset=1 << 30)), ({}, dict(rel_table=torch.zeros(32, 4), q_offset=torch.zeros(3, dtype=torch.int32))),
    ({}, dict(rel_table=torch.zeros(32, 4), q_offset=torch.zeros(2))), ({}, dict(scale=float("nan"))),
])
def test_cross_attention_refuses(shape, kw):
    with pytest.raises(ValueError):
        S.cross_attention(*_qkv(**shape), **kw)


def test_cross_attention_refuses_shapes_and_cpu_tensors():
    q, k, v = _qkv()
    for a in ((q[0], k, v), (q, k, v[:, :4]), (q, k[:1], v[:1]), (q, k[..., :16], v[..., :16]), (q, k.half(), v)):
        with pytest.raises(ValueError):
            S.cross_attention(*a)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        S.cross_attention(q, k, v)


@pytest.mark.parametrize("table,kw", [
    (torch.zeros(33, 4), {}), (torch.zeros(32), {}), (torch.zeros(32, 4).double(), {}), (torch.zeros(32, 4), dict(max_distance=8)),
    (torch.zeros(32, 4), dict(max_distance=128.0)), (torch.zeros(257, 4), dict(bidirectional=False, max_distance=900)), (torch.zeros(32, 4), dict(dtype=torch.float64)),
    (torch.zeros(32, 4), dict(q_offset=1.5)), (torch.zeros(32, 4), dict(q_offset=-(1 << 30))), (torch.zeros(32, 0), {}), (torch.zeros(32, 4), dict(q_len=-1)),
])
def test_relative_position_bias_refuses(table, kw):
    kw = dict(dict(q_len=4, k_len=4), **kw)
    with pytest.raises(ValueError):
        S.relative_position_bias(table, **kw)


def test_relative_position_bias_refuses_cpu_tensors():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        S.relative_position_bias(torch.zeros(32, 4), 4, 4)


@pytest.mark.parametrize("kw", [dict(rotary_dim=8), dict(rotary_dim=48), dict(rotary_dim=-16), dict(base=0.0), dict(eps=-1.0), dict(w_q=torch.ones(16)),
                                dict(w_k=torch.ones(32).half()), dict(q_positions=torch.zeros(3)), dict(q_positions=torch.zeros(4, dtype=torch.int64)),
                                dict(k_positions=torch.zeros(3, 5, dtype=torch.int64))])
def test_qk_norm_rope_refuses(kw):
    q, k, _ = _qkv()
    with pytest.raises(ValueError):
        S.qk_norm_rope(q, k, **kw)


def test_qk_norm_rope_refuses_shapes_and_cpu_tensors():
    q, k, _ = _qkv()
    for a in ((None, None), (q, k.half()), (q, k[:1]), (q[0], None), (q.double(), None), (torch.zeros(1, 1, 1, 264), None), (torch.zeros(1, 1, 1, 20), None),
              (torch.zeros(1, 1, 1, 24), None)):
        with pytest.raises(ValueError):
            S.qk_norm_rope(*a)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        S.qk_norm_rope(q, k)


def test_module_refuses():
    for kw in (dict(c_hidden=136), dict(c_q=12), dict(no_kv_heads=3), dict(qk_norm=False, rotary_dim=32), dict(num_buckets=7)):
        with pytest.raises(ValueError):
            S.CrossAttention(**dict(dict(c_q=64, c_kv=64, c_hidden=32, no_heads=4), **kw))


def test_launch_plans():
    # a token over a long cache: the group's heads share tiles, the keys are cut; a long prompt: neither
    pack, parts, pair = S._attn_plan(16, 1, 16384, 32, 8, 0, 256)
    assert pack == 4 and parts > 1 and not pair
    assert S._attn_plan(2, 8192, 8192, 16, 16, 0, 256) == (1, 1, 0)
    assert S._attn_plan(1, 1, 1, 8, 8, 0, 256) == (1, 1, 0) and S._attn_plan(1, 4, 0, 8, 8, 0, 256) == (1, 1, 0)
    # one workgroup per CU and many tiles: two waves per 32 rows
    assert S._attn_plan(4, 1001, 1001, 8, 8, 0, 256) == (1, 1, 1)
    # bias rows of a group that do not fit: the heads stay apart
    assert S._attn_plan(1, 1, 64, 32, 1, 2049, 256)[0] == 1
    # no part without a tile of its own
    for B, Lq, Lk, H, Hkv in ((1, 1, 100, 1, 1), (1, 17, 6001, 16, 4), (3, 200, 999, 8, 8), (1, 1, 1 << 20, 1, 1)):
        pack, s, _ = S._attn_plan(B, Lq, Lk, H, Hkv, 0, 256)
        nt = -(-Lk // 64)
        assert 1 <= s <= nt and s <= 1024


def rel_of(table, dist, both):
    return S.RelBias.from_buffer_copy(S._rel_desc(table, table.shape[0], dist, both, 0))


def test_packed_descriptors_have_the_layout_of_the_structures():
    assert S._REL.size == sizeof(S.RelBias) and S._ATTN.size + S._REL.size == sizeof(S.AttnDesc) and S._GRAD.size == sizeof(S.AttnGrad)
    assert S._PART.size == sizeof(S.RopePart) and 2 * S._PART.size + S._ROPE.size == sizeof(S.RopeDesc)
    d = S.AttnDesc.from_buffer_copy(S._ATTN.pack(*range(1, 32), 0.5) + S._NO_REL)
    assert [getattr(d, n) for n, _ in S.AttnDesc._fields_[:31]] == list(range(1, 32)) and d.scale == 0.5
    g = S.AttnGrad.from_buffer_copy(S._GRAD.pack(*range(1, 15)))
    assert [getattr(g, n) for n, _ in S.AttnGrad._fields_] == list(range(1, 15))
    r = S.RopeDesc.from_buffer_copy(S._PART.pack(*range(1, 16)) + S._PART.pack(*range(21, 36)) + S._ROPE.pack(51, 2.5, 0.25, *range(52, 57)))
    assert [getattr(r.part[1], n) for n, _ in S.RopePart._fields_] == list(range(21, 36))
    assert [getattr(r, n) for n, _ in S.RopeDesc._fields_[1:]] == [51, 2.5, 0.25, 52, 53, 54, 55, 56]
    rel = rel_of(torch.zeros(32, 4), 128, True)
    assert list(rel.far_border[:7]) == list(S.far_borders(32, 128, True)) and rel.num_buckets == 32 and rel.bidirectional == 1


def test_cabi_refuses_bad_descriptors():
    from dynamicpdb_amd import _lib
    L = _lib.lib()
    tok = 16

    def attn(**kw):
        d = S.AttnDesc()
        for n in ("q", "k", "v", "o"):
            setattr(d, n, tok)
        d.B, d.Lq, d.Lk, d.H, d.Hkv, d.D, d.splits, d.pack, d.scale = 1, 4, 4, 4, 2, 64, 1, 1, 0.1
        for n, x in kw.items():
            setattr(d, n, x)
        return d
    assert L.dfold_seq_attn_fwd(None, c_void_p(0)) == -1
    for kw in (dict(q=None), dict(k=None), dict(o=None), dict(dtype=2), dict(D=60), dict(D=136), dict(D=0), dict(H=3), dict(Hkv=0), dict(B=0), dict(Lq=0),
               dict(Lk=-1), dict(splits=0), dict(splits=2), dict(splits=1025, ws=tok), dict(pack=3), dict(q_sl=4), dict(k_sh=-8), dict(q=tok + 2), dict(mask_sb=-1)):
        assert L.dfold_seq_attn_fwd(byref(attn(**kw)), c_void_p(0)) == -1, kw
    for nb, dist, both, breakage in ((32, 128, True, lambda r: setattr(r, "num_buckets", 33)), (32, 128, True, lambda r: setattr(r, "num_buckets", 1)),
                                     (32, 128, True, lambda r: r.far_border.__setitem__(0, 3)), (32, 128, True, lambda r: r.far_border.__setitem__(6, 1025)),
                                     (32, 128, False, lambda r: setattr(r, "num_buckets", 600))):
        d = attn()
        table = torch.zeros(nb, 4)
        d.rel = rel_of(table, dist, both)
        breakage(d.rel)
        assert L.dfold_seq_attn_fwd(byref(d), c_void_p(0)) == -1
        assert L.dfold_relpos_fwd(byref(d.rel), c_void_p(tok), c_int32(0), c_int32(4), c_int32(4), c_int32(4), c_void_p(0)) == -1
    d = attn(pack=2)                                   # bias rows of the packed heads over 32 KB
    d.H, d.pack = 16, 8
    d.rel = rel_of(torch.zeros(32, 16), 1024, True)
    assert L.dfold_seq_attn_fwd(byref(d), c_void_p(0)) == -1

    def grad(**kw):
        g = S.AttnGrad()
        for n in ("d_o", "dq", "dk", "dv", "delta"):
            setattr(g, n, tok)
        g.splits_q = g.splits_k = 1
        for n, x in kw.items():
            setattr(g, n, x)
        return g
    assert L.dfold_seq_attn_bwd(byref(attn()), byref(grad()), c_void_p(0)) == -1          # no log-sums
    for kw in (dict(d_o=None), dict(dq=None), dict(dk=None), dict(delta=None), dict(splits_q=0), dict(splits_q=2), dict(splits_k=2), dict(do_sl=3), dict(dv=tok + 8)):
        assert L.dfold_seq_attn_bwd(byref(attn(lse=tok)), byref(grad(**kw)), c_void_p(0)) == -1, kw

    rel = rel_of(torch.zeros(32, 4), 128, True)
    one, st = c_void_p(tok), c_void_p(0)
    for args in ((None, 0, 4, 4, 4), (tok + 2, 0, 4, 4, 4), (tok, 3, 4, 4, 4), (tok, 0, 0, 4, 4), (tok, 0, 4, 0, 4), (tok, 0, 4, 4, 0), (tok, 0, 70000, 4, 4)):
        a = (byref(rel), c_void_p(args[0])) + tuple(c_int32(x) for x in args[1:])
        assert L.dfold_relpos_fwd(*a, st) == -1
        assert L.dfold_relpos_bwd(*a, one, one, st) == -1
    assert L.dfold_relpos_ws(c_int32(0), c_int32(1), c_int32(1)) == -1 and L.dfold_relpos_ws(c_int32(1 << 20), c_int32(1 << 20), c_int32(1 << 20)) == -1
    for blocks_of in ((1, 1, 32), (16, 4097, 64), (3000, 5, 2)):
        assert L.dfold_relpos_ws(*(c_int32(x) for x in blocks_of)) == blocks_of[0] * min(blocks_of[1], max(1280 // blocks_of[0], 1)) * blocks_of[2]

    def rope(**kw):
        d = S.RopeDesc()
        d.B, d.D, d.rotary_dim, d.base, d.eps = 1, 64, 64, 10000.0, 1e-6
        p = d.part[0]
        p.x = p.y = tok
        p.L, p.H = 4, 2
        for n, x in kw.items():
            setattr(p if hasattr(p, n) and n not in ("B", "D") else d, n, x)
        return d
    for kw in (dict(x=None), dict(y=None), dict(L=0), dict(H=0), dict(B=0), dict(D=60), dict(D=264), dict(rotary_dim=8), dict(rotary_dim=80), dict(dtype=3),
               dict(base=0.0), dict(eps=-1.0), dict(x_sl=4), dict(x_sh=-8), dict(x=tok + 4), dict(pos=tok, pos_sb=-1)):
        assert L.dfold_qk_norm_rope_fwd(byref(rope(**kw)), st) == -1, kw
    for kw in (dict(), dict(g=tok, g_sl=4), dict(g=tok, dw=tok)):
        assert L.dfold_qk_norm_rope_bwd(byref(rope(**kw)), st) == -1, kw


def test_strides_of_axes_of_one_entry_are_zero():
    """dense for torch, whatever the strides of axes of one entry: the kernels get 0 for those"""
    a = torch.zeros(1, 7, 132)[..., :128].unflatten(-1, (4, 32))[:, :1]
    b = torch.zeros(64).as_strided((1, 1, 2, 32), (3, (1 << 24) + 5, 32, 1))
    c = torch.zeros(2, 1, 36)[:1, :, :32].unflatten(-1, (1, 32))
    for t, heads in ((a, 32), (b, 32), (c, 0)):
        assert t.is_contiguous() and S._rows16(t) is t and S._strides(t) == (0, 0, heads)
    assert S._strides(torch.zeros(2, 3, 4, 8)) == (96, 32, 8) and S._strides(torch.zeros(2, 0, 4, 8)) == (0, 0, 0)


def test_forward_mode_and_tracing_are_not_silent(monkeypatch):
    """inputs with a tangent reach the autograd node, which has no forward-mode derivative and says so; a traced call records it or raises (the kernels
    replaced by empty results: no GPU)"""
    import torch.autograd.forward_ad as fw
    from ctypes import ArgumentError
    monkeypatch.setattr(S, "_require_cuda", lambda t: None)
    monkeypatch.setattr(S, "_call", lambda *a, **kw: None)
    monkeypatch.setattr(S.ops, "cu_count", lambda dev: 256)
    q, k, v = _qkv()
    table, w = torch.zeros(32, 4), torch.ones(32)
    for f, t in ((lambda t: S.cross_attention(t, k, v), q), (lambda t: S.cross_attention(q, k, v, rel_table=t), table),
                 (lambda t: S.relative_position_bias(t, 4, 4), table), (lambda t: S.qk_norm_rope(q, t)[1], k), (lambda t: S.qk_norm_rope(q, k, w_q=t)[0], w)):
        with fw.dual_level():
            f(t)
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="jvp"):
                    f(fw.make_dual(t, torch.ones_like(t)))
        try:
            graph = str(torch.jit.trace(f, (t,), check_trace=False).graph)
        except (RuntimeError, ValueError, ArgumentError):
            continue
        assert "Fn" in graph


@pytest.mark.parametrize("scale", [1e39, -1e39, 1e-50, 1e-39, 2.0 ** -121, 2.0 ** 121, float("inf"), 0.0])
def test_cross_attention_refuses_scales_outside_fp32(scale):
    """the kernels hold the scale, its product with log2 e and the inverse of that in fp32: none of them may leave its normal range"""
    with pytest.raises(ValueError):
        S.cross_attention(*_qkv(), scale=scale)
    from dynamicpdb_amd import _lib
    if abs(scale) < 1e38:
        d = S.AttnDesc()
        d.q = d.k = d.v = d.o = 16
        d.B, d.Lq, d.Lk, d.H, d.Hkv, d.D, d.splits, d.pack, d.scale = 1, 4, 4, 4, 2, 64, 1, 1, scale
        assert _lib.lib().dfold_seq_attn_fwd(byref(d), c_void_p(0)) == -1


@pytest.mark.parametrize("kw", [dict(eps=1e39), dict(eps=math.inf), dict(eps=math.nan), dict(base=math.inf), dict(base=math.nan)])
def test_qk_norm_rope_refuses_numbers_outside_fp32(kw):
    q, k, _ = _qkv()
    with pytest.raises(ValueError):
        S.qk_norm_rope(q, k, **kw)
