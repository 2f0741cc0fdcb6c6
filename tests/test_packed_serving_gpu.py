"""The packed serving operators (per-head q/k norm with rotation, attention over
packed sequences, single-token attention behind a shared prefix) against plain
implementations in 64 bits.

Tolerances. bf16 rounds by at most h = 2^-8 of a value. qk_norm_rope computes in
fp32 and rounds once: h * |y|, plus 2^-20 of the two rotated terms for the fp32
arithmetic. Attention rounds each softmax weight to bf16 for the second product,
which moves the output by at most h * sum_j p_j |v_j|, and rounds the output once,
h * |o|; 2^-12 * sum_j p_j |v_j| covers the fp32 scores and exponentials (a score
is a 128-term fp32 sum, off by about 1e-5 here). The log-sum-exp is fp32: 1e-4,
and 2^-20 of its value: the largest score is summed in eight steps of 16 products,
each of which may lose a step of 2^-23 of the partial sum where all products have
one sign (8 * 2^-23 = 2^-20), which shows once the value is in the hundreds.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

H_BF16 = 2.0 ** -8
DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    from mka_b200 import ops as _ops

    _ops.device_status()
    return _ops


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, scale=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * scale).bfloat16()


# --------------------------------------------------------------- references --
def _tables(pos):
    inv = 10000.0 ** (-torch.arange(0, 128, 2, dtype=torch.float64, device=DEV) / 128)
    a = pos.double()[..., None] * inv
    a = torch.cat([a, a], -1)
    return a.cos().float(), a.sin().float()


def _ref_norm(x, w, eps, cos, sin):
    """x [..., H, 128]; cos / sin [..., 128] or None. Returns the value and the size of its terms."""
    x = x.double()
    if w is not None:
        x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w.double()
    if cos is None:
        return x, x.abs()
    c, s = cos.double().unsqueeze(-2), sin.double().unsqueeze(-2)
    turned = torch.cat([-x[..., 64:], x[..., :64]], -1)
    return x * c + turned * s, (x * c).abs() + (turned * s).abs()


def _check_norm(got, x, w, eps, cos, sin):
    ref, size = _ref_norm(x, w, eps, cos, sin)
    err = (got.double() - ref).abs()
    assert torch.isfinite(err).all()
    assert (err <= H_BF16 * ref.abs() * (1 + 2.0 ** -8) + 2.0 ** -20 * size + 1e-30).all(), err.max().item()


def _ref_rows(q, k, v, see, scale):
    """q [R, 128], k / v [S, 128], see [R, S]: o, sum p|v|, lse in 64 bits."""
    s = (q.double() @ k.double().t()) * scale
    s = s.masked_fill(~see, -math.inf)
    m = s.amax(-1, keepdim=True) if s.shape[1] else torch.full((s.shape[0], 1), -math.inf, device=DEV)
    e = torch.exp(s - m.masked_fill(m == -math.inf, 0.0)).masked_fill(~see, 0.0)
    z = e.sum(-1, keepdim=True)
    p = e / z.masked_fill(z == 0, 1.0)
    v = torch.nan_to_num(v.double()) if not see.all() else v.double()
    return p @ v, p @ v.abs(), (z.log() + m).squeeze(-1)


def _check_attn(o, lse, ro, size, rl, what=""):
    err = (o.double() - ro).abs()
    assert torch.isfinite(o.double()).all(), what
    tol = H_BF16 * (size + ro.abs()) * (1 + 2.0 ** -8) + 2.0 ** -12 * size
    assert (err <= tol).all(), (what, (err - tol).max().item())
    if lse is not None:
        empty = torch.isinf(rl)
        assert torch.equal(torch.isinf(lse) & (lse < 0), empty), what
        assert ((lse.double() - rl).abs()[~empty] <= 1e-4 + 2.0 ** -20 * rl.abs()[~empty]).all(), what


def _check_varlen(o, lse, q, k, v, q_lens, k_lens, causal, scale=128 ** -0.5):
    G = q.shape[1] // k.shape[1]
    q0 = k0 = 0
    for i, (lq, lk) in enumerate(zip(q_lens, k_lens)):
        see = torch.ones(lq, lk, dtype=torch.bool, device=DEV)
        if causal:
            see = torch.arange(lk, device=DEV)[None] <= torch.arange(lq, device=DEV)[:, None] + lk - lq
        for h in range(q.shape[1]):
            kk, vv = k[k0:k0 + lk, h // G], v[k0:k0 + lk, h // G]
            ref = _ref_rows(q[q0:q0 + lq, h], kk, vv, see, scale)
            _check_attn(o[q0:q0 + lq, h], None if lse is None else lse[h, q0:q0 + lq], *ref, what=(i, lq, lk, h))
        q0, k0 = q0 + lq, k0 + lk


def _cu(lens):
    return torch.tensor([0] + list(lens), device=DEV).cumsum(0).int()


def _check_shared(o, lse, q, kp, vp, k, v, lens, scale=128 ** -0.5):
    G = q.shape[1] // kp.shape[0]
    for b, n in enumerate(lens):
        for h in range(q.shape[1]):
            kk = torch.cat([kp[h // G], k[b, h // G, :n]])
            vv = torch.cat([vp[h // G], v[b, h // G, :n]])
            see = torch.ones(1, kk.shape[0], dtype=torch.bool, device=DEV)
            ref = _ref_rows(q[b, h][None], kk, vv, see, scale)
            _check_attn(o[b, 0, h][None], None if lse is None else lse[b, h][None], *ref, what=(b, n, h))


# ------------------------------------------------------------- qk_norm_rope --
@pytest.mark.parametrize("T,Hq,Hkv", [(1, 1, 1), (1, 32, 8), (3, 28, 4), (64, 32, 8), (129, 5, 2), (1021, 7, 7),
                                      (77, 16, 16), (2500, 28, 4)])
@pytest.mark.parametrize("layout", ["fused", "heads"])
def test_norm_rope(ops, T, Hq, Hkv, layout):
    g = _gen(T + Hq)
    if layout == "fused":
        x = _randn(g, T, Hq + 2 * Hkv, 128, scale=3.0)
        q, k = x[:, :Hq], x[:, Hq:Hq + Hkv]
    else:
        q, k = _randn(g, Hq, T, 128).transpose(0, 1), _randn(g, Hkv, T, 128).transpose(0, 1)
    qw, kw = 1 + _randn(g, 128, scale=0.3), 1 + _randn(g, 128, scale=0.3)
    cos, sin = _tables(torch.arange(T, device=DEV) + 5000)
    qo, ko = ops.qk_norm_rope(q, k, qw, kw, 1e-6, rope=(cos, sin))
    assert qo.shape == q.shape and ko.shape == k.shape
    _check_norm(qo, q, qw, 1e-6, cos, sin)
    _check_norm(ko, k, kw, 1e-6, cos, sin)


@pytest.mark.parametrize("pos_dtype", [torch.int32, torch.int64])
def test_norm_rope_batched_positions_and_padding(ops, pos_dtype):
    g = _gen(3)
    B, T, Hq, Hkv, P = 3, 37, 6, 2, 500
    q, k = _randn(g, B, T, Hq, 128), _randn(g, B, T, Hkv, 128)
    qw, kw = torch.randn(128, device=DEV, generator=g), 1 + _randn(g, 128)  # one fp32, one bf16 weight
    cos, sin = _tables(torch.arange(P, device=DEV))
    pos = torch.randint(0, P, (B, T), device=DEV, generator=g).to(pos_dtype)
    pos[0, :5] = pos[2, -3:] = -1  # padding
    qo, ko = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    ops.qk_norm_rope(q, k, qw, kw, 1e-5, rope=(cos, sin), positions=pos, q_out=qo, k_out=ko)
    live = pos >= 0
    at = pos.clamp(min=0).long()
    _check_norm(qo[live], q[live], qw, 1e-5, cos[at][live], sin[at][live])
    _check_norm(ko[live], k[live], kw, 1e-5, cos[at][live], sin[at][live])
    assert (qo[~live] == 7).all() and (ko[~live] == 7).all()
    assert ops.device_status() == 0


def test_norm_rope_position_outside_the_table_is_reported(ops):
    g = _gen(4)
    q = _randn(g, 4, 2, 128)
    cos, sin = _tables(torch.arange(10, device=DEV))
    for bad in (10, -2, 2 ** 31 - 1):
        pos = torch.tensor([0, 9, bad, 3], device=DEV, dtype=torch.int32)
        out = torch.full_like(q, 7.0)
        ops.qk_norm_rope(q, None, rope=(cos, sin), positions=pos, q_out=out)
        assert ops.device_status() == ops.STATUS_BAD_LAUNCH
        assert (out[2] == 7).all()
        rest = torch.tensor([0, 1, 3], device=DEV)
        _check_norm(out[rest], q[rest], None, 0, cos[pos[rest].long()], sin[pos[rest].long()])
    assert ops.device_status() == 0


@pytest.mark.parametrize("B,T,rope_batch", [(2, 50, 1), (3, 17, 3), (1, 1, 1)])
def test_norm_rope_per_token_tables_of_a_batch(ops, B, T, rope_batch):
    """[1|B, T, 128] angles, into views of a head-split cache [B, H, cap, 128]."""
    g = _gen(B * T)
    q, k = _randn(g, B, 8, T, 128).transpose(1, 2), _randn(g, B, 2, T, 128).transpose(1, 2)
    kw = 1 + _randn(g, 128, scale=0.2)
    cos, sin = _tables(torch.randint(0, 9000, (rope_batch, T), device=DEV, generator=g))
    cache = torch.full((B, 2, T + 9, 128), 7.0, device=DEV, dtype=torch.bfloat16)
    qo, _ = ops.qk_norm_rope(q, k, None, kw, 1e-6, rope=(cos, sin), k_out=cache[:, :, 4:4 + T].transpose(1, 2))
    _check_norm(qo, q, None, 0, cos.expand(B, T, 128), sin.expand(B, T, 128))
    _check_norm(cache[:, :, 4:4 + T].transpose(1, 2), k, kw, 1e-6, cos.expand(B, T, 128), sin.expand(B, T, 128))
    assert (cache[:, :, :4] == 7).all() and (cache[:, :, 4 + T:] == 7).all()


def test_norm_rope_parts_in_place_and_values(ops):
    g = _gen(9)
    T = 70
    x = _randn(g, T, 12, 128)
    w = 1 + _randn(g, 128, scale=0.2)
    cos, sin = _tables(torch.arange(T, device=DEV))
    only_norm, none = ops.qk_norm_rope(x, None, w, None, 1e-6)
    assert none is None
    _check_norm(only_norm, x, w, 1e-6, None, None)
    only_rope, _ = ops.qk_norm_rope(x, None, rope=(cos, sin))
    _check_norm(only_rope, x, None, 0, cos, sin)
    assert torch.equal(ops.qk_norm_rope(x, x[:, :3])[1], x[:, :3])  # neither: a copy
    y = x.clone()
    ops.qk_norm_rope(y[:, :8], y[:, 8:], w, w, 1e-6, rope=(cos, sin), q_out=y[:, :8], k_out=y[:, 8:])
    _check_norm(y, x, w, 1e-6, cos, sin)
    # all-zero rows, tiny rows (eps matters), one bad row that must stay alone
    z = x.clone()
    z[3] = 0
    z[4] *= 1e-4
    z[5, 2, 17] = float("nan")
    z[6, 1, 100] = float("inf")
    o, _ = ops.qk_norm_rope(z, None, w, None, 1e-6, rope=(cos, sin))
    bad = torch.zeros(T, 12, dtype=torch.bool, device=DEV)
    bad[5, 2] = bad[6, 1] = True
    assert torch.isfinite(o[~bad].float()).all() and not torch.isfinite(o[5, 2].float()).any()
    keep = torch.ones(T, dtype=torch.bool, device=DEV)
    keep[5:7] = False
    _check_norm(o[keep], z[keep], w, 1e-6, cos[keep], sin[keep])
    e, _ = ops.qk_norm_rope(x[:0], x[:0, :2], w, w)
    assert e.shape == (0, 12, 128)


# -------------------------------------------------------------- attn_varlen --
@pytest.mark.parametrize("q_lens,Hq,Hkv", [
    ([1], 1, 1), ([1], 32, 8), ([5, 8, 30, 6, 7], 28, 4), ([64], 2, 2), ([65, 63, 1, 128, 129], 7, 7),
    ([127, 0, 256, 0, 0, 257, 33], 10, 2), ([511, 513], 8, 1), ([300, 20], 40, 8), ([1100], 28, 4),
    ([40] * 70, 4, 2), ([200, 90], 80, 1), ([150], 130, 1), ([33, 47], 18, 6)])
@pytest.mark.parametrize("causal", [True, False])
def test_varlen_prompts(ops, q_lens, Hq, Hkv, causal):
    g = _gen(sum(q_lens) + Hq)
    T = sum(q_lens)
    x = _randn(g, T, Hq + 2 * Hkv, 128, scale=1.3)
    q, k, v = x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]
    o, lse = ops.attn_varlen(q, k, v, _cu(q_lens), _cu(q_lens), max_k=max(q_lens), causal=causal)
    assert o.shape == (T, Hq, 128) and lse.shape == (Hq, T)
    _check_varlen(o, lse, q, k, v, q_lens, q_lens, causal)
    assert ops.device_status() == 0


@pytest.mark.parametrize("q_lens,k_lens,Hq,Hkv", [
    ([1, 1, 1, 1], [1, 64, 65, 1000], 32, 8),                # single tokens
    ([1, 37, 1, 256], [3001, 700, 0, 4096], 28, 4),          # tokens and chunks behind a history, one without keys
    ([40, 3, 0, 90], [17, 3, 50, 0], 6, 2),                  # more queries than keys: rows that see nothing
    ([130, 260], [129, 1], 4, 4), ([2], [9000], 8, 1), ([1], [20000], 5, 1), ([7], [130], 16, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_varlen_histories(ops, q_lens, k_lens, Hq, Hkv, causal):
    g = _gen(sum(k_lens))
    q, k, v = _randn(g, sum(q_lens), Hq, 128), _randn(g, sum(k_lens), Hkv, 128), _randn(g, sum(k_lens), Hkv, 128)
    o, lse = ops.attn_varlen(q, k, v, _cu(q_lens), _cu(k_lens), causal=causal)
    _check_varlen(o, lse, q, k, v, q_lens, k_lens, causal)
    # a bound on the keys changes no result beyond the order of the sums
    o2, lse2 = ops.attn_varlen(q, k, v, _cu(q_lens), _cu(k_lens), max_k=max(k_lens), causal=causal)
    _check_varlen(o2, lse2, q, k, v, q_lens, k_lens, causal)
    assert ops.device_status() == 0


def test_varlen_wrong_bound_on_the_keys_changes_nothing(ops):
    g = _gen(17)
    q_lens, k_lens = [1, 30, 1], [5000, 900, 2100]
    q, k, v = _randn(g, 32, 8, 128), _randn(g, 8000, 2, 128), _randn(g, 8000, 2, 128)
    for max_k in (0, 1, 100, 10 ** 9):
        o, lse = ops.attn_varlen(q, k, v, _cu(q_lens), _cu(k_lens), max_k=max_k)
        _check_varlen(o, lse, q, k, v, q_lens, k_lens, True)


def test_varlen_layouts_scale_and_rows_outside(ops):
    """Head-split strided inputs, output into a padded view, a scale of its own; rows outside every sequence stay."""
    g = _gen(8)
    q_lens, k_lens, Hq, Hkv = [50, 1, 77], [90, 200, 77], 12, 4
    cap_q, cap_k = 140, 400
    q = _randn(g, Hq, cap_q, 128).transpose(0, 1)
    kv = _randn(g, 2, Hkv, cap_k, 128)
    k, v = kv[0].transpose(0, 1), kv[1].transpose(0, 1)
    cu_q, cu_k = _cu(q_lens) + 3, _cu(k_lens) + 11  # the first sequence does not start at row 0
    buf = torch.full((cap_q + 2, Hq, 192), 7.0, device=DEV, dtype=torch.bfloat16)
    out = buf[1:-1, :, 32:160]
    got, lse = ops.attn_varlen(q, k, v, cu_q, cu_k, scale=0.2, out=out)
    assert got.data_ptr() == out.data_ptr()
    n = sum(q_lens)
    _check_varlen(out[3:3 + n], lse[:, 3:3 + n], q[3:3 + n], k[11:], v[11:], q_lens, k_lens, True, 0.2)
    left = buf.clone()
    left[1:-1, :, 32:160][3:3 + n] = 7.0
    assert (left == 7).all()
    no, none = ops.attn_varlen(q, k, v, cu_q, cu_k, scale=0.2, want_lse=False)
    assert none is None and torch.equal(no[3:3 + n], out[3:3 + n])


@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf")])
def test_varlen_neighbours_have_no_influence(ops, poison):
    """Bad values in other sequences, behind the last one and in keys a causal row does not see stay where they are."""
    g = _gen(12)
    lens, Hq, Hkv = [70, 130, 45, 300], 8, 2
    T = sum(lens) + 60
    q, k, v = _randn(g, T, Hq, 128), _randn(g, T, Hkv, 128), _randn(g, T, Hkv, 128)
    cu = _cu(lens)
    clean, clean_lse = ops.attn_varlen(q, k, v, cu, cu)
    clean, clean_lse = clean.clone(), clean_lse.clone()
    k2, v2, q2 = k.clone(), v.clone(), q.clone()
    k2[70:200] = v2[70:200] = q2[70:200] = poison   # the second sequence
    k2[sum(lens):] = v2[sum(lens):] = q2[sum(lens):] = poison
    o, lse = ops.attn_varlen(q2, k2, v2, cu, cu)
    rows = [i for i in range(sum(lens)) if not 70 <= i < 200]
    assert torch.equal(o[rows], clean[rows]) and torch.equal(lse[:, rows], clean_lse[:, rows])
    # the last keys of the fourth sequence: earlier rows do not see them
    for first_bad in (540, 470, 373, 300):
        k3, v3 = k.clone(), v.clone()
        k3[first_bad:545] = v3[first_bad:545] = poison
        o, lse = ops.attn_varlen(q, k3, v3, cu, cu)
        assert torch.equal(o[:first_bad], clean[:first_bad]), first_bad
        assert torch.equal(lse[:, :first_bad], clean_lse[:, :first_bad])
        # and the rows that do see a bad value show it
        assert not torch.isfinite(o[first_bad:545].float()).all(-1).any()
    assert ops.device_status() == 0


def test_varlen_extreme_scores(ops):
    """Scores far apart: one key takes all the weight, however late it comes; the lowest finite values are values."""
    g = _gen(13)
    n = 700
    q, k, v = _randn(g, 3, 4, 128), _randn(g, n, 2, 128), _randn(g, n, 2, 128)
    k = k * 0.01
    for at in (0, 63, 64, 127, 128, 300, 697):
        k2 = k.clone()
        k2[at] = q[0, :1].expand(2, 128) * 40
        o, lse = ops.attn_varlen(q, k2, v, _cu([3]), _cu([n]))
        _check_varlen(o, lse, q, k2, v, [3], [n], True)
    big = torch.full_like(k, torch.finfo(torch.bfloat16).min)
    o, lse = ops.attn_varlen(q.abs() * 1e-38, big, v, _cu([3]), _cu([n]))
    _check_varlen(o, lse, q.abs() * 1e-38, big, v, [3], [n], True)


@pytest.mark.parametrize("cu_q,cu_k", [([0, 10, 5], [0, 10, 20]), ([0, 10, 41], [0, 10, 20]), ([-1, 10, 20], [0, 1, 2]),
                                       ([0, 10, 20], [0, 30, 20]), ([0, 10, 20], [0, 10, 2 ** 31 - 1])])
def test_varlen_bad_offsets_are_reported_and_nothing_is_written(ops, cu_q, cu_k):
    g = _gen(14)
    q, k = _randn(g, 40, 4, 128), _randn(g, 40, 2, 128)
    out = torch.full_like(q, 7.0)
    i32 = lambda x: torch.tensor(x, device=DEV, dtype=torch.int32)  # noqa: E731
    ops.attn_varlen(q, k, k, i32(cu_q), i32(cu_k), out=out)
    assert ops.device_status() == ops.STATUS_BAD_LAUNCH
    assert (out == 7).all()
    assert ops.device_status() == 0


def test_varlen_bad_offsets_late_in_a_long_list(ops):
    g = _gen(15)
    n = 100
    q, k = _randn(g, n, 4, 128), _randn(g, n, 2, 128)
    cu = torch.arange(n + 1, device=DEV, dtype=torch.int32)
    bad = cu.clone()
    bad[90] = 95
    out = torch.full_like(q, 7.0)
    ops.attn_varlen(q, k, k, cu, bad, out=out)
    assert ops.device_status() == ops.STATUS_BAD_LAUNCH
    assert (out == 7).all()


def test_varlen_nothing_to_do(ops):
    q, k = torch.zeros(4, 2, 128, device=DEV, dtype=torch.bfloat16), torch.zeros(0, 2, 128, device=DEV, dtype=torch.bfloat16)
    zero = torch.zeros(2, device=DEV, dtype=torch.int32)
    out = torch.full_like(q, 7.0)
    ops.attn_varlen(q, k, k, zero[:1], zero[:1], out=out)       # no sequence
    ops.attn_varlen(q, q, q, zero, zero, out=out)               # one empty sequence
    assert (out == 7).all()
    o, lse = ops.attn_varlen(q, k, k, zero + torch.tensor([0, 4], device=DEV, dtype=torch.int32), zero, out=out)
    assert (o == 0).all() and (lse == -math.inf).all()          # rows without keys
    assert ops.attn_varlen(q[:0], q, q, zero, zero)[0].shape == (0, 2, 128)


# ------------------------------------------------------- attn_decode_shared --
@pytest.mark.parametrize("B,Hq,Hkv,P,cap", [
    (1, 1, 1, 1, 1), (1, 32, 8, 100, 3), (4, 28, 4, 1000, 64), (3, 5, 1, 129, 70), (33, 10, 2, 517, 40),
    (64, 8, 2, 4100, 130), (2, 40, 8, 20000, 600), (5, 130, 1, 300, 20), (17, 16, 16, 64, 1), (300, 4, 4, 65, 5),
    (7, 14, 2, 0, 300), (7, 14, 2, 300, 0), (9, 23, 1, 2, 1025), (128, 7, 1, 700, 33)])
def test_shared(ops, B, Hq, Hkv, P, cap):
    g = _gen(B * 7 + P)
    q = _randn(g, B, Hq, 128, scale=1.5)
    kp, vp = _randn(g, Hkv, P, 128), _randn(g, Hkv, P, 128)
    k, v = _randn(g, B, Hkv, cap, 128), _randn(g, B, Hkv, cap, 128)
    lens = torch.randint(0, cap + 1, (B,), device=DEV, generator=g, dtype=torch.int32)
    lens[0] = cap
    lens[-1] = 0 if P else min(1, cap)
    o, lse = ops.attn_decode_shared(q, kp, vp, k, v, lens)
    assert o.shape == (B, 1, Hq, 128) and lse.shape == (B, Hq)
    _check_shared(o, lse, q, kp, vp, k, v, lens.tolist())
    assert ops.device_status() == 0


def test_shared_without_lens_equals_decode_of_the_whole(ops):
    g = _gen(31)
    B, Hq, Hkv, P, cap = 6, 28, 4, 900, 77
    q = _randn(g, B, Hq, 1, 128)
    kp, vp = _randn(g, 1, Hkv, P, 128), _randn(g, 1, Hkv, P, 128)
    k, v = _randn(g, B, Hkv, cap, 128), _randn(g, B, Hkv, cap, 128)
    o, lse = ops.attn_decode_shared(q, kp, vp, k, v)
    _check_shared(o, lse, q[:, :, 0], kp[0], vp[0], k, v, [cap] * B)
    whole, whole_lse = ops.attn_decode(q, torch.cat([kp.expand(B, -1, -1, -1), k], 2),
                                       torch.cat([vp.expand(B, -1, -1, -1), v], 2))
    assert (o.float() - whole.float()).abs().max() <= 4 * H_BF16 * whole.float().abs().max()
    assert (lse - whole_lse).abs().max() <= 1e-4


def test_shared_unused_slots_and_lens_out_of_range(ops):
    g = _gen(32)
    B, Hq, Hkv, P, cap = 5, 14, 2, 200, 150
    q = _randn(g, B, Hq, 128)
    kp, vp = _randn(g, Hkv, P, 128), _randn(g, Hkv, P, 128)
    k, v = _randn(g, B, Hkv, cap, 128), _randn(g, B, Hkv, cap, 128)
    want = [0, 1, 64, 99, cap]
    for b, n in enumerate(want):
        k[b, :, n:] = float("nan")
        v[b, :, n:] = float("inf")
    lens = torch.tensor([-5, 1, 64, 99, 10 ** 6], device=DEV, dtype=torch.int32)
    o, lse = ops.attn_decode_shared(q, kp, vp, k, v, lens)
    _check_shared(o, lse, q, kp, vp, k, v, want)
    # no prefix either: the request without keys gives zeros and -inf
    o, lse = ops.attn_decode_shared(q, kp[:, :0], vp[:, :0], k, v, lens)
    assert (o[0] == 0).all() and (lse[0] == -math.inf).all()
    _check_shared(o[1:], lse[1:], q[1:], kp[:, :0], vp[:, :0], k[1:], v[1:], want[1:])
    o, lse = ops.attn_decode_shared(q, kp[:, :0], vp[:, :0], k[:, :, :0], v[:, :, :0])
    assert (o == 0).all() and (lse == -math.inf).all()


def test_shared_strided_views_and_out(ops):
    g = _gen(33)
    B, Hq, Hkv, P, cap = 9, 12, 4, 333, 50
    q = _randn(g, Hq, B, 128).transpose(0, 1)
    pre = _randn(g, P, 2 * Hkv, 128)            # token-major prefix, k and v side by side
    kp, vp = pre[:, :Hkv].transpose(0, 1), pre[:, Hkv:].transpose(0, 1)
    big = _randn(g, 2, B, Hkv, 128, 128)
    k, v = big[0][:, :, 10:10 + cap], big[1][:, :, 10:10 + cap]
    lens = torch.randint(0, cap + 1, (B,), device=DEV, generator=g, dtype=torch.int32)
    buf = torch.full((B, 2, Hq, 128), 7.0, device=DEV, dtype=torch.bfloat16)
    o, lse = ops.attn_decode_shared(q, kp, vp, k, v, lens, scale=0.15, out=buf[:, 1:])
    _check_shared(buf[:, 1:], lse, q, kp, vp, k, v, lens.tolist(), 0.15)
    assert (buf[:, 0] == 7).all()
    o2, none = ops.attn_decode_shared(q, kp, vp, k, v, lens, scale=0.15, want_lse=False)
    assert none is None and torch.equal(o2, o)


@pytest.mark.parametrize("B,Hq,Hkv,P,cap", [
    (40, 8, 2, 0, 600), (40, 8, 2, 500, 0), (37, 4, 1, 1000, 1048), (37, 4, 1, 1000, 1049), (38, 4, 1, 1000, 30),
    (1, 16, 1, 63, 1), (2, 8, 8, 2047, 1), (2, 17, 1, 200, 200), (1, 40, 2, 1, 0), (1, 4, 4, 0, 513), (6, 8, 8, 9, 1300)])
def test_shared_around_the_limits(ops, B, Hq, Hkv, P, cap):
    """Sizes on both sides of where the work is cut differently, every length of the own keys from none to all."""
    g = _gen(B * 11 + P + cap)
    q, kp, vp = _randn(g, B, Hq, 128, scale=1.5), _randn(g, Hkv, P, 128), _randn(g, Hkv, P, 128)
    k, v = _randn(g, B, Hkv, cap, 128), _randn(g, B, Hkv, cap, 128)
    n = [i * cap // max(1, B - 1) for i in range(B)]
    for b in range(B):
        k[b, :, n[b]:], v[b, :, n[b]:] = float("nan"), float("inf")
    o, lse = ops.attn_decode_shared(q, kp, vp, k, v, torch.tensor(n, device=DEV, dtype=torch.int32))
    _check_shared(o, lse, q, kp, vp, k, v, n)
    assert ops.device_status() == 0


@pytest.mark.parametrize("B,P,cap", [(3, 70, 40000), (40, 300, 9000), (24, 9000, 5000)])
def test_shared_caches_with_much_room(ops, B, P, cap):
    g = _gen(36)
    Hq, Hkv = 8, 2
    q, kp, vp = _randn(g, B, Hq, 128), _randn(g, Hkv, P, 128), _randn(g, Hkv, P, 128)
    k, v = _randn(g, B, Hkv, cap, 128), _randn(g, B, Hkv, cap, 128)
    n = torch.randint(0, cap + 1, (B,), device=DEV, generator=g, dtype=torch.int32)
    n[0], n[1], n[2] = cap, 0, 1
    for b, x in enumerate(n.tolist()):
        k[b, :, x:], v[b, :, x:] = float("nan"), float("inf")
    o, lse = ops.attn_decode_shared(q, kp, vp, k, v, n)
    _check_shared(o, lse, q, kp, vp, k, v, n.tolist())
    assert ops.device_status() == 0


@pytest.mark.parametrize("P", [333, 6000])
def test_shared_strided_views_of_a_large_batch(ops, P):
    g = _gen(34)
    B, Hq, Hkv, cap = 64, 12, 4, 50
    q = _randn(g, Hq, B, 128).transpose(0, 1)
    pre = _randn(g, P, 2 * Hkv, 128)
    kp, vp = pre[:, :Hkv].transpose(0, 1), pre[:, Hkv:].transpose(0, 1)
    big = _randn(g, 2, B, 128, Hkv, 128).transpose(2, 3)
    k, v = big[0][:, :, 10:10 + cap], big[1][:, :, 10:10 + cap]
    lens = torch.randint(0, cap + 1, (B,), device=DEV, generator=g, dtype=torch.int32)
    buf = torch.full((B, 2, Hq, 192), 7.0, device=DEV, dtype=torch.bfloat16)
    _, lse = ops.attn_decode_shared(q, kp, vp, k, v, lens, scale=0.15, out=buf[:, 1:, :, 32:160])
    _check_shared(buf[:, 1:, :, 32:160], lse, q, kp, vp, k, v, lens.tolist(), 0.15)
    buf[:, 1:, :, 32:160] = 7.0
    assert (buf == 7).all()


@pytest.mark.parametrize("B,P", [(2, 100), (60, 100), (60, 6000)])
def test_shared_bad_values_show_in_the_rows_that_see_them(ops, B, P):
    g = _gen(35)
    Hq, Hkv, cap = 8, 2, 70
    q, kp, vp = _randn(g, B, Hq, 128), _randn(g, Hkv, P, 128), _randn(g, Hkv, P, 128)
    k, v = _randn(g, B, Hkv, cap, 128), _randn(g, B, Hkv, cap, 128)
    want, want_lse = ops.attn_decode_shared(q, kp, vp, k, v)
    for poison in (float("nan"), float("inf")):
        v2, k2 = v.clone(), k.clone()
        v2[1, 0, 69, 5] = poison          # one channel of one request's kv head
        k2[0, 1, 3, 7] = float("nan")     # one key: all of its heads' channels
        o, lse = ops.attn_decode_shared(q, kp, vp, k2, v2)
        assert not torch.isfinite(o[1, 0, :4, 5].float()).any() and torch.isnan(o[0, 0, 4:].float()).all()
        o[1, 0, :4, 5], o[0, 0, 4:], lse[0, 4:] = want[1, 0, :4, 5], want[0, 0, 4:], want_lse[0, 4:]
        assert torch.equal(o, want) and torch.equal(lse, want_lse)
        vp2 = vp.clone()
        vp2[1, P // 2, 9] = poison
        o, _ = ops.attn_decode_shared(q, kp, vp2, k, v)
        assert not torch.isfinite(o[:, 0, 4:, 9].float()).any()
        o[:, 0, 4:, 9] = want[:, 0, 4:, 9]
        assert torch.equal(o, want)


# ---------------------------------------------------- long lists, large sizes --
def _check_varlen_heads(o, lse, q, k, v, q_lens, k_lens, causal=True, scale=128 ** -0.5):
    """_check_varlen with all heads of a sequence at once."""
    G = q.shape[1] // k.shape[1]
    q0 = k0 = 0
    for i, (lq, lk) in enumerate(zip(q_lens, k_lens)):
        qq = q[q0:q0 + lq].double().transpose(0, 1)
        kk = k[k0:k0 + lk].double().transpose(0, 1).repeat_interleave(G, 0)
        vv = v[k0:k0 + lk].double().transpose(0, 1).repeat_interleave(G, 0)
        sc = qq @ kk.transpose(1, 2) * scale
        if causal:
            see = torch.arange(lk, device=DEV)[None] <= torch.arange(lq, device=DEV)[:, None] + lk - lq
            sc = sc.masked_fill(~see, -math.inf)
        rl = torch.logsumexp(sc, -1)
        p = torch.exp(sc - rl.masked_fill(rl == -math.inf, 0.0)[..., None])
        _check_attn(o[q0:q0 + lq].transpose(0, 1), lse[:, q0:q0 + lq], p @ vv, p @ vv.abs(), rl, what=(i, lq, lk))
        q0, k0 = q0 + lq, k0 + lk


@pytest.mark.parametrize("n,most,hist,Hq,Hkv", [
    (1500, 30, 0, 2, 1),      # more sequences than the plan keeps on chip
    (2100, 1, 90, 4, 2),      # ... of one token
    (500, 40, 60, 32, 32),    # more items than one launch takes
    (1200, 3, 200, 4, 1)])
def test_varlen_long_lists(ops, n, most, hist, Hq, Hkv):
    g = _gen(n)
    r = torch.Generator().manual_seed(n)
    q_lens = torch.randint(0 if most > 1 else 1, most + 1, (n,), generator=r).tolist()
    k_lens = [x + y for x, y in zip(q_lens, torch.randint(0, hist + 1, (n,), generator=r).tolist())]
    q = _randn(g, sum(q_lens), Hq, 128)
    k, v = _randn(g, sum(k_lens), Hkv, 128), _randn(g, sum(k_lens), Hkv, 128)
    o, lse = ops.attn_varlen(q, k, v, _cu(q_lens), _cu(k_lens))
    _check_varlen_heads(o, lse, q, k, v, q_lens, k_lens)
    assert ops.device_status() == 0


def test_varlen_bad_offset_behind_a_thousand(ops):
    g = _gen(16)
    n = 1400
    q, k = _randn(g, n, 4, 128), _randn(g, n, 2, 128)
    cu = torch.arange(n + 1, device=DEV, dtype=torch.int32)
    for at in (1024, 1025, 1399):
        bad = cu.clone()
        bad[at] = n + 1
        out = torch.full_like(q, 7.0)
        ops.attn_varlen(q, k, k, cu, bad, out=out)
        assert ops.device_status() == ops.STATUS_BAD_LAUNCH
        assert (out == 7).all()


@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("Hq,Hkv", [(4, 1), (2, 2)])
def test_varlen_few_tokens_do_not_see_later_keys(ops, poison, Hq, Hkv):
    """Two to four tokens behind long histories: a bad last key reaches the last token only, parts and joins included."""
    g = _gen(18)
    q_lens, k_lens = [2, 4, 1, 3, 4], [700, 9000, 64, 3, 4097]
    q, k, v = _randn(g, 14, Hq, 128), _randn(g, sum(k_lens), Hkv, 128), _randn(g, sum(k_lens), Hkv, 128)
    cu_q, cu_k = _cu(q_lens), _cu(k_lens)
    want, want_lse = ops.attn_varlen(q, k, v, cu_q, cu_k)
    _check_varlen(want, want_lse, q, k, v, q_lens, k_lens, True)
    ends = (cu_k[1:] - 1).long()
    k[ends] = v[ends] = poison
    o, lse = ops.attn_varlen(q, k, v, cu_q, cu_k)
    last = (cu_q[1:] - 1).long()
    rest = [i for i in range(14) if i not in last.tolist()]
    assert torch.equal(o[rest], want[rest]) and torch.equal(lse[:, rest], want_lse[:, rest])
    assert not torch.isfinite(o[last].float()).all(-1).any()


@pytest.mark.parametrize("q_lens,k_lens,Hq,Hkv", [
    ([2, 4, 1, 3, 4], [700, 900, 64, 3, 1097], 4, 1), ([1], [8000], 32, 8), ([1], [12001], 8, 8),
    ([0, 1, 0, 7], [5, 3000, 0, 9], 20, 1), ([33], [1500], 16, 1), ([1, 1], [513, 512], 40, 8), ([40, 3], [450, 1], 4, 4),
    ([16], [4000], 32, 8), ([130], [900], 1, 1), ([1] * 8, [1000] * 7 + [1], 32, 8), ([6, 90], [400, 40], 5, 1),
    ([1] * 3, [0, 0, 4000], 8, 2), ([17, 1], [16, 2000], 7, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_varlen_few_rows(ops, q_lens, k_lens, Hq, Hkv, causal):
    """Few rows behind short to long histories, the longest given; a bad last key reaches its own row only."""
    g = _gen(sum(k_lens) + Hq)
    Tq = sum(q_lens)
    q, k, v = _randn(g, Tq, Hq, 128), _randn(g, sum(k_lens), Hkv, 128), _randn(g, sum(k_lens), Hkv, 128)
    cu_q, cu_k = _cu(q_lens), _cu(k_lens)
    buf = torch.full((Tq + 2, Hq, 128), 7.0, device=DEV, dtype=torch.bfloat16)
    o, lse = ops.attn_varlen(q, k, v, cu_q, cu_k, max_k=max(k_lens), causal=causal, out=buf[1:-1])
    _check_varlen(o, lse, q, k, v, q_lens, k_lens, causal)
    assert (buf[0] == 7).all() and (buf[-1] == 7).all()
    want, want_lse = o.clone(), lse.clone()
    ends = [int(cu_k[i + 1]) - 1 for i, (a, b) in enumerate(zip(q_lens, k_lens)) if a and b]
    last = [int(cu_q[i + 1]) - 1 for i, (a, b) in enumerate(zip(q_lens, k_lens)) if a and b]
    rest = [i for i in range(Tq) if i not in last]
    for poison in (float("nan"), -float("inf")):
        k2, v2 = k.clone(), v.clone()
        k2[ends] = v2[ends] = poison
        o, lse = ops.attn_varlen(q, k2, v2, cu_q, cu_k, max_k=max(k_lens), causal=causal)
        if causal:
            assert torch.equal(o[rest], want[rest]) and torch.equal(lse[:, rest], want_lse[:, rest])
        assert not torch.isfinite(o[last].float()).all(-1).any()
    bad = cu_k.clone()
    bad[-1] = sum(k_lens) + 1
    out = torch.full_like(q, 7.0)
    ops.attn_varlen(q, k, v, cu_q, bad, max_k=max(k_lens), causal=causal, out=out)
    assert ops.device_status() == ops.STATUS_BAD_LAUNCH and (out == 7).all()


@pytest.mark.parametrize("q_lens,k_lens", [([3, 40], [3, 40]), ([1, 1, 1], [9000, 30, 4000]), ([300, 700], [900, 800])])
def test_varlen_expanded_views(ops, q_lens, k_lens):
    """One kv head under all, one query row for all heads or tokens: strides of zero."""
    g = _gen(19)
    Tq, Tk = sum(q_lens), sum(k_lens)
    cu_q, cu_k = _cu(q_lens), _cu(k_lens)
    q, k, v = _randn(g, Tq, 8, 128), _randn(g, Tk, 4, 128), _randn(g, Tk, 4, 128)
    one_k, one_v = k[:, :1].expand(Tk, 4, 128), v[:, :1].expand(Tk, 4, 128)
    for qq, kk, vv in ((q, one_k, one_v), (q[:, :1].expand(Tq, 8, 128), k, v), (q[:1].expand(Tq, 8, 128), k, v),
                       (q, k[:1].expand(Tk, 4, 128), v[:1].expand(Tk, 4, 128))):
        o, lse = ops.attn_varlen(qq, kk, vv, cu_q, cu_k)
        _check_varlen_heads(o, lse, qq, kk, vv, q_lens, k_lens)


@pytest.mark.parametrize("B,P", [(3, 150), (40, 5000)])
def test_shared_expanded_views(ops, B, P):
    g = _gen(20)
    Hq, Hkv, cap = 8, 4, 70
    q, kp, vp = _randn(g, B, Hq, 128), _randn(g, Hkv, P, 128), _randn(g, Hkv, P, 128)
    k, v = _randn(g, B, Hkv, cap, 128), _randn(g, B, Hkv, cap, 128)
    lens = [cap] * B
    for qq, a, b in ((q[:1].expand(B, Hq, 128), kp, vp), (q, kp[:1].expand(Hkv, P, 128), vp[:1].expand(Hkv, P, 128)),
                     (q[:, :1].expand(B, Hq, 128), kp[:, :1].expand(Hkv, P, 128), vp[:, :1].expand(Hkv, P, 128))):
        for kk, vv in ((k, v), (k[:1].expand(B, Hkv, cap, 128), v[:1].expand(B, Hkv, cap, 128))):
            o, lse = ops.attn_decode_shared(qq, a, b, kk, vv)
            _check_shared(o, lse, qq, a, b, kk, vv, lens)


def test_offsets_past_32_bits(ops):
    """Rows behind the 2^31st element of a cache; every path, and a request's own slots that far out."""
    g = _gen(21)
    rows = 2 ** 31 // (8 * 128) + 4096
    cache = torch.empty(rows, 8, 128, device=DEV, dtype=torch.bfloat16)
    tail = 4000
    cache[-tail:] = _randn(g, tail, 8, 128)
    end = rows - tail
    for q_lens, k_lens in (([5], [40]), ([1, 1], [2000, 1900]), ([900, 30], [2000, 2000])):
        q = _randn(g, sum(q_lens), 16, 128)
        o, lse = ops.attn_varlen(q, cache, cache, _cu(q_lens), _cu(k_lens) + end, max_k=max(k_lens))
        _check_varlen_heads(o, lse, q, cache[end:], cache[end:], q_lens, k_lens)
    # two requests, the second one's slots at the end of the cache; the prefix there too
    own = cache.as_strided((2, 8, 100, 128), ((rows - 100) * 1024, 128, 1024, 1))
    cache[:100] = _randn(g, 100, 8, 128)
    for P in (300, 4000):
        pre = cache[-P:].transpose(0, 1)
        q = _randn(g, 2, 32, 128)
        o, lse = ops.attn_decode_shared(q, pre, pre, own, own)
        _check_shared(o, lse, q, pre, pre, own, own, [100, 100])
    big = cache[rows // 2:]
    w = 1 + _randn(g, 128, scale=0.2)
    cos, sin = _tables(torch.arange(big.shape[0], device=DEV))
    out = torch.empty(rows, 8, 128, device=DEV, dtype=torch.bfloat16)[rows // 2:]
    ops.qk_norm_rope(big, None, w, None, 1e-6, rope=(cos, sin), q_out=out)
    _check_norm(out[-tail:], big[-tail:], w, 1e-6, cos[-tail:], sin[-tail:])
    assert ops.device_status() == 0


# ---------------------------------------------------------------- refusals --
def test_refusals(ops):
    bf = lambda *s: torch.zeros(*s, device=DEV, dtype=torch.bfloat16)  # noqa: E731
    cu = torch.tensor([0, 4], device=DEV, dtype=torch.int32)
    cos = torch.zeros(4, 128, device=DEV)
    q, k = bf(4, 4, 128), bf(4, 2, 128)
    bad = [
        (ops.qk_norm_rope, (q.half(), k), {}, "bfloat16"),
        (ops.qk_norm_rope, (bf(4, 4, 64), k), {}, "128"),
        (ops.qk_norm_rope, (q, bf(5, 2, 128)), {}, "q's shape"),
        (ops.qk_norm_rope, (q, k, bf(64)), {}, "weights"),
        (ops.qk_norm_rope, (q, k, bf(128).half()), {}, "weights"),
        (ops.qk_norm_rope, (q, k), dict(positions=cu), "tables"),
        (ops.qk_norm_rope, (q, k), dict(rope=(cos, cos), positions=cu), "token shape"),
        (ops.qk_norm_rope, (q, k), dict(rope=(cos[:3], cos[:3])), "rope"),
        (ops.qk_norm_rope, (q, k), dict(q_out=bf(4, 5, 128)), "q_out"),
        (ops.qk_norm_rope, (q, k), dict(k_out=bf(1, 2, 128).expand(4, 2, 128)), "expanded"),
        (ops.qk_norm_rope, (bf(4, 4, 256)[:, :, ::2], k), {}, "contiguous"),
        (ops.qk_norm_rope, (bf(4 * 4 * 128 + 4)[4:].view(4, 4, 128), None), {}, "16-byte"),
        (ops.attn_varlen, (q, k, k, cu.long(), cu.long()), {}, "int32"),
        (ops.attn_varlen, (q, k, k, cu, torch.cat([cu, cu])), {}, "same sequences"),
        (ops.attn_varlen, (q, bf(4, 3, 128), bf(4, 3, 128), cu, cu), {}, "multiple"),
        (ops.attn_varlen, (q, k, bf(4, 4, 128)[:, :2], cu, cu), {}, "strides"),
        (ops.attn_varlen, (q, k.float(), k.float(), cu, cu), {}, "bfloat16"),
        (ops.attn_varlen, (q, k, k, cu, cu), dict(max_k=-1), "max_k"),
        (ops.attn_varlen, (q, k, k, cu, cu), dict(out=bf(4, 4, 64)), "out"),
        (ops.attn_varlen, (q, k, k, cu, cu), dict(scale=float("nan")), "scale"),
        (ops.attn_varlen, (q, k, k, cu.cpu(), cu), {}, "CUDA"),
        (ops.attn_varlen, (bf(1, 4, 4, 128), k, k, cu, cu), {}, "expected"),
        (ops.attn_decode_shared, (bf(4, 4, 2, 128), bf(2, 9, 128), bf(2, 9, 128), bf(4, 2, 5, 128), bf(4, 2, 5, 128)), {},
         "one query token"),
        (ops.attn_decode_shared, (q, bf(2, 9, 128), bf(2, 8, 128), bf(4, 2, 5, 128), bf(4, 2, 5, 128)), {}, "same shape"),
        (ops.attn_decode_shared, (q, bf(2, 9, 128), bf(2, 9, 128), bf(3, 2, 5, 128), bf(3, 2, 5, 128)), {}, "batch"),
        (ops.attn_decode_shared, (q, bf(2, 9, 128), bf(2, 9, 128), bf(4, 2, 5, 128), bf(4, 2, 5, 128), cu), {}, "lens"),
        (ops.attn_decode_shared, (q, bf(3, 9, 128), bf(3, 9, 128), bf(4, 3, 5, 128), bf(4, 3, 5, 128)), {}, "multiple"),
    ]
    for fn, args, kw, word in bad:
        with pytest.raises(RuntimeError, match=word):
            fn(*args, **kw)


# ------------------------------------------------- streams, graphs, together --
def _calls(ops, g, B=6, Hq=8, Hkv=2):
    """One call of each operator on inputs of its own, as closures over static buffers."""
    lens = [3, 100, 40, 1, 260, 17]
    T = sum(lens)
    x = _randn(g, T, Hq + 2 * Hkv, 128)
    w = 1 + _randn(g, 128, scale=0.1)
    cos, sin = _tables(torch.arange(300, device=DEV))
    pos = torch.cat([torch.arange(n, device=DEV) for n in lens]).int()
    cu, cu_k = _cu(lens), _cu([n + 2000 for n in lens])
    kv = _randn(g, 2, T + 2000 * len(lens), Hkv, 128)
    kp, k = _randn(g, 2, Hkv, 1500, 128), _randn(g, 2, B, Hkv, 90, 128)
    n_own = torch.randint(0, 91, (B,), device=DEV, generator=g, dtype=torch.int32)
    qd = _randn(g, B, Hq, 128)

    def run():
        a = ops.qk_norm_rope(x[:, :Hq], x[:, Hq:Hq + Hkv], w, w, 1e-6, rope=(cos, sin), positions=pos)
        b = ops.attn_varlen(a[0], a[1], x[:, Hq + Hkv:].contiguous(), cu, cu, max_k=260)
        c = ops.attn_varlen(a[0], kv[0], kv[1], cu, cu_k)
        d = ops.attn_decode_shared(qd, kp[0], kp[1], k[0], k[1], n_own)
        return [*a, *b, *c, *d]

    return run, (x, kv, kp, k, qd)


def test_repeated_calls_give_the_same_bits(ops):
    run, _ = _calls(ops, _gen(50))
    first = [t.clone() for t in run()]
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, run()))


def test_other_streams(ops):
    """Two streams at once, each with its own inputs, give what one stream gives."""
    runs = [_calls(ops, _gen(60 + i))[0] for i in range(2)]
    want = [[t.clone() for t in r()] for r in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in runs]
    got = [None, None]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = runs[i]()
    torch.cuda.synchronize()
    for w, o in zip(want, got):
        assert all(torch.equal(a, b) for a, b in zip(w, o))
    assert ops.device_status() == 0


def test_captured_graphs_replay_with_new_inputs_and_side_by_side(ops):
    made = [_calls(ops, _gen(70 + i)) for i in range(2)]
    graphs, outs = [], []
    for run, _ in made:
        run()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            run()
        torch.cuda.current_stream().wait_stream(s)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(run())
        graphs.append(gr)
    for step in range(3):
        for i, (_, bufs) in enumerate(made):
            g = _gen(100 * step + i)
            for b in bufs:
                b.copy_(_randn(g, *b.shape))
        want = [[t.clone() for t in run()] for run, _ in made]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for s, gr in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
                gr.replay()
        torch.cuda.synchronize()
        for w, o in zip(want, outs):
            assert all(torch.equal(a, b) for a, b in zip(w, o))
    assert ops.device_status() == 0


@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (7, 1)])
def test_a_packed_serving_step(ops, Hq, Hkv):
    """The three together, as a server uses them: a shared prompt is computed once and kept, three questions follow it
    as packed sequences, then every request decodes two tokens behind prompt and question. Each token's output has to
    be the plain causal attention over its whole sequence (roped, normed keys in bf16, as the caches hold them)."""
    g = _gen(80)
    P, q_lens, steps = 150, [5, 64, 33], 2
    B = len(q_lens)
    cap = max(q_lens) + steps
    seqs = [_randn(g, P, Hq + 2 * Hkv, 128)]                                  # the prompt's projections
    tails = [_randn(g, n + steps, Hq + 2 * Hkv, 128) for n in q_lens]         # the requests' own
    qw, kw = 1 + _randn(g, 128, scale=0.2), 1 + _randn(g, 128, scale=0.2)
    rope = _tables(torch.arange(P + cap, device=DEV))

    def norm(x, pos):
        return ops.qk_norm_rope(x[:, :Hq], x[:, Hq:Hq + Hkv], qw, kw, 1e-6, rope=rope, positions=pos)

    # the prompt: its keys and values become the shared prefix
    pq, pk = norm(seqs[0], torch.arange(P, device=DEV))
    pv = seqs[0][:, Hq + Hkv:]
    ops.attn_varlen(pq, pk.contiguous(), pv.contiguous(), _cu([P]), _cu([P]))
    k_prefix, v_prefix = pk.transpose(0, 1).contiguous(), pv.transpose(0, 1).contiguous()
    # the questions, packed, each behind the prompt
    x = torch.cat([t[:n] for t, n in zip(tails, q_lens)])
    pos = torch.cat([torch.arange(P, P + n, device=DEV) for n in q_lens])
    q, k = norm(x, pos)
    v = x[:, Hq + Hkv:]
    parts_q, parts_k, parts_v = q.split(q_lens), k.split(q_lens), v.split(q_lens)
    k_all = torch.cat([torch.cat([pk, t]) for t in parts_k])
    v_all = torch.cat([torch.cat([pv, t]) for t in parts_v])
    k_lens = [P + n for n in q_lens]
    o, lse = ops.attn_varlen(q, k_all, v_all, _cu(q_lens), _cu(k_lens), max_k=max(k_lens))
    _check_varlen(o, lse, q, k_all, v_all, q_lens, k_lens, True)
    # decode: own caches behind the shared prefix
    kc = torch.full((B, Hkv, cap, 128), float("nan"), device=DEV, dtype=torch.bfloat16)
    vc = torch.full_like(kc, float("nan"))
    for b, n in enumerate(q_lens):
        kc[b, :, :n], vc[b, :, :n] = parts_k[b].transpose(0, 1), parts_v[b].transpose(0, 1)
    lens = torch.tensor(q_lens, device=DEV, dtype=torch.int32)
    for t in range(steps):
        x1 = torch.stack([s[n + t] for s, n in zip(tails, q_lens)])
        q1, k1 = norm(x1, P + lens)
        _check_norm(k1, x1[:, Hq:Hq + Hkv], kw, 1e-6, rope[0][(P + lens).long()], rope[1][(P + lens).long()])
        at = lens.long()
        kc[torch.arange(B), :, at], vc[torch.arange(B), :, at] = k1, x1[:, Hq + Hkv:]
        lens += 1
        od, ld = ops.attn_decode_shared(q1, k_prefix, v_prefix, kc, vc, lens)
        _check_shared(od, ld, q1, k_prefix, v_prefix, kc, vc, lens.tolist())
    assert ops.device_status() == 0


# ------------------------------------------------------ scales next to zero --
# Every path: found in the kernel, clusters, plan of few rows (cut along the keys), pairs of CTAs (direct and cut).
SCALE_CASES = [
    ([5, 8, 30], [5, 8, 30], 8, 2), ([1], [4000], 32, 8), ([1] * 40, [37 * i + 11 for i in range(40)], 32, 8),
    ([1, 2], [9000, 30000], 8, 1), ([700, 300, 33], [700, 300, 33], 8, 2), ([260], [9001], 4, 4),
    ([300, 40], [100, 900], 16, 4)]


@pytest.mark.parametrize("q_lens,k_lens,Hq,Hkv", SCALE_CASES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("scale", [0.0, 1e-39, 1e-30])
def test_varlen_scales_next_to_zero(ops, q_lens, k_lens, Hq, Hkv, causal, scale):
    """Equal weights for all keys that a row sees: masked scores stay out whatever the scale multiplies them by."""
    g = _gen(sum(k_lens))
    q, k, v = _randn(g, sum(q_lens), Hq, 128), _randn(g, sum(k_lens), Hkv, 128), _randn(g, sum(k_lens), Hkv, 128)
    o, lse = ops.attn_varlen(q, k, v, _cu(q_lens), _cu(k_lens), max_k=max(k_lens), causal=causal, scale=scale)
    _check_varlen_heads(o, lse, q, k, v, q_lens, k_lens, causal, scale)
    assert ops.device_status() == 0


@pytest.mark.parametrize("B,Hq,Hkv,P,cap", [(2, 8, 2, 100, 70), (40, 8, 2, 700, 600), (60, 8, 2, 6001, 70),
                                            (33, 40, 8, 5003, 0), (1, 4, 4, 70000, 5)])
@pytest.mark.parametrize("scale", [0.0, 1e-39, 1e-30])
def test_shared_scales_next_to_zero(ops, B, Hq, Hkv, P, cap, scale):
    g = _gen(B + P)
    q, kp, vp = _randn(g, B, Hq, 128), _randn(g, Hkv, P, 128), _randn(g, Hkv, P, 128)
    k, v = _randn(g, B, Hkv, cap, 128), _randn(g, B, Hkv, cap, 128)
    n = [i * cap // B for i in range(B)]
    o, lse = ops.attn_decode_shared(q, kp, vp, k, v, torch.tensor(n, device=DEV, dtype=torch.int32), scale=scale)
    _check_shared(o, lse, q, kp, vp, k, v, n, scale)
    assert ops.device_status() == 0


# ------------------------------------- bad values in V alone, K left finite --
def _check_bad_v(ops, q, k, v, q_lens, k_lens, Hkv, spots, want, want_lse, **kw):
    """spots: (sequence, key of it, kv head, channel, value) with different channels. The value shows, in this channel
    of the rows and heads that see the key and nowhere else; everything else keeps its bits."""
    G = q.shape[1] // Hkv
    cu_q, cu_k = _cu(q_lens), _cu(k_lens)
    q0, k0 = cu_q.tolist(), cu_k.tolist()
    v2, expect = v.clone(), want.clone()
    for s, key, hk, ch, x in spots:
        v2[k0[s] + key, hk, ch] = x
        first = max(0, key + q_lens[s] - k_lens[s])
        expect[q0[s] + first:q0[s + 1], hk * G:(hk + 1) * G, ch] = x
    o, lse = ops.attn_varlen(q, k, v2, cu_q, cu_k, **kw)
    assert torch.equal(torch.nan_to_num(o, 7e4, 8e4, 9e4), torch.nan_to_num(expect, 7e4, 8e4, 9e4)), (
        (o != expect) & ~(o.isnan() & expect.isnan())).nonzero()[:8].tolist()
    assert torch.equal(lse, want_lse)


BAD = (float("nan"), float("inf"), -float("inf"))


def test_varlen_bad_values_in_the_first_tile(ops):
    """Prompts so short that their first tile holds masked keys: what the rows that see a bad value get is decided before
    the first product."""
    g = _gen(90)
    q_lens, Hq, Hkv = [5, 8, 30, 64, 17], 8, 2
    T = sum(q_lens)
    q, k, v = _randn(g, T, Hq, 128), _randn(g, T, Hkv, 128), _randn(g, T, Hkv, 128)
    want, want_lse = ops.attn_varlen(q, k, v, _cu(q_lens), _cu(q_lens), max_k=64)
    _check_varlen(want, want_lse, q, k, v, q_lens, q_lens, True)
    for i in range(60):
        spots = [(s, (7 * i + 3 * s + hk) % n, hk, (31 * i + 5 * s) % 128, BAD[(i + s + hk) % 3])
                 for s, n in enumerate(q_lens) for hk in range(Hkv)]
        _check_bad_v(ops, q, k, v, q_lens, q_lens, Hkv, spots, want, want_lse, max_k=64)
    assert ops.device_status() == 0


# Rows in one launch, in clusters, from a plan with cut keys, and pairs of CTAs (whole rows, cut keys, rows without keys).
BAD_V_CASES = [
    ([70, 5, 40], [70, 5, 40], 8, 2), ([20, 3], [90, 200], 10, 2),
    ([3], [4000], 32, 8), ([2, 4], [700, 900], 4, 1), ([9], [65], 20, 1),
    ([2, 3, 4] * 20, [150 * i + 40 for i in range(60)], 4, 1), ([4, 1, 2], [20000, 30, 3333], 12, 4),
    ([300, 700, 33], [300, 700, 33], 8, 2), ([129, 1, 64], [400, 500, 64], 32, 8), ([513], [513], 2, 2),
    ([260], [9001], 4, 4), ([100, 30], [6000, 20000], 10, 2), ([300, 140], [100, 900], 16, 4),
    ([60 + i % 70 for i in range(150)], [60 + i % 70 + (i % 3) * 50 for i in range(150)], 8, 8)]  # many per pair


@pytest.mark.parametrize("q_lens,k_lens,Hq,Hkv", BAD_V_CASES)
@pytest.mark.parametrize("seed", range(4))
def test_varlen_bad_values_in_v_show_in_the_rows_that_see_them(ops, q_lens, k_lens, Hq, Hkv, seed):
    import random

    r = random.Random(seed)
    g = _gen(91 + seed)
    q, k, v = _randn(g, sum(q_lens), Hq, 128), _randn(g, sum(k_lens), Hkv, 128), _randn(g, sum(k_lens), Hkv, 128)
    cu_q, cu_k, max_k = _cu(q_lens), _cu(k_lens), max(k_lens)
    want, want_lse = ops.attn_varlen(q, k, v, cu_q, cu_k, max_k=max_k)
    _check_varlen_heads(want, want_lse, q, k, v, q_lens, k_lens)
    for x in BAD:
        spots = []
        for s, (lq, lk) in enumerate(zip(q_lens, k_lens)):
            for hk in range(Hkv):
                # the last key, one that only some rows see, one anywhere; in both halves of the channels
                keys = {lk - 1, r.randrange(max(0, lk - lq), lk), r.randrange(lk)}
                chans = r.sample(range(64), 3) if r.random() < 0.3 else r.sample(range(128), 3)
                spots += [(s, key, hk, ch, x) for key, ch in zip(sorted(keys), chans)]
        _check_bad_v(ops, q, k, v, q_lens, k_lens, Hkv, spots, want, want_lse, max_k=max_k)
        # every channel of one key at once
        s = r.randrange(len(q_lens))
        key = r.randrange(max(0, k_lens[s] - q_lens[s]), k_lens[s])
        _check_bad_v(ops, q, k, v, q_lens, k_lens, Hkv, [(s, key, hk, slice(None), x) for hk in range(Hkv)], want,
                     want_lse, max_k=max_k)
    assert ops.device_status() == 0


@pytest.mark.parametrize("q_lens,k_lens,Hq,Hkv", [([70, 5], [70, 5], 8, 2), ([2, 4], [700, 900], 4, 1),
                                                  ([300, 33], [700, 33], 8, 2), ([260], [9001], 4, 4)])
def test_varlen_bad_values_of_both_signs_make_a_nan(ops, q_lens, k_lens, Hq, Hkv):
    """+inf and -inf in one channel: the rows between them show the first, the rows that see both a NaN."""
    g = _gen(92)
    q, k, v = _randn(g, sum(q_lens), Hq, 128), _randn(g, sum(k_lens), Hkv, 128), _randn(g, sum(k_lens), Hkv, 128)
    cu_q, cu_k = _cu(q_lens), _cu(k_lens)
    want, want_lse = ops.attn_varlen(q, k, v, cu_q, cu_k)
    v[k_lens[0] - 2, :, 77], v[k_lens[0] - 1, :, 77] = math.inf, -math.inf
    o, lse = ops.attn_varlen(q, k, v, cu_q, cu_k)
    n = q_lens[0]
    assert (o[n - 2, :, 77] == math.inf).all() and torch.isnan(o[n - 1, :, 77].float()).all()
    o[n - 2:n, :, 77] = want[n - 2:n, :, 77]
    assert torch.equal(o, want) and torch.equal(lse, want_lse)


# ----------------------------------------------- calls between the others --
@pytest.mark.parametrize("q_lens,k_lens,Hq,Hkv", [([70, 5], [70, 5], 8, 2), ([2, 4], [700, 900], 4, 1),
                                                  ([300, 33], [700, 33], 8, 2), ([260], [9001], 4, 4)])
def test_varlen_a_key_of_infinite_score(ops, q_lens, k_lens, Hq, Hkv):
    """An infinity in K alone: rows whose score it makes -inf go on without that key, the others turn NaN."""
    g = _gen(95)
    q, k, v = _randn(g, sum(q_lens), Hq, 128), _randn(g, sum(k_lens), Hkv, 128), _randn(g, sum(k_lens), Hkv, 128)
    q[:, :, 3] = q[:, :, 3].abs() + 1
    q[::2, :, 3] *= -1
    at = k_lens[0] - q_lens[0] // 2 - 1
    first = at + q_lens[0] - k_lens[0]                 # the first row that sees the key
    k[at, :, 3] = math.inf
    o, lse = ops.attn_varlen(q, k, v, _cu(q_lens), _cu(k_lens))
    n = q_lens[0]
    odd = [i for i in range(max(0, first), n) if i % 2]
    assert torch.isnan(o[odd].float()).all() and torch.isnan(lse[:, odd]).all()
    rows = [i for i in range(sum(q_lens)) if i not in odd]
    # without the key: a score of -inf has no weight
    k[at, :, 3] = 0
    see = torch.arange(k_lens[0], device=DEV)[None] <= torch.arange(n, device=DEV)[:, None] + k_lens[0] - n
    see[:, at] = False
    for h in range(Hq):
        ref = _ref_rows(q[:n, h], k[:k_lens[0], h * Hkv // Hq], v[:k_lens[0], h * Hkv // Hq], see, 128 ** -0.5)
        here = [i for i in rows if i < n]
        _check_attn(o[here, h], lse[h, here], *(t[here] for t in ref), what=h)
    assert torch.isfinite(o[n:].float()).all()


def test_shared_more_items_than_one_launch_takes(ops):
    g = _gen(96)
    B, Hq, P, cap = 20001, 128, 300, 3
    q, kp, vp = _randn(g, B, Hq, 128), _randn(g, 1, P, 128), _randn(g, 1, P, 128)
    k, v = _randn(g, B, 1, cap, 128), _randn(g, B, 1, cap, 128)
    lens = torch.randint(0, cap + 1, (B,), device=DEV, generator=g, dtype=torch.int32)
    o, lse = ops.attn_decode_shared(q, kp, vp, k, v, lens)
    at = torch.tensor([0, 1, 9999, 18943, 18944, 18945, 20000], device=DEV)
    _check_shared(o[at], lse[at], q[at], kp, vp, k[at], v[at], lens[at].tolist())
    # every request, by products of all rows at once in fp32 (which may be off by as much as the kernel)
    sc = (q.view(-1, 128).float() @ kp[0].float().t()).view(B, Hq, P) * 128 ** -0.5
    own = torch.einsum("bhd,bcd->bhc", q.float(), k[:, 0].float()) * 128 ** -0.5
    own.masked_fill_(torch.arange(cap, device=DEV)[None, None] >= lens[:, None, None], -math.inf)
    ref = torch.logsumexp(torch.cat([sc, own], -1), -1)
    assert ((lse - ref).abs() <= 2e-4 + 2.0 ** -20 * ref.abs()).all()
    assert ops.device_status() == 0


@pytest.mark.parametrize("q_lens,k_lens", [([5, 9], [30, 9]), ([1], [3000]), ([1] * 40, [500] * 40), ([300, 200], [300, 900])])
def test_varlen_overlapping_rows(ops, q_lens, k_lens):
    """Views whose rows overlap in memory (a window that slides by eight channels): read as any other strides."""
    g = _gen(97)
    Tq, Tk = sum(q_lens), sum(k_lens)
    q = _randn(g, 4, 8 * Tq + 128).as_strided((Tq, 4, 128), (8, 8 * Tq + 128, 1))
    kv = _randn(g, 2, 2, 8 * Tk + 128)
    k, v = (t.as_strided((Tk, 2, 128), (8, 8 * Tk + 128, 1), t.storage_offset()) for t in (kv[0], kv[1]))
    o, lse = ops.attn_varlen(q, k, v, _cu(q_lens), _cu(k_lens), max_k=max(k_lens))
    _check_varlen_heads(o, lse, q, k, v, q_lens, k_lens)


def test_nothing_to_see_in_a_captured_graph(ops):
    """A batch without prefix and slots behind a copy in the same graph: the join alone is launched."""
    g = _gen(98)
    B, Hq = 300, 8
    src, q = _randn(g, B, Hq, 128), torch.zeros(B, Hq, 128, device=DEV, dtype=torch.bfloat16)
    own = q.new_empty(B, 2, 0, 128)
    none = q.new_empty(2, 0, 128)
    out = torch.full((B, 1, Hq, 128), 7.0, device=DEV, dtype=torch.bfloat16)
    ops.attn_decode_shared(q, none, none, own, own, out=out)
    assert (out == 0).all()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        q.copy_(src)
        _, lse = ops.attn_decode_shared(q, none, none, own, own, out=out)
    out.fill_(7.0)
    gr.replay()
    torch.cuda.synchronize()
    assert (out == 0).all() and (lse == -math.inf).all()


def test_two_threads_at_once(ops):
    """Two host threads, each with its stream and inputs; the first calls of a path may meet."""
    import threading

    runs = [_calls(ops, _gen(200 + i))[0] for i in range(2)]
    want = [[t.clone() for t in r()] for r in runs]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i] = runs[i]()
                torch.cuda.current_stream().synchronize()
        except BaseException as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for w, o in zip(want, got):
        assert all(torch.equal(a, b) for a, b in zip(w, o))
    assert ops.device_status() == 0
