"""Attention without [T, T] intermediates and distillation from top logits (fh_op_attention_*, fh_op_distill_loss).

CPU tests: every refusal, which comes before any device work (the context is a dummy that no
refused call looks into), and the host mirror's size checks.  GPU tests: each entry point
against its formula in 64 bits on the same inputs, with bounds that are derived here from the
roundings of the kernels; `half` is half a step of a type relative to the value, 2^-24 in fp32
and 2^-8 in bf16.
"""
import ctypes

import numpy as np
import pytest

F32 = 2.0 ** -24
TINY = 2.0 ** -126  # fp32 values below it may be zeros
HALF = {"f32": F32, "bf16": 2.0 ** -8}


# ---- types ---------------------------------------------------------------------------------------

def to_bf16(x):
    """bf16 bits (round to nearest even) of a float array."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def from_bf16(u):
    return (u.astype(np.uint32) << 16).view(np.float32)


def stored(x, dtype):
    """(the bits a buffer of dtype holds for x, their values)."""
    if dtype == "f32":
        x = np.ascontiguousarray(x, np.float32)
        return x, x
    nan = np.isnan(x)
    b = np.where(nan, np.uint16(0x7FC0), to_bf16(np.where(nan, 0, x)))
    return b, from_bf16(b)


def values(raw, dtype):
    return raw if dtype == "f32" else from_bf16(raw)


@pytest.fixture(scope="module")
def be(fhp):
    with fhp.HipBackend(0) as backend:
        yield backend


# ---- attention in 64 bits, with the kernels' error bounds ------------------------------------------

def split(qkv, B, T, H, Hk, hd):
    """q [B, H, T, hd], and k, v repeated for the heads that share them."""
    x = np.asarray(qkv, np.float64).reshape(B, T, H + 2 * Hk, hd).transpose(0, 2, 1, 3)
    return x[:, :H], np.repeat(x[:, H:H + Hk], H // Hk, 1), np.repeat(x[:, H + Hk:], H // Hk, 1)


def rows(x, B, T):
    return x.transpose(0, 2, 1, 3).reshape(B * T, -1)


class Attention64:
    """Forward and backward of one call in 64 bits, and how far a kernel's values may be from them.

    A score is a sum of hd fp32 products, (hd + 4) half steps of sum |q||k|, scaled; a probability
    is off by its score's error and that of the row's log sum (the same errors, T + 8 sums, and
    the roundings of |lse| and of the exponents), which `dp` bounds per row; one below TINY is a
    zero, so it is off by TINY besides (times a gradient and a key in the tens: 1e-36).  bf16 rounds
    each probability (and its gradient) once more as it enters a product, and o, from which D comes."""

    def __init__(self, qkv, dout, lengths, B, T, H, Hk, hd, scale, dtype):
        q, k, v = split(qkv, B, T, H, Hk, hd)
        n = np.asarray(lengths).reshape(B, 1, 1, 1)
        i, j = np.arange(T).reshape(T, 1), np.arange(T).reshape(1, T)
        seen = (j <= i) & (j < n) & (i < n)
        q, k, v = (np.where(np.arange(T).reshape(1, 1, T, 1) < n, x, 0.0) for x in (q, k, v))
        s = np.where(seen, np.matmul(q, k.swapaxes(-1, -2)) * scale, -np.inf)
        m = np.max(s, -1, keepdims=True, initial=-np.inf)
        p = np.where(seen, np.exp(np.where(seen, s - np.where(np.isfinite(m), m, 0), 0)), 0.0)
        total = p.sum(-1, keepdims=True)
        self.lse = np.where(total[..., 0] > 0, np.log(np.where(total > 0, total, 1))[..., 0] + np.where(np.isfinite(m), m, 0)[..., 0],
                            -np.inf)
        p = p / np.where(total > 0, total, 1)
        o = np.matmul(p, v)
        half, r = HALF[dtype], 0.0 if dtype == "f32" else HALF[dtype]  # of the outputs; of what enters a product
        size = np.where(seen, np.matmul(np.abs(q), np.abs(k).swapaxes(-1, -2)) * scale, 0).max(-1, initial=0, keepdims=True)
        dp = F32 * (2 * (hd + 4) * size + 4 * np.abs(np.where(np.isfinite(self.lse), self.lse, 0))[..., None] + T + 16)
        self.lse_err = dp[..., 0]
        tiny = np.where(seen, TINY, 0.0)
        self.out, out_err = o, np.matmul(p, np.abs(v)) * (2 * dp + r + T * F32) + half * np.abs(o) + np.matmul(tiny, np.abs(v))
        self.out_err = rows(out_err, B, T)
        if dout is not None:
            do = np.asarray(dout, np.float64).reshape(B, T, H, hd).transpose(0, 2, 1, 3)
            do = np.where(np.arange(T).reshape(1, 1, T, 1) < n, do, 0.0)
            g = np.matmul(do, v.swapaxes(-1, -2))
            ga = np.matmul(np.abs(do), np.abs(v).swapaxes(-1, -2))
            D = (do * o).sum(-1, keepdims=True)
            ds = p * (g - D)
            # dP: hd products; D: the error of o and hd products; then p's own error and ds's rounding
            derr = (np.abs(do) * out_err).sum(-1, keepdims=True) + (hd + 2) * F32 * (np.abs(do) * np.abs(o)).sum(-1, keepdims=True)
            dserr = p * ((hd + 4) * F32 * ga + derr) + np.abs(ds) * (2 * dp + r + 4 * F32) + tiny * (ga + np.abs(D) + 1)
            fold = lambda x: x.reshape(B, Hk, H // Hk, T, hd).sum(2)  # noqa: E731
            tr = lambda x: x.swapaxes(-1, -2)  # noqa: E731
            grads = [np.matmul(ds, k) * scale, fold(np.matmul(tr(ds), q)) * scale, fold(np.matmul(tr(p), do))]
            many = H // Hk * T * F32
            errs = [np.matmul(dserr + T * F32 * np.abs(ds), np.abs(k)) * scale,
                    fold(np.matmul(tr(dserr + many * np.abs(ds)), np.abs(q))) * scale,
                    fold(np.matmul(tr(p * (2 * dp + r + many) + tiny), np.abs(do)))]
            self.dqkv = rows(np.concatenate(grads, 1), B, T)
            self.dqkv_err = rows(np.concatenate(errs, 1), B, T) + 2 * half * np.abs(self.dqkv)
        self.out = rows(o, B, T)


def check(got, want, err, what):
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape, what
    bad = ~(np.abs(got - want) <= err + 1e-37)
    assert not bad.any(), (what, int(bad.sum()), float(np.nanmax(np.abs(got - want) / (err + 1e-37))), np.argwhere(bad)[:4].tolist())


def attention_case(fhp, be, B, T, H, Hk, hd, dtype, lengths=None, scale=None, more=0, seed=0, std=1.0, past=np.nan):
    """Runs forward and backward and checks both; `more` columns beside the heads' hold a mark."""
    r = np.random.default_rng(seed)
    W, Wo = (H + 2 * Hk) * hd, H * hd
    qkv = r.normal(0, std, (B * T, W + more))
    dout = r.normal(0, 1, (B * T, Wo + more))
    n = np.full(B, T) if lengths is None else np.asarray(lengths)
    pad = (np.arange(T) >= n[:, None]).reshape(-1)
    qkv[pad], dout[pad] = past, past  # what no result may depend on
    qkv[:, W:], dout[:, Wo:] = 7.0, 7.0
    qb, qv = stored(qkv, dtype)
    db, dv = stored(dout, dtype)
    sc = 1 / np.sqrt(hd) if scale is None else scale
    ref = Attention64(qv[:, :W], dv[:, :Wo], n, B, T, H, Hk, hd, float(np.float32(sc)), dtype)
    mark, _ = stored(np.full((B * T, Wo + more), 7.0), dtype)
    bq, bd = fhp.DeviceBuffer.from_array(be, qb), fhp.DeviceBuffer.from_array(be, db)
    bo, bg = fhp.DeviceBuffer.from_array(be, mark), fhp.DeviceBuffer.from_array(be, np.where(np.ones_like(qb), stored(np.full(1, 7.0), dtype)[0][0], 0).astype(qb.dtype))
    bl = fhp.DeviceBuffer(be, 4 * B * H * T)
    kw = dict(n_kv_heads=Hk, lengths=lengths, scale=scale, qkv_cols=W + more, out_cols=Wo + more, dtype=dtype)
    be.attention_forward(bq, bo, bl, B, T, H, hd, **kw)
    out = values(bo.read(qb.dtype, B * T * (Wo + more)), dtype).reshape(B * T, -1)
    lse = bl.read(np.float32, B * H * T).reshape(B, H, T)
    np.testing.assert_array_equal(out[:, Wo:], 7.0)
    fin = np.isfinite(ref.lse)
    np.testing.assert_array_equal(np.isneginf(lse), ~fin)
    check(np.where(fin, lse, 0), np.where(fin, ref.lse, 0), ref.lse_err + 4 * F32 * np.abs(np.where(fin, ref.lse, 0)), "lse")
    check(out[:, :Wo], ref.out, ref.out_err, "out")
    be.attention_backward(bd, bq, bo, bl, bg, B, T, H, hd, **kw)
    raw = bg.read(qb.dtype, B * T * (W + more))
    dqkv = values(raw, dtype).reshape(B * T, -1)
    np.testing.assert_array_equal(dqkv[:, W:], 7.0)
    check(dqkv[:, :W], ref.dqkv, ref.dqkv_err, "dqkv")
    assert not out[pad, :Wo].any() and not dqkv[pad, :W].any()
    be.attention_backward(bd, bq, bo, bl, bg, B, T, H, hd, **kw)  # the same bits again
    np.testing.assert_array_equal(bg.read(qb.dtype, B * T * (W + more)), raw)
    for b in (bq, bd, bo, bg, bl):
        b.free()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T", [1, 2, 31, 32, 33, 64, 127, 129, 300])
def test_attention_lengths(fhp, be, T, dtype):
    attention_case(fhp, be, 2, T, 3, 3, 64, dtype, seed=T)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [1, 5, 8, 20, 32, 36, 40, 72, 80, 90, 100, 128])
def test_attention_head_sizes(fhp, be, hd, dtype):
    # 5, 90, 20 (bf16) and 36 (bf16) are no multiple of 16 bytes
    attention_case(fhp, be, 1, 75, 4, 2, hd, dtype, seed=hd)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("H,Hk", [(1, 1), (8, 8), (8, 1), (6, 2)])
def test_attention_shared_heads(fhp, be, H, Hk, dtype):
    attention_case(fhp, be, 2, 140, H, Hk, 32, dtype, seed=H + Hk)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd,Hk", [(32, 16), (64, 16), (64, 4), (128, 16)])
def test_attention_many_blocks(fhp, be, hd, Hk, dtype):
    # enough blocks of 128 rows that the four waves take rows of their own
    attention_case(fhp, be, 16, 133, 16, Hk, hd, dtype, seed=hd)


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,H,Hk,hd,dtype", [
    (16, 133, 16, 4, 128, "bf16"), (16, 133, 16, 8, 128, "bf16"),  # blocks of keys: few, as many as CUs
    (16, 133, 16, 8, 64, "bf16"), (8, 260, 32, 32, 32, "bf16"), (16, 133, 16, 8, 128, "f32"), (16, 133, 20, 20, 128, "f32"),
    (16, 260, 16, 16, 32, "f32"), (16, 260, 16, 2, 64, "f32"), (8, 260, 24, 12, 48, "f32"),  # in three parts
])
def test_attention_blocks_of_queries_and_keys(fhp, be, B, T, H, Hk, hd, dtype):
    # dq, dk and dv in one launch or in turn, in blocks of 32 and of 128 rows
    attention_case(fhp, be, B, T, H, Hk, hd, dtype, seed=hd + H)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_many_blocks_unaligned(fhp, be, dtype):
    attention_case(fhp, be, 16, 133, 16, 16, 25, dtype, seed=25, more=1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lengths", [[0, 1, 32, 97], [97, 0, 96, 33], [0, 0, 0, 0], [64, 65, 31, 97]])
def test_attention_padded(fhp, be, lengths, dtype):
    # rows past a length hold NaN: they are not read, and their outputs are zeros
    attention_case(fhp, be, 4, 97, 4, 2, 64, dtype, lengths=lengths, seed=sum(lengths))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_padded_many_blocks(fhp, be, dtype):
    r = np.random.default_rng(5)
    attention_case(fhp, be, 24, 200, 12, 12, 64, dtype, lengths=r.integers(0, 201, 24), seed=5, past=np.inf)


@pytest.mark.gpu
def test_attention_more_sequences_than_fit_a_launch(fhp, be):
    r = np.random.default_rng(6)
    attention_case(fhp, be, 100, 9, 2, 1, 16, "f32", lengths=r.integers(0, 10, 100), seed=6)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("more", [1, 8])
def test_attention_strides(fhp, be, more, dtype):
    attention_case(fhp, be, 2, 70, 3, 1, 40, dtype, more=more, seed=more)


@pytest.mark.gpu
@pytest.mark.parametrize("std,scale", [(8.0, None), (3.0, 1.0), (0.05, 2.5)])
def test_attention_sharp_and_flat_rows(fhp, be, std, scale):
    # scores of hundreds (one probability of 1 in a row) and of nearly nothing
    attention_case(fhp, be, 1, 90, 2, 2, 64, "f32", std=std, scale=scale, seed=3)


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,H,Hk,hd,lengths", [
    (6, 520, 9, 3, 64, None), (6, 520, 9, 9, 40, [520, 1, 519, 0, 300, 32]), (4, 260, 24, 24, 32, None),
    (1, 1030, 2, 1, 64, None), (2, 1100, 3, 3, 20, [1061, 97]),
])
def test_attention_fp32_in_three_parts(fhp, be, B, T, H, Hk, hd, lengths):
    # long enough that fp32 values are multiplied in bf16 parts, with the bounds of the fp32 products: of a
    # product a b the parts leave out two of mid times lo, 2^-8 2^-16 each, and add up six exact ones for
    # every 16 dims, fewer roundings than the hd that the bound counts
    attention_case(fhp, be, B, T, H, Hk, hd, "f32", lengths=lengths, seed=T + hd)


@pytest.mark.gpu
def test_attention_largest_values_in_parts(fhp, be):
    # values that would round to infinity in bf16: v and dout alone, so that every sum is in range
    B, T, H, hd = 1, 1030, 1, 32
    qkv, dout = np.zeros((T, 3 * hd), np.float32), np.zeros((T, hd), np.float32)
    top = np.finfo(np.float32).max
    qkv[:, 2 * hd], dout[-1, 1] = top, top
    qkv[0, hd + 1], qkv[:, 1] = -1e4, 1.0  # no weight on the first key, but for the first query
    bq, bd = fhp.DeviceBuffer.from_array(be, qkv), fhp.DeviceBuffer.from_array(be, dout)
    bo, bl, bg = fhp.DeviceBuffer(be, dout.nbytes), fhp.DeviceBuffer(be, 4 * T), fhp.DeviceBuffer(be, qkv.nbytes)
    be.attention_forward(bq, bo, bl, B, T, H, hd)
    be.attention_backward(bd, bq, bo, bl, bg, B, T, H, hd)
    dv = bg.read(np.float32, T * 3 * hd).reshape(T, -1)[:, 2 * hd + 1].astype(np.float64)
    want = np.where(np.arange(T) == 0, 0.0, float(top) / (T - 1))  # of the last query, which all others' dout leave alone
    np.testing.assert_allclose(dv, want, rtol=(T + 40) * F32)
    for b in (bq, bd, bo, bl, bg):
        b.free()


@pytest.mark.gpu
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("which", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("B,T,H,Hk,hd,dtype", [
    (1, 75, 4, 2, 64, "f32"), (1, 75, 4, 2, 64, "bf16"), (1, 75, 2, 2, 128, "bf16"), (1, 75, 2, 1, 25, "f32"),
    (16, 133, 16, 8, 64, "bf16"), (16, 133, 16, 16, 32, "f32"), (1, 1030, 2, 2, 32, "f32"), (9, 520, 6, 6, 16, "f32"),
])
def test_attention_rows_depend_on_what_they_see_alone(fhp, be, B, T, H, Hk, hd, dtype, which, value):
    # row 41 of the last sequence is not finite: o and dq of the rows before it, and what a query's q or
    # dout cannot reach, are as without it
    W, Wo, at = (H + 2 * Hk) * hd, H * hd, (B - 1) * T + 41
    r = np.random.default_rng(8)
    qkv, dout = r.normal(0, 1, (B * T, W)), r.normal(0, 1, (B * T, Wo))
    _, qv = stored(qkv, dtype)
    _, dv = stored(dout, dtype)
    ref = Attention64(qv, dv, np.full(B, T), B, T, H, Hk, hd, float(np.float32(1 / np.sqrt(hd))), dtype)
    cols = {"q": slice(0, H * hd), "k": slice(H * hd, (H + Hk) * hd), "v": slice((H + Hk) * hd, W)}
    if which == "dout":
        dout[at] = value
    else:
        qkv[at, cols[which]] = value
    raw = lambda x: stored(x, dtype)[0] if dtype == "f32" else np.where(  # noqa: E731
        np.isinf(x), np.where(x > 0, np.uint16(0x7F80), np.uint16(0xFF80)), stored(np.where(np.isinf(x), 0, x), dtype)[0])
    qb, db = raw(qkv), raw(dout)
    bq, bd = fhp.DeviceBuffer.from_array(be, qb), fhp.DeviceBuffer.from_array(be, db)
    bo, bl, bg = fhp.DeviceBuffer(be, db.nbytes), fhp.DeviceBuffer(be, 4 * B * H * T), fhp.DeviceBuffer(be, qb.nbytes)
    be.attention_forward(bq, bo, bl, B, T, H, hd, n_kv_heads=Hk, dtype=dtype)
    be.attention_backward(bd, bq, bo, bl, bg, B, T, H, hd, n_kv_heads=Hk, dtype=dtype)
    out = values(bo.read(db.dtype, B * T * Wo), dtype).reshape(B * T, Wo)
    lse = bl.read(np.float32, B * H * T).reshape(B, H, T)
    g = values(bg.read(qb.dtype, B * T * W), dtype).reshape(B * T, W)
    row = np.arange(B * T)
    other = row < (B - 1) * T                      # of other sequences
    before, after = row < at, other | (row > at)
    o_ok = np.ones(B * T, bool) if which == "dout" else row != at if which == "q" else before
    dq_ok = row != at if which in ("q", "dout") else before
    kv_ok = after if which in ("q", "dout") else other
    check(out[o_ok], ref.out[o_ok], ref.out_err[o_ok], "out")
    fine = o_ok.reshape(B, 1, T) & np.ones((B, H, T), bool)
    check(lse[fine], ref.lse[fine], (ref.lse_err + 4 * F32 * np.abs(ref.lse))[fine], "lse")
    for c, ok, what in ((cols["q"], dq_ok, "dq"), (cols["k"], kv_ok, "dk"), (cols["v"], kv_ok, "dv")):
        check(g[ok, c], ref.dqkv[ok, c], ref.dqkv_err[ok, c], what)
    if np.isnan(value):  # and what sees it shows it
        assert not np.isfinite(out[at] if which != "dout" else g[at, cols["q"]]).any()
    for b in (bq, bd, bo, bl, bg):
        b.free()


@pytest.mark.gpu
def test_attention_gradient_by_differences(fhp, be):
    B, T, H, hd = 1, 5, 2, 4
    r = np.random.default_rng(1)
    qkv, dout = r.normal(0, 1, (B * T, 3 * H * hd)).astype(np.float32), r.normal(0, 1, (B * T, H * hd)).astype(np.float32)
    bo, bl, bg = fhp.DeviceBuffer(be, dout.nbytes), fhp.DeviceBuffer(be, 4 * B * H * T), fhp.DeviceBuffer(be, qkv.nbytes)
    bq, bd = fhp.DeviceBuffer(be, qkv.nbytes), fhp.DeviceBuffer.from_array(be, dout)

    def loss(x):
        bq.write(x)
        be.attention_forward(bq, bo, bl, B, T, H, hd)
        return float((bo.read(np.float32, dout.size).astype(np.float64) * dout.reshape(-1)).sum())

    loss(qkv)
    be.attention_backward(bd, bq, bo, bl, bg, B, T, H, hd)
    got = bg.read(np.float32, qkv.size)
    for i in range(qkv.size):
        x = qkv.reshape(-1).copy()
        x[i] = qkv.reshape(-1)[i] + 1e-2
        up, hi = loss(x), float(x[i])
        x[i] = qkv.reshape(-1)[i] - 1e-2
        num = (up - loss(x)) / (hi - float(x[i]))
        # third derivatives of order one by h^2 / 6, and rounding by 2 h: far below 2e-3
        assert abs(num - got[i]) <= 2e-3 * max(1.0, abs(num)), (i, num, got[i])


@pytest.mark.gpu
def test_attention_rows_past_32_bit_offsets(fhp, be):
    # 2^20 columns: the last sequence's rows start past 2^31 elements of qkv and dqkv
    B, T, H, hd, W = 1060, 2, 1, 8, 1 << 20
    L = fhp.lib()
    bq, bg = fhp.DeviceBuffer(be, 2 * W * B * T), fhp.DeviceBuffer(be, 2 * W * B * T)
    bo, bd, bl = fhp.DeviceBuffer(be, 2 * B * T * hd), fhp.DeviceBuffer(be, 2 * B * T * hd), fhp.DeviceBuffer(be, 4 * B * T)
    r = np.random.default_rng(2)
    x, _ = stored(r.normal(0, 1, (T, 3 * hd)), "bf16")
    d, dv = stored(r.normal(0, 1, (B * T, hd)), "bf16")
    bd.write(d)
    lengths = np.zeros(B, np.int32)
    lengths[-1] = T
    for t in range(T):
        at = bq.ptr.value + 2 * W * ((B - 1) * T + t)
        fhp._native.check(L.fh_buffer_write(be.handle, at, np.ascontiguousarray(x[t]).ctypes.data, x[t].nbytes))
    kw = dict(lengths=lengths, qkv_cols=W, dtype="bf16")
    be.attention_forward(bq, bo, bl, B, T, H, hd, **kw)
    be.attention_backward(bd, bq, bo, bl, bg, B, T, H, hd, **kw)
    ref = Attention64(from_bf16(x), dv[-T:], [T], 1, T, H, H, hd, float(np.float32(1 / np.sqrt(hd))), "bf16")
    check(from_bf16(bo.read(np.uint16, B * T * hd)).reshape(-1, hd)[-T:], ref.out, ref.out_err, "out")
    got = np.empty((T, 3 * hd), np.uint16)
    for t in range(T):
        at = bg.ptr.value + 2 * W * ((B - 1) * T + t)
        fhp._native.check(L.fh_buffer_read(be.handle, got[t].ctypes.data, at, got[t].nbytes))
    check(from_bf16(got), ref.dqkv, ref.dqkv_err, "dqkv")
    for b in (bq, bg, bo, bd, bl):
        b.free()


# ---- distillation ------------------------------------------------------------------------------------

def distill64(z, targets, ids, top, tau, alpha, ignore):
    """Loss, gradient, and the bound of the gradient's error before its last rounding.

    An exponential is off by the roundings of its argument (|z - max| / tau and the product with
    log2 e) and its own step; a sum over V by the elements a thread adds and the joins (V / 256 +
    32 at the most)."""
    T, V = z.shape
    z = np.asarray(z, np.float64)
    on = np.asarray(targets) != ignore
    count = int(on.sum())
    g, err, loss, lerr = np.zeros((T, V)), np.zeros((T, V)), 0.0, 0.0
    for t in range(T):
        if not on[t]:
            continue
        used = (ids[t] >= 0) & (ids[t] < V) & (np.asarray(top[t]) != -np.inf)
        x = z[t] / tau
        m = x.max()
        lse = m + np.log(np.exp(x - m).sum())
        p = np.exp(x - lse)
        m1 = z[t].max()
        lse1 = m1 + np.log(np.exp(z[t] - m1).sum())
        p1 = np.exp(z[t] - lse1)
        fin = np.abs(np.where(np.isfinite(z[t]), z[t], m1) - m1)
        rel = F32 * (4 * fin * max(1, 1 / tau) + V / 256 + 40)
        kl = 0.0
        q = np.zeros(V)
        if used.any():
            u = np.asarray(top[t], np.float64)[used] / tau
            lq = u - (u.max() + np.log(np.exp(u - u.max()).sum()))
            kl = float((np.exp(lq) * (lq - (x - lse)[ids[t][used]])).sum())
            np.add.at(q, ids[t][used], np.exp(lq))
            g[t] += alpha * tau * (p - q)
            qrel = F32 * (4 * np.abs(u - u.max()).max() + len(u) + 40)
            err[t] += alpha * tau * (p * (rel + rel[fin.argmin()]) + q * qrel)
            lerr += alpha * tau * tau * F32 * (8 * (np.abs(u).max() + np.abs(x[ids[t][used]] - m).max()) + V / 256 + len(u) + 60)
        hot = np.zeros(V)
        hot[targets[t]] = 1
        g[t] += (1 - alpha) * (p1 - hot)
        err[t] += (1 - alpha) * (p1 * (rel + rel[fin.argmin()]) + hot * 4 * F32)
        loss += alpha * tau * tau * kl + (1 - alpha) * (lse1 - z[t, targets[t]])
        lerr += (1 - alpha) * F32 * (4 * abs(z[t, targets[t]] - m1) + V / 256 + 60)
    return loss / max(1, count), g / max(1, count), err / max(1, count), lerr / max(1, count)


def distill_case(fhp, be, T, V, K, dtype, tau, alpha, seed=0, ignore=-1, in_place=False, edit=None):
    r = np.random.default_rng(seed)
    zb, z = stored(r.normal(0, 3, (T, V)), dtype)
    ids = r.integers(0, V, (T, K)).astype(np.int32)  # an id may come twice
    top = r.normal(0, 3, (T, K)).astype(np.float32)
    ids[r.random((T, K)) < 0.2] = -1
    targets = r.integers(0, V, T).astype(np.int32)
    targets[r.random(T) < 0.2] = ignore
    if edit:
        edit(z, ids, top, targets)
        zb, z = stored(z, dtype)
    loss, g, err, lerr = distill64(z, targets, ids, top, tau, alpha, ignore)
    bz, bi, bt = (fhp.DeviceBuffer.from_array(be, a) for a in (zb, ids, top))
    bg = bz if in_place else fhp.DeviceBuffer(be, zb.nbytes)
    kw = dict(ignore_index=ignore, temperature=tau, alpha=alpha, dtype=dtype)
    alone = be.distill_loss(bz, targets, bi, bt, None, T, V, K, **kw)
    got = be.distill_loss(bz, targets, bi, bt, bg, T, V, K, **kw)
    assert alone == got
    if np.isfinite(loss):
        assert abs(got - loss) <= lerr + 2 * F32 * abs(loss) + 1e-30, (got, loss, lerr)
    else:
        assert got == loss
    dz = values(bg.read(zb.dtype, T * V), dtype).reshape(T, V)
    check(dz, g, err + 4 * F32 * np.abs(g) + HALF[dtype] * np.abs(g) * (1 + 2 ** -7) + 1e-30, "dlogits")
    assert not dz[targets == ignore].any()
    for b in {id(x): x for x in (bz, bi, bt, bg)}.values():
        b.free()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [1, 2, 7, 100, 1027, 2256, 4099, 8200, 16257, 33000, 50257, 110001])
def test_distill_vocabularies(fhp, be, V, dtype):
    # a row in 256 or 1024 threads' registers, or (110001) read again; odd V: rows start anywhere
    distill_case(fhp, be, 5, V, min(9, V), dtype, 2.0, 0.5, seed=V)


@pytest.mark.gpu
@pytest.mark.parametrize("tau,alpha", [(1.0, 1.0), (1.0, 0.0), (1.0, 0.3), (4.0, 1.0), (0.5, 0.0), (0.5, 0.7)])
def test_distill_weights(fhp, be, tau, alpha):
    distill_case(fhp, be, 9, 777, 5, "f32", tau, alpha, seed=4)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [1, 64, 300, 1024])
def test_distill_slots(fhp, be, K):
    # more slots than ids: most ids come several times
    distill_case(fhp, be, 4, 90, K, "f32", 2.0, 0.6, seed=K)
    distill_case(fhp, be, 4, 5000, K, "bf16", 2.0, 0.6, seed=K)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_distill_in_place(fhp, be, dtype):
    distill_case(fhp, be, 6, 4097, 8, dtype, 2.0, 0.5, in_place=True)
    distill_case(fhp, be, 6, 120001, 8, dtype, 2.0, 0.5, in_place=True)


@pytest.mark.gpu
def test_distill_empty_rows_and_infinite_logits(fhp, be):
    def edit(z, ids, top, targets):
        targets[:] = np.arange(len(targets)) % 50 + 10
        ids[0] = -1               # no slot of the row is used
        top[1] = -np.inf          # all of them without weight
        ids[2], top[2, 0] = ids[2, 0], 0.0
        ids[3, 0], ids[3, 1] = 2 ** 31 - 1, z.shape[1]  # outside the vocabulary
        z[4, :10] = -np.inf       # a student's masked tokens
        ids[4] = 30
        top[5, 1:] = -np.inf      # one slot with all the weight
        ids[5, 0] = targets[5]
    distill_case(fhp, be, 7, 1500, 6, "f32", 2.0, 0.5, edit=edit)
    distill_case(fhp, be, 7, 200, 6, "bf16", 1.0, 1.0, edit=edit)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [2048, 2049, 20000])
def test_distill_many_rows(fhp, be, T):
    # few targets go to the device with the call's work, more are copied first
    distill_case(fhp, be, T, 33, 4, "f32", 2.0, 0.5, seed=T)


@pytest.mark.gpu
def test_distill_every_row_ignored(fhp, be):
    def edit(z, ids, top, targets):
        targets[:] = 5
    distill_case(fhp, be, 3, 300, 4, "f32", 2.0, 0.5, ignore=5, edit=edit)


@pytest.mark.gpu
def test_distill_repeats_its_bits(fhp, be):
    r = np.random.default_rng(0)
    T, V, K = 40, 3001, 200
    z, top = r.normal(0, 2, (T, V)).astype(np.float32), r.normal(0, 2, (T, K)).astype(np.float32)
    ids, tg = r.integers(0, 60, (T, K)).astype(np.int32), r.integers(0, V, T)
    bz, bt, bi = (fhp.DeviceBuffer.from_array(be, a) for a in (z, top, ids))
    bg, seen = fhp.DeviceBuffer(be, z.nbytes), []
    for _ in range(3):
        loss = be.distill_loss(bz, tg, bi, bt, bg, T, V, K, temperature=2.0, alpha=0.5)
        seen.append((loss, bg.read(np.uint32, T * V)))
    for loss, g in seen[1:]:
        assert loss == seen[0][0]
        np.testing.assert_array_equal(g, seen[0][1])


@pytest.mark.gpu
def test_distill_in_a_loss_accumulation(fhp):
    ops = fhp.HipTensorBackend(0)
    r = np.random.default_rng(3)
    total = n = 0
    ops.BeginLossAccumulation()
    for T, V in ((7, 200), (3, 5000)):
        z, top = fhp.Tensor(r.normal(0, 2, (T, V)), T, V), fhp.Tensor(r.normal(0, 2, (T, 4)), T, 4)
        ids = r.integers(0, V, (T, 4)).astype(np.int32)
        tg = r.integers(0, V, T).astype(np.int32)
        tg[0] = -1
        g = fhp.Tensor(T, V)
        assert ops.DistillLoss(z, tg, fhp.DeviceBuffer.from_array(ops.backend, ids), top, g, T, V, 4, -1, 2.0, 0.5) == 0.0
        loss, dz, err, _ = distill64(z.Data.reshape(T, V), tg, ids, top.Data.reshape(T, 4), 2.0, 0.5, -1)
        ops.EnsureHostCurrent(g)
        check(g.Data.reshape(T, V), dz, err + 6 * F32 * np.abs(dz) + 1e-30, "dlogits")
        total, n = total + loss * (T - 1), n + T - 1
    mean = ops.EndLossAccumulation()
    assert abs(mean - total / n) <= 1e-5 * abs(total / n)
    ops.Dispose()


# ---- together -------------------------------------------------------------------------------------------

@pytest.mark.gpu
def test_a_training_step_with_both(fhp):
    """x -> qkv -> attention -> logits -> distillation, and back to every weight, against differences in
    64 bits of the same step."""
    B, T, H, hd, V, K = 2, 9, 2, 8, 40, 5
    D = H * hd
    r = np.random.default_rng(11)
    x, wq, wo = r.normal(0, 1, (B * T, D)), r.normal(0, 0.4, (D, 3 * D)), r.normal(0, 0.4, (V, D))
    x, wq, wo = (a.astype(np.float32) for a in (x, wq, wo))
    ids, top = r.integers(0, V, (B * T, K)).astype(np.int32), r.normal(0, 2, (B * T, K)).astype(np.float32)
    lengths = [T, 6]
    tg = r.integers(0, V, B * T).astype(np.int32)
    tg[T + 6:] = -1  # the padding has no loss

    def step64(wq, wo):
        a = Attention64(x @ wq, None, lengths, B, T, H, H, hd, 1 / np.sqrt(hd), "f32")
        return distill64(a.out @ wo.T, tg, ids, top, 2.0, 0.4, -1)[0]

    ops = fhp.HipTensorBackend(0)
    t = {k: fhp.Tensor(v, *v.shape) for k, v in dict(x=x, wq=wq, wo=wo, top=top).items()}
    e = {k: fhp.Tensor(*s) for k, s in dict(qkv=(B * T, 3 * D), o=(B * T, D), lse=(B * H, T), z=(B * T, V), do=(B * T, D),
                                            dqkv=(B * T, 3 * D), dwq=(D, 3 * D), dwo=(V, D)).items()}
    ops.MatMulNN(t["x"], t["wq"], e["qkv"], B * T, D, 3 * D)
    ops.AttentionForward(e["qkv"], e["o"], e["lse"], B, T, H, hd, lengths=lengths)
    ops.MatMulNT(e["o"], t["wo"], e["z"], B * T, D, V)
    loss = ops.DistillLoss(e["z"], tg, fhp.DeviceBuffer.from_array(ops.backend, ids), t["top"], e["z"], B * T, V, K, -1, 2.0, 0.4)
    ops.MatMulTN(e["z"], e["o"], e["dwo"], V, B * T, D)
    ops.MatMulNN(e["z"], t["wo"], e["do"], B * T, V, D)
    ops.AttentionBackward(e["do"], e["qkv"], e["o"], e["lse"], e["dqkv"], B, T, H, hd, lengths=lengths)
    ops.MatMulTN(t["x"], e["dqkv"], e["dwq"], D, B * T, 3 * D)
    ops.EnsureHostCurrent(e["dwq"])
    ops.EnsureHostCurrent(e["dwo"])
    w64, o64 = wq.astype(np.float64), wo.astype(np.float64)
    assert abs(loss - step64(w64, o64)) <= 1e-5 * abs(loss)
    for got, w, other in ((e["dwq"], w64, lambda m: step64(m, o64)), (e["dwo"], o64, lambda m: step64(w64, m))):
        for i in r.choice(w.size, 40, replace=False):
            d = np.zeros(w.size)
            d[i] = 1e-5
            d = d.reshape(w.shape)
            num = (other(w + d) - other(w - d)) / 2e-5
            # differences in 64 bits: 1e-9; the fp32 step: some hundred roundings of terms of order one
            assert abs(got.Data[i] - num) <= 1e-5, (i, got.Data[i], num)
    ops.Dispose()


@pytest.mark.gpu
def test_two_contexts_at_once(fhp, be):
    # each has its own stream, scratch and result: interleaved calls of two threads give what each gives alone
    import threading

    def work(b, seed, out):
        r = np.random.default_rng(seed)
        B, T, H, hd, V, K = 2, 300, 3, 64, 900, 4
        x = fhp.DeviceBuffer.from_array(b, r.normal(0, 1, (B * T, 3 * H * hd)).astype(np.float32))
        d = fhp.DeviceBuffer.from_array(b, r.normal(0, 1, (B * T, H * hd)).astype(np.float32))
        z = fhp.DeviceBuffer.from_array(b, r.normal(0, 2, (T, V)).astype(np.float32))
        ids = fhp.DeviceBuffer.from_array(b, r.integers(0, V, (T, K)).astype(np.int32))
        top = fhp.DeviceBuffer.from_array(b, r.normal(0, 2, (T, K)).astype(np.float32))
        o, l, g = fhp.DeviceBuffer(b, d.nbytes), fhp.DeviceBuffer(b, 4 * B * H * T), fhp.DeviceBuffer(b, x.nbytes)
        targets = r.integers(0, V, T)
        for _ in range(20):
            b.attention_forward(x, o, l, B, T, H, hd)
            loss = b.distill_loss(z, targets, ids, top, None, T, V, K, temperature=2.0, alpha=0.5)
            b.attention_backward(d, x, o, l, g, B, T, H, hd)
            out.append((loss, g.read(np.float32, x.nbytes // 4).tobytes()))
        for buf in (x, d, z, ids, top, o, l, g):
            buf.free()

    with fhp.HipBackend(0) as other:
        alone, together = [[], []], [[], []]
        for b, seed, out in ((be, 1, alone[0]), (other, 2, alone[1])):
            work(b, seed, out)
        threads = [threading.Thread(target=work, args=(b, s, out)) for b, s, out in ((be, 1, together[0]), (other, 2, together[1]))]
        for th in threads:
            th.start()
        for th in threads:
            th.join()
    for a, g in zip(alone, together):
        assert len(g) == 20 and all(x == a[0] for x in a + g)


# ---- refusals (before any device work) --------------------------------------------------------------------

class Calls:
    """The entry points with arguments that would be accepted, each replaceable; the context and the
    buffers are host memory that a refused call does not look into."""

    def __init__(self, fhp):
        self.L, self.N = fhp.lib(), fhp._native
        self.mem = (ctypes.c_char * 65536)()
        self.at = lambda k: (ctypes.addressof(self.mem) + 63) // 64 * 64 + 4096 * k

    def attention(self, back=False, **kw):
        a = dict(ctx=self.at(0), dout=self.at(1), qkv=self.at(2), qkv_cols=48, out=self.at(3), out_cols=16, lse=self.at(4),
                 dqkv=self.at(5), lengths=None, batch=2, T=5, H=2, Hk=2, hd=8, scale=0.5, dtype=0)
        a.update(kw)
        ln = None if a["lengths"] is None else np.asarray(a["lengths"], np.int32)
        tail = [None if ln is None else ln.ctypes.data] + [a[k] for k in ("batch", "T", "H", "Hk", "hd", "scale", "dtype")]
        front = [a[k] for k in ("qkv", "qkv_cols", "out", "out_cols", "lse")]
        if back:
            return self.L.fh_op_attention_backward(a["ctx"], a["dout"], *front, a["dqkv"], *tail)
        return self.L.fh_op_attention_forward(a["ctx"], *front, *tail)

    def distill(self, **kw):
        a = dict(ctx=self.at(0), z=self.at(1), targets=[1, 2, 3], ids=self.at(2), top=self.at(3), dz=self.at(4), T=3, V=9, K=4,
                 ignore=-1, tau=2.0, alpha=0.5, dtype=0)
        a.update(kw)
        tg = None if a["targets"] is None else np.asarray(a["targets"], np.int32)
        loss = ctypes.c_float()
        return self.L.fh_op_distill_loss(a["ctx"], a["z"], None if tg is None else tg.ctypes.data, a["ids"], a["top"], a["dz"],
                                         a["T"], a["V"], a["K"], a["ignore"], a["tau"], a["alpha"], a["dtype"],
                                         ctypes.byref(loss))


@pytest.fixture(scope="module")
def calls(fhp):
    return Calls(fhp)


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("bad,code,words", [
    (dict(ctx=None), "FH_ERR_INVALID", "null context"),
    (dict(qkv=None), "FH_ERR_INVALID", "null buffer"),
    (dict(out=None), "FH_ERR_INVALID", "null buffer"),
    (dict(lse=None), "FH_ERR_INVALID", "null buffer"),
    (dict(batch=0), "FH_ERR_INVALID", "positive"),
    (dict(T=-1), "FH_ERR_INVALID", "positive"),
    (dict(H=0), "FH_ERR_INVALID", "positive"),
    (dict(Hk=0), "FH_ERR_INVALID", "positive"),
    (dict(hd=0), "FH_ERR_INVALID", "positive"),
    (dict(H=3, Hk=2), "FH_ERR_INVALID", "multiple"),
    (dict(H=1, Hk=2), "FH_ERR_INVALID", "multiple"),
    (dict(qkv_cols=47), "FH_ERR_INVALID", "do not hold"),
    (dict(out_cols=15), "FH_ERR_INVALID", "do not hold"),
    (dict(H=2 ** 30, Hk=2 ** 30, hd=100), "FH_ERR_INVALID", "do not hold"),
    (dict(hd=129, qkv_cols=1000, out_cols=1000), "FH_ERR_UNSUPPORTED", "head_dim"),
    (dict(qkv_cols=2 ** 20 + 1), "FH_ERR_UNSUPPORTED", "limits"),
    (dict(out_cols=2 ** 20 + 1), "FH_ERR_UNSUPPORTED", "limits"),
    (dict(T=2 ** 24 + 1), "FH_ERR_UNSUPPORTED", "limits"),
    (dict(batch=2 ** 30), "FH_ERR_UNSUPPORTED", "limits"),
    (dict(scale=0.0), "FH_ERR_INVALID", "scale"),
    (dict(scale=-1.0), "FH_ERR_INVALID", "scale"),
    (dict(scale=float("nan")), "FH_ERR_INVALID", "scale"),
    (dict(scale=float("inf")), "FH_ERR_INVALID", "scale"),
    (dict(dtype=2), "FH_ERR_INVALID", "dtype"),
    (dict(lengths=[5, 6]), "FH_ERR_RANGE", "sequence 1"),
    (dict(lengths=[-1, 5]), "FH_ERR_RANGE", "sequence 0"),
])
def test_attention_refusals(calls, back, bad, code, words):
    assert calls.attention(back, **bad) == getattr(calls.N, code)
    assert words in calls.N.last_error()


def test_attention_refuses_outputs_over_inputs_and_odd_addresses(calls):
    at = calls.at
    for back, bad in [(False, dict(out=at(2))), (False, dict(lse=at(3))), (True, dict(dqkv=at(1))), (True, dict(dqkv=at(2))),
                      (True, dict(dqkv=at(3))), (True, dict(dqkv=at(4)))]:
        assert calls.attention(back, **bad) == calls.N.FH_ERR_INVALID
        assert "of its own" in calls.N.last_error() or "of their own" in calls.N.last_error()
    for back, bad in [(False, dict(qkv=at(2) + 2)), (False, dict(out=at(3) + 1, dtype=1)), (False, dict(lse=at(4) + 2, dtype=1)),
                      (True, dict(dout=at(1) + 2)), (True, dict(dqkv=at(5) + 1, dtype=1))]:
        assert calls.attention(back, **bad) == calls.N.FH_ERR_INVALID
        assert "aligned" in calls.N.last_error()
    assert calls.attention(True, dout=None) == calls.attention(True, dqkv=None) == calls.N.FH_ERR_INVALID


@pytest.mark.parametrize("bad,code,words", [
    (dict(ctx=None), "FH_ERR_INVALID", "null context"),
    (dict(z=None), "FH_ERR_INVALID", "null buffer"),
    (dict(targets=None), "FH_ERR_INVALID", "null buffer"),
    (dict(ids=None), "FH_ERR_INVALID", "null buffer"),
    (dict(top=None), "FH_ERR_INVALID", "null buffer"),
    (dict(T=0), "FH_ERR_INVALID", "positive"),
    (dict(V=0), "FH_ERR_INVALID", "positive"),
    (dict(K=0), "FH_ERR_INVALID", "positive"),
    (dict(tau=0.0), "FH_ERR_INVALID", "temperature"),
    (dict(tau=float("inf")), "FH_ERR_INVALID", "temperature"),
    (dict(alpha=-0.1), "FH_ERR_INVALID", "alpha"),
    (dict(alpha=1.1), "FH_ERR_INVALID", "alpha"),
    (dict(alpha=float("nan")), "FH_ERR_INVALID", "alpha"),
    (dict(dtype=7), "FH_ERR_INVALID", "dtype"),
    (dict(K=1025), "FH_ERR_UNSUPPORTED", "1024"),
    (dict(T=2 ** 24), "FH_ERR_UNSUPPORTED", "2^24"),
    (dict(targets=[0, 9, 1]), "FH_ERR_RANGE", "position 1"),
    (dict(targets=[0, 1, -2]), "FH_ERR_RANGE", "position 2"),
])
def test_distill_refusals(calls, bad, code, words):
    assert calls.distill(**bad) == getattr(calls.N, code)
    assert words in calls.N.last_error()


def test_distill_refuses_odd_addresses(calls):
    for bad in (dict(z=calls.at(1) + 2), dict(dz=calls.at(4) + 1, dtype=1), dict(ids=calls.at(2) + 2), dict(top=calls.at(3) + 1)):
        assert calls.distill(**bad) == calls.N.FH_ERR_INVALID
        assert "aligned" in calls.N.last_error()


def test_host_mirror_checks_sizes_before_the_call(fhp):
    class Buf(fhp.DeviceBuffer):
        def __init__(self, nbytes):
            self.nbytes = nbytes
            self.ptr = ctypes.c_void_p(0)
    be = fhp.HipBackend.__new__(fhp.HipBackend)
    be._ctx = ctypes.c_void_p(0)
    ok = dict(qkv=Buf(2 * 5 * 48 * 4), out=Buf(2 * 5 * 16 * 4), lse=Buf(2 * 2 * 5 * 4))
    for name in ok:
        small = {**ok, name: Buf(ok[name].nbytes - 1)}
        with pytest.raises(ValueError, match=name):
            be.attention_forward(*small.values(), 2, 5, 2, 8)
    with pytest.raises(ValueError, match="dqkv"):
        be.attention_backward(ok["out"], *ok.values(), Buf(1), 2, 5, 2, 8)
    with pytest.raises(ValueError, match="lengths"):
        be.attention_forward(*ok.values(), 2, 5, 2, 8, lengths=[5])
    with pytest.raises(fhp.ArgumentError, match="null context"):
        be.attention_forward(*ok.values(), 2, 5, 2, 8)
    z, ids, top = Buf(3 * 9 * 4), Buf(3 * 4 * 4), Buf(3 * 4 * 4)
    for bad in ((Buf(4), ids, top, None), (z, Buf(4), top, None), (z, ids, Buf(4), None), (z, ids, top, Buf(4))):
        with pytest.raises(ValueError, match="needs"):
            be.distill_loss(bad[0], [0, 1, 2], bad[1], bad[2], bad[3], 3, 9, 4)
    with pytest.raises(ValueError, match="targets"):
        be.distill_loss(z, [0, 1], ids, top, None, 3, 9, 4)
