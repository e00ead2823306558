"""GPU tests of the few-row operators on block-float weights (bfp_matvec, moe_route, moe_experts, moe_layer) against plain
64-bit implementations on the oracle-decoded weights.

Tolerances, derived: a product of two stored operands (8 bits each) is exact in binary32.  Adding n of them in any order,
each addition off by at most one last place of a partial sum that no sum of magnitudes exceeds, is off by at most
n 2^-23 sum |products|.  Rounding the result to bfloat16 adds 2^-8 of it, to binary32 2^-24.  The experts' intermediate
is carried in two bfloat16 pieces, off by at most 2^-16 of it; the slope of silu and gelu stays below 1.13, and their
binary32 evaluation is off by a few units of 2^-24, for which 2^-19 of the value is allowed."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

FORMATS = ["Bfp8_b", "Bfp4_b", "Bfp2_b"]


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.fail("these tests need a CUDA device; there is no CPU fallback to test")
    from pybuda import cuda_ops

    return cuda_ops


def _pad32(n):
    return -(-n // 32) * 32


def _store(oracle, w, df):
    """(queue image as CUDA bytes, float64 values it stands for) of a [K,N] matrix, zero-padded to tiles."""
    k, n = w.shape
    p = np.zeros((1, 1, _pad32(k), _pad32(n)), np.float32)
    p[0, 0, :k, :n] = w
    code = getattr(oracle, df)
    img = oracle.tilize_pack(p, code)
    return torch.from_numpy(img).cuda(), oracle.unpack_untilize(img, code, p.shape)[0, 0, :k, :n].astype(np.float64)


def _rand(shape, seed, scale=1.0):
    return (np.random.default_rng(seed).standard_normal(shape) * scale).astype(np.float32)


def _bf16(x):
    return torch.from_numpy(np.ascontiguousarray(x)).bfloat16()


def _check_sum(got, a, w, dtype):
    """got = a @ w for exact operands a, w (float64 numpy)."""
    ref, mag = a @ w, np.abs(a) @ np.abs(w)
    tol = (a.shape[1] + 16) * 2.0 ** -23 * mag + np.abs(ref) * (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24) + 2.0 ** -133
    err = np.abs(got.double().cpu().numpy() - ref)
    assert got.dtype == dtype and (err <= tol).all(), f"worst {np.max(err / tol)} of the tolerance at {np.unravel_index(np.argmax(err / tol), err.shape)}"


# ------------------------------------------------------------------------------------------------ matvec
@pytest.mark.parametrize("df", FORMATS)
@pytest.mark.parametrize("m,k,n", [(1, 32, 32), (1, 1, 1), (2, 17, 33), (3, 64, 128), (8, 100, 130), (9, 256, 96), (16, 544, 288), (17, 96, 160),
                                   (33, 320, 64), (64, 70, 40), (1, 4096, 256), (5, 2080, 1100)])
def test_matvec_shapes(ops, oracle, df, m, k, n):
    img, w = _store(oracle, _rand((k, n), m + k + n, 0.05), df)
    a = _bf16(_rand((m, k), 1))
    for dtype in (torch.bfloat16, torch.float32):
        got = ops.bfp_matvec(a.cuda(), img, n, getattr(ops.DF, df), out_dtype=dtype)
        _check_sum(got, a.double().numpy(), w, dtype)
    rc, st = ops._cabi.device_status()
    assert rc == 0 and st == 0


@pytest.mark.parametrize("df", FORMATS)
def test_matvec_one_hot_rows_copy_the_stored_values(ops, oracle, df):
    k, n = 96, 160
    img, w = _store(oracle, _rand((k, n), 3), df)      # magnitudes on both sides of 2: shared exponents on both sides of 128
    a = torch.eye(k)[:64].bfloat16()
    got = ops.bfp_matvec(a.cuda(), img, n, getattr(ops.DF, df), out_dtype=torch.float32).cpu().numpy()
    assert np.array_equal(got, w[:64].astype(np.float32))
    got = ops.bfp_matvec(torch.eye(k)[32:].bfloat16().cuda(), img, n, getattr(ops.DF, df)).cpu()
    assert torch.equal(got.float(), torch.from_numpy(w[32:].astype(np.float32)))


@pytest.mark.parametrize("df", FORMATS)
@pytest.mark.parametrize("exponent", [1, 2, 7, 64, 126, 127, 128, 129, 190, 253])
def test_matvec_shared_exponents_of_the_whole_range(ops, oracle, df, exponent):
    """Images of one shared exponent and all data patterns; the activation brings the product back to the middle."""
    code, m = getattr(ops.DF, df), {"Bfp8_b": 7, "Bfp4_b": 3, "Bfp2_b": 1}[df]
    rec = {"Bfp8_b": 1088, "Bfp4_b": 576, "Bfp2_b": 320}[df]
    raw = np.random.default_rng(exponent).integers(0, 256, rec, dtype=np.uint8)
    raw[:64] = exponent
    w = oracle.unpack_untilize(raw, getattr(oracle, df), (1, 1, 32, 32))[0, 0].astype(np.float64)
    back = 2.0 ** min(127, max(-120, 127 - exponent))
    a = torch.eye(32).mul(back).bfloat16()
    got = ops.bfp_matvec(a.cuda(), torch.from_numpy(raw).cuda(), 32, code, out_dtype=torch.float32).cpu().numpy()
    assert np.array_equal(got.astype(np.float64), w * back)
    assert np.abs(w).max() >= 2.0 ** (exponent - 127) * (1 if m > 1 else 0.5)


@pytest.mark.parametrize("df", FORMATS)
@pytest.mark.parametrize("exponent", [1, 2, 7, 64, 126, 127, 128, 129, 190, 253])
def test_matvec_one_row_over_the_whole_range(ops, oracle, df, exponent):
    """The same for a single row, whose activations are scaled in place of the weights: each of the 32 rows on its own, with
    activations from the smallest normal number to the largest that keeps the product finite."""
    code, m = getattr(ops.DF, df), {"Bfp8_b": 7, "Bfp4_b": 3, "Bfp2_b": 1}[df]
    rec = {"Bfp8_b": 1088, "Bfp4_b": 576, "Bfp2_b": 320}[df]
    raw = np.random.default_rng(exponent).integers(0, 256, rec, dtype=np.uint8)
    raw[:64] = exponent
    w = oracle.unpack_untilize(raw, getattr(oracle, df), (1, 1, 32, 32))[0, 0].astype(np.float64)
    img = torch.from_numpy(raw).cuda()
    for power in (-126, -100, -30, 0, 30, 100, 127):
        if not -110 <= exponent - 127 + power <= 126:
            continue                        # the product leaves binary32, or is small enough to be rounded at 2^-125
        for k in (0, 5, 14, 31):
            a = torch.zeros(1, 32)
            a[0, k] = -(2.0 ** power)
            got = ops.bfp_matvec(a.bfloat16().cuda(), img, 32, code, out_dtype=torch.float32).cpu().numpy()
            assert np.array_equal(got[0].astype(np.float64), -w[k] * 2.0 ** power), (power, k)


@pytest.mark.parametrize("df", FORMATS)
def test_matvec_one_row_of_mixed_magnitudes(ops, oracle, df):
    """Blocks of very unlike shared exponents in one matrix against activations that undo them: every step takes the wide path."""
    k, n = 160, 200
    rng = np.random.default_rng(2)
    power = rng.integers(-60, 61, (k, 1))
    w0 = rng.standard_normal((k, n)) * 2.0 ** power * np.repeat(2.0 ** rng.integers(-8, 9, (k, -(-n // 16))), 16, 1)[:, :n]
    img, w = _store(oracle, w0.astype(np.float32), df)
    for rows in (1, 3):
        a = torch.from_numpy(rng.standard_normal((rows, k)) * 2.0 ** (-power[:, 0] + 20)).bfloat16()
        got = ops.bfp_matvec(a.cuda(), img, n, getattr(ops.DF, df), out_dtype=torch.float32)
        _check_sum(got, a.double().numpy(), w, torch.float32)


def test_matvec_not_finite_activations_stay_in_their_row(ops, oracle):
    k, n = 64, 96
    img, w = _store(oracle, _rand((k, n), 5) + 0.1, "Bfp4_b")
    a = _bf16(_rand((4, k), 6))
    a[1, 7], a[2, 63], a[2, 0] = float("nan"), float("inf"), float("-inf")
    got = ops.bfp_matvec(a.cuda(), img, n, ops.DF.Bfp4_b, out_dtype=torch.float32).cpu()
    assert torch.isnan(got[1]).all() and not torch.isfinite(got[2]).any()
    _check_sum(got[[0, 3]], a.double().numpy()[[0, 3]], w, torch.float32)
    assert torch.isnan(ops.bfp_matvec(a[1:2].cuda(), img, n, ops.DF.Bfp4_b)).all()
    assert not torch.isfinite(ops.bfp_matvec(a[2:3].cuda(), img, n, ops.DF.Bfp4_b)).any()


def test_matvec_strides_alignment_and_neighbours(ops, oracle):
    k, n = 75, 70
    img, w = _store(oracle, _rand((k, n), 8, 0.1), "Bfp8_b")
    for offset, pitch in ((0, 75), (1, 76), (1, 81), (2, 128), (3, 77)):
        big = _bf16(_rand((5, 256), offset)).reshape(-1).cuda()
        a = big[offset:offset + 4 * pitch + k].as_strided((5, k), (pitch, 1))
        wide = torch.full((9, n + 5), 7.0, dtype=torch.bfloat16, device="cuda")
        ops.bfp_matvec(a, img, n, ops.DF.Bfp8_b, out=wide[2:7, 3:3 + n])
        _check_sum(wide[2:7, 3:3 + n], a.double().cpu().numpy(), w, torch.bfloat16)
        wide[2:7, 3:3 + n] = 7.0
        assert torch.all(wide == 7.0)       # rows behind the last one and columns beside them keep what they held
    same = a[:1].expand(6, k)               # a row stride of zero
    got = ops.bfp_matvec(same, img, n, ops.DF.Bfp8_b)
    assert torch.equal(got, got[:1].expand_as(got))
    assert ops.bfp_matvec(a[:0], img, n, ops.DF.Bfp8_b).shape == (0, n)


def test_matvec_rows_do_not_depend_on_their_company(ops, oracle):
    k, n = 512, 256
    img, _ = _store(oracle, _rand((k, n), 9, 0.1), "Bfp4_b")
    a = _bf16(_rand((8, k), 2)).cuda()
    all8 = ops.bfp_matvec(a, img, n, ops.DF.Bfp4_b, out_dtype=torch.float32)
    for i in (0, 5):
        assert torch.equal(all8[i], ops.bfp_matvec(a[i:i + 1], img, n, ops.DF.Bfp4_b, out_dtype=torch.float32)[0])
    for _ in range(20):
        assert torch.equal(all8, ops.bfp_matvec(a, img, n, ops.DF.Bfp4_b, out_dtype=torch.float32))


# ------------------------------------------------------------------------------------------------ router
def _route_ref(x, w, top, renorm):
    l = x.double().numpy() @ w.double().numpy().T
    ids = np.argsort(-l, axis=1, kind="stable")[:, :top]
    p = np.exp(l - l.max(1, keepdims=True))
    c = np.take_along_axis(p, ids, 1)
    return c / (c.sum(1, keepdims=True) if renorm else p.sum(1, keepdims=True)), ids


@pytest.mark.parametrize("router", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t,h,e,top", [(1, 1, 1, 1), (1, 8, 2, 2), (2, 33, 5, 3), (3, 1024, 8, 2), (17, 100, 7, 7), (19, 257, 64, 8), (37, 512, 65, 16),
                                       (64, 96, 256, 16), (40, 2048, 128, 1)])
def test_route_shapes(ops, router, t, h, e, top):
    g = torch.Generator().manual_seed(t + h + e)
    x, w = torch.randn(t, h, generator=g).bfloat16(), (torch.randn(e, h, generator=g) * 2 * h ** -0.5).to(router)
    for renorm in (True, False):
        weights, ids = ops.moe_route(x.cuda(), w.cuda(), top, renorm)
        ref, rid = _route_ref(x, w, top, renorm)
        assert ids.dtype == torch.int32 and np.array_equal(ids.cpu().numpy(), rid)
        # scores below 16 in magnitude, exponentials and the sum in binary32: a few units of 2^-24 each, h / 8 group sums exact to 2^-24
        assert np.abs(weights.double().cpu().numpy() - ref).max() <= 2.0 ** -18 * ref.max()


def test_route_ties_go_to_the_lowest_index(ops):
    x = torch.ones(3, 64).bfloat16().cuda()
    w = torch.zeros(40, 64, device="cuda")
    w[[7, 9, 33], 0] = 2.0
    w[3, 0] = -0.0
    weights, ids = ops.moe_route(x, w, 6, True)
    assert ids.cpu().tolist() == [[7, 9, 33, 0, 1, 2]] * 3
    w.zero_()
    weights, ids = ops.moe_route(x, w, 5, False)
    assert ids.cpu().tolist() == [[0, 1, 2, 3, 4]] * 3
    assert torch.equal(weights.cpu(), torch.full((3, 5), 1 / 40))


def test_route_scores_that_are_not_numbers(ops):
    x = torch.ones(2, 16).bfloat16().cuda()
    w = torch.arange(6, device="cuda").float().view(6, 1).expand(6, 16).contiguous()
    w[4, 3] = float("nan")
    w[5, 3] = -float("inf")
    weights, ids = ops.moe_route(x, w, 6, True)
    assert ids.cpu().tolist() == [[3, 2, 1, 0, 5, 4]] * 2       # a NaN score behind every number
    assert torch.isnan(weights).all()
    weights, ids = ops.moe_route(x, w, 4, True)
    assert ids.cpu().tolist() == [[3, 2, 1, 0]] * 2 and torch.allclose(weights.sum(1), torch.ones(2, device="cuda"))
    w[:] = float("nan")
    _, ids = ops.moe_route(x, w, 3, False)
    assert ids.cpu().tolist() == [[0, 1, 2]] * 2                # distinct experts whatever the scores are


def test_route_strides_and_alignment(ops):
    g = torch.Generator().manual_seed(4)
    buf, wbuf = torch.randn(4000, generator=g).bfloat16().cuda(), torch.randn(9000, generator=g).cuda()
    for off, h, pitch in ((1, 120, 128), (0, 121, 121), (8, 64, 72), (3, 99, 130)):
        x = buf[off:].as_strided((6, h), (pitch, 1), off)
        w = wbuf.as_strided((24, h), (pitch + 4, 1), off)
        _, ids = ops.moe_route(x, w, 4, True)
        assert np.array_equal(ids.cpu().numpy(), _route_ref(x.cpu(), w.cpu(), 4, True)[1])


# ------------------------------------------------------------------------------------------------ experts
def _make_experts(oracle, e, h, i, df, seed, gated=True):
    out = []
    for which, (r, c) in enumerate(((h, i), (h, i), (i, h))):
        if which == 1 and not gated:
            out.append((None, None))
            continue
        pairs = [_store(oracle, _rand((r, c), seed + 10 * which + 100 * k, r ** -0.5), df) for k in range(e)]
        out.append((torch.stack([p[0] for p in pairs]), np.stack([p[1] for p in pairs])))
    return [o[0] for o in out], [o[1] for o in out]


def _experts_ref(x, weights, ids, vals, act):
    """(reference, tolerance) in float64."""
    gate, up, down = vals
    x, weights, ids = x.double().numpy(), weights.double().cpu().numpy(), ids.cpu().numpy()
    y, tol = np.zeros(x.shape), np.zeros(x.shape)
    erf = lambda v: torch.erf(torch.from_numpy(v)).numpy()
    h_n, i_n = gate.shape[1], gate.shape[2]
    for t in range(x.shape[0]):
        for s in range(ids.shape[1]):
            e = ids[t, s]
            if e < 0 or e >= gate.shape[0]:
                continue
            w = weights[t, s]
            gt, dg = x[t] @ gate[e], (h_n + 16) * 2.0 ** -23 * (np.abs(x[t]) @ np.abs(gate[e]))
            a = gt / (1 + np.exp(-gt)) if act == "silu" else 0.5 * gt * (1 + erf(gt / np.sqrt(2)))
            da = 1.13 * dg + 2.0 ** -19 * np.abs(a) + 2.0 ** -100
            u, du = (1.0, 0.0) if up is None else (x[t] @ up[e], (h_n + 16) * 2.0 ** -23 * (np.abs(x[t]) @ np.abs(up[e])))
            h = a * u
            dh = da * (np.abs(u) + du) + np.abs(a) * du
            dh += 2.0 ** -16 * (np.abs(h) + dh)
            y[t] += w * (h @ down[e])
            tol[t] += abs(w) * ((dh + (2 * i_n * ids.shape[1] + 16) * 2.0 ** -23 * (np.abs(h) + dh)) @ np.abs(down[e]))
    return y, tol + 2.0 ** -8 * (np.abs(y) + tol)


def _check_experts(got, x, weights, ids, vals, act):
    ref, tol = _experts_ref(x, weights, ids, vals, act)
    err = np.abs(got.double().cpu().numpy() - ref)
    assert (err <= tol).all(), f"worst {np.max(err / np.maximum(tol, 1e-300))} of the tolerance"


def _routing(t, e, top, seed, drop=0.0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.rand(t, e, generator=g).argsort(1)[:, :top].int()
    weights = torch.rand(t, top, generator=g)
    if drop:
        ids[torch.rand(t, top, generator=g) < drop] = -1
    return weights, ids


@pytest.mark.parametrize("df", FORMATS)
@pytest.mark.parametrize("t,h,i,e,top,act,gated", [(1, 32, 32, 1, 1, "silu", True), (1, 64, 96, 4, 2, "gelu", True), (3, 100, 50, 5, 3, "silu", True),
                                                  (8, 128, 160, 3, 2, "gelu", False), (9, 96, 64, 6, 2, "silu", True), (20, 70, 33, 2, 1, "gelu", True),
                                                  (40, 64, 40, 3, 3, "silu", False), (64, 33, 65, 20, 4, "gelu", True), (2, 300, 700, 2, 2, "silu", True)])
def test_experts_shapes(ops, oracle, df, t, h, i, e, top, act, gated):
    images, vals = _make_experts(oracle, e, h, i, df, t + h, gated)
    x = _bf16(_rand((t, h), 7))
    weights, ids = _routing(t, e, top, t, drop=0.2 if top > 2 else 0.0)
    got = ops.moe_experts(x.cuda(), weights.cuda(), ids.cuda(), *images, i, getattr(ops.DF, df), act)
    assert got.dtype == torch.bfloat16 and got.shape == (t, h)
    _check_experts(got, x, weights, ids, vals, act)
    rc, st = ops._cabi.device_status()
    assert rc == 0 and st == 0


def test_experts_dropped_repeated_and_foreign_slots(ops, oracle):
    e, h, i, t = 5, 96, 80, 6
    images, vals = _make_experts(oracle, e, h, i, "Bfp4_b", 11)
    x = _bf16(_rand((t, h), 12))
    weights = torch.rand(t, 4, generator=torch.Generator().manual_seed(5))
    ids = torch.tensor([[0, 1, 2, 3], [4, 4, 4, 4], [-1, -1, -1, -1], [2, -1, 2, 0], [5, 1000000, -7, 3], [1, 1, -1, 0]], dtype=torch.int32)
    got = ops.moe_experts(x.cuda(), weights.cuda(), ids.cuda(), *images, i)
    _check_experts(got, x, weights, ids, vals, "silu")
    assert torch.all(got[2] == 0)
    for rows in (1, 6, 12):
        none = ops.moe_experts(x.repeat(2, 1)[:rows].cuda(), weights.repeat(2, 1)[:rows].cuda(), torch.full((rows, 4), -1, dtype=torch.int32, device="cuda"),
                               *images, i)
        assert torch.all(none == 0) and none.shape == (rows, h)


@pytest.mark.parametrize("df", FORMATS)
@pytest.mark.parametrize("t", [1, 3, 12])
def test_experts_infinite_weights_reach_their_own_tokens_only(ops, oracle, df, t):
    """Images packed from matrices with infinities: their experts' tokens get numbers that are not finite, all others what they get
    without that expert.  (Few tokens run through all experts as one sum, with zeros in the other experts' rows.)"""
    e, h, i = 3, 96, 64
    images, vals = _make_experts(oracle, e, h, i, df, 24)
    broken = _rand((i, h), 25, 0.1)
    broken[3, :] = np.inf
    images[2][1] = _store(oracle, broken, df)[0]
    x = _bf16(_rand((t, h), 26))
    ids = torch.tensor([[k % 3, (k + 2) % 3] for k in range(t)], dtype=torch.int32)     # every third pair has no expert 1
    weights = torch.rand(t, 2, generator=torch.Generator().manual_seed(27)) + 0.1
    got = ops.moe_experts(x.cuda(), weights.cuda(), ids.cuda(), *images, i, getattr(ops.DF, df))
    clean = [k for k in range(t) if 1 not in ids[k]]
    dirty = [k for k in range(t) if 1 in ids[k]]
    assert not dirty or not torch.isfinite(got[dirty]).any()
    _check_experts(got[clean], x[clean], weights[clean], ids[clean], vals, "silu")


def test_experts_many_experts_one_token_each(ops, oracle):
    e, h, i, t = 256, 32, 32, 64
    images, vals = _make_experts(oracle, e, h, i, "Bfp2_b", 13)
    x = _bf16(_rand((t, h), 14))
    ids = torch.arange(256, dtype=torch.int32).view(64, 4).flip(0).contiguous()
    weights = torch.rand(t, 4, generator=torch.Generator().manual_seed(6))
    got = ops.moe_experts(x.cuda(), weights.cuda(), ids.cuda(), *images, i, ops.DF.Bfp2_b)
    _check_experts(got, x, weights, ids, vals, "silu")
    one = torch.full((t, 1), 255, dtype=torch.int32)            # all tokens to the last expert
    got = ops.moe_experts(x.cuda(), weights[:, :1].contiguous().cuda(), one.cuda(), *images, i, ops.DF.Bfp2_b, "gelu")
    _check_experts(got, x, weights[:, :1], one, vals, "gelu")


def test_experts_strides_neighbours_and_in_place(ops, oracle):
    e, h, i, t = 3, 70, 40, 5
    images, vals = _make_experts(oracle, e, h, i, "Bfp8_b", 15)
    big = _bf16(_rand((8, 91), 16)).cuda()
    x = big[1:6, 3:3 + h]
    weights, ids = _routing(t, e, 2, 3)
    wide = torch.full((7, 90), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.moe_experts(x, weights.cuda(), ids.cuda(), *images, i, ops.DF.Bfp8_b, out=wide[1:6, 5:5 + h])
    _check_experts(wide[1:6, 5:5 + h], x.cpu(), weights, ids, vals, "silu")
    want = wide[1:6, 5:5 + h].clone()
    wide[1:6, 5:5 + h] = 7.0
    assert torch.all(wide == 7.0)
    before = big.clone()
    ops.moe_experts(x, weights.cuda(), ids.cuda(), *images, i, ops.DF.Bfp8_b, out=x)
    assert torch.equal(x, want)
    big[1:6, 3:3 + h] = before[1:6, 3:3 + h]
    assert torch.equal(big, before)


# ------------------------------------------------------------------------------------------------ the layer, and the operators together
@pytest.mark.parametrize("t,h,i,e,top,df,router", [(1, 64, 96, 8, 2, "Bfp4_b", torch.float32), (7, 100, 40, 12, 3, "Bfp8_b", torch.bfloat16),
                                                   (33, 64, 64, 40, 4, "Bfp2_b", torch.float32)])
def test_layer_is_route_then_experts(ops, oracle, t, h, i, e, top, df, router):
    images, vals = _make_experts(oracle, e, h, i, df, 17)
    g = torch.Generator().manual_seed(18)
    x, wr = torch.randn(t, h, generator=g).bfloat16(), (torch.randn(e, h, generator=g) * 2 * h ** -0.5).to(router)
    for renorm in (True, False):
        weights, ids = ops.moe_route(x.cuda(), wr.cuda(), top, renorm)
        two = ops.moe_experts(x.cuda(), weights, ids, *images, i, getattr(ops.DF, df), "gelu")
        for _ in range(5):
            assert torch.equal(two, ops.moe_layer(x.cuda(), wr.cuda(), top, *images, i, getattr(ops.DF, df), "gelu", renorm))
        rw, rid = _route_ref(x, wr, top, renorm)
        _check_experts(two, x, torch.from_numpy(rw), torch.from_numpy(rid), vals, "gelu")


def _block(ops, x, proj, wr, images, i):
    """A decoding step's use: a projection, the layer on its result, a projection of the sum back to binary32."""
    a = ops.bfp_matvec(x, proj, x.shape[1], ops.DF.Bfp4_b)
    y = ops.moe_layer(a, wr, 2, *images, i)
    return ops.bfp_matvec(a + y, proj, x.shape[1], ops.DF.Bfp4_b, out_dtype=torch.float32), y


def test_operators_together_eager_captured_and_on_side_streams(ops, oracle):
    h, i, e = 128, 96, 8
    images, _ = _make_experts(oracle, e, h, i, "Bfp4_b", 19)
    proj, pv = _store(oracle, _rand((h, h), 20, h ** -0.5), "Bfp4_b")
    wr = torch.randn(e, h, generator=torch.Generator().manual_seed(21)).cuda() * 0.2
    xs = [_bf16(_rand((3, h), 30 + k)).cuda() for k in range(6)]
    want = [_block(ops, x, proj, wr, images, i) for x in xs]
    a = ops.bfp_matvec(xs[0], proj, h, ops.DF.Bfp4_b)
    _check_sum(a, xs[0].double().cpu().numpy(), pv, torch.bfloat16)
    # two graphs, replayed at the same time on two streams
    graphs, bufs, outs, streams = [], [], [], [torch.cuda.Stream() for _ in range(2)]
    for k in range(2):
        buf = xs[k].clone()
        gr = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(gr):
            out = _block(ops, buf, proj, wr, images, i)
        graphs.append(gr), bufs.append(buf), outs.append(out)
    for r in range(3):
        for k in range(2):
            bufs[k].copy_(xs[2 * r + k])
        torch.cuda.synchronize()
        for _ in range(10):
            for k in range(2):
                with torch.cuda.stream(streams[k]):
                    graphs[k].replay()
        torch.cuda.synchronize()
        for k in range(2):
            assert torch.equal(outs[k][0], want[2 * r + k][0]) and torch.equal(outs[k][1], want[2 * r + k][1])
    # eager calls on two streams at once
    got = [[], []]
    for r in range(20):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(_block(ops, xs[k], proj, wr, images, i))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(o[0], want[k][0]) and torch.equal(o[1], want[k][1]) for o in got[k])
    rc, st = ops._cabi.device_status()
    assert rc == 0 and st == 0


def test_images_from_the_pack_of_a_stacked_tensor(ops, oracle):
    """The documented way to the images: tilize_pack of [1,E,H,I], one row of bytes for each expert."""
    e, h, i = 3, 64, 96
    w = _rand((1, e, h, i), 22, 0.1)
    img = ops.tilize_pack(torch.from_numpy(w).cuda(), ops.DF.Bfp4_b).view(e, -1)
    for k in range(e):
        assert torch.equal(img[k], _store(oracle, w[0, k], "Bfp4_b")[0])


def test_image_past_4_gib(ops):
    """Records whose offsets pass 32 bits: 512 experts' worth of bytes in a 256-expert set, only the ends filled."""
    e, h, i = 256, 4096, 4096
    per = (h // 32) * (i // 32) * 1088
    images = torch.zeros(e, per, dtype=torch.uint8, device="cuda")
    assert images.numel() > 1 << 32
    g = torch.Generator().manual_seed(23)
    x = torch.randn(2, h, generator=g).bfloat16().cuda()
    small = torch.randn(1, 1, h, i, generator=g) * h ** -0.5
    img = ops.tilize_pack(small.cuda(), ops.DF.Bfp8_b)
    images[255] = img
    images[3] = img
    weights = torch.ones(2, 1, device="cuda")
    last = ops.moe_experts(x, weights, torch.tensor([[255], [255]], dtype=torch.int32, device="cuda"), images, images, images, i, ops.DF.Bfp8_b)
    low = ops.moe_experts(x, weights, torch.tensor([[3], [3]], dtype=torch.int32, device="cuda"), images, images, images, i, ops.DF.Bfp8_b)
    assert torch.equal(last, low) and last.float().abs().max() > 0.01


# ------------------------------------------------------------------------------------------------ what a caller may do, and may not
def test_empty_batches(ops, oracle):
    images, _ = _make_experts(oracle, 3, 64, 32, "Bfp4_b", 40)
    x = torch.zeros(0, 64, dtype=torch.bfloat16, device="cuda")
    wr = torch.ones(3, 64, device="cuda")
    weights, ids = ops.moe_route(x, wr, 2)
    assert weights.shape == ids.shape == (0, 2)
    assert ops.moe_experts(x, weights, ids, *images, 32).shape == (0, 64)
    assert ops.moe_layer(x, wr, 2, *images, 32).shape == (0, 64)


def test_refusals(ops, oracle):
    images, _ = _make_experts(oracle, 3, 64, 32, "Bfp4_b", 41)
    x, wr = torch.zeros(2, 64, dtype=torch.bfloat16, device="cuda"), torch.ones(3, 64, device="cuda")
    weights, ids = torch.ones(2, 2, device="cuda"), torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    big = torch.zeros(4 * 576 + 32, dtype=torch.uint8, device="cuda")
    bad = [
        lambda: ops.bfp_matvec(x, big[16:], 64),                                          # image not 32-byte aligned
        lambda: ops.bfp_matvec(x, big[:3 * 576], 64),                                     # too small
        lambda: ops.bfp_matvec(x, big, 0),
        lambda: ops.bfp_matvec(x, big.view(torch.int8), 64),
        lambda: ops.bfp_matvec(x.expand(65, 2, 64)[:, 0], big, 64),                       # 65 rows
        lambda: ops.bfp_matvec(x, big, 64, out_dtype=torch.float16),
        lambda: ops.bfp_matvec(x, big, 64, out=torch.empty(2, 65, dtype=torch.bfloat16, device="cuda")),
        lambda: ops.bfp_matvec(x, big, 64, out=torch.empty(64, 2, dtype=torch.bfloat16, device="cuda").t()),
        lambda: ops.bfp_matvec(x, big, 64, out=torch.empty(1, 64, dtype=torch.bfloat16, device="cuda").expand(2, 64)),   # rows on one another
        lambda: ops.moe_route(x, wr, 4),                                                  # more than there are
        lambda: ops.moe_route(x, wr, 0),
        lambda: ops.moe_route(x, wr[:, :63], 1),
        lambda: ops.moe_route(x, wr.half(), 1),
        lambda: ops.moe_route(x, wr.expand(90, 3, 64).reshape(270, 64), 1),               # 270 experts
        lambda: ops.moe_experts(x, weights, ids.long(), *images, 32),
        lambda: ops.moe_experts(x, weights[:, :1], ids, *images, 32),
        lambda: ops.moe_experts(x, weights.t(), ids, *images, 32),
        lambda: ops.moe_experts(x, weights, ids, images[0], images[1][:2], images[2], 32),
        lambda: ops.moe_experts(x, weights, ids, *images, 33),
        lambda: ops.moe_experts(x, weights, ids, *images, 32, activation="tanh"),
        lambda: ops.moe_layer(x, wr[:2], 2, *images, 32),
        lambda: ops.moe_layer(x.cpu(), wr, 2, *images, 32),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was not refused")
    prev = ops.get_bfp_policy()
    try:
        ops.set_bfp_policy(ops._cabi.BfpPolicy(face_order=(0, 2, 1, 3)))
        with pytest.raises(ops._cabi.BudaError, match="byte layout"):
            ops.bfp_matvec(x, big, 64)
    finally:
        ops.set_bfp_policy(prev)
    ops.bfp_matvec(x, big, 64)


@pytest.mark.parametrize("df", FORMATS)
@pytest.mark.parametrize("t,h,i,e", [(40, 1024, 40, 2), (64, 1056, 200, 3)])
def test_experts_of_many_tokens_over_clusters(ops, oracle, df, t, h, i, e):
    """Several passes over one expert's tokens, each joined over a cluster of CTAs."""
    images, vals = _make_experts(oracle, e, h, i, df, 42)
    x = _bf16(_rand((t, h), 43))
    weights, ids = _routing(t, e, 2, 44)
    got = ops.moe_experts(x.cuda(), weights.cuda(), ids.cuda(), *images, i, getattr(ops.DF, df))
    _check_experts(got, x, weights, ids, vals, "silu")


@pytest.mark.parametrize("captured", [False, True])
def test_weights_that_another_stream_has_just_packed(ops, oracle, captured):
    """A launch may ask for its weights while the launch in front of it still runs; not before an event that the stream waits for."""
    k = n = 512
    a = _bf16(_rand((1, k), 45)).cuda()
    other, _ = _store(oracle, _rand((k, n), 46, 0.1), "Bfp4_b")
    w = [torch.from_numpy(_rand((1, 1, k, n), 47 + r, 0.1)).cuda() for r in range(4)]
    want = [ops.bfp_matvec(a, ops.tilize_pack(x, ops.DF.Bfp4_b), n) for x in w]
    src, img = w[0].clone(), torch.zeros_like(other)
    main, side = torch.cuda.Stream(), torch.cuda.Stream()

    def step():
        side.wait_stream(torch.cuda.current_stream())
        ops.bfp_matvec(a, other, n)
        with torch.cuda.stream(side):
            torch.cuda._sleep(200000)
            ops.tilize_pack(src, ops.DF.Bfp4_b, out=img)
        torch.cuda.current_stream().wait_stream(side)
        return ops.bfp_matvec(a, img, n)

    torch.cuda.synchronize()
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=main):
            got = step()
    for r in range(4):
        img.zero_()
        src.copy_(w[r])
        torch.cuda.synchronize()
        if captured:
            graph.replay()
        else:
            with torch.cuda.stream(main):
                got = step()
        torch.cuda.synchronize()
        assert torch.equal(got, want[r]), r


_FIRST_CALL_CAPTURED = """
import sys
sys.path[:0] = {path!r}
import torch
from pybuda import cuda_ops as ops
x = torch.ones(3, 64, device="cuda").bfloat16()
img = torch.zeros(2, 4 * 576, dtype=torch.uint8, device="cuda")
img[:, :64] = 120
img[:, 64:] = 0x21
wr = torch.ones(2, 64, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = ops.moe_layer(ops.bfp_matvec(x, img[0], 64), wr, 1, img, img, img, 64)
g.replay()
torch.cuda.synchronize()
assert torch.equal(y, ops.moe_layer(ops.bfp_matvec(x, img[0], 64), wr, 1, img, img, img, 64)) and y.float().abs().max() > 0
print("captured ok")
"""


def test_first_call_of_a_process_inside_a_capture():
    import subprocess
    import sys

    r = subprocess.run([sys.executable, "-c", _FIRST_CALL_CAPTURED.format(path=[p for p in sys.path if p])], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured ok" in r.stdout, r.stderr[-2000:]


# ------------------------------------------------------------------------------------------------ what the launch in front writes
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("e,k", [(8, 4096), (64, 2048)])
def test_router_weights_that_a_few_row_product_has_just_written(ops, oracle, e, k, captured):
    """Launches overlap: the router may begin while the product that writes its weights still runs, and must not read them yet."""
    h, t = 512, 3
    img, _ = _store(oracle, _rand((k, h), 50, k ** -0.5), "Bfp8_b")
    images, _ = _make_experts(oracle, e, h, 32, "Bfp4_b", 51)
    rows = [_bf16(_rand((e, k), 52 + r)).cuda() for r in range(3)]
    x = _bf16(_rand((t, h), 56)).cuda()
    want = []
    for r in rows:
        w = ops.bfp_matvec(r, img, h, ops.DF.Bfp8_b, out_dtype=torch.float32)
        torch.cuda.synchronize()
        want.append((*ops.moe_route(x, w, 2), ops.moe_layer(x, w, 2, *images, 32)))
        torch.cuda.synchronize()
    assert not torch.equal(want[0][1], want[1][1])
    buf, src = torch.zeros(e, h, device="cuda"), rows[0].clone()

    def step():
        ops.bfp_matvec(src, img, h, ops.DF.Bfp8_b, out=buf)
        chosen = ops.moe_route(x, buf, 2)
        ops.bfp_matvec(src, img, h, ops.DF.Bfp8_b, out=buf)
        return (*chosen, ops.moe_layer(x, buf, 2, *images, 32))

    torch.cuda.synchronize()
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
    for r in range(60):
        src.copy_(rows[r % 3])
        if captured:
            graph.replay()
        else:
            got = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want[r % 3])), r


def test_router_weights_that_the_experts_have_just_written(ops, oracle):
    """The same behind the launch that adds up the slots of more than 8 tokens."""
    e, h, i, t = 4, 256, 64, 12
    images, _ = _make_experts(oracle, e, h, i, "Bfp4_b", 57)
    xs = [_bf16(_rand((t, h), 58 + r)).cuda() for r in range(3)]
    weights, ids = (v.cuda() for v in _routing(t, e, 2, 61))
    q = _bf16(_rand((5, h), 62)).cuda()
    want = []
    for x in xs:
        w = ops.moe_experts(x, weights, ids, *images, i)
        torch.cuda.synchronize()
        want.append(ops.moe_route(q, w, 3))
        torch.cuda.synchronize()
    buf = torch.zeros(t, h, dtype=torch.bfloat16, device="cuda")
    for r in range(60):
        ops.moe_experts(xs[r % 3], weights, ids, *images, i, out=buf)
        got = ops.moe_route(q, buf, 3)
        assert all(torch.equal(a, b) for a, b in zip(got, want[r % 3])), r


@pytest.mark.parametrize("m", [1, 5, 40])
def test_images_that_the_launch_in_front_has_just_written(ops, oracle, m):
    """An image whose bytes are the result of a product: bfloat16 numbers of [2, 4) are exponents and data of finite weights.  One-hot
    rows pick which, over blocks with exponents of 128, so that the product in front takes its time."""
    k, n, rows, side = 2048, 2304, 8, 256
    assert 2 * rows * n == (side // 32) ** 2 * 576
    img, _ = _store(oracle, 2 + 1.9 * np.random.default_rng(63).random((k, n), np.float32), "Bfp8_b")
    picks = [torch.zeros(rows, k).index_put_((torch.arange(rows), torch.arange(rows) + 100 * r), torch.ones(())).bfloat16().cuda() for r in range(3)]
    x = _bf16(_rand((m, side), 64)).cuda()
    weights, ids = torch.ones(m, 1, device="cuda"), torch.zeros(m, 1, dtype=torch.int32, device="cuda")
    buf = torch.zeros(rows, n, dtype=torch.bfloat16, device="cuda")
    image = buf.view(torch.uint8).view(1, -1)

    def use(which):
        if which == 0:
            return ops.bfp_matvec(x, image.view(-1), side, out_dtype=torch.float32)
        images = [image.clone() if i != which else image for i in range(1, 4)]      # the copies are made of an older image
        return images, lambda: ops.moe_experts(x, weights, ids, *images, side)

    def fill(r):
        ops.bfp_matvec(picks[r], img, n, ops.DF.Bfp8_b, out=buf)

    want = []
    for r in range(3):
        fill(r)
        torch.cuda.synchronize()
        want.append(use(0))
        torch.cuda.synchronize()
    assert torch.isfinite(want[0]).all() and not torch.equal(want[0], want[1])
    for r in range(30):
        fill(r % 3)
        assert torch.equal(use(0), want[r % 3]), r
    fill(0)
    for which in (1, 2, 3):
        images, call = use(which)
        for r in range(3):
            fill(r)
            torch.cuda.synchronize()
            want[r] = call()
            torch.cuda.synchronize()
        for r in range(30):
            fill(r % 3)
            assert torch.equal(call().view(torch.int16), want[r % 3].view(torch.int16)), (which, r)


# ------------------------------------------------------------------------------------------------ the ends of the number range
@pytest.mark.parametrize("df", FORMATS)
@pytest.mark.parametrize("exponent", [0, 128, 200, 254, 255])
@pytest.mark.parametrize("rows", [1, 3, 12, 20])
def test_matvec_outermost_shared_exponents(ops, oracle, df, exponent, rows):
    """One weight row of the exponent among ordinary ones, met by activations of all sizes that leave the product in binary32, the
    smallest subnormal ones among them.  Weights that unpack to infinities give infinities."""
    code = getattr(ops.DF, df)
    rec = {"Bfp8_b": 1088, "Bfp4_b": 576, "Bfp2_b": 320}[df]
    powers = [p for p in (-133, -126, -115, -103, -60, -1, 0, 20, 60, 126) if -110 <= exponent - 127 + p <= 126 or (exponent == 255 and p <= -1)]
    for k in (0, 14, 31):
        raw = np.random.default_rng(exponent + k).integers(0, 256, rec, dtype=np.uint8)
        raw[:64] = 127
        for face in (2 * (k // 16), 2 * (k // 16) + 1):
            raw[16 * face + k % 16] = exponent
        w = oracle.unpack_untilize(raw, getattr(oracle, df), (1, 1, 32, 32))[0, 0].astype(np.float64)
        img = torch.from_numpy(raw).cuda()
        for first in range(len(powers)):
            a = torch.zeros(rows, 32)
            a[:, k] = torch.tensor([(-1.0) ** (r + first) * 2.0 ** powers[(r + first) % len(powers)] for r in range(rows)])
            a = a.bfloat16()
            got = ops.bfp_matvec(a.cuda(), img, 32, code, out_dtype=torch.float32).cpu().numpy()
            want = (a[:, k].double().numpy()[:, None] * w[k]).astype(np.float32)
            assert np.array_equal(got, want), (k, first)
    if exponent == 255 and df != "Bfp2_b":
        assert np.isinf(w).any() and np.isfinite(w[k]).any()


@pytest.mark.parametrize("df", FORMATS)
@pytest.mark.parametrize("t", [1, 3, 12])
def test_experts_infinite_weights_keep_their_sign(ops, oracle, df, t):
    """A row of infinities of both signs in one expert's second matrix: h times them is an infinity of the product's sign, whatever
    pieces h is carried in."""
    e, h, i = 3, 96, 64
    images, vals = _make_experts(oracle, e, h, i, df, 65)
    broken = _rand((i, h), 66, 0.1)
    broken[3, :] = np.where(np.arange(h) % 3 == 0, -np.inf, np.inf)
    images[2][1], stored = _store(oracle, broken, df)
    assert np.isinf(stored[3]).all() and np.isfinite(np.delete(stored, 3, 0)).all()
    x = _bf16(_rand((t, h), 67))
    for other in (0, 2):
        ids = torch.tensor([[other, 1]] * t, dtype=torch.int32)
        weights = torch.rand(t, 2, generator=torch.Generator().manual_seed(68)) + 0.1
        got = ops.moe_experts(x.cuda(), weights.cuda(), ids.cuda(), *images, i, getattr(ops.DF, df))
        a, u = x.double().numpy() @ vals[0][1][:, 3], x.double().numpy() @ vals[1][1][:, 3]
        h3 = a / (1 + np.exp(-a)) * u
        assert np.abs(h3).min() > 1e-4
        assert np.array_equal(got.double().cpu().numpy(), np.sign(h3)[:, None] * stored[3])


@pytest.mark.parametrize("t", [1, 3, 12])
def test_experts_intermediate_keeps_binary32(ops, oracle, t):
    """Results that are the difference of two intermediate values within 2^-12 to 2^-14 of one another.  One-hot tokens make
    h = silu(g) u of single stored values.  The exponential is good to 2 units of the last place and carries 0.27 of the value, the
    addition, the division and the product round once each, 2^-22 h in all; three additions of pieces lose up to 2^-23 of the larger
    value each; the result is rounded to bfloat16."""
    h, i = 32, 64
    grid = np.arange(64, 128) / 64                    # what Bfp8_b stores of [1, 2)
    hs = (grid / (1 + np.exp(-grid)))[:, None] * grid[None, :]
    order = np.argsort(hs, axis=None)
    flat = hs.reshape(-1)[order]
    gap = (flat[1:] - flat[:-1]) / flat[1:]
    at = np.flatnonzero((gap > 2.0 ** -14) & (gap < 2.0 ** -12))
    assert len(at) > 32 * 32
    rng = np.random.default_rng(69)
    gate, up, down = np.zeros((h, i), np.float32), np.zeros((h, i), np.float32), np.zeros((i, h), np.float32)
    for k in range(h):
        for n in range(h):
            p = rng.choice(at)
            for c, which in enumerate((order[p], order[p + 1])):
                gate[k, 2 * n + c], up[k, 2 * n + c] = grid[which // 64], grid[which % 64]
    down[np.arange(0, i, 2), np.arange(h)], down[np.arange(1, i, 2), np.arange(h)] = 1, -1
    images = [_store(oracle, m, "Bfp8_b") for m in (gate, up, down)]
    assert all(np.array_equal(v, m) for (_, v), m in zip(images, (gate, up, down)))
    want = gate.astype(np.float64)
    want = want / (1 + np.exp(-want)) * up
    tol = 2 * 2.0 ** -22 * want[:, ::2] + 3 * 2.0 ** -23 * want[:, ::2]
    want = want[:, ::2] - want[:, 1::2]
    tol = tol + 2.0 ** -8 * (np.abs(want) + tol)
    images = [m[0].view(1, -1) for m in images]
    for first in range(0, h, t):
        x = torch.eye(h)[first:first + t].bfloat16().cuda()
        rows = x.shape[0]
        got = ops.moe_experts(x, torch.ones(rows, 1, device="cuda"), torch.zeros(rows, 1, dtype=torch.int32, device="cuda"), *images, i, ops.DF.Bfp8_b)
        err = np.abs(got.double().cpu().numpy() - want[first:first + t])
        assert (err <= tol[first:first + t]).all(), np.max(err / tol[first:first + t])


@pytest.mark.parametrize("df", ["Bfp8_b", "Bfp4_b"])
@pytest.mark.parametrize("t", [1, 3, 12, 40])
def test_experts_not_finite_activations_stay_in_their_token(ops, oracle, df, t):
    """Tokens with a NaN, an infinity, or values that overflow on the way, among ordinary ones of the same experts."""
    e, h, i = 2, 64, 96
    images, vals = _make_experts(oracle, e, h, i, df, 70)
    x = _bf16(_rand((t, h), 71))
    weights, ids = torch.rand(t, 2, generator=torch.Generator().manual_seed(72)) + 0.1, torch.tensor([[0, 1]] * t, dtype=torch.int32)
    bad = {0: float("nan"), t // 2: float("inf"), t - 1: 3e38}
    for row, v in bad.items():
        y = x.clone()
        y[row, 5] = v
        got = ops.moe_experts(y.cuda(), weights.cuda(), ids.cuda(), *images, i, getattr(ops.DF, df), "gelu").cpu()
        assert not torch.isfinite(got[row]).any(), (row, v)
        if v != v:
            assert torch.isnan(got[row]).all()
        rest = [r for r in range(t) if r != row]
        if rest:
            _check_experts(got[rest], y[rest], weights[rest], ids[rest], vals, "gelu")


@pytest.mark.parametrize("t", [1, 3, 12])
def test_experts_infinite_intermediate_gives_infinities(ops, oracle, t):
    """An intermediate value beyond binary32 is an infinity, and its products with weights of one sign are."""
    h, i = 32, 32
    gate, up, down = np.zeros((h, i), np.float32), np.zeros((h, i), np.float32), np.full((i, h), 0.5, np.float32)
    gate[0, :] = up[0, :] = 1.5
    down[:, ::3] = -1.0
    images = [_store(oracle, m, "Bfp8_b")[0].view(1, -1) for m in (gate, up, down)]
    x = torch.zeros(t, h)
    x[:, 0] = 2.0 ** 100
    got = ops.moe_experts(x.bfloat16().cuda(), torch.ones(t, 1, device="cuda"), torch.zeros(t, 1, dtype=torch.int32, device="cuda"), *images, i,
                          ops.DF.Bfp8_b).double().cpu().numpy()
    assert np.array_equal(got, np.broadcast_to(np.sign(down[0]) * np.inf, got.shape))


@pytest.mark.parametrize("router", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("e", [7, 64, 256])
def test_route_orders_scores_that_binary32_cannot_tell_apart(ops, router, e):
    """Scores of thousands that differ by 2^-9 to 2^-15.  At most one product of each 8 is not zero, so that every sum is exact in
    64 bits."""
    h, top = 512, min(e, 16)
    rng = np.random.default_rng(73 + e)
    w = np.zeros((e, h), np.float32)
    w[:, 0:128:8] = (rng.integers(128, 256, 16) * 4).astype(np.float32)      # the same for all experts
    place = rng.permutation(e)
    for b in range(8):
        w[:, 128 + 8 * b] = (place >> b & 1) * 2.0 ** (b - 15)
    x = torch.ones(3, h)
    x[1] *= -1
    x[2] *= 2
    weights, ids = ops.moe_route(x.bfloat16().cuda(), torch.from_numpy(w).to(router).cuda(), top, True)
    descending = np.argsort(-place)
    for row, order in ((0, descending), (1, descending[::-1]), (2, descending)):
        assert ids[row].cpu().tolist() == order[:top].tolist()
    score = place[descending] * 2.0 ** -15
    p = np.exp(score[:top] - score[0])
    # the exponential and the sum of up to 16 of them: 2 and 16 units of 2^-23, the quotient one rounding
    assert np.abs(weights[0].double().cpu().numpy() * p.sum() / p - 1).max() <= 19 * 2.0 ** -23


@pytest.mark.parametrize("t", [1, 4, 16])
def test_experts_gelu_of_negative_values_keeps_its_digits(ops, oracle, t):
    """gelu(v) for v from -2 to -8, where 1 + erf is a small difference: results, not sums, for the second matrix is the unit matrix.
    z = v / sqrt 2 is off by 2 * 2^-24 of itself, which erfc turns into 2 z^2 times that; erfc is good to 4 units of 2^-23; two
    products and the rounding to bfloat16."""
    h = i = 32
    gate = -(64 + np.random.default_rng(74).integers(0, 64, (h, i))).astype(np.float32) / 64
    images = [_store(oracle, m, "Bfp8_b") for m in (gate, np.eye(i, h, dtype=np.float32))]
    assert np.array_equal(images[0][1], gate) and np.array_equal(images[1][1], np.eye(i, h))
    gate_i, down_i = (m[0].view(1, -1) for m in images)
    for first in range(0, h, t):
        x = torch.eye(h)[first:first + t] * torch.linspace(2, 4, t).view(t, 1)
        x = x.bfloat16()
        got = ops.moe_experts(x.cuda(), torch.ones(t, 1, device="cuda"), torch.zeros(t, 1, dtype=torch.int32, device="cuda"), gate_i, None, down_i, i,
                              ops.DF.Bfp8_b, "gelu")
        v = x.double() @ torch.from_numpy(gate).double()
        want = (0.5 * v * torch.erfc(-v / 2 ** 0.5)).numpy()
        rel = 2 * (v.numpy() ** 2 / 2) * 2 * 2.0 ** -24 + 4 * 2.0 ** -23 + 2 * 2.0 ** -24
        assert (np.abs(got.double().cpu().numpy() - want) <= (2.0 ** -8 + 1.01 * rel) * np.abs(want)).all()


# ------------------------------------------------------------------------------------------------ forms that a caller meets
@pytest.mark.parametrize("df", FORMATS)
@pytest.mark.parametrize("offset", [1, 2, 3])
def test_one_unaligned_row(ops, oracle, df, offset):
    """A single row whose values begin at any element: the product, and the experts."""
    k, n = 333, 150
    img, w = _store(oracle, _rand((k, n), 75, 0.1), df)
    buf = _bf16(_rand((k + 8,), 76)).cuda()
    a = buf[offset:offset + k].view(1, k)
    for dtype in (torch.bfloat16, torch.float32):
        _check_sum(ops.bfp_matvec(a, img, n, getattr(ops.DF, df), out_dtype=dtype), a.double().cpu().numpy(), w, dtype)
    e, i = 3, 70
    images, vals = _make_experts(oracle, e, k, i, df, 77)
    weights, ids = torch.tensor([[0.4, 0.7]]), torch.tensor([[2, 0]], dtype=torch.int32)
    got = ops.moe_experts(a, weights.cuda(), ids.cuda(), *images, i, getattr(ops.DF, df))
    _check_experts(got, a.cpu(), weights, ids, vals, "silu")


@pytest.mark.parametrize("df", FORMATS)
@pytest.mark.parametrize("t", [7, 12, 40])
def test_experts_of_unaligned_rows(ops, oracle, df, t):
    e, h, i = 3, 101, 70
    images, vals = _make_experts(oracle, e, h, i, df, 78)
    x = _bf16(_rand((t * h + 1,), 79)).cuda()[1:].view(t, h)
    weights, ids = _routing(t, e, 2, 80)
    got = ops.moe_experts(x, weights.cuda(), ids.cuda(), *images, i, getattr(ops.DF, df))
    _check_experts(got, x.cpu(), weights, ids, vals, "silu")


@pytest.mark.parametrize("df", FORMATS)
@pytest.mark.parametrize("t", [1, 3, 12, 40])
@pytest.mark.parametrize("scale", [2.0, 0.6])
def test_experts_with_large_weights(ops, oracle, df, t, scale):
    """All three matrices with shared exponents of 128 and more: nearly all of them, or some."""
    e, h, i = 2, 160, 96
    parts = [[_store(oracle, _rand(s, 81 + 10 * which + k, scale), df) for k in range(e)] for which, s in enumerate(((h, i), (h, i), (i, h)))]
    images, vals = [torch.stack([p[0] for p in m]) for m in parts], [np.stack([p[1] for p in m]) for m in parts]
    assert all(int(m[:, :64].max()) >= 128 and (scale > 1 or int(m[:, :64].min()) < 128) for m in images)
    x = _bf16(_rand((t, h), 84, 0.05))
    weights, ids = torch.rand(t, 2, generator=torch.Generator().manual_seed(85)), torch.tensor([[0, 1]] * t, dtype=torch.int32)
    got = ops.moe_experts(x.cuda(), weights.cuda(), ids.cuda(), *images, i, getattr(ops.DF, df), "gelu")
    _check_experts(got, x, weights, ids, vals, "gelu")


@pytest.mark.parametrize("df", FORMATS)
@pytest.mark.parametrize("rows", [9, 16, 17, 32, 64])
def test_matvec_rows_of_mixed_magnitudes(ops, oracle, df, rows):
    """Blocks of very unlike shared exponents against activations that undo them, in wider passes."""
    k, n = 160, 200
    rng = np.random.default_rng(86)
    power = rng.integers(-60, 61, (k, 1))
    w0 = rng.standard_normal((k, n)) * 2.0 ** power * np.repeat(2.0 ** rng.integers(-8, 9, (k, -(-n // 16))), 16, 1)[:, :n]
    img, w = _store(oracle, w0.astype(np.float32), df)
    a = torch.from_numpy(rng.standard_normal((rows, k)) * 2.0 ** (-power[:, 0] + 20)).bfloat16()
    got = ops.bfp_matvec(a.cuda(), img, n, getattr(ops.DF, df), out_dtype=torch.float32)
    _check_sum(got, a.double().numpy(), w, torch.float32)


@pytest.mark.parametrize("t", [1, 6, 12, 40])
def test_weights_of_dropped_slots_are_not_looked_at(ops, oracle, t):
    """A padded batch: slots without an expert hold whatever was there."""
    e, h, i = 4, 96, 64
    images, vals = _make_experts(oracle, e, h, i, "Bfp4_b", 87)
    x = _bf16(_rand((t, h), 88))
    weights, ids = _routing(t, e, 3, 89)
    ids[:, 1] = torch.tensor([-1, 4, -2 ** 31, 2 ** 31 - 1], dtype=torch.int32).repeat(t)[:t]
    weights[:, 1] = torch.tensor([float("nan"), float("inf")]).repeat(t)[:t]
    got = ops.moe_experts(x.cuda(), weights.cuda(), ids.cuda(), *images, i)
    _check_experts(got, x, weights, ids, vals, "silu")


@pytest.mark.parametrize("t", [1, 8, 12, 64])
def test_layer_in_place(ops, oracle, t):
    e, h, i = 6, 128, 64
    images, _ = _make_experts(oracle, e, h, i, "Bfp8_b", 90)
    wr = torch.randn(e, h, generator=torch.Generator().manual_seed(91)).cuda()
    x = _bf16(_rand((t, h), 92)).cuda()
    want = ops.moe_layer(x, wr, 2, *images, i, ops.DF.Bfp8_b)
    for _ in range(10):
        y = x.clone()
        assert ops.moe_layer(y, wr, 2, *images, i, ops.DF.Bfp8_b, out=y) is y
        assert torch.equal(y, want)


def test_calls_from_two_threads_at_once(ops, oracle):
    import threading

    e, h, i = 6, 128, 96
    images, _ = _make_experts(oracle, e, h, i, "Bfp4_b", 93)
    proj, _ = _store(oracle, _rand((h, h), 94, h ** -0.5), "Bfp4_b")
    wr = torch.randn(e, h, generator=torch.Generator().manual_seed(95)).cuda()
    xs = [_bf16(_rand((t, h), 96 + t)).cuda() for t in (1, 3, 12, 40)]
    want = [_block(ops, x, proj, wr, images, i) for x in xs]
    torch.cuda.synchronize()
    wrong, errors = [], []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for r in range(40):
                    got = _block(ops, xs[k], proj, wr, images, i)
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[k])):
                        wrong.append((k, r))
        except Exception as ex:           # noqa: BLE001 -- shown below
            errors.append(ex)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    [t.start() for t in threads], [t.join() for t in threads]
    assert not errors and not wrong, (errors, wrong)


@pytest.mark.parametrize("router", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t,h,e,top", [(1, 16384, 8, 2), (2, 20001, 3, 1), (30, 7168, 16, 4), (64, 4104, 16, 4), (37, 4001, 9, 3)])
def test_route_rows_too_long_to_be_staged(ops, router, t, h, e, top):
    g = torch.Generator().manual_seed(t + h + e)
    x, w = torch.randn(t, h, generator=g).bfloat16(), (torch.randn(e, h, generator=g) * 2 * h ** -0.5).to(router)
    weights, ids = ops.moe_route(x.cuda(), w.cuda(), top, True)
    ref, rid = _route_ref(x, w, top, True)
    assert np.array_equal(ids.cpu().numpy(), rid)
    # a score is off by 7 * 2^-24 of its products' magnitudes at most, a weight by twice that and a few units of 2^-24
    mag = (x.double().abs() @ w.double().abs().T).max().item()
    assert (np.abs(weights.double().cpu().numpy() - ref) <= (14 * mag + 8) * 2.0 ** -24 * ref).all()


_OUT_OF_MEMORY = """
import sys
sys.path[:0] = {path!r}
import torch
from pybuda import cuda_ops as ops
a, img = torch.ones(64, 32, device="cuda").bfloat16(), torch.zeros(1 << 15, 320, dtype=torch.uint8, device="cuda").view(-1)
torch.cuda.set_per_process_memory_fraction(2 ** 26 / torch.cuda.get_device_properties(0).total_memory)
try:
    ops.bfp_matvec(a, img, 1 << 20, ops.DF.Bfp2_b, out_dtype=torch.float32)
except torch.OutOfMemoryError:
    y = ops.bfp_matvec(a, img, 1 << 10, ops.DF.Bfp2_b)
    assert torch.all(y == 0)
    print("out of memory said so")
"""


def test_results_that_do_not_fit_raise_torchs_out_of_memory_error():
    """The allocator's limit for this process stands in for a full device."""
    import subprocess
    import sys

    r = subprocess.run([sys.executable, "-c", _OUT_OF_MEMORY.format(path=[p for p in sys.path if p])], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "out of memory said so" in r.stdout, r.stderr[-2000:]
