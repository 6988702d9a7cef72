"""The 8-bit products and the drawing of tokens against their definitions in
64 bits.

Tolerances.  A code is a definite number, so codes are compared for equality.
u = 2^-24 is half a step of FP32 relative to the value.  A product is
fl(fl(fl(sum) sx) sw), 3 u, each addition after it one u of its result, the
output type's half step once.  A normed row's scale holds a sum of squares (at
most 64 additions on the way of any of them up to 8192 values, K / 256 more
beyond), a square root's reciprocal (2 steps) and three more roundings:
(64 + 10) u / 2 < 2^-18.7 in all, so 2^-18 is allowed.
"""

from __future__ import annotations

import math
import threading
import time

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
NORM_REL = 2.0 ** -18
EPS = 1e-6
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def K():
    from soraku_tts_b200 import kernels

    return kernels


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def codes_of(x, nw=None):
    """Codes and steps by the definition: FP32 products and quotients, in numpy.  The step is the largest times FP32's
    1 / 127, as `x.abs().amax(1) / 127` gives it on the device (test_codes_are_those_of_elementary_operations)."""
    y = x.float().cpu().numpy()
    if nw is not None:
        y = (y * nw.cpu().numpy()).astype(np.float32)
    with np.errstate(invalid="ignore", over="ignore"):
        top = np.abs(y).max(1)
        s = np.maximum(top * (np.float32(1) / np.float32(127)), np.float32(2.0 ** -126)).astype(np.float32)
        q = np.rint(y / s[:, None])
    bad = ~np.isfinite(top)
    q[bad] = 0
    s[bad] = np.nan
    return q, s


def scale_of(x, s, nw):
    if nw is None:
        return s.astype(np.float64)
    x = x.double().cpu().numpy()
    return s.astype(np.float64) / np.sqrt((x ** 2).mean(1) + EPS)


def rows_in(shape, seed, dtype, pad=0):
    """Rows with channels that stand out; with `pad`, a view into wider rows that begins off 16 bytes."""
    g = gen(seed)
    wide = torch.randn(shape[0], shape[1] + pad, device="cuda", generator=g)
    wide *= torch.where(torch.rand(shape[1] + pad, device="cuda", generator=g) < 0.02, 15.0, 1.0)
    return wide.to(dtype)[:, pad // 2:pad // 2 + shape[1]]


# ------------------------------------------------------------ quantize_rows
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 7), (1, 16), (5, 100), (9, 1024), (2, 1025), (3, 2048), (2, 8192), (3, 8195), (2, 20000),
                                    (1, 131071), (700, 64)])
@pytest.mark.parametrize("norm", [False, True])
def test_quantize_rows(K, rows, k, dtype, norm):
    for pad in (0, 5):
        x = rows_in((rows, k), rows + k, DT[dtype], pad)
        nw = 1 + 0.3 * torch.randn(k, device="cuda", generator=gen(1)) if norm else None
        got = K.quantize_rows(x, norm_weight=nw, eps=EPS)
        q, s = codes_of(x, nw)
        assert got.q.shape == x.shape and got.q.stride(0) % 16 == 0
        assert np.array_equal(got.q.cpu().numpy(), q)
        # behind a row's end its codes are zeros
        whole = torch.as_strided(got.q, (rows, got.q.stride(0)), (got.q.stride(0), 1))
        assert not whole[:, k:].any()
        want, scale = scale_of(x, s, nw), got.scale.double().cpu().numpy()
        # beyond 8192 values the sum of squares has K / 256 more additions in a row
        more = max(0, k - 8192) / 256 * U
        assert np.all(np.abs(scale - want) <= (NORM_REL + more) * want if norm else scale == want)


def test_quantize_rows_of_all_kinds(K):
    inf, nan, tiny = float("inf"), float("nan"), 2.0 ** -149
    x = torch.zeros(9, 40, device="cuda")
    x[1, 3] = 5.0
    x[2, 3] = inf
    x[3, 39] = -inf
    x[4, 0] = nan
    x[5, 7] = tiny
    x[6] = 3.0e38
    x[7, :20], x[7, 20:] = 127.0, 0.5  # halves go to even
    x[7, 30:] = 1.5
    x[8, ::2], x[8, 1::2] = 1e-40, -2e-40
    got = K.quantize_rows(x)
    q, s = codes_of(x)
    assert np.array_equal(got.q.cpu().numpy(), q)
    assert np.array_equal(got.scale.cpu().numpy(), s, equal_nan=True)
    assert not got.q[[0, 2, 3, 4]].any() and got.q[7, 25] == 0 and got.q[7, 35] == 2
    # a norm's weight that makes something not finite
    w = torch.ones(40, device="cuda")
    w[3] = inf
    got = K.quantize_rows(x[:2], norm_weight=w)
    assert torch.isnan(got.scale).all() and not got.q.any()


def test_codes_at_every_border(K):
    """Values at and next to every half step, where a quotient by way of a reciprocal would go wrong."""
    for top in (127.0, 1.0, 0.7315, 3.1e-5, 8.87e30):
        s = np.float32(top) / np.float32(127)
        half = ((np.arange(-127, 127) + 0.5) * np.float64(s)).astype(np.float32)
        y = np.concatenate([np.nextafter(half, np.float32(-np.inf)), half, np.nextafter(half, np.float32(np.inf)), [np.float32(top)]])
        x = torch.from_numpy(y.astype(np.float32))[None].cuda()
        assert np.array_equal(K.quantize_rows(x).q.cpu().numpy(), codes_of(x)[0])


def test_codes_are_those_of_elementary_operations(K):
    """To the last one, where quotients next to a half are many: 6.7 million values a time."""
    for seed in range(12):
        x, nw = rows_in((6541, 1024), seed, torch.float32), 1 + 0.2 * torch.randn(1024, device="cuda", generator=gen(seed))
        y = x * nw
        s = torch.clamp(y.abs().amax(1) / 127, min=2.0 ** -126)
        assert torch.equal(K.quantize_rows(x, norm_weight=nw).q.float(), torch.round(y / s[:, None]))
        assert torch.equal(K.quantize_rows(y).scale, s)


# ---------------------------------------------------------------- products
def weights(n, k, seed, ld=0, low=-127):
    g = gen(seed)
    ld = (max(ld, k) + 15) // 16 * 16
    q = torch.randint(low, 128, (n, ld), device="cuda", generator=g, dtype=torch.int32).to(torch.int8)[:, :k]
    return q, 0.001 + 0.02 * torch.rand(n, device="cuda", generator=g)


def product(q, scale, w):
    """Sums in whole numbers, then 64 bits: [T, N] values, without rounding."""
    acc = torch.from_numpy(q).double().cuda() @ w[0].double().T
    return acc.cpu().numpy() * scale[:, None] * w[1].double().cpu().numpy()


def check_linear(K, t, n, k, dtype="f32", norm=False, bias=False, residual=False, pad=0, codes=False, out_dtype=None, ld=0,
                 in_place=False):
    x = rows_in((t, k), t + n + k, DT[dtype], pad)
    nw = 1 + 0.3 * torch.randn(k, device="cuda", generator=gen(2)) if norm else None
    od = DT[out_dtype or dtype]
    w = weights(n, k, n + k, ld)
    b = torch.randn(n, device="cuda", generator=gen(3)) if bias else None
    r = torch.randn(t, n + pad, device="cuda", generator=gen(4)).to(od)[:, pad:] if residual else None
    arg = K.quantize_rows(x, norm_weight=nw, eps=EPS) if codes else x
    kw = dict(norm_weight=None if codes else nw, eps=EPS, bias=b, residual=r)
    rd = r.double().cpu().numpy() if residual else 0.0
    got = K.int8_linear(arg, w, out_dtype=od, **kw, **({"out": r} if in_place else {}))
    assert got.dtype is od and tuple(got.shape) == (t, n)
    q, s = codes_of(x, nw)
    p = product(q, scale_of(x, s, nw), w)
    with_bias = p + (b.double().cpu().numpy() if bias else 0.0)
    want = with_bias + rd
    tol = (3 * U + (NORM_REL if norm else 0)) * np.abs(p) + U * (np.abs(with_bias) * bias + np.abs(want) * residual)
    tol = 1.01 * tol + torch.finfo(od).eps / 2 * np.abs(want) * (od is not torch.float32) + 2.0 ** -24
    err = np.abs(got.double().cpu().numpy() - want)
    assert np.all(err <= tol), f"worst {np.max(err - tol)} of {np.abs(want).max()}"
    return got


# tokens about the borders between the variants, widths and lengths about the tiles'
TOKENS = [1, 2, 3, 4, 5, 8, 9, 16, 17, 31, 33, 64, 65, 100, 128, 129, 200, 256, 257, 300]


@pytest.mark.parametrize("t", TOKENS)
@pytest.mark.parametrize("n,k", [(128, 128), (1, 1), (130, 100), (515, 1000), (64, 2053)])
def test_linear(K, t, n, k):
    check_linear(K, t, n, k)


@pytest.mark.parametrize("t", [1, 2, 4, 7, 16, 40, 130, 300])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("codes", [False, True])
def test_linear_with_everything(K, t, dtype, codes):
    check_linear(K, t, 259, 328, dtype, norm=True, bias=True, residual=True, pad=3, codes=codes, ld=400)
    check_linear(K, t, 256, 1024, dtype, norm=not codes, bias=False, residual=True, codes=codes, in_place=True)


@pytest.mark.parametrize("t,n,k", [(2, 4096, 1024), (128, 4096, 1024), (1500, 2051, 1024), (2, 32816, 1024), (700, 257, 8192),
                                   (1, 9, 131071), (8, 40, 40000), (20, 300, 20000), (4100, 384, 64), (3, 20000, 33)])
def test_linear_at_size(K, t, n, k):
    check_linear(K, t, n, k, norm=k <= 8192, bias=True)
    check_linear(K, t, n, k, "bf16", residual=True, out_dtype="f32")


# more tiles than SMs: pairs of CTAs, with edges in every direction, and outputs off and on 16 bytes
@pytest.mark.parametrize("t,n,k", [(1500, 2048, 1024), (2111, 2052, 1000), (1281, 2304, 130), (1300, 2049, 256), (6541, 1024, 64),
                                   (300, 20008, 96)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_linear_of_many_tiles(K, t, n, k, dtype):
    check_linear(K, t, n, k, dtype, norm=True, bias=True)
    check_linear(K, t, n, k, dtype, codes=True)
    check_linear(K, t, n, k, dtype, residual=True, in_place=n % 8 == 0)


@pytest.mark.parametrize("t,n,k", [(5281, 64, 384), (531, 1727, 104), (40, 700, 130), (9000, 64, 96), (181, 4736, 64), (300, 2048, 520)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_linear_with_and_without_residual(K, t, n, k, dtype):
    """Tiles of every width; a residual that is not there is not read."""
    check_linear(K, t, n, k, dtype, norm=True, bias=False)
    check_linear(K, t, n, k, dtype, residual=True)


@pytest.mark.parametrize("t,n,k", [(1500, 1536, 1024), (2111, 1028, 1000), (1281, 2001, 130), (5003, 520, 64)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_swiglu_of_many_tiles(K, t, n, k, dtype):
    check_swiglu(K, t, n, k, dtype, norm=True)
    check_swiglu(K, t, n, k, dtype, codes=True)
    wide = torch.full((t + 1, n + 24), 7.0, device="cuda").to(DT[dtype])
    check_swiglu(K, t, n, k, dtype, out=wide[:t, 8:8 + n])
    wide[:t, 8:8 + n] = 7.0
    assert (wide == 7.0).all()


def test_the_largest_sums_are_exact(K):
    """All codes at their ends: sums near 2^31, which FP32 or a 16-bit step on the way would not hold."""
    for t in (1, 5, 33, 140):
        k = 131071
        q = torch.full((t, (k + 15) // 16 * 16), -128, dtype=torch.int8, device="cuda")[:, :k]
        w = torch.full((3, (k + 15) // 16 * 16), -128, dtype=torch.int8, device="cuda")[:, :k]
        w[1] = 127
        w[2, ::2] = 127
        one, three = torch.ones(t, device="cuda"), torch.ones(3, device="cuda")
        got = K.int8_linear((q, one), (w, three)).double()
        want = (q.double() @ w.double().T)
        assert ((got - want).abs() <= U * want.abs()).all()


def test_what_lies_behind_a_row_counts_for_nothing(K):
    for t in (1, 3, 20, 200):
        q = torch.randint(-127, 128, (t, 64), device="cuda", generator=gen(5), dtype=torch.int32).to(torch.int8)
        w, ws = weights(70, 64, 6)
        got = K.int8_linear((q[:, :37], torch.ones(t, device="cuda")), (w[:, :37], ws))
        want = product(q[:, :37].cpu().numpy().astype(np.float64), np.ones(t), (w[:, :37], ws))
        assert np.all(np.abs(got.double().cpu().numpy() - want) <= 3.01 * U * np.abs(want))


@pytest.mark.parametrize("t", [2, 40, 300])
def test_rows_that_are_not_finite(K, t):
    x = rows_in((t, 256), 8, torch.float32)
    x[0, 5], x[1, 255] = float("nan"), float("-inf")
    w = weights(130, 256, 9)
    got = K.int8_linear(x, w)
    assert torch.isnan(got[:2]).all() and torch.isfinite(got[2:]).all()
    assert torch.isnan(K.int8_swiglu(x, w, w)[:2]).all()


@pytest.mark.parametrize("t", [1, 6, 20, 150, 300])
def test_rows_of_zeros(K, t):
    w, b = weights(130, 256, 9), torch.randn(130, device="cuda", generator=gen(1))
    x = torch.zeros(t, 256, device="cuda")
    nw = torch.ones(256, device="cuda")
    assert torch.equal(K.int8_linear(x, w, norm_weight=nw, bias=b), b.expand(t, 130))
    assert not K.int8_swiglu(x, w, w, norm_weight=nw).any()


def check_swiglu(K, t, n, k, dtype="f32", norm=False, codes=False, pad=0, out=None):
    x = rows_in((t, k), t + n + k, DT[dtype], pad)
    nw = 1 + 0.3 * torch.randn(k, device="cuda", generator=gen(2)) if norm else None
    gate, up = weights(n, k, 1), weights(n, k, 2, ld=k + 64)
    # products of ordinary size
    for w in (gate, up):
        w[1].mul_(40 / (127 * math.sqrt(k)))
    arg = K.quantize_rows(x, norm_weight=nw, eps=EPS) if codes else x
    od = torch.float32 if codes else DT[dtype]
    got = K.int8_swiglu(arg, gate, up, norm_weight=None if codes else nw, eps=EPS, out=out)
    assert got.dtype is od
    q, s = codes_of(x, nw)
    sc = scale_of(x, s, nw)
    g, u = product(q, sc, gate), product(q, sc, up)
    with np.errstate(over="ignore"):
        want = g / (1 + np.exp(-g)) * u
    rel = 3 * U + (NORM_REL if norm else 0)
    # silu's condition is at most 1 + |g|; exp two steps, quotient and product one rounding each
    tol = np.abs(want) * 1.01 * ((2 + np.abs(g)) * rel + 8 * U)
    tol += torch.finfo(od).eps / 2 * np.abs(want) * (od is not torch.float32) + 2.0 ** -24
    err = np.abs(got.double().cpu().numpy() - want)
    assert np.all(err <= tol), f"worst {np.max(err - tol)}"


@pytest.mark.parametrize("t", TOKENS)
@pytest.mark.parametrize("n,k", [(128, 128), (1, 3), (131, 100), (300, 1000)])
def test_swiglu(K, t, n, k):
    check_swiglu(K, t, n, k)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("t,n,k", [(2, 2048, 1024), (77, 2048, 1024), (1000, 1031, 777), (5, 64, 20000), (64, 65, 20000)])
def test_swiglu_at_size(K, t, n, k, dtype):
    check_swiglu(K, t, n, k, dtype, norm=k <= 8192, pad=2)
    check_swiglu(K, t, n, k, dtype, codes=True)


def test_strided_outputs_leave_the_rest(K):
    for t in (2, 50, 300):
        x, w = rows_in((t, 96), 1, torch.float32), weights(70, 96, 2)
        wide = torch.full((t + 2, 80), 7.0, device="cuda")
        got = K.int8_linear(x, w, out=wide[1:t + 1, 3:73])
        assert torch.equal(got, K.int8_linear(x, w)) and got.data_ptr() == wide[1, 3:].data_ptr()
        wide[1:t + 1, 3:73] = 7.0
        assert (wide == 7.0).all()
        K.int8_swiglu(x, w, w, out=wide[1:t + 1, 3:73])
        assert torch.equal(wide[1:t + 1, 3:73], K.int8_swiglu(x, w, w))
        wide[1:t + 1, 3:73] = 7.0
        assert (wide == 7.0).all()


def test_a_row_goes_by_itself(K):
    """A token's result is the same in any batch, to the bit, when it comes as codes."""
    x, w = K.quantize_rows(rows_in((300, 512), 3, torch.float32)), weights(200, 512, 4)
    whole, glu = K.int8_linear(x, w), K.int8_swiglu(x, w, w)
    more = K.Int8Rows(x.q.repeat(40, 1), x.scale.repeat(40))
    assert torch.equal(K.int8_linear(more, w), whole.repeat(40, 1)) and torch.equal(K.int8_swiglu(more, w, w), glu.repeat(40, 1))
    for a, b in ((0, 1), (5, 7), (10, 26), (0, 100), (17, 217)):
        part = K.Int8Rows(x.q[a:b], x.scale[a:b])
        assert torch.equal(K.int8_linear(part, w), whole[a:b])
        assert torch.equal(K.int8_swiglu(part, w, w), glu[a:b])


def test_products_refuse(K):
    x, w = rows_in((4, 64), 1, torch.float32), weights(20, 64, 2)
    cut = torch.zeros(20, 70, dtype=torch.int8, device="cuda")[:, :64]  # rows that begin off 16 bytes
    for call in (lambda: K.int8_linear(x.double(), w), lambda: K.int8_linear(x, weights(20, 63, 2)),
                 lambda: K.int8_linear(x, (w[0].int(), w[1])), lambda: K.int8_linear(x, (w[0], w[1][:19])),
                 lambda: K.int8_linear(x, w[0]), lambda: K.int8_linear(x, (cut, w[1])), lambda: K.int8_linear(x.T, w),
                 lambda: K.int8_linear(x, w, bias=torch.zeros(19, device="cuda")),
                 lambda: K.int8_linear(x, w, residual=torch.zeros(4, 20, device="cuda", dtype=torch.bfloat16)),
                 lambda: K.int8_linear(x, w, norm_weight=torch.ones(63, device="cuda")),
                 lambda: K.int8_linear(K.quantize_rows(x), w, norm_weight=torch.ones(64, device="cuda")),
                 lambda: K.int8_linear(x, w, out=torch.zeros(4, 21, device="cuda")),
                 lambda: K.int8_linear(x, w, out_dtype=torch.int8), lambda: K.int8_swiglu(x, w, weights(21, 64, 2)),
                 lambda: K.int8_linear(x, (w[0].cpu(), w[1])), lambda: K.quantize_rows(x.int()),
                 lambda: K.quantize_rows(x, norm_weight=torch.ones(64)), lambda: K.quantize_rows(x[:, :0]),
                 lambda: K.int8_linear(x.expand(3, 4, 64), w), lambda: K.int8_linear(x[:1].expand(4, 64), w)):
        with pytest.raises(ValueError):
            call()
    assert K.int8_linear(x[:0], w).shape == (0, 20) and K.int8_swiglu(x[:0], w, w).shape == (0, 20)
    assert K.quantize_rows(x[:0]).q.shape == (0, 64)


# ----------------------------------------------------------- drawing tokens
def draw(line, u, T, k, p, m):
    """One row by the definition: (token, logarithm of its share)."""
    line = line.astype(np.float64)
    if np.isnan(line).any() or not (line > -np.inf).any():
        return -1, math.nan
    order = np.argsort(-line, kind="stable")
    v = line[order]
    if T <= 0:
        return int(order[0]), 0.0
    with np.errstate(invalid="ignore"):
        score = np.where(v == v[0], 0.0, (v - v[0]) / T)
    e = np.exp(score)
    n = len(v) if k <= 0 else min(k, len(v))
    sums = np.cumsum(e[:n])
    if p < 1:
        n = min(n, 1 + int((sums[:-1] < p * sums[-1]).sum()))
    n = max(1, min(n, int((e >= min(m, 1.0)).sum())))
    sums = sums[:n]
    at = min(int((sums <= u * sums[-1]).sum()), n - 1)
    return int(order[at]), score[at] - math.log(sums[-1])


def check_sample(K, logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    tokens, logprob = K.sample_tokens(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    rows = logits.shape[0]

    def each(x, whole=False):
        if isinstance(x, torch.Tensor):
            return x.tolist()
        return [x if whole else float(np.float32(x))] * rows

    want = [draw(*a) for a in zip(logits.float().cpu().numpy(), u.tolist(), each(temperature), each(top_k, True), each(top_p),
                                  each(min_p))]
    assert tokens.tolist() == [w[0] for w in want]
    lp = np.array([w[1] for w in want])
    got = logprob.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(lp))
    ok = ~np.isnan(lp)
    # one FP32 rounding; weights are whole multiples of 2^-44: V 2^-45 of the largest at most
    assert np.all(np.abs(got[ok] - lp[ok]) <= U * np.abs(lp[ok]) + 2.0 ** -26)
    return tokens, logprob


def some_logits(rows, v, seed, dtype=torch.float32, spread=3.0):
    return (torch.randn(rows, v, device="cuda", generator=gen(seed)) * spread).to(dtype)


def uniforms(rows, seed):
    return torch.rand(rows, device="cuda", generator=gen(seed))


@pytest.mark.parametrize("v", [1, 2, 5, 31, 100, 2051, 8192, 8193, 16385, 33000, 151936, 262144])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_sample(K, v, dtype):
    for n, (k, p, m) in enumerate([(0, 1.0, 0.0), (50, 0.95, 0.05), (0, 0.9, 0.0), (0, 1.0, 0.02), (1000, 0.7, 0.0), (1, 0.5, 0.5),
                                   (128, 1.0, 0.0), (129, 1.0, 0.0), (v, 0.99, 0.0)]):
        x = some_logits(5, v, v + n, DT[dtype])
        check_sample(K, x, uniforms(5, n), 0.9, k, p, m)


@pytest.mark.parametrize("spread", [0.0, 1e-3, 0.3, 30.0, 1e4])
@pytest.mark.parametrize("v", [700, 20000, 100000])
def test_sample_of_flat_and_sharp_rows(K, spread, v):
    for t in (1e-3, 1.0, 50.0, 1e6):
        for k, p, m in ((0, 1.0, 0.0), (0, 0.8, 0.0), (40, 0.9, 0.0), (5000, 0.9, 0.3)):
            check_sample(K, some_logits(3, v, v, spread=spread), uniforms(3, 7), t, k, p, m)


@pytest.mark.parametrize("v", [2051, 151936])
def test_sample_of_equal_logits(K, v):
    """Rows of few different values: order and borders go by the index."""
    for levels in (1, 2, 3, 40):
        x = torch.randint(0, levels, (6, v), device="cuda", generator=gen(levels), dtype=torch.int32).float()
        for k, p, m in ((0, 1.0, 0.0), (0, 0.5, 0.0), (700, 0.5, 0.0), (60, 0.5, 0.0), (0, 0.25, 0.9)):
            u = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.3, 1 - 2.0 ** -24], device="cuda")
            check_sample(K, x, u, 1.0, k, p, m)


@pytest.mark.parametrize("v", [64, 9000])
def test_sample_of_masked_rows(K, v):
    inf, nan, low = float("inf"), float("nan"), torch.finfo(torch.float32).min
    x = some_logits(12, v, 3)
    x[0] = -inf
    x[1, 1:] = -inf
    x[2, 7] = nan
    x[3, ::2] = -inf
    x[4] = low
    x[5, 3:] = low
    x[6, [5, 9]] = inf
    x[7] = inf
    x[8, 10:] = -inf
    x[9], x[9, 20], x[9, 30] = -0.0, 0.0, -inf
    x[10], x[10, 50] = -inf, low
    x[11, 0] = 3e38
    for k, p, m in ((0, 1.0, 0.0), (5, 0.9, 0.0), (0, 0.9, 0.1), (1000, 1.0, 0.0)):
        for t in (1.0, 0.01, 1e30):
            tokens, _ = check_sample(K, x, uniforms(12, k), t, k, p, m)
            assert tokens[0] == -1 and tokens[2] == -1 and tokens[1] == 0 and tokens[10] == 50
    # what is masked is never drawn, not by the largest number either
    u = torch.full((12,), 1 - 2.0 ** -24, device="cuda")
    tokens, _ = check_sample(K, x, u)
    assert tokens[3] % 2 == 1 and tokens[8] < 10


def test_sample_takes_each_rows_own_settings(K):
    rows = 40
    g = gen(5)
    t = 0.2 + torch.rand(rows, device="cuda", generator=g)
    t[::7] = 0.0
    k = torch.randint(0, 400, (rows,), device="cuda", generator=g, dtype=torch.int32)
    k[3::5] = 0
    p = 0.3 + torch.rand(rows, device="cuda", generator=g)
    m = 0.1 * torch.rand(rows, device="cuda", generator=g)
    p[4], p[5], m[6], m[8], t[9] = 0.0, -1.0, 1.0, 7.0, -3.0
    for v in (2051, 40000):
        check_sample(K, some_logits(rows, v, 6), uniforms(rows, 6), t, k, p, m)


def test_sample_at_the_ends_of_the_uniform_range(K):
    x = some_logits(4, 3000, 1)
    for u in (0.0, 2.0 ** -24, 1 - 2.0 ** -24, 1e-38):
        check_sample(K, x, torch.full((4,), u, device="cuda"), 0.7, 0, 0.9, 0.0)
    # outside of it: the first and the last of the kept ones
    inside, _ = K.sample_tokens(x, torch.zeros(4, device="cuda"), top_k=9)
    for u in (-1.0, float("-inf"), float("nan")):
        assert torch.equal(K.sample_tokens(x, torch.full((4,), u, device="cuda"), top_k=9)[0], inside)
        assert torch.equal(K.sample_tokens(x, torch.full((4,), u, device="cuda"))[0], inside)
    for u in (1.0, 5.0, float("inf")):
        got, _ = K.sample_tokens(x, torch.full((4,), u, device="cuda"), top_k=9)
        assert torch.equal(got, torch.sort(x, dim=1, descending=True, stable=True).indices[:, 8])


def test_sample_rows_anywhere(K):
    """Rows at every place mod 16 bytes, in wider rows."""
    for dtype in (torch.float32, torch.bfloat16):
        wide = some_logits(7, 10011, 2, dtype)
        for a, v in ((0, 10000), (1, 2051), (3, 9999), (5, 8), (7, 10004), (2, 1)):
            check_sample(K, wide[:, a:a + v], uniforms(7, a), 1.0, 0, 0.95, 0.0)
            check_sample(K, wide[:, a:a + v], uniforms(7, a), 1.0, 30, 0.95, 0.01)


def test_sample_many_rows(K):
    check_sample(K, some_logits(1000, 300, 4), uniforms(1000, 4), 0.8, 20, 0.9, 0.0)
    check_sample(K, some_logits(300, 12000, 4), uniforms(300, 4), 0.8, 0, 0.9, 0.0)


@pytest.mark.parametrize("rows", [5, 40])
@pytest.mark.parametrize("v", [8193, 16385, 50001, 151936])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sample_by_clusters_and_streams(K, dtype, v, rows):
    """Few and many rows of long lines, with one top-k and with each row's own."""
    k = torch.tensor([50, 1000, 1, 0, 1280], dtype=torch.int32, device="cuda").repeat(rows // 5)
    x = some_logits(rows, v, rows + v, DT[dtype])
    x[1] = (x[1] * 2).round()  # many equal ones
    x[2, ::3] = float("-inf")
    x[3, 77], x[3, v - 1] = float("inf"), float("inf")
    u = uniforms(rows, v)
    for top_k in (k, 20, 0):
        check_sample(K, x, u, 0.8, top_k, 0.9, 0.001)
    x[0] = 1.5
    check_sample(K, x, u, 1.0, k, 1.0, 0.0)
    check_sample(K, x, u, 1.0, 1000, 1.0, 0.0)


def test_sample_draws_as_the_frame_sampler_does(K):
    n, v = 64, 2051
    x = some_logits(n, v, 9)
    params = K.pack_sample_params([dict(temperature=0.9, top_k=50, top_p=0.95, seed=3, request=i, V=v) for i in range(n)])
    codes, uni = K.cfg_sample(x, params, rows_per_req=1, bos_id=2048, pad_id=2050, eos_id=2049, return_uniform=True)
    masked = x.clone()
    masked[:, [2048, 2050]] = -float("inf")
    tokens, _ = K.sample_tokens(masked, uni, temperature=0.9, top_k=50, top_p=0.95)
    assert torch.equal(tokens, codes)


def test_sample_frequencies(K):
    """A grid of numbers draws each token as often as its share says."""
    x = some_logits(1, 40, 8, spread=1.0)
    n = 4096
    tokens, _ = K.sample_tokens(x.expand(n, 40).contiguous(), (torch.arange(n, device="cuda") + 0.5) / n, temperature=0.8, top_k=30)
    e = torch.exp((x[0].double() - x.max().double()) / float(np.float32(0.8)))
    e[torch.sort(x[0], descending=True, stable=True).indices[30:]] = 0
    share = torch.bincount(tokens, minlength=40).double() / n
    assert ((share - e / e.sum()).abs() <= 1.0 / n + 1e-9).all()  # points of a grid in an interval: off by less than one


def test_sample_refuses(K):
    x, u = some_logits(4, 100, 1), uniforms(4, 1)
    for call in (lambda: K.sample_tokens(x.double(), u), lambda: K.sample_tokens(x, u[:3]), lambda: K.sample_tokens(x.T, u),
                 lambda: K.sample_tokens(x, u.double()), lambda: K.sample_tokens(x, u.cpu()), lambda: K.sample_tokens(x[:, :0], u),
                 lambda: K.sample_tokens(x, u, top_k=1.5), lambda: K.sample_tokens(x, u, top_k=torch.zeros(4, device="cuda")),
                 lambda: K.sample_tokens(x, u, top_p=torch.zeros(3, device="cuda")), lambda: K.sample_tokens(x, u, top_p=float("nan")),
                 lambda: K.sample_tokens(torch.zeros(1, (1 << 18) + 1, device="cuda"), u[:1])):
        with pytest.raises(ValueError):
            call()
    tokens, logprob = K.sample_tokens(x[:0], u[:0])
    assert tokens.shape == (0,) and logprob.shape == (0,)


# ------------------------------------------------------------ used together
def depth_step(K, hidden, prefix, norm_in, norm_out, gate, up, down, table, bias, u):
    """The depth head's step for one codebook in 8 bits, up to its code."""
    d = hidden.shape[1]
    a = K.add_rmsnorm(hidden.shape[0], d, EPS)(hidden, prefix, norm_in)
    act = K.int8_swiglu(a, gate, up)
    body = K.int8_linear(act, down, residual=a)
    logits = K.int8_linear(body, table, norm_weight=norm_out, eps=EPS, bias=bias)
    return (act, body, logits) + K.sample_tokens(logits, u, temperature=0.9, top_k=50, top_p=0.95, min_p=0.02)


def head_weights(K, d, inner, v):
    g = gen(11)

    def normal(*s):
        return torch.randn(*s, device="cuda", generator=g)

    return dict(norm_in=1 + 0.1 * normal(d), norm_out=1 + 0.1 * normal(d), gate=K.quantize_rows(0.05 * normal(inner, d)),
                up=K.quantize_rows(0.05 * normal(inner, d)), down=K.quantize_rows(0.05 * normal(d, inner)),
                table=K.quantize_rows(0.1 * normal(v, d)), bias=0.1 * normal(v))


@pytest.mark.parametrize("rows", [1, 2, 16, 130])
def test_depth_step(K, rows):
    d, inner, v = 1024, 2048, 2051
    w = head_weights(K, d, inner, v)
    hidden, prefix = rows_in((rows, d), 1, torch.float32).contiguous(), some_logits(rows, d, 2, spread=0.3)
    u = uniforms(rows, 3)
    act, body, logits, tokens, logprob = depth_step(K, hidden, prefix, u=u, **w)
    # each step by its own inputs, in 64 bits; wide of a code's border no code differs
    a = K.add_rmsnorm(rows, d, EPS)(hidden, prefix, w["norm_in"])
    q, s = codes_of(a)
    g, up = product(q, s.astype(np.float64), w["gate"]), product(q, s.astype(np.float64), w["up"])
    want = g / (1 + np.exp(-g)) * up
    assert np.all(np.abs(act.double().cpu().numpy() - want) <= np.abs(want) * (3 + np.abs(g)) * 9 * U + U)
    q, s = codes_of(act)
    want = product(q, s.astype(np.float64), w["down"])
    total = want + a.double().cpu().numpy()
    assert np.all(np.abs(body.double().cpu().numpy() - total) <= 3.1 * U * np.abs(want) + U * np.abs(total))
    q, s = codes_of(body, w["norm_out"])
    want = product(q, scale_of(body, s, w["norm_out"]), w["table"])
    total = want + w["bias"].double().cpu().numpy()
    assert np.all(np.abs(logits.double().cpu().numpy() - total) <= (NORM_REL + 4 * U) * np.abs(want) + U * np.abs(total))
    check_sample(K, logits, u, 0.9, 50, 0.95, 0.02)


def test_on_another_stream_and_in_graphs(K):
    """The step captured once per stream, two graphs replayed at a time, with inputs that change."""
    d, inner, v, rows = 256, 384, 2051, 20
    w = head_weights(K, d, inner, v)
    graphs = []
    for i in range(2):
        st = torch.cuda.Stream()
        inputs = dict(hidden=some_logits(rows, d, i), prefix=some_logits(rows, d, 10 + i), u=uniforms(rows, 20 + i))
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            depth_step(K, **inputs, **w)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            out = depth_step(K, **inputs, **w)
        graphs.append((graph, st, inputs, out))
    for turn in range(3):
        for i, (graph, st, inputs, out) in enumerate(graphs):
            inputs["hidden"].copy_(some_logits(rows, d, 100 + 10 * turn + i))
            inputs["u"].copy_(uniforms(rows, 200 + 10 * turn + i))
        torch.cuda.synchronize()
        for graph, st, _, _ in graphs:
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for _, _, inputs, out in graphs:
            for x, y in zip(out, depth_step(K, **inputs, **w)):
                assert torch.equal(x, y)


def test_the_same_call_twice_gives_the_same(K):
    x, w = rows_in((150, 700), 1, torch.float32), weights(300, 700, 2)
    assert torch.equal(K.int8_linear(x, w), K.int8_linear(x, w))
    lg, u = some_logits(30, 50000, 3), uniforms(30, 3)
    a, b = K.sample_tokens(lg, u, top_p=0.9), K.sample_tokens(lg, u, top_p=0.9)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("k", [1, 37, 256, 300, 520, 1024, 2048, 4100, 8192, 20000])
def test_a_normed_row_goes_by_itself(K, dtype, k):
    """A row's scale holds its sum of squares, added in the same order whatever stands beside it: by a product's own
    CTAs for one or two tokens, by 32 to 256 threads a row in a batch.  To the bit."""
    t = 700
    x, nw = rows_in((t, k), k, DT[dtype], 3), 1 + 0.3 * torch.randn(k, device="cuda", generator=gen(1))
    w, w2 = weights(70, k, 2), weights(70, k, 3)
    kw = dict(norm_weight=nw, eps=EPS)
    rows, lin, glu = K.quantize_rows(x, **kw), K.int8_linear(x, w, **kw), K.int8_swiglu(x, w, w2, **kw)
    for a, b in ((0, 1), (699, 700), (5, 7), (0, 3), (10, 26), (300, 333), (17, 313), (17, 314)):
        part = K.quantize_rows(x[a:b], **kw)
        assert torch.equal(part.scale, rows.scale[a:b]) and torch.equal(part.q, rows.q[a:b])
        assert torch.equal(K.int8_linear(x[a:b], w, **kw), lin[a:b])
        assert torch.equal(K.int8_swiglu(x[a:b], w, w2, **kw), glu[a:b])


@pytest.mark.parametrize("n,k", [(1024, 131071), (4096, 40000)])
def test_fewer_tokens_take_no_longer(K, n, k):
    """Rows so long that the tensor cores have them: one to four tokens in hardly more time than eight (they took up to
    eight times as long, where every few tokens read all weights again)."""
    weight = weights(n, k, 1)
    rows = {t: K.quantize_rows(rows_in((t, k), t, torch.float32)) for t in (1, 2, 3, 4, 8)}
    times = {t: [] for t in rows}
    for turn in range(9):
        for t, x in rows.items():
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            K.int8_linear(x, weight)
            a.record()
            for _ in range(4):
                K.int8_linear(x, weight)
            b.record()
            torch.cuda.synchronize()
            times[t].append(a.elapsed_time(b))
    best = {t: min(v) for t, v in times.items()}
    assert max(best[t] for t in (1, 2, 3, 4)) < 1.5 * best[8], best


@pytest.mark.parametrize("t", [1, 2, 3, 4, 5, 16, 17])
@pytest.mark.parametrize("k", [8192, 8193, 16384, 16385, 24576, 24577, 33000, 66000])
def test_few_tokens_of_long_rows(K, t, k):
    """About the borders at which long rows go to the tensor cores, with few channels and with many."""
    check_linear(K, t, 37, k, bias=True)
    check_linear(K, t, 700, k, "bf16", residual=True, codes=True)
    check_swiglu(K, t, 21, k)
    check_swiglu(K, t, 300, k, "f16")


@pytest.mark.parametrize("call", ["sample_tokens", "int8_linear", "quantize_rows"])
def test_other_threads_run_while_a_launch_waits(K, call):
    """More calls than a stream's queue holds, behind half a second of other work: the launch that waits for room keeps
    no other Python thread from running."""
    x, u = torch.randn(4, 512, device="cuda", generator=gen(1)), torch.rand(4, device="cuda", generator=gen(2))
    w = weights(64, 512, 3)
    once = {"sample_tokens": lambda: K.sample_tokens(x, u), "int8_linear": lambda: K.int8_linear(x, w),
            "quantize_rows": lambda: K.quantize_rows(x)}[call]
    once()
    torch.cuda.synchronize()
    stop, longest = threading.Event(), [0.0]

    def tick():
        last = time.perf_counter()
        while not stop.is_set():
            time.sleep(0.001)
            now = time.perf_counter()
            longest[0], last = max(longest[0], now - last), now

    other = threading.Thread(target=tick)
    other.start()
    try:
        torch.cuda._sleep(1_000_000_000)
        for _ in range(3000):
            once()
        torch.cuda.synchronize()
    finally:
        stop.set()
        other.join()
    assert longest[0] < 0.2, longest[0]


def test_the_longer_way_gives_the_same(K, monkeypatch):
    """Through ctypes, where the short way was not built."""
    from soraku_tts_b200 import _lib

    x, nw, u = rows_in((40, 512), 1, torch.bfloat16), torch.rand(512, device="cuda", generator=gen(1)), torch.rand(40, device="cuda")
    w, b = weights(96, 512, 2), torch.randn(96, device="cuda", generator=gen(3))

    def step():
        y = K.int8_linear(x, w, norm_weight=nw, bias=b, residual=x[:, :96])
        q = K.quantize_rows(x, norm_weight=nw)
        return y, *q, K.int8_swiglu(q, w, w), *K.sample_tokens(y, u, temperature=0.8, top_k=20, top_p=0.9, min_p=0.01)

    short = step()
    monkeypatch.setattr(_lib, "_bind", _lib._NoBind)
    assert all(torch.equal(a, c) for a, c in zip(short, step()))
