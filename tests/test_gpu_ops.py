"""The device-buffer operators (include/czg_ops.h) against their definitions in 64 bits.

Tolerances.  u is half a step of the output type (fp32 2^-24, bf16 2^-8 / 2 ... as
torch.finfo(t).eps / 2); a result's error is bounded by u |y| for its one rounding plus what the
arithmetic before it may lose, written out at each comparison.
"""
import math
import os

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    from compress_zip_b200 import ops

    return ops


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def u(t):
    return torch.finfo(t).eps / 2


# ---- quantize_rows ------------------------------------------------------------------


def codes_of(x):
    """(codes, scales) by the definition; the quotients of 16-bit values are exact to 2^-53."""
    x = x.double()
    a = x.abs().amax(1, keepdim=True)
    return torch.where(a > 0, 127 * x / a, 0).round().to(torch.int8), (a / 127).float()[:, 0]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 16), (3, 17), (5, 384), (2, 4097), (300, 63), (64, 1024), (7, 10007),
                                 (2401, 40), (2370, 1000), (2368, 4096), (5001, 2049), (3000, 300), (2370, 5000)])
def test_quantize_rows(ops, dtype, m, k):
    g = gen(m * k)
    x = randn(g, m, k + 5).to(dtype)[:, 2:k + 2]   # rows that begin off any boundary
    if k > 2:
        x[0, 1] = x[0].abs().max()
        x[0, 2] = -x[0, 1] / 2                     # 127 x / max = -63.5: the even neighbour
    got = ops.quantize_rows(x)
    codes, scales = codes_of(x)
    assert got.codes.shape == (m, k) and got.codes.stride(0) % 16 == 0
    if dtype == FP32:   # 127 x and the quotient round (2^-23 in all): codes may differ next to a half alone
        q = 127 * x.double() / x.double().abs().amax(1, keepdim=True)
        assert ((got.codes.double() - q).abs() <= 0.5 + 128 * 2.0 ** -23).all()
    else:
        assert torch.equal(got.codes, codes)
    assert torch.equal(got.scales, scales)
    if k % 16:   # the bytes behind a row are zeros
        full = got.codes.as_strided((m, got.codes.stride(0)), (got.codes.stride(0), 1))
        assert not full[:, k:].any()


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_quantize_rows_at_the_halves(ops, dtype):
    """Rows whose maxima have 127 as a factor, or are twice an entry, are full of exact halves;
    their neighbours by one step of the type are not."""
    rows = []
    for e in (-20, -3, 0, 9) if dtype == FP16 else (-130, -100, -3, 0, 60, 118):
        for m in (127, 254, 255, 129, 200, 191, 131):
            top = torch.tensor(m * 2.0 ** (e if dtype == BF16 else max(e, -14) - 7), dtype=torch.float64, device=DEV)
            k = torch.arange(-127, 128, dtype=torch.float64, device=DEV)
            v = torch.cat([top[None], top * (k + 0.5) / 127, top * k / 254]).to(dtype)
            up = torch.nextafter(v.cpu(), torch.full_like(v.cpu(), math.inf)).to(DEV)
            down = torch.nextafter(v.cpu(), torch.full_like(v.cpu(), -math.inf)).to(DEV)
            rows.append(torch.cat([v, up, down]).clamp(-top.item(), top.item()))
    x = torch.stack(rows)
    assert torch.isfinite(x).all()
    codes, scales = codes_of(x)
    for copies in (1, 60):       # a CTA a row, a warp a row
        got = ops.quantize_rows(x.repeat(copies, 1))
        assert torch.equal(got.codes, codes.repeat(copies, 1)) and torch.equal(got.scales, scales.repeat(copies))


def test_quantize_rows_special(ops):
    x = torch.zeros(10, 40, device=DEV)
    x[1] = 3.0
    x[2, 5] = float("nan")
    x[3, 39] = float("inf")
    x[4, 0] = -float("inf")
    x[5] = torch.linspace(-3e38, 3e38, 40)             # its step overflows: the row is not finite
    x[9] = torch.linspace(-1, 1, 40) * 3e38
    x[6] = 1e-45
    x[7, 3] = -1e-20
    x[8] = -0.0
    for dtype in (FP32, BF16):
        got = ops.quantize_rows(x.to(dtype))
        s = got.scales
        assert s[0] == 0 and s[8] == 0 and not got.codes[[0, 8]].any()
        assert (got.codes[1] == 127).all()
        assert not torch.isfinite(x[5]).all()
        assert torch.isnan(s[2:6]).all() and not got.codes[2:6].any()
        want, scale = codes_of(x.to(dtype)[9:])
        assert (got.codes[9] - want[0]).abs().max() <= (1 if dtype == FP32 else 0) and s[9] == scale[0]
        assert got.codes[7, 3] == -127 and got.codes[7].ne(0).sum() == 1
        if dtype == FP32:
            assert (got.codes[6] == 127).all()
    assert ops.quantize_rows(torch.zeros(0, 7, device=DEV)).codes.shape == (0, 7)
    empty = ops.quantize_rows(torch.zeros(3, 0, device=DEV))
    assert empty.codes.shape == (3, 0) and not empty.scales.any()


# ---- linear_i8 ------------------------------------------------------------------------


def rand_codes(ops, g, n, k, pad=0):
    """Codes whose rows are followed by bytes that must not count."""
    ld = (k + 15) // 16 * 16 + pad
    full = torch.randint(-127, 128, (n, ld), generator=g, device=DEV, dtype=torch.int8)
    return ops.QRows(full[:, :k], 0.001 * (0.5 + torch.rand(n, generator=g, device=DEV)))


def check_linear(y, x, w, bias):
    acc = x.codes.double() @ w.codes.double().t()
    prod = acc * x.scales.double()[:, None] * w.scales.double()
    want = prod if bias is None else prod + bias.double()
    # float(sum), two products and the sum with the bias round once each; then the output type's one
    tol = u(y.dtype) * want.abs() + 4 * 2.0 ** -24 * (prod.abs() + want.abs())
    if y.dtype == FP16:
        tol = tol + 2.0 ** -25   # half a step of its subnormal numbers
    assert ((y.double() - want).abs() <= tol).all(), ((y.double() - want).abs() - tol).max()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 512, 384), (2, 129, 17), (5, 64, 16), (16, 130, 100), (17, 100, 1100),
                                   (33, 257, 640), (64, 300, 129), (65, 96, 512), (130, 257, 128), (200, 1000, 48),
                                   (257, 513, 1000), (600, 640, 2048), (1, 4096, 4096), (24, 4096, 8200), (128, 1100, 3000),
                                   (2500, 2100, 200), (2049, 2500, 1000), (5000, 1000, 129), (2560, 8192, 64), (300, 20000, 400)])
def test_linear_i8(ops, dtype, m, n, k):
    g = gen(m + n + k)
    x, w = rand_codes(ops, g, m, k, 32), rand_codes(ops, g, n, k)
    bias = randn(g, n) if (m + n) % 2 else None
    check_linear(ops.linear_i8(x, w, bias=bias, out_dtype=dtype), x, w, bias)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,n,k", [(1, 512, 384), (3, 70, 33), (50, 1024, 512), (300, 384, 1024), (16, 200, 2048), (15, 64, 1),
                                   (2, 130, 11264), (2, 130, 11265), (2, 130, 12288), (1, 20000, 1100), (17, 300, 640), (5, 1, 4100)])
def test_linear_i8_from_floats(ops, dtype, m, n, k):
    """Quantising in the call is quantize_rows and then the product, bit for bit."""
    g = gen(m * n)
    x, w = randn(g, m, k).to(dtype), rand_codes(ops, g, n, k)
    y = ops.linear_i8(x, w)
    assert y.dtype == dtype
    q = ops.quantize_rows(x)
    assert torch.equal(y, ops.linear_i8(q, w, out_dtype=dtype))
    check_linear(y, q, w, None)
    batched = ops.linear_i8(x.view(1, m, k), w)
    assert batched.shape == (1, m, n) and torch.equal(batched[0], y)
    assert torch.equal(ops.linear_i8(x.t().contiguous().t().contiguous(), w), y)


@pytest.mark.parametrize("m", [1, 7, 40, 150])
def test_linear_i8_into_a_view(ops, m):
    """out may be columns of a wider tensor: what lies beside them stays."""
    g = gen(m)
    x, w = rand_codes(ops, g, m, 96), rand_codes(ops, g, 45, 96)
    wide = torch.full((m, 64), 7.0, device=DEV, dtype=BF16)
    y = ops.linear_i8(x, w, out=wide[:, 3:48])
    assert y.data_ptr() == wide[:, 3:].data_ptr()
    check_linear(y, x, w, None)
    assert (wide[:, :3] == 7).all() and (wide[:, 48:] == 7).all()


@pytest.mark.parametrize("m", [3, 40])
def test_linear_i8_beside_its_operand(ops, m):
    """Columns of one buffer: x in some, out in others; over one another they are refused."""
    g = gen(m)
    w = rand_codes(ops, g, 45, 64)
    buf = randn(g, m, 128).to(BF16)
    x = buf[:, 64:]
    want = ops.linear_i8(x.clone(), w)
    before = buf[:, 64:].clone()
    assert torch.equal(ops.linear_i8(x, w, out=buf[:, 8:53]), want) and torch.equal(buf[:, 64:], before)
    with pytest.raises(RuntimeError, match="over x"):
        ops.linear_i8(x, w, out=buf[:, 30:75])


def test_attend_in_place(ops):
    """out may be q itself, or other heads of the buffer that q lies in."""
    r = gen(21)
    c = noise_cache(ops, r, 3, 2, 1200, 64, False)
    for lens in ((100, 7, 40), (1200, 3, 600)):
        buf = randn(r, 3, 2, 20, 64).to(BF16)
        want = c.attend(buf[:, :, :8].clone(), int32(0, 1, 2), int32(*lens))
        c.attend(buf[:, :, :8], int32(0, 1, 2), int32(*lens), out=buf[:, :, 10:18])
        assert torch.equal(buf[:, :, 10:18], want)
        c.attend(buf[:, :, :8], int32(0, 1, 2), int32(*lens), out=buf[:, :, :8])
        assert torch.equal(buf[:, :, :8], want)
        with pytest.raises(RuntimeError, match="over q"):
            c.attend(buf[:, :, :8], int32(0, 1, 2), int32(*lens), out=buf[:, :, 4:12])


def test_linear_i8_sums_are_exact(ops):
    """The longest row at the largest codes: 131,071 * 127 * 127 stays below 2^31."""
    k = 131071
    x = ops.QRows(torch.full((3, 131072), 127, dtype=torch.int8, device=DEV)[:, :k], torch.ones(3, device=DEV))
    w = ops.QRows(torch.full((5, 131072), 127, dtype=torch.int8, device=DEV)[:, :k], torch.ones(5, device=DEV))
    w.codes[1] = -127
    w.codes[2, ::2] = -127
    y = ops.linear_i8(x, w, out_dtype=FP32)
    want = (x.codes.double() @ w.codes.double().t()).float()
    assert torch.equal(y, want)
    with pytest.raises(RuntimeError, match="MAX_K"):
        big = ops.QRows(torch.zeros(1, 131072, dtype=torch.int8, device=DEV), torch.ones(1, device=DEV))
        ops.linear_i8(big, big)


def test_linear_i8_not_finite(ops):
    g = gen(4)
    x, w = rand_codes(ops, g, 40, 64), rand_codes(ops, g, 30, 64)
    x.scales[3] = float("nan")
    w.scales[7] = float("inf")
    y = ops.linear_i8(x, w, out_dtype=FP32)
    assert torch.isnan(y[3]).all()
    rest = torch.arange(40, device=DEV) != 3
    assert not torch.isfinite(y[rest][:, 7]).any()
    cols = torch.arange(30, device=DEV) != 7
    assert torch.isfinite(y[rest][:, cols]).all()


@pytest.mark.parametrize("n,k", [(512, 384), (130, 100), (4096, 1024)])
def test_linear_i8_does_not_depend_on_the_batch(ops, n, k):
    """A row alone gives the bits that it gives among others, wherever it stands."""
    g = gen(n)
    x, w, bias = rand_codes(ops, g, 700, k), rand_codes(ops, g, n, k), randn(g, n)
    full = ops.linear_i8(x, w, bias=bias, out_dtype=FP32)
    for a, b in ((0, 1), (5, 6), (3, 12), (100, 133), (690, 700), (64, 264)):
        part = ops.linear_i8(ops.QRows(x.codes[a:b], x.scales[a:b]), w, bias=bias, out_dtype=FP32)
        assert torch.equal(part, full[a:b])


def test_linear_i8_is_the_models_projection(ops, shipped_path, oracle_mod):
    """With a channel scale of mult / 2^shift (exact powers and small integers) the rounded and
    clamped product is the engine's requantised projection, on the shipped model's weights."""
    from compress_zip_b200 import czm

    t = czm.ModelFile.load(shipped_path).tensors
    wq = torch.from_numpy(np.array(t["layers.0.attn.qkv.weight"])).to(DEV)
    mult, shift = 819, 20
    g = gen(1)
    x = torch.randint(-127, 128, (90, wq.shape[1]), generator=g, device=DEV, dtype=torch.int8)
    y = ops.linear_i8(ops.QRows(x, torch.full((90,), float(mult), device=DEV)),
                      ops.QRows(wq, torch.full((wq.shape[0],), 2.0 ** -shift, device=DEV)), out_dtype=FP32)
    acc = (x.double() @ wq.double().t()).long() * mult
    down = acc >> shift
    rest = acc - (down << shift)
    half = 1 << (shift - 1)
    rne = down + ((rest > half) | ((rest == half) & (down & 1 == 1))).long()
    # acc * mult < 2^34 may need more than 24 bits: away from a half by less than 2^-24 of the value
    # the fp32 product may round onto it, so those places are left out
    near = (rest - half).abs().double() <= acc.abs().double() * 2.0 ** -23
    assert near.double().mean() < 0.01
    got = y.round().clamp(-127, 127).long()
    assert torch.equal(got[~near], rne.clamp(-127, 127)[~near])


# ---- the 4-bit cache --------------------------------------------------------------------


def bf16_below(x):
    m, e = torch.frexp(x)
    return torch.ldexp(torch.floor(m * 256), e - 8)


def held(x):
    """What an entry holds of rows x, in float64."""
    x = x.double()
    lo = bf16_below(x.amin(-1, keepdim=True))
    step = -bf16_below((lo - x.amax(-1, keepdim=True)) / 15)
    return lo + step * torch.where(step > 0, (x - lo) / step.clamp(min=1e-300), 0).round(), step[..., 0], lo[..., 0]


def int32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def entries(c, slot):
    """All entries of a slot in float64: k, v [heads, capacity, d]."""
    out = []
    for x, col in ((c.k, 0), (c.v, 2)):
        b = x[slot].int()
        codes = torch.stack([b & 15, b >> 4], -1).flatten(-2).double()
        s = c.scales[slot].double()
        out.append(s[..., col + 1:col + 2] + s[..., col:col + 1] * codes)
    return out


def noise_cache(ops, g, n_slots, heads, capacity, d, track):
    """A cache of arbitrary codes and ranges: what no sequence has written yet is not zero."""
    def codes():
        return torch.randint(0, 256, (n_slots, heads, capacity, d // 2), generator=g, device=DEV, dtype=torch.uint8)

    step = 0.05 + 0.3 * torch.rand(n_slots, heads, capacity, 2, generator=g, device=DEV)
    lo = -step * (6 + 3 * torch.rand(step.shape, generator=g, device=DEV))
    scales = torch.stack([step[..., 0], lo[..., 0], step[..., 1], lo[..., 1]], -1).to(BF16)
    w = torch.rand(n_slots, heads, capacity, generator=g, device=DEV) if track else None
    return ops.KV4Cache(codes(), codes(), scales, w)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_append_and_read(ops, dtype, d):
    g = gen(d)
    c = noise_cache(ops, g, 6, 3, 50, d, True)
    before = [t.clone() for t in (c.k, c.v, c.scales, c.weights)]
    t = 5
    # full, one row, a padded place, all padding, up to the end of the slot
    slots, lengths = int32(4, 0, -1, 2, 5), int32(9, 1, 7, 0, 50)
    big = randn(g, 5, 3, t + 2, 2 * d + 4).to(dtype)
    k = big[:, :, 1:t + 1, 2:d + 2].transpose(1, 2)       # strides of its own for every dimension
    v = randn(g, 5, t, 3, d).to(dtype)
    k[0, 0, 0] = 0.75                                      # a constant row: exact
    v[1, 4, 2] = 0                                         # a row of zeros
    k[4, 1, 1, 7] = float("nan")
    v[4, 2, 0, 0] = float("inf")
    c.append(k, v, slots, lengths)
    c.check()
    written = torch.zeros(6, 50, dtype=torch.bool, device=DEV)
    for i, (s, n) in enumerate(zip(slots.tolist(), lengths.tolist())):
        if s < 0:
            continue
        for r in range(t):
            e = n - t + r
            if e < 0:
                continue
            written[s, e] = True
            for x, col, name in ((k, 0, "k"), (v, 2, "v")):
                want, step, lo = held(x[i, r])
                got = entries(c, s)[0 if name == "k" else 1][:, e]
                bad = ~torch.isfinite(x[i, r]).all(-1)
                assert torch.isnan(got[bad]).all()
                assert torch.equal(got[~bad], want[~bad])
                assert torch.equal(c.scales[s, :, e, col].double()[~bad], step[~bad])
                # half a step, and the rounding of the quotient (15 * 2^-24 of a step) next to a half
                assert ((got - x[i, r].double()).abs() <= step[:, None] * (0.5 + 2.0 ** -20))[~bad].all()
            assert not c.weights[s, :, e].any()
    assert torch.equal(entries(c, 4)[0][0, 4], torch.full((d,), 0.75, dtype=torch.float64, device=DEV))
    assert not entries(c, 0)[1][2, 0].any()
    for now, old in zip((c.k, c.v, c.scales, c.weights), before):   # nothing else is touched
        keep = ~written[:, None, :].expand(6, 3, 50)
        assert torch.equal(now[keep], old[keep])
    rk, rv = c.read(int32(4, -3, 5), int32(3, 0, 46), 6, dtype=dtype)
    for got, which in ((rk, 0), (rv, 1)):
        assert got.shape == (3, 6, 3, d) and not got[1].any() and not got[2, 4:].any()
        for i, (s, a, n) in enumerate(((4, 3, 6), (-1, 0, 0), (5, 46, 4))):
            want = entries(c, s)[which][:, a:a + n].transpose(0, 1)
            ok = torch.isfinite(want)
            assert torch.equal(torch.isfinite(got[i, :n]), ok)
            # step * code is exact, the sum rounds to fp32 and then to the output type
            tol = (u(dtype) + 2.0 ** -24) * want.abs() + (2.0 ** -25 if dtype == FP16 else 0)
            assert ((got[i, :n].double() - want).abs() <= tol)[ok].all()
    with pytest.raises(RuntimeError, match="length"):      # the read past the slot's end was reported
        c.check()
    c.check()


def test_append_extremes(ops):
    c = ops.KV4Cache.empty(1, 1, 8, 64)
    x = torch.zeros(1, 4, 1, 64, device=DEV)
    x[0, 0, 0, 3] = 3e38
    x[0, 0, 0, 5] = -3e38          # the range overflows fp32
    x[0, 1] = 1e-30
    x[0, 1, 0, 9] = -2e-30
    x[0, 2] = 65504.0
    x[0, 3, 0, ::2] = 1.0
    c.append(x, -x, int32(0), int32(4))
    k, v = entries(c, 0)
    assert torch.isnan(k[0, 0]).all() and torch.isnan(v[0, 0]).all()
    for i in (1, 2, 3):
        assert torch.equal(k[0, i], held(x[0, i])[0][0]) and torch.equal(v[0, i], held(-x[0, i])[0][0])
    # 1 / 15 rounded up to bf16 is 137 / 2048: the upper end is held as 15 of those
    assert torch.equal(k[0, 3], x[0, 3, 0].double() * (15 * 137 / 2048))


def test_append_out_of_range_is_left_out_and_reported(ops):
    g = gen(3)
    for slots, lengths, text in (((0, 3), (2, 2), "slot beyond"), ((0, 1), (2, 11), "length"), ((0, 1), (2, -1), "length"),
                                 ((1, 1), (2, 2), "twice")):
        c = noise_cache(ops, g, 3, 2, 10, 64, False)
        old = c.k.clone()
        rows = randn(g, 2, 2, 2, 64)
        c.append(rows, rows, int32(*slots), int32(*lengths))
        with pytest.raises(RuntimeError, match=text):
            c.check()
        assert torch.equal(c.k[2], old[2])
        if text != "twice":
            assert torch.equal(entries(c, 0)[0][:, :2], held(rows[0])[0].transpose(0, 1))
            where = c.k[1] == old[1]
            assert where[:, :9].all() and (slots != (0, 1) or lengths[1] == 11 or where.all())


# ---- attention ---------------------------------------------------------------------------


def attention(c, q, slots, lengths, scale, max_len):
    """(out, its tolerance, added weights, their tolerance) in float64.

    A score's fp32 error is at most (D + 16) 2^-24 E, E the sum of its terms' magnitudes, and the
    exponential adds 2^-21 (of it and its argument's product with log2 e): a weight is off by the
    factor 1 + r, r = 2 (D + 16) 2^-24 E + 2^-20, numerator and denominator together twice that.
    The weights are held in fp16 for the product with the values: 2^-11 of each value's terms."""
    b, t, hq, d = q.shape
    g = hq // c.n_heads
    out, tol = torch.zeros(q.shape, dtype=torch.float64, device=DEV), torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    add = torch.zeros(c.n_slots, c.n_heads, c.capacity, dtype=torch.float64, device=DEV)
    add_tol = torch.zeros_like(add)
    for i, (s, n) in enumerate(zip(slots.tolist(), lengths.tolist())):
        if not 0 <= s < c.n_slots:
            continue
        n = max(0, min(n, max_len, c.capacity))
        k, v = entries(c, s)
        sc = c.scales[s].double().abs()
        k_abs, v_abs = 15 * sc[..., 0] + sc[..., 1], 15 * sc[..., 2] + sc[..., 3]
        for r in range(t):
            seen = n - (t - 1 - r)
            if seen <= 0:
                continue
            qr = q[i, r].double().view(c.n_heads, g, d)
            p = torch.softmax(scale * torch.einsum("hgd,hnd->hgn", qr, k[:, :seen]), -1)
            e = abs(scale) * qr.abs().sum(-1, keepdim=True) * k_abs[:, None, :seen]
            rel = 2 * (2 * (d + 16) * 2.0 ** -24 * e.amax(-1, keepdim=True) + 2.0 ** -20)
            y = torch.einsum("hgn,hnd->hgd", p, v[:, :seen]).reshape(hq, d)
            out[i, r] = y
            terms = torch.einsum("hgn,hn->hg", p * (rel + 2.0 ** -11), v_abs[:, :seen]).reshape(hq, 1)
            tol[i, r] = u(q.dtype) * y.abs() + terms + (2.0 ** -25 if q.dtype == FP16 else 0)
            add[s, :, :seen] += p.sum(1)
            add_tol[s, :, :seen] += (p * rel).sum(1)
    return out, tol, add, add_tol


def check_attend(ops, c, q, slots, lengths, max_len=None, scale=None):
    before = None if c.weights is None else c.weights.clone()
    y = c.attend(q, slots, lengths, max_len=max_len, scale=scale)
    out, tol, add, add_tol = attention(c, q, slots, lengths, q.shape[3] ** -0.5 if scale is None else scale,
                                       c.capacity if max_len is None else max_len)
    assert y.shape == q.shape and y.dtype == q.dtype
    assert torch.isfinite(y).all()
    worst = ((y.double() - out).abs() - tol).max()
    assert worst <= 0, worst
    if before is not None:
        want = before.double() + add
        rows = q.shape[1] * q.shape[2] // c.n_heads
        tol = add_tol + (rows + 2) * 2.0 ** -24 * (want.abs() + add)
        worst = ((c.weights.double() - want).abs() - tol).max()
        assert worst <= 0, worst
        same = add == 0
        assert torch.equal(c.weights[same], before[same])   # entries that no row sees keep their bits
    return y


@pytest.mark.parametrize("track", [False, True])
@pytest.mark.parametrize("d,heads,g,t,dtype,lens,capacity", [
    (64, 1, 6, 1, BF16, (1,), 64),
    (64, 1, 6, 1, BF16, (77, 0, 2, 31, 32, 33), 100),
    (64, 1, 8, 1, FP16, (512, 511, 513, 64, 63, 65), 520),
    (64, 2, 1, 1, BF16, (1023, 1, 1024, 1025, 900), 1025),
    (128, 2, 4, 1, BF16, (300, 17, 0, 129), 300),
    (128, 1, 8, 1, FP16, (5000, 2047, 1, 2048), 5003),
    (64, 4, 4, 1, BF16, (20000,), 20000),
    (128, 1, 16, 1, BF16, (700, 3), 700),
    (64, 2, 3, 5, BF16, (4, 0, 5, 6, 1, 700, 1030), 1100),
    (128, 2, 2, 7, FP16, (40, 7, 3, 1500), 1501),
    (64, 1, 6, 33, BF16, (40, 1, 600), 640),
    (64, 3, 5, 2, FP16, (95, 96, 97, 128, 160), 161),
    (128, 8, 7, 3, BF16, (513, 2, 64), 513),
    (64, 1, 8, 1, FP16, (70000, 65537, 500, 65536), 70001),
    (128, 1, 2, 2, BF16, (131073, 66001), 131073),
    (64, 1, 2, 1, BF16, (300000,), 300000),
    (64, 1, 8, 150, BF16, (300, 5, 149, 151), 300),
    (128, 1, 3, 40, FP16, (1100, 39), 1100),
    (64, 96, 1, 1, BF16, (70, 1), 70),
    (64, 1, 40, 1, FP16, (600, 20), 600),
    (128, 2, 2, 1, BF16, (1, 1, 0), 1),
])
def test_attend(ops, d, heads, g, t, dtype, lens, capacity, track):
    r = gen(capacity + t)
    b = len(lens)
    c = noise_cache(ops, r, b + 2, heads, capacity, d, track)
    slots = torch.randperm(b + 2, generator=r, device=DEV)[:b].int()
    lengths = int32(*lens)
    for i, n in enumerate(lens):   # what lies behind a sequence's end must not matter
        c.scales[slots[i].item(), :, n:] = float("nan")
    q = randn(r, b, t, heads * g, d).to(dtype)
    y = check_attend(ops, c, q, slots, lengths)
    c.check()
    if track:
        return
    # the bound of the lengths is no part of the result, nor the batch around a sequence
    assert torch.equal(c.attend(q, slots, lengths, max_len=max(max(lens), 1)), y)
    for i in range(b):
        assert torch.equal(c.attend(q[i:i + 1], slots[i:i + 1], lengths[i:i + 1]), y[i:i + 1])


def test_many_sequences(ops):
    """More sequences than any grid dimension's usual size, slots in any order, some of them padding;
    a cache of slots beyond what one pass of the check for repeated slots covers."""
    r = gen(40)
    b, n_slots = 60000, 70000
    c = noise_cache(ops, r, n_slots, 1, 4, 64, True)
    before = c.weights.clone()
    slots = torch.randperm(n_slots, generator=r, device=DEV)[:b].int()
    slots[::7] = -1
    lengths = torch.randint(0, 5, (b,), generator=r, device=DEV, dtype=torch.int32)
    rows, q = randn(r, b, 1, 1, 64).to(BF16), randn(r, b, 1, 2, 64).to(BF16)
    c.append(rows, -rows, slots, lengths)
    y = c.attend(q, slots, lengths)
    c.check()
    some = (slots >= 0) & (lengths > 0)
    assert not y[~some].any()
    at, last = slots[some].long(), lengths[some].long() - 1
    code = torch.stack([c.k & 15, c.k >> 4], -1).flatten(-2)[:, 0].double()
    sc = c.scales[:, 0].double()
    k = sc[..., 1:2] + sc[..., :1] * code
    code = torch.stack([c.v & 15, c.v >> 4], -1).flatten(-2)[:, 0].double()
    v = sc[..., 3:] + sc[..., 2:3] * code
    assert torch.equal(k[at, last], held(rows[some, 0, 0])[0]) and torch.equal(v[at, last], held(-rows[some, 0, 0])[0])
    s = torch.einsum("bgd,bnd->bgn", q[some, 0].double(), k[at]) / 8
    s = torch.where(torch.arange(4, device=DEV) <= last[:, None, None], s, -math.inf)
    p = torch.softmax(s, -1)
    want = torch.einsum("bgn,bnd->bgd", p, v[at])
    terms = torch.einsum("bgn,bn->bg", p, (15 * sc[..., 2] + sc[..., 3].abs())[at])[..., None]
    # attention()'s 2^-11 of the values' terms and 2^-20 of a weight, with room for its scores' rounding
    assert ((y[some, 0].double() - want).abs() <= u(BF16) * want.abs() + 2.0 ** -10 * terms).all()
    grown = c.weights.double()[at, 0] - torch.where(torch.arange(4, device=DEV) == last[:, None], 0.0, before[at, 0].double())
    assert (grown - p.sum(1)).abs().max() < 2.0 ** -18
    untouched = torch.ones(n_slots, dtype=torch.bool, device=DEV)
    untouched[at] = False
    assert torch.equal(c.weights[untouched], before[untouched])
    kept, new = c.evict(slots, lengths, 2, 1)
    assert torch.equal(new, torch.where(slots >= 0, lengths, 0).clamp(max=2))
    slots[b - 1] = slots[1]
    c.append(rows, rows, slots, lengths)
    with pytest.raises(RuntimeError, match="twice"):
        c.check()


@pytest.mark.parametrize("g,t", [(4, 1), (2, 3)])
def test_attend_strides_scale_and_padding(ops, g, t):
    r = gen(g)
    c = noise_cache(ops, r, 4, 2, 300, 64, True)
    big = randn(r, 4, 2 * g, t + 1, 70).to(BF16)
    q = big[:, :, 1:, 3:67].transpose(1, 2)
    slots, lengths = int32(2, -1, 0, 3), int32(300, 50, 0, 7)
    y = check_attend(ops, c, q, slots, lengths, scale=0.31)
    assert not y[1].any() and not y[2].any()
    out = torch.full((4, 2 * g, t, 80), 9.0, device=DEV, dtype=BF16)
    view = out[..., 8:72].transpose(1, 2)
    c.weights.zero_()
    got = c.attend(q, slots, lengths, scale=0.31, out=view)
    assert got.data_ptr() == view.data_ptr() and torch.equal(view, y)
    assert (out[..., :8] == 9).all() and (out[..., 72:] == 9).all()
    check_attend(ops, c, q, slots, lengths, scale=-0.2)
    c.attend(q, slots, lengths, scale=0.0)
    c.check()


def test_attend_peaked_and_flat(ops):
    """Scores far apart, equal scores, and value ranges that lie far apart."""
    r = gen(8)
    c = noise_cache(ops, r, 3, 1, 700, 64, True)
    c.scales[1, :, :, :2] = 0                      # keys all zero: a plain mean of the values
    c.scales[2, :, ::3, 2:] *= 1024                # a third of the values far above the others
    c.scales[2, :, 1::3, 2:] *= 2.0 ** -20
    c.scales[2, :, 5, 2] = 0                       # a constant row of values
    q = 12 * randn(r, 3, 1, 8, 64).to(BF16)
    check_attend(ops, c, q, int32(0, 1, 2), int32(700, 699, 640))
    tiny = (q * 2.0 ** -60).to(BF16)               # exponents that fp16 does not have
    check_attend(ops, c, tiny, int32(2, 1, 0), int32(513, 1, 30))
    huge = (q * 2.0 ** 60).to(BF16)
    check_attend(ops, c, huge, int32(0, 1, 2), int32(512, 20, 1), scale=2.0 ** -66)


def test_attend_ranges_that_grow_along_a_long_sequence(ops):
    """Later entries' steps far above the earlier ones', which may be 0 at first."""
    r = gen(18)
    c = noise_cache(ops, r, 4, 1, 70000, 64, True)
    for slot, powers in ((0, (0, 9)), (1, (-60, 3)), (2, (0, 60)), (3, (4, -30))):
        late = (torch.arange(70000, device=DEV) % 1024 >= 512)
        for part, p in ((~late, powers[0]), (late, powers[1])):
            c.scales[slot, 0, part, 2:] *= 2.0 ** p
    c.scales[2, 0, torch.arange(70000, device=DEV) % 1024 < 512, 2] = 0
    q = 2 * randn(r, 4, 1, 8, 64).to(BF16)
    check_attend(ops, c, q, int32(0, 1, 2, 3), int32(70000, 69999, 66666, 68000))


def test_attend_not_finite(ops):
    r = gen(9)
    c = noise_cache(ops, r, 2, 2, 100, 64, False)
    q = randn(r, 2, 1, 4, 64).to(BF16)
    y0 = c.attend(q, int32(0, 1), int32(60, 60))
    c.scales[0, 1, 10, 0] = float("nan")           # one key of head 1 of sequence 0
    c.scales[1, 0, 59, 3] = float("nan")           # one value of head 0 of sequence 1
    y = c.attend(q, int32(0, 1), int32(60, 60))
    assert torch.isnan(y[0, 0, 2:]).all() and torch.equal(y[0, 0, :2], y0[0, 0, :2])
    assert torch.isnan(y[1, 0, :2]).all() and torch.equal(y[1, 0, 2:], y0[1, 0, 2:])
    assert torch.isfinite(c.attend(q, int32(0, 1), int32(10, 59))).all()    # neither is seen
    q[0, 0, 1, 3] = float("nan")
    q[1, 0, 3, 0] = float("inf")
    y = c.attend(q, int32(0, 1), int32(10, 59))
    assert torch.isnan(y[0, 0, 1]).all() and not torch.isfinite(y[1, 0, 3]).any()
    assert torch.isfinite(y[0, 0, [0, 2, 3]]).all() and torch.isfinite(y[1, 0, :3]).all()


def test_attend_out_of_range_is_cut_and_reported(ops):
    r = gen(10)
    q = randn(r, 2, 1, 4, 64).to(BF16)
    for slots, lengths, max_len, text in (((0, 9), (20, 20), None, "slot beyond"), ((0, 1), (20, 51), None, "length"),
                                          ((0, 1), (20, -5), None, "length"), ((0, 1), (20, 31), 30, "length")):
        c = noise_cache(ops, r, 2, 2, 50, 64, False)
        check_attend(ops, c, q, int32(*slots), int32(*lengths), max_len=max_len)
        with pytest.raises(RuntimeError, match=text):
            c.check()
    c = noise_cache(ops, r, 2, 2, 50, 64, False)
    check_attend(ops, c, q, int32(1, 1), int32(20, 30))   # two sequences may read one slot
    c.check()
    c = noise_cache(ops, r, 2, 2, 50, 64, True)
    c.attend(q, int32(1, 1), int32(20, 30))                # but not add to its weights
    with pytest.raises(RuntimeError, match="twice"):
        c.check()


def test_offsets_beyond_32_bits(ops):
    """The last slot of a cache whose codes take more than 2^32 bytes."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB of device memory")
    slots, heads, capacity, d = 35, 8, 262144, 128
    shape = (slots, heads, capacity)
    assert math.prod(shape) * d // 2 > 1 << 32
    k, v = (torch.empty(*shape, d // 2, dtype=torch.uint8, device=DEV) for _ in range(2))
    c = ops.KV4Cache(k, v, torch.empty(*shape, 4, dtype=BF16, device=DEV), torch.empty(shape, device=DEV))
    g = gen(12)
    n = 300
    rows_k, rows_v = randn(g, 1, n, heads, d).to(BF16), randn(g, 1, n, heads, d).to(BF16)
    c.weights[slots - 1].zero_()
    c.append(rows_k, rows_v, int32(slots - 1), int32(n))
    rk, rv = c.read(int32(slots - 1), int32(0), n)
    assert (rk.double()[0] - held(rows_k[0])[0]).abs().max() <= 2.0 ** -8 * 8
    q = randn(g, 1, 1, 16, d).to(BF16)
    y = c.attend(q, int32(slots - 1), int32(n))
    small = ops.KV4Cache(*(x[slots - 1:, :, :512].contiguous() for x in (c.k, c.v, c.scales)))
    assert torch.equal(y, small.attend(q, int32(0), int32(n)))
    w = c.weights[slots - 1, :, :n].clone()
    kept, new = c.evict(int32(slots - 1), int32(n), 200, recent=10)
    assert new.tolist() == [200]
    want = torch.cat([w[:, :n - 10].topk(190, dim=1).indices.sort(1).values,
                      torch.arange(n - 10, n, device=DEV).expand(heads, 10)], 1)
    assert torch.equal(kept[0].long(), want)


# ---- eviction ----------------------------------------------------------------------------


def evicted(w, n, budget, recent):
    """The places that stay, in order, of one head's weights."""
    if n <= budget:
        return list(range(n))
    key = [math.inf if math.isnan(x) else x for x in w[:n - recent].tolist()]
    nan = [math.isnan(x) for x in w[:n - recent].tolist()]
    best = sorted(range(n - recent), key=lambda j: (not nan[j], -key[j], j))[:budget - recent]
    return sorted(best) + list(range(n - recent, n))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens,budget,recent,kind", [
    ((1, 2, 3, 0), 1, 0, "random"), ((1, 2, 3, 40), 1, 1, "random"), ((100, 64, 65, 63), 64, 10, "random"),
    ((513, 512, 1024, 1025), 300, 0, "random"), ((700, 30), 512, 512, "random"), ((900, 850, 13), 511, 100, "equal"),
    ((600, 601), 257, 3, "few"), ((400,), 100, 20, "special"), ((5000, 3000), 1000, 128, "random"), ((40000,), 20000, 77, "few"),
])
def test_evict(ops, d, lens, budget, recent, kind):
    g = gen(budget)
    b, heads, capacity = len(lens), 3, max(lens) + 9
    c = noise_cache(ops, g, b + 1, heads, capacity, d, True)
    w = c.weights
    if kind == "random":
        w.copy_(torch.exp(4 * randn(g, *w.shape)))
    elif kind == "equal":
        w.fill_(0.25)
    elif kind == "few":
        w.copy_(torch.randint(0, 4, w.shape, generator=g, device=DEV).float())
    else:
        w.copy_(randn(g, *w.shape))
        w[:, :, 3::50] = float("nan")
        w[:, :, 4::50] = float("inf")
        w[:, :, 5::50] = -0.0
        w[:, :, 6::50] = 0.0
        w[:, :, 7::50] = -float("inf")
    slots = torch.randperm(b + 1, generator=g, device=DEV)[:b].int()
    old = [x.clone() for x in (c.k, c.v, c.scales, c.weights)]
    kept, new = c.evict(slots, int32(*lens), budget, recent)
    c.check()
    assert new.tolist() == [min(n, budget) for n in lens]
    want = [x.clone() for x in old]
    for i, n in enumerate(lens):
        s = slots[i].item()
        for h in range(heads):
            stay = evicted(old[3][s, h], n, budget, recent)
            row = kept[i, h].tolist()
            assert row[:len(stay)] == stay and all(x == -1 for x in row[len(stay):])
            at = torch.tensor(stay, dtype=torch.long, device=DEV)
            for x, y in zip(want, old):
                x[s, h, :len(stay)] = y[s, h, at]
    for x, y in zip((c.k, c.v, c.scales, c.weights), want):   # the rest is left as it was
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_evict_padding_and_reports(ops):
    g = gen(2)
    c = noise_cache(ops, g, 3, 2, 40, 64, True)
    kept, new = c.evict(int32(-1, 2), int32(40, 40), 30, 5)
    c.check()
    assert new.tolist() == [0, 30] and (kept[0] == -1).all() and (kept[1] >= 0).all()
    for slots, lengths, text in (((0, 3), (40, 40), "slot beyond"), ((0, 1), (40, 41), "length"), ((0, 0), (40, 40), "twice")):
        c = noise_cache(ops, g, 3, 2, 40, 64, True)
        old = c.k.clone()
        kept, new = c.evict(int32(*slots), int32(*lengths), 30, 5)
        assert kept[0].max() < 40 and torch.equal(c.k[2], old[2])
        with pytest.raises(RuntimeError, match=text):
            c.check()
    with pytest.raises(ValueError, match="weights"):
        noise_cache(ops, g, 1, 1, 8, 64, False).evict(int32(0), int32(8), 4)


# ---- together ------------------------------------------------------------------------------


class Layer:
    """A serving step of one attention layer: projection, append, attention, projection."""

    def __init__(self, ops, seed, streams=3, heads=8, kv_heads=2, d=64, width=384, capacity=40):
        g = gen(seed)
        self.ops, self.h, self.hk, self.d = ops, heads, kv_heads, d
        rows = (heads + 2 * kv_heads) * d
        self.w_in = ops.quantize_rows(randn(g, rows, width) / width ** 0.5)
        self.w_out = ops.quantize_rows(randn(g, width, heads * d) / (heads * d) ** 0.5)
        self.cache = ops.KV4Cache.empty(streams, kv_heads, capacity, d, track_weights=True)

    def step(self, x, slots, lengths):
        b, t, width = x.shape
        qkv = self.ops.linear_i8(x, self.w_in).view(b, t, self.h + 2 * self.hk, self.d)
        q, k, v = qkv.split([self.h, self.hk, self.hk], 2)
        self.cache.append(k, v, slots, lengths)
        return self.ops.linear_i8(self.cache.attend(q, slots, lengths).flatten(2), self.w_out)


def test_a_serving_run(ops):
    """Prompts, single tokens and evictions in turn; every step's attention is compared with the
    formula on what the cache then holds, and the cache with what was appended and kept."""
    layer = Layer(ops, 5)
    c, g = layer.cache, gen(6)
    slots = int32(2, 0, 1)
    n = torch.tensor([9, 4, 0], dtype=torch.int32, device=DEV)       # a ragged prompt, padded on the left
    layer.step(randn(g, 3, 9, 384).to(BF16), slots, n)
    held_k = {s: entries(c, s)[0].clone() for s in range(3)}
    for step in range(60):
        n = n + 1
        x = randn(g, 3, 1, 384).to(BF16)
        qkv = ops.linear_i8(x, layer.w_in).view(3, 1, 12, 64)
        q, k, v = qkv.split([8, 2, 2], 2)
        c.append(k, v, slots, n)
        for i, s in enumerate(slots.tolist()):
            e = n[i].item() - 1
            assert torch.equal(entries(c, s)[0][:, e], held(k[i, 0])[0])
            held_k[s][:, e] = entries(c, s)[0][:, e]
            assert torch.equal(entries(c, s)[0][:, :e], held_k[s][:, :e])
        check_attend(ops, c, q, slots, n)
        if step % 15 == 14:
            kept, n = c.evict(slots, n, budget=16, recent=4)
            for i, s in enumerate(slots.tolist()):
                for h in range(2):
                    at = kept[i, h][kept[i, h] >= 0].long()
                    held_k[s][h, :len(at)] = held_k[s][h, at]
    c.check()


def test_two_streams_and_graph(ops):
    """The same steps on another stream and from a captured graph give the same bits; replays go
    on from what the cache holds."""
    g = gen(7)
    slots, xs = int32(1, 0, 2), [randn(g, 3, 2, 384).to(BF16) for _ in range(4)]

    def lengths(i):
        return torch.full((3,), 2 * (i + 1), dtype=torch.int32, device=DEV)

    eager = Layer(ops, 9)
    want = [eager.step(x, slots, lengths(i)) for i, x in enumerate(xs)]
    side = Layer(ops, 9)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = [side.step(x, slots, lengths(i)) for i, x in enumerate(xs)]
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(side.cache.weights, eager.cache.weights)
    layer = Layer(ops, 9)
    x, n = xs[0].clone(), lengths(0)
    warm = Layer(ops, 9)
    with torch.cuda.stream(stream):
        warm.step(x, slots, n)
    stream.synchronize()
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer.step(x, slots, n)
    with torch.cuda.graph(second):       # a second graph of the same cache, with a workspace of its own
        z = layer.step(x, slots, n)
    for i in range(4):
        x.copy_(xs[i])
        n.copy_(lengths(i))
        (graph if i % 2 == 0 else second).replay()
        torch.cuda.synchronize()
        assert torch.equal(y if i % 2 == 0 else z, want[i])
    assert torch.equal(layer.cache.weights, eager.cache.weights)


def test_graph_of_copies_and_operators(ops):
    """Copies, fills and torch's kernels before and between the operators of a captured graph."""
    g = gen(31)
    layer, slots, n = Layer(ops, 12), int32(0, 1, 2), int32(0, 0, 0)
    src, x = [randn(g, 3, 1, 384).to(BF16) for _ in range(5)], torch.zeros(3, 1, 384, dtype=BF16, device=DEV)
    feed, total = torch.zeros_like(x), torch.zeros(3, 1, 384, device=DEV)

    def step():
        x.copy_(feed)
        n.add_(1)
        total.zero_()
        y = layer.step(x, slots, n)
        total.add_(y.float())
        feed.zero_()
        return y

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    n.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    got = []
    for s in src:
        feed.copy_(s)
        graph.replay()
        got.append((y.clone(), total.clone()))
    torch.cuda.synchronize()
    layer.cache.check()
    ref, m = Layer(ops, 12), int32(0, 0, 0)
    for s, (a, b) in zip(src, got):
        m.add_(1)
        want = ref.step(s, slots, m)
        assert torch.equal(a, want) and torch.equal(b, want.float())
    assert torch.equal(layer.cache.weights[:, :, :5], ref.cache.weights[:, :, :5])


def test_every_call_gives_the_same_bits_again(ops):
    g = gen(13)
    c = noise_cache(ops, g, 20, 2, 3000, 128, True)
    q = randn(g, 20, 1, 16, 128).to(BF16)
    slots = torch.randperm(20, generator=g, device=DEV).int()
    lengths = torch.randint(0, 3001, (20,), generator=g, device=DEV, dtype=torch.int32)
    w0 = c.weights.clone()
    y0 = c.attend(q, slots, lengths)
    w1 = c.weights.clone()
    for _ in range(3):
        c.weights.copy_(w0)
        assert torch.equal(c.attend(q, slots, lengths), y0) and torch.equal(c.weights, w1)


# ---- attention over values of any size -----------------------------------------------------------
#
# The tolerances are attention()'s: rounding to fp16 is off by 2^-11 of a weight or by 2^-25 of what the
# row's largest weight times step, or (steps alike) the largest step, was brought to, 2^7 at least: for the
# 512 entries of a unit 2^-23 of the first and, with steps that differ by 2^6, 2^-16 of the second, both far
# inside what the formula leaves beside 2^-11 of all the terms.


def rising_cache(ops, g, n, heads, d, rise, track=False):
    """A cache of one slot, and a query for it, whose scores (to base 2) rise from 0 to `rise` along n entries."""
    c = noise_cache(ops, g, 1, heads, n, d, track)
    s = torch.linspace(0, rise * math.log(2), n, device=DEV)
    c.scales[0, :, :, 0] = 0
    c.scales[0, :, :, 1] = (s / d ** 0.5).to(BF16)
    return c


ones = lambda t, hq, d, dtype: torch.ones(1, t, hq, d, device=DEV, dtype=dtype)


@pytest.mark.parametrize("track", [False, True])
@pytest.mark.parametrize("d,dtype", [(64, BF16), (64, FP16), (128, BF16), (128, FP16)])
@pytest.mark.parametrize("n", [1, 77, 512, 1024, 70000])
def test_attend_constant_values(ops, n, d, dtype, track):
    """Value rows whose dimensions are all equal have a step of 0: their mean, whatever they are."""
    r = gen(n + d)
    big = torch.finfo(dtype).max if dtype == FP16 else 1e30
    for rise in (0.0, 7.9, 40.0, -40.0):
        c = rising_cache(ops, r, n, 1, d, rise, track)
        sign = torch.where(torch.rand(n, generator=r, device=DEV) < 0.5, -1.0, 1.0)
        for value in (8192.0, -65504.0, big, 100.0, 64.0 * sign, 8192 * sign, 60000 * sign, big * sign, 2.0 ** -30 * sign):
            c.scales[0, :, :, 2] = 0
            c.scales[0, 0, :, 3] = value.to(BF16) if torch.is_tensor(value) else value
            if dtype == FP16:      # bf16 rounds 65504 up, past what fp16 holds
                c.scales[0, 0, :, 3] = c.scales[0, 0, :, 3].clamp(-65280, 65280)
            check_attend(ops, c, ones(1, 2, d, dtype), int32(0), int32(n))
    c.check()


@pytest.mark.parametrize("d,power", [(64, 100), (128, 108), (64, -100), (128, -116)])
def test_attend_values_of_any_size(ops, d, power):
    """Weights from 1 to 2^-30 of the largest count alike whatever the values' exponent."""
    r = gen(power + 200 + d)
    c = rising_cache(ops, r, 900, 2, d, 30.0)
    c.scales[0, :, :, 2:] = (c.scales[0, :, :, 2:].double() * 2.0 ** power).to(BF16)
    check_attend(ops, c, ones(1, 4, d, BF16), int32(0), int32(900))


@pytest.mark.parametrize("d,g,t", [(64, 2, 1), (128, 3, 4)])
def test_attend_largest_values(ops, d, g, t):
    """Values up to the end of bf16: sums of many of them stay inside fp32."""
    r = gen(d)
    top = torch.finfo(BF16).max
    for n in (1, 512, 3000, 70000):
        for rise in (0.0, 7.9, 60.0):
            c = rising_cache(ops, r, n, 1, d, rise)
            q = ones(t, g, d, BF16)
            c.scales[0, :, :, 2] = 0
            c.scales[0, :, :, 3] = top
            y = c.attend(q, int32(0), int32(n))
            seen = torch.arange(t, device=DEV) >= t - n
            assert not y[0, ~seen].any()
            assert ((y[0, seen].double() - top).abs() <= 2 * u(BF16) * top).all()
            c.scales[0, :, ::2, 3] = -top / 4
            c.scales[0, :, 1::2, 3] = top / 8
            check_attend(ops, c, q, int32(0), int32(n))
            c.scales[0, :, 1::2, 2] = 2.0 ** 119          # steps too
            c.scales[0, :, 1::2, 3] = -(2.0 ** 122)
            check_attend(ops, c, q, int32(0), int32(n))
            c.scales[0, :, ::2, 2:] = 1.0
            check_attend(ops, c, q, int32(0), int32(n))


@pytest.mark.parametrize("d,power,far", [(64, 0, -50), (64, 100, -40), (128, 118, -30), (64, -100, -10), (128, -118, -4)])
def test_attend_small_weights_of_large_values(ops, d, power, far):
    """Entries of weights 2^far whose values are 2^-2 far times those of the heavy ones, at values' sizes
    from one end of bf16 to the other: what a weight is held to does not depend on them."""
    r = gen(power + 200 + d)
    c = rising_cache(ops, r, 900, 2, d, 0.0)
    c.scales[0, :, 500:, 1] = -far * math.log(2) / d ** 0.5
    c.scales[0, :, :, 2:] = (c.scales[0, :, :, 2:].double() * 2.0 ** power).to(BF16)
    if power >= 0:
        c.scales[0, :, 500:, 2:] = (c.scales[0, :, 500:, 2:].double() * 2.0 ** (2 * far)).to(BF16)
    check_attend(ops, c, ones(1, 4, d, BF16), int32(0), int32(900))


@pytest.mark.parametrize("dtype,ratio", [(t, p) for t in (BF16, FP16) for p in (6, 7, 12, 26, 60)] + [(BF16, 100)])
def test_attend_small_step_beside_large_ones(ops, ratio, dtype):
    """A row's result is as exact beside entries of far larger steps as without them: ones that it does
    not see, and ones whose scores are far below."""
    r = gen(ratio)
    # in one block of ranges, in two of one unit (either order), in two units
    for d, n, heavy, other in ((64, 40, 3, 1), (128, 700, 650, 600), (64, 70000, 700, 350), (64, 70000, 300, 800),
                               (128, 66000, 65998, 32000)):
        # one key far above the others (2^46 and more), whose values have small steps around 0
        c = noise_cache(ops, r, 1, 1, n, d, False)
        c.scales[0, 0, :, 0] = 0
        c.scales[0, 0, :, 1] = 0
        c.scales[0, 0, heavy, 1] = 1.0
        c.scales[0, 0, heavy, 2:] = (c.scales[0, 0, heavy, 2:].double() * 2.0 ** (-6 if dtype == FP16 else -30)).to(BF16)
        q = ones(2, 2, d, dtype) * 4
        before = c.scales[0, 0, other].clone()
        c.scales[0, 0, other, 2:] = (c.scales[0, 0, heavy, 2:].double() * 2.0 ** ratio).to(BF16)
        check_attend(ops, c, q, int32(0), int32(n))
        c.scales[0, 0, other] = before
        c.scales[0, 0, n - 1, 2:] = (c.scales[0, 0, heavy, 2:].double() * 2.0 ** ratio).to(BF16)   # the first row does not see it
        check_attend(ops, c, q, int32(0), int32(n))
    c.check()


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_attend_beside_rows_of_zeros(ops, dtype):
    """An entry with nearly all the weight whose value is 0: what the others add is all there is."""
    r = gen(77)
    for d, n in ((64, 33), (128, 600), (64, 70000)):
        for above in (10, 20, 28, 45):
            if dtype == FP16 and above > 10:
                continue                          # the result itself leaves fp16's range
            c = noise_cache(ops, r, 1, 2, n, d, True)
            c.scales[0, :, :, 0] = 0
            c.scales[0, :, :, 1] = 0
            c.scales[0, :, 2, 1] = above * math.log(2) / d ** 0.5 + math.log(n) / d ** 0.5
            c.scales[0, :, 2, 2:] = 0
            check_attend(ops, c, ones(1, 4, d, dtype), int32(0), int32(n))


@pytest.mark.parametrize("g,t", [(8, 1), (2, 9)])
@pytest.mark.parametrize("d", [64, 128])
def test_attend_ranges_of_any_exponent(ops, d, g, t):
    """Every entry's values of a size of their own, from 2^-80 to 2^80, and scores up to 2^60 apart."""
    r = gen(d + g)
    for n in (20, 500, 1300, 70000):
        c = noise_cache(ops, r, 1, 1, n, d, True)
        power = torch.randint(-80, 81, (n, 1), generator=r, device=DEV).double()
        c.scales[0, 0, :, 2:] = (c.scales[0, 0, :, 2:].double() * 2.0 ** power).to(BF16)
        c.scales[0, 0, torch.rand(n, generator=r, device=DEV) < 0.1, 2] = 0
        for q in (0.3, 4.0):
            check_attend(ops, c, (q * randn(r, 1, t, g, d)).to(BF16), int32(0), int32(n))
        # and as large as it goes where the weights are small
        order = c.scales[0, 0, :, 2].double().argsort(descending=True)
        ramp = rising_cache(ops, r, n, 1, d, 60.0)
        ramp.scales[0, 0, :, 2:] = c.scales[0, 0, order, 2:]
        check_attend(ops, ramp, ones(t, g, d, BF16), int32(0), int32(n))
        ramp.scales[0, 0, :, 2:] = c.scales[0, 0, order.flip(0), 2:]
        check_attend(ops, ramp, ones(t, g, d, BF16), int32(0), int32(n))
    c.check()


# ---- types, strides and scales that the tests above leave out --------------------------------------


@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("out_dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_linear_i8_from_floats_of_every_type(ops, dtype, out_dtype, with_bias):
    """Quantising in the call, by one kernel (at most 16 short rows) and by two, for every pair of types, from
    rows of a wider tensor, with rows of zeros and rows that are not finite."""
    for m, n, k in ((1, 512, 384), (5, 70, 33), (16, 200, 2048), (9, 130, 1500), (50, 300, 640), (17, 33, 1000)):
        g = gen(m + n)
        x = (3 * randn(g, m, k + 11)).to(dtype)[:, 3:k + 3]
        w, bias = rand_codes(ops, g, n, k), randn(g, n) if with_bias else None
        fine = torch.ones(m, dtype=torch.bool, device=DEV)
        if m >= 5:
            x[1] = 0
            x[2, k // 2] = float("nan")
            x[3, k - 1] = float("inf")
            x[4, 0] = -float("inf")
            fine[2:5] = False
        y = ops.linear_i8(x, w, bias=bias, out_dtype=out_dtype)
        q = ops.quantize_rows(x)
        two = ops.linear_i8(q, w, bias=bias, out_dtype=out_dtype)
        assert y.dtype == out_dtype and torch.equal(y[fine], two[fine])
        assert torch.isnan(y[~fine]).all() and torch.isnan(two[~fine]).all()
        check_linear(y[fine], ops.quantize_rows(x[fine]), w, bias)
        if m >= 5:
            assert torch.equal(y[1], (torch.zeros(n, device=DEV) if bias is None else bias).to(out_dtype))


@pytest.mark.parametrize("g,t", [(4, 1), (2, 3)])
def test_attend_scale_of_zero(ops, g, t):
    """The plain mean of what a row sees."""
    r = gen(g + 70)
    c = noise_cache(ops, r, 4, 2, 900, 64, True)
    check_attend(ops, c, randn(r, 3, t, 2 * g, 64).to(BF16), int32(2, 0, 3), int32(900, 1, 77), scale=0.0)
    c.check()


def test_attend_one_query_for_all(ops):
    """Expanded queries (strides of 0) and a bound of the lengths above the capacity."""
    r = gen(71)
    c = noise_cache(ops, r, 3, 2, 700, 128, False)
    q = randn(r, 1, 1, 1, 128).to(FP16).expand(3, 4, 6, 128)
    y = check_attend(ops, c, q, int32(0, 1, 2), int32(700, 5, 300), max_len=100000)
    assert torch.equal(y, c.attend(q.contiguous(), int32(0, 1, 2), int32(700, 5, 300)))
    c.check()


def test_two_caches_on_two_streams_at_once(ops):
    r = gen(72)
    caches = [noise_cache(ops, r, 40, 2, 2100, 64, True) for _ in range(2)]
    first = [c.weights.clone() for c in caches]
    q = randn(r, 40, 1, 8, 64).to(BF16)
    slots = torch.randperm(40, generator=r, device=DEV).int()
    lengths = torch.randint(0, 2101, (40,), generator=r, device=DEV, dtype=torch.int32)
    want = [[c.attend(q, slots, lengths) for _ in range(6)] for c in caches]
    grown = [c.weights.clone() for c in caches]
    for c, w in zip(caches, first):
        c.weights.copy_(w)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in caches], [[], []]
    for _ in range(6):
        for i, c in enumerate(caches):
            with torch.cuda.stream(streams[i]):
                got[i].append(c.attend(q, slots, lengths))
    torch.cuda.synchronize()
    for i, c in enumerate(caches):
        assert all(torch.equal(a, b) for a, b in zip(got[i], want[i])) and torch.equal(c.weights, grown[i])
        c.check()


@pytest.mark.parametrize("m,n,k", [(1, 128000, 384), (8, 20000, 2048), (2, 5000, 11264), (16, 40000, 1000)])
def test_linear_i8_few_rows_on_many_channels(ops, m, n, k):
    """One kernel or two, with a workspace or without: the same bits."""
    g = gen(n)
    x, w, bias = randn(g, m, k).to(BF16), rand_codes(ops, g, n, k), randn(g, n)
    y = ops.linear_i8(x, w, bias=bias)
    q = ops.quantize_rows(x)
    assert torch.equal(y, ops.linear_i8(q, w, bias=bias))
    check_linear(y, q, w, bias)
    L, none = ops.lib(), torch.empty_like(y)
    assert L.czg_linear_i8_dynamic_workspace(m, n, k) > 0 and L.czg_linear_i8_workspace(m, k) == 0
    st = L.czg_linear_i8_dynamic(x.data_ptr(), 1, k, w.codes.data_ptr(), w.ld, w.scales.data_ptr(), bias.data_ptr(), m, n, k,
                                 none.data_ptr(), 1, n, None, 0, torch.cuda.current_stream().cuda_stream)
    assert st == 0 and torch.equal(none, y)
