"""8-bit block-scaled operators (gfx950) against plain implementations in 64 bits.

Tolerances, from the roundings that each operator makes:
  * a quantized value is off by half a step at most: 2^-4 of it, or 2^-10 scales below e4m3's normals;
  * the norm's float32 chain: at most 54 additions of squares (halved by the root), the mean, eps, root,
    inverse and two products: under 64 roundings of 2^-24, 2^-18 relative;
  * the 8-bit matrix instruction sums eight neighbouring products in fixed point, whose last place is
    2^-13 of the largest one's power of two; what lies below is cut off (the test of its sums pins
    this). The largest is exact (it has 6 bits after the first), so a group loses less than 7 * 2^-13
    of its largest product. The rest is a float32 sum of at most K terms in any order, truncated or
    rounded: 2 K 2^-24 of the sum of magnitudes. Then half a step of the output's type.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
NORM_TOL = 2.0 ** -18
TYPES = [torch.bfloat16, torch.float16, torch.float32]
OUT = [torch.bfloat16, torch.float16]
E8M0, E4M3 = torch.float8_e8m0fnu, torch.float8_e4m3fn


def _ops():
    from yoda_scheduler_amd.ops import fp8
    return fp8


def _randn(shape, seed, dtype=torch.float32, spread=0.7):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * torch.exp(torch.randn(shape[-1], generator=g) * spread)
    return x.to(dtype)


def _pow2_scale(amax):
    """The least 2^p >= amax / 448, p from -126 on, in float64."""
    r = amax.double() / 448
    f, e = torch.frexp(r)
    p = torch.where(f == 0.5, e - 1, e).clamp_min(-126)
    return ((p.long() + 1023) << 52).view(torch.float64)


def _tiles(x, block_rows):
    """float x [R, K] -> [row blocks, block_rows, K blocks, 128], padded with zeros."""
    r, k = x.shape
    rb, kb = -(-r // block_rows), -(-k // 128)
    p = torch.zeros(rb * block_rows, kb * 128, dtype=x.dtype)
    p[:r, :k] = x
    return p.view(rb, block_rows, kb, 128)


def _quantized(x, pow2, block_rows):
    """The definition, each step in float32 as it is written: amax / 448, 1 / s, v * (1 / s), to nearest even."""
    t = _tiles(x.float(), block_rows)
    fin = torch.where(t.isfinite(), t, torch.zeros_like(t)).abs().amax(dim=(1, 3))
    s = _pow2_scale(fin).float() if pow2 else (fin / 448).clamp_min(2.0 ** -126)
    s = torch.where(fin > 0, s, torch.ones_like(s))
    v = t * (1.0 / s)[:, None, :, None]
    v = torch.where(t.isfinite(), v, torch.full_like(v, float("nan")))
    q = v.to(E4M3).view(t.shape[0] * block_rows, -1)[:x.shape[0]]
    return q, s


def _dequantized(m):
    """A block matrix's values in float64, on the CPU, unpadded."""
    r, k = m.shape
    s = m.scales.cpu().float().double().repeat_interleave(m.block_rows, 0)[:r].repeat_interleave(128, 1)[:, :k]
    return m.values.cpu().float().double() * s


def _same(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0), b.nan_to_num(0))


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 127), (5, 129), (17, 72), (130, 257), (257, 1000),
                                       (9, 4096), (2, 5001)])
def test_quantize_is_the_definition_bit_by_bit(require_gpu, rows, cols, dtype, pow2, block_rows):
    x = _randn((rows, cols), rows * 7 + cols, dtype)
    m = _ops().quantize(x.to(DEV), block_rows, E8M0 if pow2 else torch.float32)
    q, s = _quantized(x, pow2, block_rows)
    assert m.data.dtype == E4M3 and m.scales.dtype == (E8M0 if pow2 else torch.float32)
    assert torch.equal(m.scales.cpu().float(), s)
    assert torch.equal(m.data.cpu().float(), q.float())            # the padding's zeros too


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("pow2", [False, True])
def test_quantize_edges(require_gpu, pow2, block_rows):
    """Blocks of zeros, of subnormals, of the largest values, of NaN and infinities beside numbers."""
    x = torch.zeros(256, 640)
    x[:, 128:256] = _randn((256, 128), 3) * 2.0 ** -140
    x[:, 256:384] = _randn((256, 128), 4).clamp(-4, 4) * 2.0 ** 125
    x[:, 384:512] = _randn((256, 128), 5)
    x[3, 400], x[4, 401], x[200, 402] = float("nan"), float("inf"), -float("inf")
    x[5, 384:512] = float("nan")
    x[:, 512:] = 448.0 * 2.0 ** -3                                  # exactly at a power's border
    m = _ops().quantize(x.to(DEV), block_rows, E8M0 if pow2 else torch.float32)
    q, s = _quantized(x, pow2, block_rows)
    assert torch.equal(m.scales.cpu().float(), s)
    assert _same(m.data.cpu().float(), q.float())


def test_quantize_strides_and_no_rows(require_gpu):
    fp8 = _ops()
    wide = _randn((40, 700), 11, torch.bfloat16).to(DEV)
    for view in (wide[:, 3:260], wide[::3, 1:130], wide[5:6].expand(9, 700), wide[::2][:, 256:512]):
        for br in (1, 128):
            got, want = fp8.quantize(view, br), fp8.quantize(view.contiguous(), br)
            assert torch.equal(got.data.float(), want.data.float()) and torch.equal(got.scales, want.scales)
    for br in (1, 128):
        m = fp8.quantize(wide[:0], br)
        assert m.shape == (0, 700) and m.scales.shape == (0, 6)
    with pytest.raises(ValueError):
        fp8.quantize(wide[:, :0])


def _check_norm(q, h, x, w, res, eps, pow2):
    hh = x.float()
    if res is not None:
        hh = (x.float() + res.float()).to(x.dtype)
        assert torch.equal(h.cpu(), hh)
    else:
        assert h is None
    f = hh.double()
    y = f / torch.sqrt(f.square().mean(1, keepdim=True) + eps) * w.double()
    amax = _tiles(y, 1).abs().amax(dim=(1, 3))
    s = q.scales.cpu().float().double()
    if pow2:
        low, high = _pow2_scale(amax * (1 - NORM_TOL)), _pow2_scale(amax * (1 + NORM_TOL))
        low, high = (torch.where(amax > 0, v, torch.ones_like(v)) for v in (low, high))
        assert ((s == low) | (s == high)).all()
    else:
        want = torch.where(amax > 0, (amax / 448).clamp_min(2.0 ** -126), torch.ones_like(amax))
        assert ((s - want).abs() <= want * (NORM_TOL + 2.0 ** -24)).all()
    each = s.repeat_interleave(128, 1)[:, :y.shape[1]]
    room = torch.maximum(y.abs() * 2.0 ** -4, each * 2.0 ** -10) + y.abs() * 2 * NORM_TOL
    assert ((_dequantized(q) - y).abs() <= room).all()
    assert not q.data.cpu().float()[:, q.cols:].any()


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,residual", [(1, 1, True), (1, 4096, True), (7, 127, False), (9, 129, True),
                                                (33, 513, False), (5, 2049, True), (3, 5001, True), (2, 8193, False),
                                                (2, 16400, True), (2, 32769, True), (1, 40000, False)])
def test_norm(require_gpu, rows, cols, residual, dtype, pow2):
    x = _randn((rows, cols), rows + cols, dtype)
    r = _randn((rows, cols), rows + cols + 1, dtype) if residual else None
    for wtype in {dtype, torch.float32}:
        w = (1 + 0.1 * _randn((cols,), cols, spread=0)).to(wtype)
        q, h = _ops().add_rms_norm(x.to(DEV), w.to(DEV), None if r is None else r.to(DEV), 1e-5,
                                   E8M0 if pow2 else torch.float32)
        _check_norm(q, h, x, w, r, 1e-5, pow2)


@pytest.mark.parametrize("rows", [1024, 1025])
@pytest.mark.parametrize("cols", [1500, 2500, 5001, 9000])
def test_norm_of_few_and_of_many_rows(require_gpu, rows, cols):
    """Few rows take more lanes each."""
    x, w, res = _randn((rows, cols), cols, torch.bfloat16), _randn((cols,), 3, torch.bfloat16), _randn((rows, cols), 4, torch.bfloat16)
    q, h = _ops().add_rms_norm(x.to(DEV), w.to(DEV), res.to(DEV))
    _check_norm(q, h, x, w, res, 1e-6, False)


def test_norm_strides_zero_rows_and_nan(require_gpu):
    fp8 = _ops()
    wide, other = _randn((30, 700), 1, torch.bfloat16), _randn((30, 900), 2, torch.bfloat16)
    x, r = wide[::3, 5:405], other[10:20, 100:500]
    xd, rd = wide.to(DEV)[::3, 5:405], other.to(DEV)[10:20, 100:500]
    w = torch.ones(400, dtype=torch.bfloat16)
    q, h = fp8.add_rms_norm(xd, w.to(DEV), rd, 1e-6)
    _check_norm(q, h, x, w, r, 1e-6, False)
    q, h = fp8.add_rms_norm(xd[:0], w.to(DEV), rd[:0])
    assert q.shape == (0, 400) and h.shape == (0, 400)
    # a row of zeros (eps alone), a row that holds NaN, and its neighbours
    z = _randn((4, 300), 9)
    z[1] = 0
    z[2, 7] = float("nan")
    one = torch.ones(300)
    q, _ = fp8.add_rms_norm(z.to(DEV), one.to(DEV))
    got = _dequantized(q)
    assert not got[1].any() and got[2].isnan().all()
    want, _ = fp8.add_rms_norm(z[[0, 3]].to(DEV), one.to(DEV))
    assert torch.equal(got[[0, 3]], _dequantized(want))


def _matmul_inputs(m, n, k, pow2, seed=0):
    fp8 = _ops()
    sd = E8M0 if pow2 else torch.float32
    a = fp8.quantize(_randn((m, k), seed + 1).to(DEV), 1, sd)
    b = fp8.quantize((_randn((n, k), seed + 2, spread=0) / k ** 0.5).to(DEV), 128, sd)
    return a, b


def _check_matmul(out, a, b, bias=None):
    da, db = _dequantized(a), _dequantized(b)
    want = da @ db.t()
    mass = da.abs() @ db.abs().t()
    if bias is not None:
        want, mass = want + bias.double(), mass + bias.double().abs()
    largest = torch.zeros(a.rows, b.rows, device=DEV)                # of each group of eight, summed
    xa, xb = (torch.nn.functional.pad(d.abs(), (0, -d.shape[1] % 8)).float().to(DEV) for d in (da, db))
    for k in range(0, xa.shape[1], 8):
        largest += (xa[:, None, k:k + 8] * xb[None, :, k:k + 8]).amax(2)
    room = 7 * 2.0 ** -13 * largest.cpu().double() * (1 + 2.0 ** -12) + 2 * (a.cols + 2) * 2.0 ** -24 * mass
    room = room + (want.abs() + room) * torch.finfo(out.dtype).eps / 2
    if out.dtype == torch.float16:
        room = room + 2.0 ** -25                                     # its subnormals' half step
    off = (out.cpu().double() - want).abs()
    assert (off <= room).all(), (off - room).max()


SIZES = [(1, 1, 1), (1, 16, 128), (1, 4096, 1000), (2, 130, 129), (5, 200, 2500), (15, 48, 256), (16, 16, 4096),
         (17, 300, 640), (31, 1000, 384), (33, 128, 128), (64, 256, 512), (65, 257, 1025), (100, 96, 3000),
         (128, 128, 128), (129, 640, 300), (255, 513, 200), (256, 256, 1024), (257, 511, 700), (300, 1100, 1500),
         (600, 777, 256)]


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_matmul(require_gpu, m, n, k, pow2):
    a, b = _matmul_inputs(m, n, k, pow2)
    for t in OUT:
        _check_matmul(_ops().matmul(a, b, t), a, b)
    bias = _randn((n,), 5, torch.float16)
    _check_matmul(_ops().matmul(a, b, torch.float16, bias.to(DEV)), a, b, bias)


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 300, 5000), (7, 33, 260), (48, 500, 1300), (200, 300, 700), (300, 600, 1000),
                                   (513, 1025, 384)])
def test_matmul_of_whole_numbers_is_exact(require_gpu, m, n, k, pow2):
    """Small whole numbers times powers of two sum without a rounding, whatever the order (products up to 2^4 in
    steps of 1 fit the instruction's 13 places): a value or a scale from the wrong place cannot hide in a tolerance."""
    fp8 = _ops()
    g = torch.Generator().manual_seed(m + n + k)
    kb = fp8.blocks(k)
    qa = torch.randint(-4, 5, (m, k), generator=g).float()
    qb = torch.randint(-4, 5, (n, k), generator=g).float()
    sa = 2.0 ** torch.randint(-3, 4, (m, kb), generator=g).float()
    sb = 2.0 ** torch.randint(-3, 4, (fp8.blocks(n), kb), generator=g).float()
    sd = E8M0 if pow2 else torch.float32
    a = fp8.BlockMatrix(qa.to(E4M3).to(DEV), sa.to(sd).to(DEV))
    b = fp8.BlockMatrix(qb.to(E4M3).to(DEV), sb.to(sd).to(DEV), block_rows=128)
    da = qa.double() * sa.double().repeat_interleave(128, 1)[:, :k]
    db = qb.double() * sb.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    bias = torch.randint(-8, 9, (n,), generator=g).float()
    want = da @ db.t() + bias.double()
    assert want.abs().max() < 65504 and (want * 64 == (want * 64).round()).all() and (want.abs() * 64).max() < 2 ** 24
    for t in OUT:
        got = fp8.matmul(a, b, t, bias.to(t).to(DEV))
        assert torch.equal(got.cpu(), want.float().to(t))           # exact in float32, then rounded once


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("k", [100, 250, 380, 1300, 1500])
def test_matmul_large(require_gpu, k, pow2):
    """Sizes that take the large tiles, at the edges of rows, columns and K; the reference in float64 on the GPU."""
    fp8 = _ops()
    m, n = 3900, 4001
    sd = E8M0 if pow2 else torch.float32
    a = fp8.quantize(_randn((m, k), k).to(DEV), 1, sd)
    b = fp8.quantize((_randn((n, k), k + 1, spread=0) / k ** 0.5).to(DEV), 128, sd)
    bias = _randn((n,), 7, torch.bfloat16)
    da, db = (_dequantized(x).to(DEV) for x in (a, b))
    want = torch.mm(da, db.t().contiguous()) + bias.to(DEV).double()
    mass = torch.mm(da.abs(), db.abs().t().contiguous()) + bias.to(DEV).double().abs()
    largest = torch.zeros(m, n, device=DEV)
    xa, xb = (torch.nn.functional.pad(d.abs(), (0, -k % 8)).float() for d in (da, db))
    for i in range(0, xa.shape[1], 8):
        largest += (xa[:, None, i:i + 8] * xb[None, :, i:i + 8]).amax(2)
    room = 7 * 2.0 ** -13 * largest.double() * (1 + 2.0 ** -12) + 2 * (k + 2) * 2.0 ** -24 * mass
    room = room + (want.abs() + room) * 2.0 ** -8
    out = fp8.matmul(a, b, torch.bfloat16, bias.to(DEV))
    assert ((out.double() - want).abs() <= room).all()


@pytest.mark.parametrize("m,n,k,pow2", [(3000, 4001, 8500, False), (2900, 3900, 33_000, True), (2900, 3900, 16_700, False),
                                        (200, 2000, 9000, False), (40, 3000, 40_000, True), (3900, 4001, 3 * 128, True),
                                        # every shape of tile, whole and in parts of K
                                        (3, 17_000, 700, True), (20, 100, 20_000, True), (20, 100, 20_000, False),
                                        (31, 9000, 1500, False), (64, 512, 16_384, True), (64, 512, 16_384, False),
                                        (50, 9000, 900, True), (100, 200, 12_000, True), (100, 200, 12_000, False),
                                        (128, 9000, 640, False), (130, 130, 9000, True), (500, 900, 5000, False),
                                        (512, 8192, 1000, True), (777, 5000, 500, False), (1024, 2000, 700, True),
                                        # whole rounds of large tiles, the columns behind them in smaller ones
                                        (2300, 7700, 2000, True), (2300, 7700, 2000, False), (4096, 4100, 900, False),
                                        (4608, 4096, 1400, True), (256, 65_800, 600, True)])
def test_matmul_of_whole_numbers_is_exact_over_long_sums(require_gpu, m, n, k, pow2):
    """Scales are held for 64 or 256 steps at a time: sums longer than that, exact as above."""
    fp8 = _ops()
    g = torch.Generator(device=DEV).manual_seed(k)
    kb = fp8.blocks(k)

    def whole(low, high, *shape):
        return torch.randint(low, high + 1, shape, generator=g, device=DEV)

    qa, qb = whole(-1, 1, m, k).float(), whole(-1, 1, n, k).float()
    sa, sb = 2.0 ** whole(-1, 1, m, kb).float(), 2.0 ** whole(-1, 1, fp8.blocks(n), kb).float()
    sd = E8M0 if pow2 else torch.float32
    a = fp8.BlockMatrix(qa.to(E4M3), sa.to(sd))
    b = fp8.BlockMatrix(qb.to(E4M3), sb.to(sd), block_rows=128)
    da = qa.double() * sa.double().repeat_interleave(128, 1)[:, :k]
    db = qb.double() * sb.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    want = torch.mm(da, db.t().contiguous())
    assert want.abs().max() * 4 < 2 ** 24 and (want * 4 == (want * 4).round()).all()
    got = fp8.matmul(a, b, torch.bfloat16)
    assert torch.equal(got, want.float().to(torch.bfloat16))


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("m,n,first", [(2300, 7700, 7168), (4090, 4101, 4096)])
def test_the_columns_behind_whole_rounds(require_gpu, m, n, first, pow2):
    """Two kernels share a product: each column as in a product of its part alone, into a wider buffer, with a bias."""
    fp8 = _ops()
    k = 900
    a, b = _matmul_inputs(m, n, k, pow2)
    bias = _randn((n,), 9, torch.float16).to(DEV)
    buf = torch.full((m + 2, n + 5), 7.0, dtype=torch.float16, device=DEV)
    out = fp8.matmul(a, b, torch.float16, bias, buf[1:m + 1, 3:n + 3])
    for part in (slice(0, first), slice(first, n)):
        blocks = slice(part.start // 128, -(-part.stop // 128))
        piece = fp8.BlockMatrix(b.data[part], b.scales[blocks], cols=k, block_rows=128)
        assert torch.equal(out[:, part], fp8.matmul(a, piece, torch.float16, bias[part]))
    assert (buf[0] == 7).all() and (buf[-1] == 7).all() and (buf[:, :3] == 7).all() and (buf[:, n + 3:] == 7).all()


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("m,n", [(3, 70), (40, 200), (130, 520), (300, 300)])
def test_matmul_writes_its_rows_alone(require_gpu, m, n, pow2):
    """A wider, longer buffer: what lies beside and behind the output stays."""
    a, b = _matmul_inputs(m, n, 500, pow2)
    for t in OUT:
        buf = torch.full((m + 5, n + 9), 7.0, dtype=t, device=DEV)
        out = buf[1:m + 1, 3:n + 3]
        assert _ops().matmul(a, b, t, out=out) is out
        assert torch.equal(out, _ops().matmul(a, b, t))
        buf[1:m + 1, 3:n + 3] = 7.0
        assert (buf == 7.0).all()


def test_the_sums_of_the_matrix_instruction(require_gpu):
    """What the tolerance rests on: beside a product of 2^16, one of 2^3 (2^-13 of it) counts and one of
    6 is lost if it is among the same eight, and counts otherwise. Seen in differences of two outputs."""
    fp8 = _ops()
    w = fp8.BlockMatrix(torch.cat([torch.full((1, 128), 256.0), torch.zeros(1, 128)]).to(E4M3).to(DEV),
                        torch.ones(1, 1, device=DEV), block_rows=128)

    def out(values):
        """sum of 256 * values, as what is left after 256 * 256 is taken off in the other groups"""
        v = torch.zeros(1, 128)
        for k, x in values.items():
            v[0, k] = x
        return fp8.matmul(fp8.BlockMatrix(v.to(E4M3).to(DEV), torch.ones(1, 1, device=DEV)), w, torch.float16)[0, 0].item()

    # 256 * 256 at k = 0 in a group, -(256 * 256) in another, and a small one beside the first or apart
    for other in (8, 64, 127):
        assert out({0: 256, other: -256}) == 0
        for near in (1, 7):
            assert out({0: 256, near: 0.03125, other: -256}) == 8.0
            assert out({0: 256, near: 0.0234375, other: -256}) == 0.0
        far = 16 if other != 16 else 24
        assert out({0: 256, far: 0.0234375, other: -256}) == 6.0


def test_matmul_nan_stays_in_its_row_and_column(require_gpu):
    fp8 = _ops()
    for m, n in ((4, 300), (70, 300), (300, 300)):
        x, w = _randn((m, 400), 1), _randn((n, 400), 2)
        x[2, 130], w[200, 5] = float("nan"), float("inf")
        for sd in (torch.float32, E8M0):
            out = fp8.matmul(fp8.quantize(x.to(DEV), 1, sd), fp8.quantize(w.to(DEV), 128, sd)).cpu()
            bad = torch.zeros(m, n, dtype=torch.bool)
            bad[2], bad[:, 200] = True, True
            assert torch.equal(out.isnan(), bad)


def test_matmul_nothing_to_do(require_gpu):
    fp8 = _ops()
    a, b = _matmul_inputs(4, 200, 300, False)
    none = fp8.quantize(torch.zeros(0, 300, device=DEV))
    assert fp8.matmul(none, b).shape == (0, 200)
    assert fp8.matmul(a, fp8.quantize(torch.zeros(0, 300, device=DEV), 128)).shape == (4, 0)


def test_refusals_on_a_gpu(require_gpu):
    fp8 = _ops()
    a, b = _matmul_inputs(4, 200, 300, False)
    x = torch.zeros(4, 300, device=DEV)
    with pytest.raises(TypeError):
        fp8.matmul(a, b, torch.float32)
    with pytest.raises(TypeError):
        fp8.matmul(a, b, torch.bfloat16, torch.zeros(200, device=DEV, dtype=torch.float16))
    with pytest.raises(ValueError):
        fp8.matmul(a, b, torch.float16, torch.zeros(201, device=DEV, dtype=torch.float16))
    with pytest.raises(ValueError):
        fp8.matmul(a, b, out=torch.zeros(4, 201, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        fp8.matmul(a, b, out=torch.zeros(200, 4, device=DEV, dtype=torch.bfloat16).t())
    with pytest.raises(ValueError):
        fp8.matmul(a, b, out=torch.zeros(1, 200, device=DEV, dtype=torch.bfloat16).expand(4, 200))
    with pytest.raises(TypeError):
        fp8.quantize(x, scale_dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        fp8.quantize(x, block_rows=2)
    with pytest.raises(ValueError):
        fp8.add_rms_norm(x, torch.ones(299, device=DEV))
    with pytest.raises(TypeError):
        fp8.add_rms_norm(x, torch.ones(300, device=DEV, dtype=torch.float16))
    with pytest.raises(ValueError):
        fp8.add_rms_norm(x, torch.ones(300, device=DEV), x[:2])
    with pytest.raises(TypeError):
        fp8.add_rms_norm(x, torch.ones(300, device=DEV), x.half())
    with pytest.raises(ValueError):
        fp8.add_rms_norm(x, torch.ones(300))
    with pytest.raises(RuntimeError):
        fp8.add_rms_norm(x, torch.ones(300, device=DEV, requires_grad=True))


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("rows", [1, 40, 300])
def test_a_layer_together(require_gpu, rows, pow2):
    """Residual + norm, the product with a quantized weight, its output quantized for the next product."""
    fp8 = _ops()
    sd = E8M0 if pow2 else torch.float32
    k, n, k2 = 700, 900, 300
    x, r = _randn((rows, k), 1, torch.bfloat16), _randn((rows, k), 2, torch.bfloat16)
    g = (1 + 0.1 * _randn((k,), 3, spread=0)).bfloat16()
    up = fp8.quantize((_randn((n, k), 4, spread=0) / k ** 0.5).to(DEV), 128, sd)
    down = fp8.quantize((_randn((k2, n), 5, spread=0) / n ** 0.5).to(DEV), 128, sd)
    q, h = fp8.add_rms_norm(x.to(DEV), g.to(DEV), r.to(DEV), 1e-6, sd)
    u = fp8.matmul(q, up)
    q2 = fp8.quantize(u, 1, sd)
    out = fp8.matmul(q2, down, torch.float16)
    _check_norm(q, h, x, g, r, 1e-6, pow2)
    _check_matmul(u, q, up)
    want, s = _quantized(u.cpu(), pow2, 1)
    assert torch.equal(q2.data.cpu().float(), want.float()) and torch.equal(q2.scales.cpu().float(), s)
    _check_matmul(out, q2, down)


@pytest.mark.parametrize("rows", [1, 20, 70, 260])
def test_captured_and_replayed(require_gpu, rows):
    """A layer in a graph: every replay, with eager work in between, gives what an eager call gives."""
    fp8 = _ops()
    k, n = 640, 1100
    w = fp8.quantize((_randn((n, k), 4, spread=0) / k ** 0.5).to(DEV), 128)
    g = torch.ones(k, device=DEV, dtype=torch.bfloat16)
    x, r = (torch.zeros(rows, k, device=DEV, dtype=torch.bfloat16) for _ in range(2))

    def layer():
        q, h = fp8.add_rms_norm(x, g, r)
        return fp8.matmul(q, w), h

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer()
    torch.cuda.current_stream().wait_stream(side)
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, h = layer()
    with torch.cuda.graph(second):
        out2, _ = layer()
    for i in range(4):
        x.copy_(_randn((rows, k), 10 + i, torch.bfloat16))
        r.copy_(_randn((rows, k), 20 + i, torch.bfloat16))
        graph.replay()
        second.replay()
        want, wh = layer()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(out2, want) and torch.equal(h, wh)


def test_two_streams_at_once(require_gpu):
    fp8 = _ops()
    pairs = [_matmul_inputs(m, 2000, 3000, pow2, seed=m) for m, pow2 in ((8, False), (8, True), (150, False), (260, True))]
    want = [fp8.matmul(a, b) for a, b in pairs]
    streams = [torch.cuda.Stream() for _ in pairs]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for st, (a, b) in zip(streams, pairs):
            with torch.cuda.stream(st):
                got.append([fp8.matmul(a, b) for _ in range(4)])
        torch.cuda.synchronize()
        for w, gs in zip(want, got):
            assert all(torch.equal(w, x) for x in gs)


@pytest.mark.parametrize("m", [3, 130])
def test_offsets_past_32_bits(require_gpu, m):
    """A weight of 4.4 GB: rows on both sides of the 2^32th byte."""
    fp8 = _ops()
    n, k = 270_000, 16_384
    w = torch.zeros(n, k, dtype=torch.uint8, device=DEV)
    some = torch.tensor([0, 1, 131_071, 131_072, 262_143, 262_144, 262_145, 269_999])
    codes = _randn((len(some), k), 1, spread=0).to(E4M3)
    w[some.to(DEV)] = codes.view(torch.uint8).to(DEV)
    b = fp8.BlockMatrix(w.view(E4M3), torch.ones(fp8.blocks(n), k // 128, device=DEV), block_rows=128)
    a = fp8.quantize(_randn((m, k), 2).to(DEV))
    out = fp8.matmul(a, b, torch.float16)
    small = fp8.BlockMatrix(codes.to(DEV), torch.ones(1, k // 128, device=DEV), block_rows=128)
    _check_matmul(out[:, some.to(DEV)], a, small)
    out[:, some.to(DEV)] = 0
    assert not out.any()


@pytest.mark.parametrize("pow2", [False, True])
def test_norm_of_small_and_large_rows(require_gpu, pow2):
    """Squares that float32 does not hold, an eps that it does not hold, and a root that nothing holds."""
    fp8 = _ops()
    x = _randn((6, 640), 77).double()
    x[0] *= 2.0 ** -90
    x[1] *= 2.0 ** 100
    x[2] *= 2.0 ** -64
    x[4:] = 0
    x, w = x.float(), torch.ones(640)
    sd = E8M0 if pow2 else torch.float32
    q, h = fp8.add_rms_norm(x[:4].to(DEV), w.to(DEV), None, 0.0, sd)
    _check_norm(q, h, x[:4], w, None, 0.0, pow2)
    q, h = fp8.add_rms_norm(x[:5].to(DEV), w.to(DEV), None, 1e-60, sd)
    _check_norm(q, h, x[:5], w, None, 1e-60, pow2)
    q, _ = fp8.add_rms_norm(x[4:].to(DEV), w.to(DEV), None, 0.0, sd)
    assert q.values.float().isnan().all() and (q.scales.float() == 1).all()


@pytest.mark.parametrize("pow2", [False, True])
def test_more_rows_than_a_launch_takes(require_gpu, pow2):
    fp8 = _ops()
    sd = E8M0 if pow2 else torch.float32
    rows, cut = (1 << 21) + 13, (1 << 21) - 5
    g = torch.Generator(DEV).manual_seed(5)
    x, r = (torch.randn(rows, 40, generator=g, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    w = torch.randn(40, generator=g, device=DEV, dtype=torch.bfloat16)
    for all_, end, start in ((fp8.quantize(x, 1, sd), fp8.quantize(x[cut:], 1, sd), fp8.quantize(x[:40], 1, sd)),
                             tuple(fp8.add_rms_norm(a, w, b, 1e-6, sd)[0]
                                   for a, b in ((x, r), (x[cut:], r[cut:]), (x[:40], r[:40])))):
        for part, piece in ((slice(cut, None), end), (slice(0, 40), start)):
            assert torch.equal(all_.data[part].view(torch.uint8), piece.data.view(torch.uint8))
            assert torch.equal(all_.scales.float()[part], piece.scales.float())
    h = fp8.add_rms_norm(x, w, r)[1]
    assert torch.equal(h, (x.float() + r.float()).to(x.dtype))


@pytest.mark.parametrize("m", [2, 20])
def test_more_columns_than_a_launch_takes(require_gpu, m):
    """2^27 columns of 32 a workgroup: the choice goes to larger tiles."""
    fp8 = _ops()
    n = (1 << 27) + 70
    g = torch.Generator(DEV).manual_seed(6)
    values = torch.randint(0, 0x60, (n, 128), dtype=torch.uint8, device=DEV, generator=g).view(E4M3)
    scales = torch.rand(-(-n // 128), 1, device=DEV, generator=g)
    a = fp8.quantize(torch.randn(m, 128, device=DEV, generator=g))
    out = fp8.matmul(a, fp8.BlockMatrix(values, scales, block_rows=128))
    for first in (0, (1 << 26), n - 70 - 128):
        first = first // 128 * 128
        part = fp8.BlockMatrix(values[first:first + 198], scales[first // 128:first // 128 + -(-len(values[first:first + 198]) // 128)],
                               block_rows=128)
        want = _dequantized(a) @ _dequantized(part).T
        got = out[:, first:first + want.shape[1]].cpu().double()
        mass = _dequantized(a).abs() @ _dequantized(part).abs().T
        assert ((got - want).abs() <= mass * (7 * 2.0 ** -13 + 256 * 2.0 ** -24) + want.abs() * 2.0 ** -8).all()


def test_values_and_scales_are_views(require_gpu):
    fp8 = _ops()
    x = _randn((5, 200), 8).to(DEV)
    for m in (fp8.quantize(x), fp8.quantize(x, 128), fp8.quantize(x, 1, E8M0)):
        for view, whole, like in ((m.values, m.data, m.data[:5, :200]), (m.scales, m._room, m._room[:m.scales.shape[0], :2])):
            assert view.shape == like.shape and view.stride() == like.stride() and view.data_ptr() == whole.data_ptr()
            assert view.dtype == whole.dtype and not view.requires_grad
            assert torch.equal(view.float(), like.float())
    m = fp8.quantize(x)
    scales, before = m.scales, m._room._version
    m._room.mul_(2)                                            # what is written to the whole is seen in its views
    assert torch.equal(scales, m._room[:5]) and scales._version == m._room._version > before
    with torch.inference_mode():
        inner = fp8.quantize(x)
        assert torch.equal(inner.scales, fp8.quantize(x).scales) and inner.values.shape == (5, 200)
    learned = fp8.BlockMatrix(m.values, m.scales.clone().requires_grad_())
    (grad,) = torch.autograd.grad(learned.scales.sum(), learned._room)
    assert torch.equal(grad[:5], torch.ones_like(grad[:5])) and not grad[5:].any()


def test_out_counts_as_written(require_gpu):
    fp8 = _ops()
    a, b = fp8.quantize(torch.ones(4, 128, device=DEV)), fp8.quantize(torch.ones(8, 128, device=DEV), 128)
    out = torch.empty(4, 8, device=DEV, dtype=torch.bfloat16)
    before = out._version
    assert fp8.matmul(a, b, out=out) is out and out._version > before
    with torch.inference_mode():
        assert (fp8.matmul(a, b, out=torch.empty_like(out)) == 128).all()
    learned = fp8.BlockMatrix(b.values, b.scales.clone().requires_grad_(), block_rows=128)
    with pytest.raises(RuntimeError):
        fp8.matmul(a, learned)
    for x in (torch._neg_view(torch.ones(4, 128, device=DEV)), torch.ones(4, 128, device=DEV).to_sparse()):
        with pytest.raises(ValueError):
            fp8.quantize(x)


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("rows,cols,inner", [(1, 256, 128), (37, 512, 384), (300, 768, 1024), (1, 8192, 2048)])
def test_matrix_check_is_clean(require_gpu, rows, cols, inner, pow2):
    from yoda_scheduler_amd.ops import hip
    r = hip.matrix_check(0, rows, cols, inner, iters=3, pow2=pow2)
    assert r["errors"] == 0 and r["tflops"] > 0, r


def test_matrix_check_compares(require_gpu):
    """Checkers that go by another seed's inputs: nearly every value of the norm and the weight is off, and the
    checkers of a verifier that compares say so."""
    from yoda_scheduler_amd.ops import hip
    rows, cols, inner = 64, 512, 512
    bad = hip.matrix_check(0, rows, cols, inner, iters=1, seed=1, verify_seed=77)
    assert bad["errors"] > 0.8 * (rows + cols) * inner, bad
    with pytest.raises(ValueError):
        hip.matrix_check(0, 16, 300, 512)


def test_matrix_check_rate(require_gpu):
    from yoda_scheduler_amd.ops import hip
    r = hip.matrix_check(0, iters=10)
    # 4096 x 4096 x 4096 reaches 2500 TFLOP/s (float32 vector code would stay under 160)
    assert r["errors"] == 0 and r["tflops"] > 1000, r
    assert hip.matrix_check_bytes() > 4096 * 4096 * 14


def test_prober_runs_the_matrix_check(require_gpu):
    from yoda_scheduler_amd.sniffer.publisher import HipProber
    wrong, rate = HipProber().matrix(0)
    assert wrong == 0 and rate > 1000


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("small", [1e-36, 1e-37, 2.0 ** -126, 2.0 ** -133])
def test_norm_of_a_tiny_block_in_a_normal_row(require_gpu, small, dtype, pow2):
    """root / s of such a block is beyond float32: its values stay finite, and zeros beside them zeros."""
    x = (0.02 * _randn((5, 384), 31, spread=0)).to(dtype)
    x[:, :128] = 0
    x[0, 3] = small
    x[1, :128] = small
    x[2, 0], x[2, 127] = -small, small / 4
    x[3, 256:] = 0                                                  # tiny beside nothing and something
    x[3, 5] = small
    for w in (torch.ones(384, dtype=dtype), (1 + 0.1 * _randn((384,), 32, spread=0)).to(dtype)):
        q, h = _ops().add_rms_norm(x.to(DEV), w.to(DEV), None, 1e-6, E8M0 if pow2 else torch.float32)
        assert not q.data.float().isnan().any()
        _check_norm(q, h, x, w, None, 1e-6, pow2)


@pytest.mark.parametrize("pow2", [False, True])
def test_norm_beyond_what_float32_holds_on_the_way(require_gpu, pow2):
    """Products h * weight, roots and scales out of float32's range, of values that float32 holds."""
    sd = E8M0 if pow2 else torch.float32
    base = _randn((6, 512), 33, spread=0)
    x, w = base.clone(), torch.ones(512)
    x[0] *= 2.0 ** 124                                              # h * w beyond 2^128 in the second block
    x[1] *= 2.0 ** -140                                             # a root beyond it
    x[2, 128:256] *= 2.0 ** -100                                    # h * w below 2^-149 in the third
    x[3] *= 2.0 ** 60
    x[4] = 0
    w[128:256], w[256:384], w[384:] = 2.0 ** 40, 2.0 ** -100, 2.0 ** -20
    for eps in (0.0, 1e-300):
        q, h = _ops().add_rms_norm(x[:4].to(DEV), w.to(DEV), None, eps, sd)
        _check_norm(q, h, x[:4], w, None, eps, pow2)
    q, h = _ops().add_rms_norm(x.to(DEV), w.to(DEV), None, 1e-6, sd)
    _check_norm(q, h, x, w, None, 1e-6, pow2)


@pytest.mark.parametrize("infinite", [float("inf"), -float("inf")])
@pytest.mark.parametrize("pow2", [False, True])
def test_norm_of_infinities(require_gpu, pow2, infinite):
    """An infinite weight leaves its column NaN and its block's scale to the others; an infinite value its row."""
    sd = E8M0 if pow2 else torch.float32
    x, w = _randn((4, 256), 34, spread=0), torch.ones(256)
    w[7] = infinite
    q, _ = _ops().add_rms_norm(x.to(DEV), w.to(DEV), None, 1e-6, sd)
    got, clean = _dequantized(q), w.clone()
    clean[7] = 0
    want, _ = _ops().add_rms_norm(x.to(DEV), clean.to(DEV), None, 1e-6, sd)
    assert got[:, 7].isnan().all()
    keep = [i for i in range(256) if i != 7]
    assert torch.equal(q.scales.float(), want.scales.float()) and torch.equal(got[:, keep], _dequantized(want)[:, keep])
    x[2, 200] = float("inf")
    q, _ = _ops().add_rms_norm(x.to(DEV), torch.ones(256, device=DEV), None, 1e-6, sd)
    assert _dequantized(q)[2, 200].isnan() and not _dequantized(q)[[0, 1, 3]].isnan().any()


def test_tangents_are_refused_on_a_gpu(require_gpu):
    from torch.autograd import forward_ad
    fp8 = _ops()
    x, w = torch.ones(4, 300, device=DEV), torch.ones(300, device=DEV)
    a, b = _matmul_inputs(4, 200, 300, False)
    out = torch.zeros(4, 200, device=DEV, dtype=torch.bfloat16)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: fp8.quantize(dual(x)), lambda: fp8.add_rms_norm(dual(x), w),
                     lambda: fp8.add_rms_norm(x, dual(w)), lambda: fp8.add_rms_norm(x, w, dual(x)),
                     lambda: fp8.matmul(a, b, bias=dual(torch.zeros(200, device=DEV, dtype=torch.bfloat16))),
                     lambda: fp8.matmul(a, b, out=dual(out)),
                     lambda: fp8.matmul(a, fp8.BlockMatrix(b.values, dual(b.scales), block_rows=128))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
        q = fp8.quantize(forward_ad.unpack_dual(dual(x)).primal)
        learned = fp8.BlockMatrix(q.values, dual(q.scales.clone()))
        assert forward_ad.unpack_dual(learned.scales).tangent is not None        # its views keep it
        with torch.inference_mode():
            fp8.quantize(dual(x))


@pytest.mark.parametrize("pow2", [False, True])
def test_each_checker_of_the_matrix_check_compares(require_gpu, pow2):
    """Checkers that go by another seed's layer find nearly every value of the norm, the weight and the product off,
    and nearly every pair of values changed in each repetition. Two independent results agree within a checker's
    bound (a few parts in 2^8 of a value) for a few values in a hundred."""
    from yoda_scheduler_amd.ops import hip
    rows, cols, inner, iters = 64, 512, 512, 3
    keys = ("norm_errors", "weight_errors", "product_errors", "unstable")
    good = hip.matrix_check(0, rows, cols, inner, iters, pow2, seed=1)
    assert [good[k] for k in keys] == [0] * 4 and good["errors"] == 0, good
    bad = hip.matrix_check(0, rows, cols, inner, iters, pow2, seed=1, verify_seed=77)
    for k, count in zip(keys, (rows * inner, cols * inner, rows * cols, rows * cols // 2 * iters)):
        # (each of the 256 threads of a block of the weight counts its scale once more)
        assert 0.8 * count < bad[k] <= count + cols // 128 * (inner // 128) * 256, (k, bad)
    assert bad["errors"] == sum(bad[k] for k in keys)


def test_float_scales_held_beyond_256_steps(require_gpu):
    """Large tiles with float scales take up the columns' scales of 256 steps at a time: exact whole numbers over more."""
    test_matmul_of_whole_numbers_is_exact_over_long_sums(None, 2900, 3900, 66_000, False)
