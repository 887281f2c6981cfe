"""The 8-bit operators against plain forms in 64 bits: the quantisers bit for bit, the norm and
SwiGLU that quantise, the product with a scale per block of 128."""
import pytest
import torch

pytestmark = pytest.mark.gpu

FLOOR = 2.0 ** -100
HALF_E4M3 = 2.0 ** -4            # half a step of an e4m3 value, relative to the value
HALF_SUB = 2.0 ** -10            # half a step among e4m3's subnormals, in units of the scale
HALF_BF16 = 2.0 ** -8


def bf(shape, seed, scale=1.0, spread=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * scale
    if spread:
        x = x * torch.exp(spread * torch.randn(shape[-1], generator=g))
    return x.to(torch.bfloat16)


def blocked(x, rows):
    m, k = x.shape
    x = torch.nn.functional.pad(x, (0, -k % 128, 0, -m % rows))
    return x.view(-1, rows, x.shape[1] // 128, 128)


def quantize_ref(x, rows):
    """Codes and scales by the definition, in correctly rounded fp32 on the CPU."""
    m, k = x.shape
    b = blocked(x.float(), rows)
    a = b.abs().amax((1, 3)).clamp_min(FLOOR)
    # a tensor over a tensor: one rounding (a number over a tensor is the reciprocal times the number)
    code = (b * torch.full_like(a, 448.0).div(a)[:, None, :, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return code.view(-1, b.shape[2] * 128)[:m, :k], a / 448.0


def decode(q, scale, rows):
    m, k = q.shape
    wide = scale.double().repeat_interleave(rows, 0)[:m].repeat_interleave(128, 1)[:, :k]
    return q.double() * wide, wide


def check_against(y, q, scale, fp32_error):
    """Decoded values within half a step of `y` (64 bits), on top of y's own fp32 error."""
    got, wide = decode(q.cpu(), scale.cpu(), 1)
    assert bool(((got - y).abs() <= (HALF_E4M3 + fp32_error) * y.abs() * 1.001 + wide * HALF_SUB).all())


# ------------------------------------------------------------------ quantiser
@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 16), (3, 127), (2, 128), (5, 129), (130, 301), (128, 256), (257, 1000), (64, 5120)])
def test_quantize_is_the_definition_bit_for_bit(rows, m, k):
    from lcgemm import ops

    x = bf((m, k), m * 1000 + k, spread=0.5)
    q, s = ops.quantize_fp8(x.cuda(), block_rows=rows)
    want_q, want_s = quantize_ref(x, rows)
    assert q.shape == (m, k) and q.dtype == torch.float8_e4m3fn and q.stride(0) % 16 == 0
    assert torch.equal(s.cpu(), want_s)
    assert torch.equal(q.cpu().view(torch.uint8), want_q.view(torch.uint8))
    got, wide = decode(q.cpu(), s.cpu(), rows)
    assert bool(((got - x.double()).abs() <= HALF_E4M3 * 1.001 * x.double().abs() + wide * HALF_SUB).all())
    # the pad columns of the codes are zero
    pad = torch.as_strided(q.view(torch.uint8), (m, q.stride(0) - k), (q.stride(0), 1), q.storage_offset() + k) \
        if q.stride(0) > k else None
    assert pad is None or not bool(pad.any())


@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_strides_and_alignment(rows):
    from lcgemm import ops

    big = bf((40, 700), 5).cuda()
    for view in (big[:, 3:303], big[1:, 8:264], big[::2, 16:400], big[:, :1], big[:1, 1:130]):
        q, s = ops.quantize_fp8(view, block_rows=rows)
        want_q, want_s = quantize_ref(view.cpu(), rows)
        assert torch.equal(s.cpu(), want_s) and torch.equal(q.cpu().view(torch.uint8), want_q.view(torch.uint8))


@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_zeros_tiny_huge_and_not_finite(rows):
    from lcgemm import ops

    x = bf((256, 128 * 6), 9)
    x[:, 0:128] = 0.0
    x[:, 128:256] = (torch.randn(256, 128) * 1e-38).to(torch.bfloat16)       # below the floor, subnormals among them
    x[:, 256:384] = (x[:, 256:384].float() * 1e38).to(torch.bfloat16)
    x[3, 400] = float("inf")
    x[5, 530] = float("nan")
    x[7, 540] = -float("inf")
    q, s = ops.quantize_fp8(x.cuda(), block_rows=rows)
    want_q, want_s = quantize_ref(x, rows)
    assert torch.equal(s.cpu().view(torch.int32) & 0x7F800000, want_s.view(torch.int32) & 0x7F800000)
    finite = torch.isfinite(want_s)
    assert torch.equal(s.cpu()[finite], want_s[finite])
    got, _ = decode(q.cpu(), s.cpu(), rows)
    want, _ = decode(want_q, want_s, rows)
    assert torch.equal(got.isnan(), want.isnan()) and bool(got.isnan().any())
    assert torch.equal(got.nan_to_num(), want.nan_to_num())
    # the bad blocks decode to NaN throughout, the others not at all
    hit = blocked(got, rows).isnan()
    assert torch.equal(hit.all(3).all(1), hit.any(3).any(1))
    assert not bool(got[:, :256].isnan().any())


# -------------------------------------------------------------- norm, SwiGLU
@pytest.mark.parametrize("with_delta", [True, False])
@pytest.mark.parametrize("m,k", [(1, 8), (3, 24), (2, 128), (5, 136), (7, 1000), (4, 5120), (3, 8192), (2, 8200), (2, 16384), (1, 24576)])
def test_add_rmsnorm_fp8(m, k, with_delta):
    from lcgemm import ops

    eps = 1e-6
    delta, residual, w = bf((m, k), 1, spread=0.5), bf((m, k), 2, 3.0, 0.5), bf((k,), 3, 0.1)
    h = (delta.float() + residual.float()).to(torch.bfloat16) if with_delta else residual
    res = residual.cuda()
    q, s, got_h = ops.add_rmsnorm_fp8(delta.cuda() if with_delta else None, res, w.cuda(), eps)
    assert torch.equal(got_h.cpu(), h)
    assert (got_h is res) == (not with_delta)
    hd = h.double()
    y = hd * torch.rsqrt((hd * hd).mean(-1, keepdim=True) + eps) * (w.double() + 1.0)
    # fp32: the sum of squares carries at most (8 values a thread * vectors + two trees of 32) roundings, halved by
    # the root; rsqrtf 2 ulp; 1 + w, two products and the scaling one rounding each
    err = (24 + 10) * 2.0 ** -25 + 8 * 2.0 ** -24
    check_against(y, q, s, err)
    want_s = blocked(y, 1).abs().amax((1, 3)).clamp_min(FLOOR) / 448.0
    assert bool(((s.cpu().double() - want_s).abs() <= err * want_s).all())


def test_add_rmsnorm_fp8_in_place_zero_and_nan_rows():
    from lcgemm import ops

    m, k = 6, 512
    delta, residual, w = bf((m, k), 4).cuda(), bf((m, k), 5).cuda(), bf((k,), 6, 0.1).cuda()
    delta[1], residual[1] = 0, 0
    residual[2, 7] = float("nan")
    want = (delta.float() + residual.float()).to(torch.bfloat16)
    q0, s0, h0 = ops.add_rmsnorm_fp8(delta, residual, w, 1e-6)
    assert torch.equal(h0.nan_to_num(), want.nan_to_num())
    q1, s1, h1 = ops.add_rmsnorm_fp8(delta, residual, w, 1e-6, residual_out=residual)
    assert h1 is residual and torch.equal(residual.nan_to_num(), want.nan_to_num())
    assert torch.equal(q0.view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s0.nan_to_num(), s1.nan_to_num())
    assert not bool(q0[1].float().any()) and bool(torch.isfinite(s0[1]).all())
    assert bool(decode(q0.cpu(), s0.cpu(), 1)[0][2].isnan().all())
    assert not bool(decode(q0.cpu(), s0.cpu(), 1)[0][[0, 1, 3, 4, 5]].isnan().any())


@pytest.mark.parametrize("m,i", [(1, 8), (3, 24), (2, 128), (5, 136), (7, 1000), (33, 1024), (4, 17408)])
def test_swiglu_fp8(m, i):
    from lcgemm import ops

    z = bf((m, 2 * i), 7, 2.0, 0.5)
    z[0, 0], z[-1, 1 % i] = -90.0, 80.0
    q, s = ops.swiglu_fp8(z.cuda())
    g, u = z.double()[:, :i], z.double()[:, i:]
    y = g * torch.sigmoid(g) * u
    # fp32: __expf is off by 2 ulp plus the rounding of its scaled argument, |g| * 1.45 * 2^-24 <= 2^-17 for
    # |g| <= 90; the quotient 2 ulp, the sum, the product and the scaling one rounding each
    err = 2.0 ** -17 + 8 * 2.0 ** -24
    check_against(y, q, s, err)
    want_s = blocked(y, 1).abs().amax((1, 3)).clamp_min(FLOOR) / 448.0
    assert bool(((s.cpu().double() - want_s).abs() <= err * want_s).all())
    # a view with a wider pitch gives the same
    wide = torch.zeros((m, 2 * i + 8), dtype=torch.bfloat16, device="cuda")
    wide[:, :2 * i] = z.cuda()
    q2, s2 = ops.swiglu_fp8(wide[:, :2 * i])
    assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2)


# -------------------------------------------------------------------- product
def operands(m, n, k, seed):
    qa, sa = quantize_ref(bf((m, k), seed, spread=0.5), 1)
    qb, sb = quantize_ref(bf((n, k), seed + 1, 0.02), 128)
    return qa, sa, qb, sb


def pitched(q, pitch=None):
    m, k = q.shape
    out = torch.full((m, pitch or (k + 15) // 16 * 16), 0x55, dtype=torch.uint8)      # what lies past K is not read as data
    out[:, :k] = q.view(torch.uint8)
    return out.cuda().view(torch.float8_e4m3fn)[:, :k]


def check_product(got, qa, sa, qb, sb):
    a, b = decode(qa, sa, 1)[0], decode(qb, sb, 128)[0]
    want, size = a @ b.T, a.abs() @ b.abs().T
    blocks = sa.shape[1]
    # every addition of fp32 values may be off by 2^-23 of the magnitudes added so far: 128 in a block, then one for
    # each block and the scales' product; bf16 rounds the result once
    tol = HALF_BF16 * want.abs() + (128 + blocks + 2) * 2.0 ** -23 * size * (1 + HALF_BF16) + 1e-30
    off = (got.double().cpu() - want).abs()
    assert bool((off <= tol).all()), float((off - tol).max())


SHAPES = [(1, 1, 1), (1, 8, 16), (1, 128, 128), (1, 130, 301), (2, 257, 129), (3, 15, 640), (7, 300, 256), (8, 512, 1024),
          (9, 129, 127), (16, 256, 384), (17, 513, 160), (31, 64, 2048), (33, 1000, 500), (64, 384, 512), (65, 640, 144),
          (77, 257, 1280), (128, 256, 256), (129, 300, 400), (200, 1024, 384), (255, 130, 896), (256, 512, 640),
          (257, 257, 257), (300, 96, 2176), (513, 777, 1000), (1030, 520, 272)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_gemm_fp8(m, n, k):
    from lcgemm import ops

    qa, sa, qb, sb = operands(m, n, k, m + n + k)
    got = ops.gemm_fp8(pitched(qa), sa.cuda(), pitched(qb), sb.cuda())
    ops.check_status()
    assert got.shape == (m, n) and got.dtype == torch.bfloat16
    check_product(got, qa, sa, qb, sb)
    # the scales in the quantisers' order, and twice the same call: the same bits
    again = ops.gemm_fp8(pitched(qa), sa.cuda().t().contiguous().t(), pitched(qb), sb.cuda().t().contiguous().t())
    assert torch.equal(again, got)


@pytest.mark.parametrize("m,n,k", [(1, 300, 256), (20, 200, 300), (300, 700, 300), (600, 250, 512)])
def test_gemm_fp8_writes_its_block_of_a_larger_buffer(m, n, k):
    from lcgemm import ops

    qa, sa, qb, sb = operands(m, n, k, 3)
    big = torch.full((m + 3, (n + 7) // 8 * 8 + 16), 7.0, dtype=torch.bfloat16, device="cuda")
    out = big[1:m + 1, 8:8 + n]
    got = ops.gemm_fp8(pitched(qa, 512), sa.cuda(), pitched(qb, 768), sb.cuda(), out=out)
    assert got is out
    check_product(out, qa, sa, qb, sb)
    keep = torch.ones_like(big, dtype=torch.bool)
    keep[1:m + 1, 8:8 + n] = False
    assert bool((big[keep] == 7.0).all())


def test_gemm_fp8_nan_stays_in_its_row_and_column():
    from lcgemm import ops

    for m, n, k in ((5, 300, 256), (300, 520, 256)):
        qa, sa, qb, sb = operands(m, n, k, 11)
        qa.view(torch.uint8)[2, 130] = 0x7F          # NaN
        sb[1, 0] = float("inf")
        got = ops.gemm_fp8(pitched(qa), sa.cuda(), pitched(qb), sb.cuda()).cpu()
        assert bool(got[2].isnan().all())
        rest = [i for i in range(m) if i != 2]
        cols = [j for j in range(n) if not 128 <= j < 256]
        assert not bool(torch.isfinite(got[rest][:, 128:256]).any())
        assert bool(torch.isfinite(got[rest][:, cols]).all())


def test_gemm_fp8_sign_and_position():
    """Whole numbers that fit: every product exact, so every element has one right value."""
    from lcgemm import ops

    for m, n, k in ((3, 260, 272), (270, 390, 400)):
        g = torch.Generator().manual_seed(4)
        a = torch.randint(-4, 5, (m, k), generator=g).float()
        b = torch.randint(-4, 5, (n, k), generator=g).float()
        sa = torch.exp2(torch.randint(-3, 1, (m, -(-k // 128)), generator=g).float())
        sb = torch.exp2(torch.randint(-3, 1, (-(-n // 128), -(-k // 128)), generator=g).float())
        qa, qb = a.to(torch.float8_e4m3fn), b.to(torch.float8_e4m3fn)
        want = decode(qa, sa, 1)[0] @ decode(qb, sb, 128)[0].T
        got = ops.gemm_fp8(pitched(qa), sa.cuda(), pitched(qb), sb.cuda())
        assert torch.equal(got.cpu(), want.to(torch.bfloat16))


def test_empty_batches():
    from lcgemm import ops

    x = torch.empty((0, 256), dtype=torch.bfloat16, device="cuda")
    q, s = ops.quantize_fp8(x)
    assert q.shape == (0, 256) and s.shape == (0, 2)
    w, ws = ops.quantize_fp8(bf((64, 256), 1).cuda(), block_rows=128)
    assert ops.gemm_fp8(q, s, w, ws).shape == (0, 64)
    assert ops.swiglu_fp8(x)[0].shape == (0, 128)
    assert ops.add_rmsnorm_fp8(None, x, bf((256,), 1).cuda(), 1e-6)[0].shape == (0, 256)


def test_refusals_on_the_gpu():
    from lcgemm import ops

    x = bf((4, 256), 1).cuda()
    q, s = ops.quantize_fp8(x)
    w, ws = ops.quantize_fp8(bf((64, 256), 2).cuda(), block_rows=128)
    for call in (lambda: ops.quantize_fp8(x.float()), lambda: ops.quantize_fp8(x, block_rows=64),
                 lambda: ops.quantize_fp8(x.t()), lambda: ops.quantize_fp8(x[:, :0]),
                 lambda: ops.quantize_fp8(x[0].expand(4, 256)),
                 lambda: ops.add_rmsnorm_fp8(x, x, x[0, :128], 1e-6),
                 lambda: ops.add_rmsnorm_fp8(x[:, :252], x[:, :252].contiguous(), x[0, :252].contiguous(), 1e-6),
                 lambda: ops.add_rmsnorm_fp8(None, x[:, :250].contiguous(), x[0, :250].contiguous(), 1e-6),
                 lambda: ops.swiglu_fp8(x[:, :252]), lambda: ops.swiglu_fp8(x[:, 1:129]),
                 lambda: ops.gemm_fp8(q, s, w[:, :128], ws), lambda: ops.gemm_fp8(q, s[:2], w, ws),
                 lambda: ops.gemm_fp8(q, s, w, ws.double()), lambda: ops.gemm_fp8(x, s, w, ws),
                 lambda: ops.gemm_fp8(q[:, 1:129], s[:, :1], w[:, 1:129], ws[:, :1]),
                 lambda: ops.gemm_fp8(q, s, w, ws, out=torch.empty((4, 65), dtype=torch.bfloat16, device="cuda")),
                 lambda: ops.gemm_fp8(q, s, w, ws, out=torch.empty((4, 68), dtype=torch.bfloat16, device="cuda")[:, :64]),
                 lambda: ops.gemm_fp8(q, s, w, ws, out=torch.empty((4, 72), dtype=torch.bfloat16, device="cuda")[:, 1:65])):
        with pytest.raises(ValueError):
            call()
