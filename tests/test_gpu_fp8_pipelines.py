"""The product where its pipelines turn over: several tiles to a pair, operand rings that wrap, accumulator stages and
scale slots that are used again, cluster shares of many blocks.  Whole-number operands, so that every element has one
right value, from 64 bits.

On 148 SMs (74 pairs): the 256-wide form takes 1000 x 9400 as 148 tiles, two to a pair, and 1400 x 9400 as 222, three to
a pair; the 128-wide form takes 700 x 6300 as 150, up to three to a pair.  1024, 1100, 1200 and 1300 values of K are 8, 9,
10 and 11 blocks: every remainder of the four whose scales travel together, even and odd for two accumulator stages, all
remainders for four.  For few rows K = 16384 is 128 blocks, at most eight ways split, and 40000 columns are not split."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def whole(rows, k, block_rows, g):
    """Codes -4..4 with scales 1/8..1 and the values they stand for, in 64 bits."""
    q = torch.randint(-4, 5, (rows, k), generator=g, device="cuda").float()
    scale = torch.exp2(torch.randint(-3, 1, (-(-rows // block_rows), -(-k // 128)), generator=g, device="cuda").float())
    codes = torch.zeros((rows, (k + 15) // 16 * 16), dtype=torch.float8_e4m3fn, device="cuda")
    codes.view(torch.uint8)[:, :k] = q.to(torch.float8_e4m3fn).view(torch.uint8)
    wide = scale.double().repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :k]
    return codes[:, :k], scale, q.double() * wide


def check(m, n, k, times=1):
    from lcgemm import ops

    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    a, sa, wide_a = whole(m, k, 1, g)
    b, sb, wide_b = whole(n, k, 128, g)
    # the largest sum, 16 K, is a whole number of 1/64ths of at most 2^24: exact in fp32 whatever the order
    assert 16 * k * 64 <= 2 ** 24
    want = (wide_a @ wide_b.t()).to(torch.bfloat16)
    for _ in range(times):
        got = ops.gemm_fp8(a, sa.t().contiguous().t(), b, sb)
        ops.check_status()
        bad = (got != want).nonzero()
        assert bad.shape[0] == 0, f"{bad.shape[0]} elements, the first at {bad[0].tolist()}"


@pytest.mark.parametrize("k", [1024, 1100, 1200, 1300])
@pytest.mark.parametrize("m,n", [(1000, 9400), (1000, 9401), (1400, 9400)])
def test_256_wide_tiles(m, n, k):
    check(m, n, k, times=2)


@pytest.mark.parametrize("k", [1024, 1100, 1200, 1300])
@pytest.mark.parametrize("m,n", [(700, 6300), (700, 6304)])
def test_128_wide_tiles(m, n, k):
    check(m, n, k, times=2)


@pytest.mark.parametrize("m,n,k", [(300, 18900, 2176), (4000, 4800, 700), (129, 5120, 8200)])
def test_other_grids(m, n, k):
    check(m, n, k)


@pytest.mark.parametrize("n,k", [(1500, 16384), (1501, 10000), (9000, 10000), (40000, 1300)])
@pytest.mark.parametrize("m", [1, 10, 16, 20, 32, 50, 64, 100, 128])
def test_few_rows(m, n, k):
    check(m, n, k, times=2)
