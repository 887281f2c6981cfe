"""The C entries of the 8-bit operators and of the log probabilities refuse what is not aligned to its own type: such a
load or store would fault on the GPU.  Nothing is launched."""
import pytest

from lcgemm import _native as nat

P = 4096                                # a non-null, aligned address; never dereferenced


def refused(fn, args, at, by):
    args = list(args)
    args[at] += by
    return fn(*args) == nat.ERR_MISALIGNED


@pytest.mark.parametrize("rows", [1, 128])
def test_quantise(native_lib, rows):
    ok = (P, 4, 128, 128, rows, P, 128, P, 1, 4, None)
    assert refused(native_lib.lcg_quantize_fp8, ok, 0, 1) and refused(native_lib.lcg_quantize_fp8, ok, 7, 2)


def test_norm_and_swiglu(native_lib):
    assert refused(native_lib.lcg_add_rmsnorm_fp8, (P, P, P, 4, 128, 1e-6, P, P, 128, P, 1, 4, None), 9, 2)
    assert refused(native_lib.lcg_swiglu_fp8, (P, 4, 128, 256, P, 128, P, 1, 4, None), 6, 1)


def test_product(native_lib):
    ok = (P, 128, P, 1, 4, P, 128, P, 1, 1, P, 64, 4, 64, 128, P, None)
    for at in (2, 7, 15):
        assert refused(native_lib.lcg_gemm_fp8, ok, at, 2)


@pytest.mark.parametrize("token_bytes", [4, 8])
def test_logprobs(native_lib, token_bytes):
    ok = (P, nat.DTYPE_BF16, 4, 100, 100, P, token_bytes, 5, P, P, P, P, None)
    assert refused(native_lib.lcg_token_logprobs, ok, 5, token_bytes // 2)
    for at in (8, 9, 10):
        assert refused(native_lib.lcg_token_logprobs, ok, at, 2)
    assert refused(native_lib.lcg_token_logprobs, ok, 11, 4)
