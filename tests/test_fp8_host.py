"""Refusals of the 8-bit operators and of the log probabilities that need no GPU: CPU tensors, and
the C entry points' own checks of pointers, extents, pitches and alignment (nothing is launched)."""
import pytest
import torch

from lcgemm import _native as nat
from lcgemm import ops

P = 4096                                # a non-null, aligned address; never dereferenced


def test_cpu_tensors_are_refused():
    x = torch.zeros((4, 128), dtype=torch.bfloat16)
    q, s = x.to(torch.float8_e4m3fn), torch.zeros((4, 1))
    for call in (lambda: ops.quantize_fp8(x), lambda: ops.swiglu_fp8(x), lambda: ops.add_rmsnorm_fp8(x, x, x[0], 1e-6),
                 lambda: ops.gemm_fp8(q, s, q, s[:1]), lambda: ops.token_logprobs(x, torch.zeros(4, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="no CPU implementation"):
            call()


def test_quantisers_check_their_arguments(native_lib):
    q = native_lib.lcg_quantize_fp8
    ok = (P, 4, 128, 128, 1, P, 128, P, 1, 4, None)

    def bad(i, v, fn=q, base=ok):
        a = list(base)
        a[i] = v
        return fn(*a)

    for i in (0, 5, 7):
        assert bad(i, None) == nat.ERR_BAD_ARG
    assert bad(1, 0) == bad(2, 0) == nat.ERR_UNSUPPORTED_SHAPE
    assert bad(3, 127) == nat.ERR_BAD_ARG                    # rows overlap
    assert bad(4, 64) == nat.ERR_BAD_ARG
    assert bad(6, 120) == bad(6, 136) == nat.ERR_BAD_ARG     # pitch of the codes
    assert bad(5, P + 8) == nat.ERR_MISALIGNED
    assert bad(1, 1 << 50) == nat.ERR_UNSUPPORTED_SHAPE
    assert q(P, 1 << 30, 128, 128, 128, P, 128, P, 1, 4, None) == nat.ERR_UNSUPPORTED_SHAPE

    n = native_lib.lcg_add_rmsnorm_fp8
    ok = (P, P, P, 4, 128, 1e-6, P, P, 128, P, 1, 4, None)
    for i in (1, 2, 6, 7, 9):
        assert bad(i, None, n, ok) == nat.ERR_BAD_ARG
    assert bad(4, 132, n, ok) == bad(4, 24584, n, ok) == bad(3, 0, n, ok) == nat.ERR_UNSUPPORTED_SHAPE
    for i in (0, 1, 2, 6, 7):
        assert bad(i, P + 8, n, ok) == nat.ERR_MISALIGNED

    g = native_lib.lcg_swiglu_fp8
    ok = (P, 4, 128, 256, P, 128, P, 1, 4, None)
    for i in (0, 4, 6):
        assert bad(i, None, g, ok) == nat.ERR_BAD_ARG
    assert bad(2, 132, g, ok) == bad(3, 248, g, ok) == bad(3, 260, g, ok) == nat.ERR_UNSUPPORTED_SHAPE
    assert bad(0, P + 2, g, ok) == nat.ERR_MISALIGNED


def test_product_checks_its_arguments(native_lib):
    ok = (P, 128, P, 1, 4, P, 128, P, 1, 1, P, 64, 4, 64, 128, None, None)

    def bad(i, v):
        a = list(ok)
        a[i] = v
        return native_lib.lcg_gemm_fp8(*a)

    for i in (0, 2, 5, 7, 10):
        assert bad(i, None) == nat.ERR_BAD_ARG
    for i in (12, 13, 14):
        assert bad(i, 0) == nat.ERR_UNSUPPORTED_SHAPE
    assert bad(1, 112) == bad(6, 112) == bad(11, 56) == nat.ERR_BAD_ARG
    assert bad(1, 136) == bad(6, 136) == bad(11, 68) == nat.ERR_MISALIGNED
    assert bad(0, P + 8) == bad(5, P + 8) == bad(10, P + 8) == nat.ERR_MISALIGNED


def test_logprobs_check_their_arguments(native_lib):
    ok = (P, nat.DTYPE_BF16, 4, 100, 100, P, 8, 5, P, P, P, P, None)

    def bad(i, v):
        a = list(ok)
        a[i] = v
        return native_lib.lcg_token_logprobs(*a)

    for i in (0, 5, 8, 9, 10, 11):
        assert bad(i, None) == nat.ERR_BAD_ARG
    assert bad(1, 3) == bad(4, 99) == bad(6, 2) == bad(7, 33) == bad(7, -1) == nat.ERR_BAD_ARG
    assert bad(2, 0) == bad(3, 0) == nat.ERR_UNSUPPORTED_SHAPE
    assert bad(3, (1 << 20) + 1) == bad(2, 1 << 31) == nat.ERR_UNSUPPORTED_SHAPE
    assert bad(0, P + 1) == nat.ERR_MISALIGNED
    assert native_lib.lcg_token_logprobs(P + 2, nat.DTYPE_FP32, 4, 100, 100, P, 8, 0, P, P, None, None,
                                         None) == nat.ERR_MISALIGNED
    assert native_lib.lcg_token_logprobs(P, nat.DTYPE_BF16, 4, 3, 3, P, 8, 4, P, P, P, P, None) == nat.ERR_BAD_ARG
