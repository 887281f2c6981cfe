"""The 8-bit operators at the ends of what their documentation allows: padding beside NaN, gates whose exponential
leaves fp32's range, empty batches, another current device."""
import pytest
import torch

from gpu_util import seeded

pytestmark = pytest.mark.gpu


def padding(q):
    m, k = q.shape
    return torch.as_strided(q.view(torch.uint8), (m, q.stride(0) - k), (q.stride(0), 1), q.storage_offset() + k)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("k", [1, 8, 120, 129, 301, 1001])
@pytest.mark.parametrize("rows", [1, 128])
def test_padding_is_zero_beside_bad_values(rows, k, bad):
    from lcgemm import ops

    x = seeded((5, k), k)
    x[2, k - 1] = bad
    q, s = ops.quantize_fp8(x, block_rows=rows)
    assert q.stride(0) % 16 == 0 and q.stride(0) > k and not bool(padding(q).any())
    got = q.float() * s.repeat_interleave(rows, 0)[:5].repeat_interleave(128, 1)[:, :k]
    last = k - 1 - (k - 1) % 128
    assert bool(got[2, last:].isnan().all()) and not bool(got[:, :last].isnan().any())
    # the codes of a block with a NaN are NaN by the definition, x * (448 / NaN)
    assert bad == bad or bool(q[2, last:].float().isnan().all())


@pytest.mark.parametrize("inter", [8, 136, 1000])
def test_swiglu_padding_is_zero_beside_bad_values(inter):
    from lcgemm import ops

    z = seeded((4, 2 * inter), inter)
    z[1, inter - 1], z[3, 2 * inter - 1] = float("nan"), float("inf")
    q, s = ops.swiglu_fp8(z)
    assert q.stride(0) > inter and not bool(padding(q).any())
    got = q.float() * s.repeat_interleave(128, 1)[:, :inter]
    last = inter - 1 - (inter - 1) % 128
    assert bool(got[[1, 3], last:].isnan().all()) and not bool(got[[0, 2]].isnan().any())


def test_swiglu_of_far_gates_and_large_products():
    """silu(g) * u where e^-g or silu(g) alone leaves fp32's normal range and the product does not."""
    from lcgemm import ops

    gates = torch.cat([-torch.arange(60.0, 200.0, 0.5), -torch.tensor([300.0, 1e4, 3e38]), torch.tensor([0.0, 1.0, 88.0, 1e4])])
    ups = torch.tensor([1.0, -1e6, 1e10, 1e20, -1e30, 3e38])
    g = gates.to(torch.bfloat16)[:, None].expand(-1, len(ups)).reshape(-1)
    u = ups.to(torch.bfloat16)[None, :].expand(len(gates), -1).reshape(-1)
    keep = (g.double() * torch.sigmoid(g.double()) * u.double()).abs() < 3e38
    g, u = g[keep], u[keep]
    # a value to a row, so that each has a block and a scale of its own; seven small ones beside it
    m = g.shape[0]
    z = torch.zeros((m, 16), dtype=torch.bfloat16)
    z[:, 0], z[:, 8] = g, u
    z[:, 1:8] = -90.0
    q, s = ops.swiglu_fp8(z.cuda())
    y = z[:, :8].double() * torch.sigmoid(z[:, :8].double()) * z[:, 8:].double()
    got = q.double().cpu() * s.double().cpu()
    # The half exponential: its argument's rounding and constant 2^-18 each of at most 126 in base 2, its own 2^-22; it
    # enters twice.  Four products, a sum, a reciprocal and the scaling: 2^-24 each, 2^-23 for the reciprocal.
    err = 2 * (0.7 * (2.0 ** -18 + 2.0 ** -18) + 2.0 ** -22) + 8 * 2.0 ** -24
    assert bool(((got - y).abs() <= (2.0 ** -4 + err) * y.abs() * 1.001 + s.double().cpu() * 2.0 ** -10).all())
    want_s = y.abs().amax(1, keepdim=True).clamp_min(2.0 ** -100) / 448.0
    assert bool(((s.double().cpu() - want_s).abs() <= (err + 2.0 ** -24) * want_s).all())


def test_an_empty_batch_through_the_layer():
    from lcgemm.layer import Fp8MlpLayer

    layer = Fp8MlpLayer(4, seeded((256,), 3, 0.01), seeded((512, 256), 4, 0.02), seeded((256, 256), 5, 0.02))
    for delta in (None, seeded((0, 256), 2)):
        assert layer(seeded((0, 256), 1), delta).shape == (0, 256)


def test_a_prompt_on_the_host():
    from lcgemm.model import DecoderConfig, RandomInitDecoder

    model = RandomInitDecoder(DecoderConfig(layers=1, hidden=256, q_heads=4, kv_heads=2, head_dim=64, inter=256, vocab=999, seed=1))
    tokens = torch.randint(0, 999, (40,), generator=torch.Generator().manual_seed(2))
    want = model.prompt_logprobs(tokens.cuda(), top=3)
    got = model.prompt_logprobs(tokens, top=3)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_another_current_device(monkeypatch):
    """Every operator sets its tensors' device and calls itself when another one is current: the first question after
    the current device is answered with one that is not the tensors'."""
    from lcgemm import ops

    x, nw = seeded((5, 256), 1), seeded((256,), 3, 0.1)
    w, ws = ops.quantize_fp8(seeded((64, 256), 2), block_rows=128)
    q, s = ops.quantize_fp8(x)
    ids = torch.arange(5, device="cuda")
    residual, out = x.clone(), torch.empty((5, 64), dtype=torch.bfloat16, device="cuda")
    calls = (lambda: ops.quantize_fp8(x), lambda: ops.quantize_fp8(x, 128), lambda: ops.swiglu_fp8(x),
             lambda: ops.add_rmsnorm_fp8(x, residual, nw, 1e-6), lambda: ops.add_rmsnorm_fp8(None, residual, nw, 1e-6),
             lambda: (ops.gemm_fp8(q, s, w, ws),), lambda: (ops.gemm_fp8(q, s, w, ws, out),),
             lambda: ops.token_logprobs(x, ids, 4))
    real = ops._current_device
    for call in calls:
        want = [t.clone() for t in call()]
        asked = []

        def other():
            asked.append(None)
            return real() + 1 if len(asked) == 1 else real()

        monkeypatch.setattr(ops, "_current_device", other)
        got = call()
        monkeypatch.setattr(ops, "_current_device", real)
        assert len(asked) == 2 and torch.cuda.current_device() == 0
        assert all(torch.equal(a.float(), b.float()) for a, b in zip(got, want))


def test_the_norm_repeats_itself():
    """A long prefill's norm: the same bits every time, and codes that are off from 64 bits only where the scaled
    value lies within fp32's error of a border between two codes."""
    from lcgemm import ops

    m, k = 8192, 5120
    g = torch.Generator(device="cuda").manual_seed(7)
    spread = torch.exp(0.5 * torch.randn(k, generator=g, device="cuda"))
    delta = (torch.randn((m, k), generator=g, device="cuda") * spread).to(torch.bfloat16)
    residual = (3.0 * torch.randn((m, k), generator=g, device="cuda") * spread).to(torch.bfloat16)
    w = (0.1 * torch.randn(k, generator=g, device="cuda")).to(torch.bfloat16)
    q, s, h = ops.add_rmsnorm_fp8(delta, residual, w, 1e-6)
    for _ in range(20):
        again = ops.add_rmsnorm_fp8(delta, residual, w, 1e-6)
        assert torch.equal(again[0].view(torch.uint8), q.view(torch.uint8))
        assert torch.equal(again[1], s) and torch.equal(again[2], h)
    assert torch.equal(h, (delta.float() + residual.float()).to(torch.bfloat16))
    # err as in test_add_rmsnorm_fp8: its derivation holds for this K
    err = (24 + 10) * 2.0 ** -25 + 8 * 2.0 ** -24
    for i in range(0, m, 1024):
        hd = h[i:i + 1024].double()
        y = hd * torch.rsqrt((hd * hd).mean(-1, keepdim=True) + 1e-6) * (w.double() + 1.0)
        blocks = y.view(1024, k // 128, 128)
        scale = blocks.abs().amax(-1, keepdim=True) / 448.0
        scaled = (blocks / scale).view(1024, k)
        low, high = ((scaled * (1 + e)).clamp(-448.0, 448.0).float().to(torch.float8_e4m3fn).float() for e in (-2 * err, 2 * err))
        got = q[i:i + 1024].float()
        assert bool(((got == low) | (got == high)).all())
        assert float((low != high).float().mean()) < 1e-3       # so nearly every code has one right value


@pytest.mark.parametrize("m", [3, 300])
def test_scale_products_at_the_ends_of_their_range(m):
    """The product of a block's two scales may be anything in fp32's normal range, the scales themselves too."""
    from lcgemm import ops

    n, k = 260, 384
    g = torch.Generator(device="cuda").manual_seed(5)
    a = torch.randint(-1, 2, (m, k), generator=g, device="cuda").to(torch.float8_e4m3fn)
    b = torch.randint(-1, 2, (n, k), generator=g, device="cuda").to(torch.float8_e4m3fn)
    for low, high in ((-63, -63), (-126, 0), (7, -126), (63, 55), (127, -9), (-9, 127)):
        sa, sb = torch.full((m, 3), 2.0 ** low, device="cuda"), torch.full((3, 3), 2.0 ** high, device="cuda")
        want = ((a.double() @ b.double().t()) * 2.0 ** (low + high)).to(torch.bfloat16)
        assert torch.equal(ops.gemm_fp8(a, sa, b, sb), want)


@pytest.mark.parametrize("m", [1, 70, 129, 300])
@pytest.mark.parametrize("n", [1, 3, 7, 8, 9, 63, 64, 65, 127, 129])
def test_narrow_products(m, n):
    """Fewer columns than a 16-byte piece, and around the edges of a staged store; one K value to a block and a bit."""
    from lcgemm import ops

    g = torch.Generator(device="cuda").manual_seed(m + n)
    for k in (1, 16, 31, 128, 129):
        pitch = (k + 15) // 16 * 16
        a, b = (torch.randint(-4, 5, (rows, pitch), generator=g, device="cuda").to(torch.float8_e4m3fn)[:, :k] for rows in (m, n))
        sa = torch.exp2(torch.randint(-3, 1, (m, -(-k // 128)), generator=g, device="cuda").float())
        sb = torch.exp2(torch.randint(-3, 1, (-(-n // 128), -(-k // 128)), generator=g, device="cuda").float())
        wide_a = a.double() * sa.double().repeat_interleave(128, 1)[:, :k]
        wide_b = b.double() * sb.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
        big = torch.full((m + 2, (n + 7) // 8 * 8 + 8), 7.0, dtype=torch.bfloat16, device="cuda")
        out = ops.gemm_fp8(a, sa, b, sb, out=big[1:m + 1, :n])
        assert torch.equal(out, (wide_a @ wide_b.t()).to(torch.bfloat16))
        assert bool((big[0] == 7.0).all() and (big[m + 1] == 7.0).all() and (big[:, n:] == 7.0).all())
    ops.check_status()
