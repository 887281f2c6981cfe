"""The 8-bit operators as they are used together: a layer, a decoder arm, prompt log probabilities; on other
streams, in a captured graph, with the row counts of a decode step."""
import pytest
import torch

from gpu_util import seeded

pytestmark = pytest.mark.gpu


def decode(q, scale, rows):
    m, k = q.shape
    return q.double().cpu() * scale.double().cpu().repeat_interleave(rows, 0)[:m].repeat_interleave(128, 1)[:, :k]


def weights(hidden, inter):
    return seeded((hidden,), 3, 0.01), seeded((2 * inter, hidden), 4, 0.02), seeded((hidden, inter), 5, 0.02)


@pytest.mark.parametrize("m", [1, 5, 77, 300])
@pytest.mark.parametrize("with_delta", [True, False])
def test_layer_stage_by_stage(m, with_delta):
    from lcgemm import ops
    from lcgemm.layer import Fp8MlpLayer

    hidden, inter, eps = 384, 640, 1e-6
    nw, wgu, wd = weights(hidden, inter)
    x, delta = seeded((m, hidden), 10), seeded((m, hidden), 11) if with_delta else None
    layer = Fp8MlpLayer(300, nw, wgu, wd, eps)
    out = layer(x, delta)
    ops.check_status()
    h = (x.float() + delta.float()).to(torch.bfloat16) if with_delta else x
    # the same operators one by one: the same bits
    q, s, h_ops = ops.add_rmsnorm_fp8(delta, x, nw, eps)
    z = ops.gemm_fp8(q, s, layer.w_gu, layer.w_gu_scale)
    q2, s2 = ops.swiglu_fp8(z)
    d = ops.gemm_fp8(q2, s2, layer.w_down, layer.w_down_scale)
    assert torch.equal(h_ops, h) and torch.equal(out, (h.float() + d.float()).to(torch.bfloat16))
    # each stage against 64 bits of the stage before it
    hd = h.double().cpu()
    y = hd * torch.rsqrt((hd * hd).mean(-1, keepdim=True) + eps) * (nw.double().cpu() + 1.0)
    got = decode(q, s, 1)
    assert bool(((got - y).abs() <= 2.0 ** -4 * 1.001 * y.abs() + s.double().cpu().repeat_interleave(128, 1)[:, :hidden] * 2.0 ** -10).all())
    for a, w, c, k in ((got, decode(layer.w_gu, layer.w_gu_scale, 128), z, hidden),
                       (decode(q2, s2, 1), decode(layer.w_down, layer.w_down_scale, 128), d, inter)):
        want, size = a @ w.T, a.abs() @ w.abs().T
        tol = 2.0 ** -8 * want.abs() + (128 + k / 128 + 2) * 2.0 ** -23 * size * 1.004
        assert bool(((c.double().cpu() - want).abs() <= tol).all())


def test_layer_is_near_the_bf16_layer():
    """Rounding to e4m3 is off by at most 2^-4 of a value, on average over a binade about 0.026 of it in the mean
    square; a product of two such operands is off by sqrt(2) * 0.026 = 0.037 of its norm where the errors are
    independent, SwiGLU of two such inputs by at most 1.1 * sqrt(2) times that (|d silu| <= 1.1), 0.057, and the second product by
    sqrt(0.057^2 + 2 * 0.026^2) = 0.068.  Held to twice that."""
    from lcgemm.layer import DenseMlpLayer, Fp8MlpLayer

    hidden, inter, m = 512, 1024, 256
    nw, wgu, wd = weights(hidden, inter)
    x = seeded((m, hidden), 12)
    want, _ = DenseMlpLayer(m, nw, wgu, wd).chain(None, x)
    got, h = Fp8MlpLayer(m, nw, wgu, wd).chain(None, x)
    assert h is x
    rel = ((got.double() - want.double()).norm() / want.double().norm()).item()
    assert rel <= 0.136


def test_layer_refuses_more_rows_than_it_was_built_for():
    from lcgemm.layer import Fp8MlpLayer

    nw, wgu, wd = weights(256, 256)
    layer = Fp8MlpLayer(4, nw, wgu, wd)
    with pytest.raises(ValueError, match="at most 4 rows"):
        layer(seeded((5, 256), 1))
    with pytest.raises(ValueError, match="intermediate"):
        Fp8MlpLayer(4, nw, wgu[:-2], wd)


@pytest.mark.parametrize("m", [3, 300])
def test_captured_layer_and_replay_with_new_inputs(m):
    from lcgemm.layer import CapturedLayer, Fp8MlpLayer

    nw, wgu, wd = weights(384, 640)
    layer = Fp8MlpLayer(m, nw, wgu, wd)
    x = seeded((m, 384), 20)
    graph = CapturedLayer(layer, x)
    for seed in (20, 21, 22):
        new = seeded((m, 384), seed)
        x.copy_(new)
        got = graph().clone()
        assert torch.equal(got, layer(new))


def test_two_streams_at_once():
    """Two layers' calls in flight on two streams, each with its own buffers: the results of one stream."""
    from lcgemm import ops
    from lcgemm.layer import Fp8MlpLayer

    nw, wgu, wd = weights(512, 1024)
    layers = [Fp8MlpLayer(600, nw, wgu, wd) for _ in range(2)]
    xs = [seeded((m, 512), 30 + m) for m in (600, 8)]
    logits = torch.randn((40, 30001), device="cuda")
    ids = torch.arange(40, device="cuda")
    want = [layer(x).clone() for layer, x in zip(layers, xs)]
    want_lp = ops.token_logprobs(logits, ids, top=8)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        got, lps = [], []
        for layer, x, stream in zip(layers, xs, streams):
            with torch.cuda.stream(stream):
                got.append(layer(x))
                lps.append(ops.token_logprobs(logits, ids, top=8))
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))
        assert all(torch.equal(g, w) for lp in lps for g, w in zip(lp, want_lp))
    ops.check_status()


def test_logprobs_in_a_graph():
    from lcgemm import ops

    logits = torch.randn((3, 40000), device="cuda").to(torch.bfloat16)
    ids = torch.tensor([1, 2, 3], device="cuda")
    ops.token_logprobs(logits, ids, top=20)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.token_logprobs(logits, ids, top=20)
    for seed in (1, 2):
        g = torch.Generator(device="cuda").manual_seed(seed)
        logits.copy_(torch.randn((3, 40000), device="cuda", generator=g))
        ids.copy_(torch.randint(0, 40000, (3,), device="cuda", generator=g))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, ops.token_logprobs(logits, ids, top=20)))


def test_decoder_arm_and_prompt_logprobs():
    from lcgemm import ops
    from lcgemm.model import DecoderConfig, RandomInitDecoder, compare_arms

    cfg = DecoderConfig(layers=3, hidden=512, q_heads=8, kv_heads=2, head_dim=64, inter=1024, vocab=4099, seed=1)
    model = RandomInitDecoder(cfg)
    tokens = torch.randint(0, cfg.vocab, (301,), generator=torch.Generator().manual_seed(2)).cuda()
    with pytest.raises(RuntimeError, match="quantize"):
        model.prefill(tokens, arm="fp8")
    assert model.quantize()["layers"] == 3
    stock_logits, stock_hidden = model.prefill(tokens, arm="stock")
    logits, hidden = model.prefill(tokens, arm="fp8")
    ops.check_status()
    assert model.calls["fp8"] == cfg.layers
    # each of the 3 layers adds an MLP branch that is off by at most 0.136 of itself (see above)
    assert compare_arms(stock_logits, logits, stock_hidden, hidden)["hidden_rel_fro"] < 0.136
    for arm in ("stock", "fp8"):
        got = model.prompt_logprobs(tokens, arm=arm, top=20, rows=100)
        final = model.prefill(tokens, arm=arm)[1]
        logp = torch.log_softmax(torch.nn.functional.linear(final[:-1], model.lm_head).double(), -1)
        assert got.logprob.shape == (300,) and got.top_ids.shape == (300, 20)
        # the head's products in batches of 100 and of 300 rows may round differently: one bf16 step of a logit
        step = 2.0 ** -7 * torch.nn.functional.linear(final[:-1], model.lm_head).abs().max().double()
        assert float((got.logprob.double() - logp.gather(1, tokens[1:, None])[:, 0]).abs().max()) <= 2 * step + 1e-5
        assert float((got.entropy.double() + (logp.exp() * logp).sum(-1)).abs().max()) <= 2 * step + 1e-4
        assert bool((got.top_logprobs[:, :-1] >= got.top_logprobs[:, 1:]).all())
    with pytest.raises(ValueError):
        model.prompt_logprobs(tokens[:1])


def test_offsets_past_32_bits():
    """Matrices of more than 2^31 elements: the last rows are where they belong."""
    from lcgemm import ops

    # quantiser and log probabilities: 2^31 bf16 values and some
    v, m = 131075, 16400
    big = torch.zeros((m, v), dtype=torch.bfloat16, device="cuda")
    tail = seeded((3, v), 41, 2.0)
    big[-3:] = tail
    ids = torch.full((m,), 7, device="cuda")
    got = ops.token_logprobs(big, ids, top=4)
    want = ops.token_logprobs(tail, ids[:3], top=4)
    # 3 rows are split over clusters and 16400 are not, so the sums associate differently: each is within
    # (V / 256 + 64) 2^-24 + 2^-21 of the exact S and T (tests/test_gpu_logprobs.py), twice that of the other
    rel = 2 * ((v / 256 + 64) * 2.0 ** -24 + 2.0 ** -21)
    assert torch.equal(got.top_ids[-3:], want.top_ids)
    assert bool(((got.logprob[-3:] - want.logprob).abs() <= rel + 2.0 ** -21 * want.logprob.abs()).all())
    assert bool(((got.top_logprobs[-3:] - want.top_logprobs).abs() <= rel + 2.0 ** -21 * want.top_logprobs.abs()).all())
    assert bool(((got.entropy[-3:] - want.entropy).abs() <= rel * (2 + want.entropy)).all())
    assert torch.equal(got.top_ids[0].cpu(), torch.arange(4))
    q, s = ops.quantize_fp8(big)
    want_q, want_s = ops.quantize_fp8(tail)
    assert torch.equal(q[-3:].view(torch.uint8), want_q.view(torch.uint8)) and torch.equal(s[-3:], want_s)
    del big, q, s, got
    # the product: an output of 2^31 values and some, for many rows; for few rows a weight of as many
    m, n = 65600, 32776
    a, sa = ops.quantize_fp8(seeded((m, 32), 42))
    b, sb = ops.quantize_fp8(seeded((n, 32), 43), block_rows=128)
    out = ops.gemm_fp8(a, sa, b, sb)
    assert torch.equal(out[-300:], ops.gemm_fp8(a[-300:], sa[-300:], b, sb))
    del out
    n, k = 131200, 16400
    w = torch.zeros((n, k), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    last, last_s = ops.quantize_fp8(seeded((128, k), 44), block_rows=128)
    w[-128:].view(torch.uint8).copy_(last.view(torch.uint8))
    ws = torch.ones((n // 128, -(-k // 128)), device="cuda")
    ws[-1] = last_s[0]
    x, sx = ops.quantize_fp8(seeded((2, k), 45))
    got = ops.gemm_fp8(x, sx, w, ws)
    ops.check_status()
    want = decode(x, sx, 1) @ decode(last, last_s, 128).T
    size = decode(x, sx, 1).abs() @ decode(last, last_s, 128).abs().T
    assert bool(((got[:, -128:].double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + (128 + 129 + 2) * 2.0 ** -23 * size).all())
    assert not bool(got[:, :-128].any())


def test_first_product_inside_a_capture_is_refused():
    from lcgemm import ops

    q, s = ops.quantize_fp8(seeded((4, 256), 1))
    w, ws = ops.quantize_fp8(seeded((64, 256), 2), block_rows=128)
    word = ops._STATUS.pop(q.device, None)
    try:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="before a graph capture"):
            with torch.cuda.graph(graph):
                ops.gemm_fp8(q, s, w, ws)
    finally:
        if word is not None:
            ops._STATUS[q.device] = word
    torch.cuda.synchronize()
    assert torch.isfinite(ops.gemm_fp8(q, s, w, ws)).all()


def test_tensors_on_another_device():
    from lcgemm import ops

    if torch.cuda.device_count() < 2:
        pytest.skip("needs two devices")
    x = seeded((5, 256), 1)
    other = x.to("cuda:1")
    assert torch.cuda.current_device() == 0
    q, s = ops.quantize_fp8(other)
    w, ws = ops.quantize_fp8(seeded((64, 256), 2).to("cuda:1"), block_rows=128)
    c = ops.gemm_fp8(q, s, w, ws)
    lp = ops.token_logprobs(c, torch.zeros(5, dtype=torch.int64, device="cuda:1"), top=3)
    torch.cuda.synchronize(1)
    assert c.device == lp.logprob.device == other.device and torch.cuda.current_device() == 0
    q0, s0 = ops.quantize_fp8(x)
    assert torch.equal(q.cpu().view(torch.uint8), q0.cpu().view(torch.uint8)) and torch.equal(s.cpu(), s0.cpu())
    with pytest.raises(ValueError, match="one device"):
        ops.gemm_fp8(q0, s0, w, ws)


def test_scales_of_stride_zero():
    """One scale for a whole matrix is a tensor of stride 0."""
    from lcgemm import ops

    for m in (4, 300):
        q, _ = ops.quantize_fp8(seeded((m, 300), 1))
        w, _ = ops.quantize_fp8(seeded((200, 300), 2), block_rows=128)
        one = torch.full((1, 1), 0.25, device="cuda")
        got = ops.gemm_fp8(q, one.expand(m, 3), w, one.expand(2, 3))
        want = ops.gemm_fp8(q, one.repeat(m, 3), w, one.repeat(2, 3))
        assert torch.equal(got, want)
