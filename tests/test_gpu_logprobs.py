"""Log probabilities, entropy and top alternatives against 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def reference(x, tokens, top):
    """In 64 bits, for rows that have a distribution; ids by value, then by id."""
    x = x.double()
    logp = torch.log_softmax(x, -1)
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    ids = torch.sort(x + 0.0, dim=-1, descending=True, stable=True).indices[:, :top]
    return logp.gather(1, tokens[:, None])[:, 0], entropy, logp.gather(1, ids), ids


def tolerance(x, want_lp, want_h):
    """S and T are sums of at most V / 256 + 64 terms in any one chain of fp32 additions, each off by 2^-24 of what it
    adds to; a term carries its exponential's error, 2^-22, and its argument's; the logarithms and differences round once."""
    v = x.shape[1]
    rel = (v / 256 + 64) * 2.0 ** -24 + 2.0 ** -21
    return rel + 2.0 ** -22 * want_lp.abs(), rel * (2 + want_h) + 2.0 ** -22


def check(x, tokens, top, device_x=None):
    from lcgemm import ops

    got = ops.token_logprobs(x.cuda() if device_x is None else device_x, tokens.cuda(), top=top)
    lp, h, tlp, ids = (t.cpu() for t in got)
    want_lp, want_h, want_tlp, want_ids = reference(x, tokens.long(), top)
    assert torch.equal(ids, want_ids)
    for g, w in ((lp, want_lp), (tlp, want_tlp)):
        finite = torch.isfinite(w)
        assert torch.equal(torch.isfinite(g), finite) and torch.equal(g[~finite].double(), w[~finite])
        tol = tolerance(x, w, want_h)[0]
        assert bool(((g.double() - w).abs()[finite] <= tol[finite]).all())
    assert bool(((h.double() - want_h).abs() <= tolerance(x, want_lp, want_h)[1]).all())
    return got


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("m,v,top", [(1, 1, 1), (1, 1, 0), (2, 2, 2), (3, 31, 5), (2, 32, 32), (5, 33, 20), (4, 255, 7),
                                     (4, 257, 32), (3, 1000, 20), (2, 4099, 32), (7, 8192, 0), (3, 50257, 5), (1, 151936, 20),
                                     (9, 65537, 20), (700, 999, 3)])
def test_sizes(kind, m, v, top):
    g = torch.Generator().manual_seed(m + v)
    x = (torch.randn((m, v), generator=g) * 3).to(TYPES[kind])
    tokens = torch.randint(0, v, (m,), generator=g)
    check(x, tokens, top)
    check(x, tokens.int(), min(top, 1))


@pytest.mark.parametrize("kind", list(TYPES))
def test_rows_of_any_pitch_and_alignment(kind):
    g = torch.Generator().manual_seed(5)
    big = (torch.randn((6, 3001), generator=g) * 4).to(TYPES[kind])
    dev = big.cuda()
    for rows, cols in ((slice(None), slice(0, 3001)), (slice(None), slice(1, 2000)), (slice(0, 6, 2), slice(3, 1026)),
                       (slice(1, 5), slice(7, 263)), (slice(2, 3), slice(5, 6)), (slice(None), slice(2, 40))):
        x = big[rows, cols]
        tokens = torch.randint(0, x.shape[1], (x.shape[0],), generator=g)
        check(x, tokens, min(20, x.shape[1]), dev[rows, cols])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("v", [300, 20001])
def test_orders_and_ties(kind, v):
    t = TYPES[kind]
    rows = [torch.arange(v).float() / v * 20,                       # rising: every value a new best
            -torch.arange(v).float() / v * 20,                      # falling
            torch.zeros(v),                                         # all equal
            torch.where(torch.arange(v) % 2 == 0, 0.0, -0.0),       # equal, of both signs
            (torch.arange(v) // 7 % 3).float(),                     # many ties
            torch.full((v,), -5.0)]
    rows[5][v - 1] = 3.0                                            # the best is the last
    x = torch.stack(rows).to(t)
    check(x, torch.randint(0, v, (len(rows),), generator=torch.Generator().manual_seed(1)), 32)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("v", [40, 300, 20001])
def test_masked_values(kind, v):
    t = TYPES[kind]
    g = torch.Generator().manual_seed(v)
    x = (torch.randn((6, v), generator=g) * 2).to(t)
    x[0, v // 2:] = -math.inf                       # a masked tail
    x[1, :v // 2] = -math.inf                       # a masked head
    x[2, torch.randperm(v, generator=g)[:v - 1]] = -math.inf     # one value left
    x[3] = torch.finfo(t).min                       # all at the type's lowest value
    x[4, ::2] = torch.finfo(t).min                  # half of them
    x[5, 1:] = -math.inf
    x[5, 0] = torch.finfo(t).max
    tokens = torch.tensor([v - 1, 0, 3, 7, 2, 0])   # masked tokens among them
    got = check(x, tokens, 20)
    assert got.logprob[0].item() == -math.inf and got.logprob[1].item() == -math.inf
    assert got.entropy[2].item() == 0.0 and got.entropy[5].item() == 0.0


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("v", [9, 300, 20001])
def test_rows_without_a_distribution(kind, v):
    from lcgemm import ops

    g = torch.Generator().manual_seed(v)
    x = (torch.randn((5, v), generator=g) * 2).to(TYPES[kind])
    x[0] = -math.inf
    x[1, 3] = math.inf
    x[2, v - 1] = math.nan
    x[3] = math.nan
    tokens = torch.randint(0, v, (5,), generator=g)
    top = min(v, 20)
    got = ops.token_logprobs(x.cuda(), tokens.cuda(), top=top)
    assert bool(got.logprob[:4].isnan().all()) and bool(got.entropy[:4].isnan().all())
    assert bool(got.top_logprobs[:4].isnan().all())
    want_lp, want_h, want_tlp, want_ids = reference(x[4:], tokens[4:], top)
    assert torch.equal(got.top_ids[4:].cpu(), want_ids) and abs(got.logprob[4].item() - want_lp.item()) < 1e-4
    # ids by the stated order: a NaN ranks with -inf
    ranked = torch.where(x.isnan(), -math.inf, x.double())
    ids = torch.sort(ranked + 0.0, dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(got.top_ids.cpu(), ids)


def test_tokens_out_of_range_are_not_read():
    from lcgemm import ops

    x = torch.randn((5, 100), generator=torch.Generator().manual_seed(2))
    tokens = torch.tensor([-1, 100, 2 ** 40, -2 ** 60, 99])
    got = ops.token_logprobs(x.cuda(), tokens.cuda(), top=2)
    assert bool(got.logprob[:4].isnan().all()) and bool(torch.isfinite(got.logprob[4]))
    assert bool(torch.isfinite(got.entropy).all()) and bool(torch.isfinite(got.top_logprobs).all())
    got = ops.token_logprobs(x.cuda(), torch.tensor([-1, 100, 2 ** 31 - 1, -2 ** 31, 99], dtype=torch.int32).cuda())
    assert bool(got.logprob[:4].isnan().all()) and bool(torch.isfinite(got.logprob[4]))


def test_peaked_rows_keep_their_small_numbers():
    """A row that knows its token: log probabilities near 0 and -1000, an entropy near 0."""
    x = torch.zeros((2, 5000))
    x[0, 17], x[1, 4999] = 30.0, 1000.0
    check(x, torch.tensor([17, 4999]), 5)
    check(x, torch.tensor([0, 0]), 5)


def test_empty_batch_and_refusals():
    from lcgemm import ops

    x = torch.randn((4, 64), device="cuda")
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    got = ops.token_logprobs(x[:0], t[:0], top=3)
    assert got.logprob.shape == (0,) and got.top_ids.shape == (0, 3)
    for call in (lambda: ops.token_logprobs(x.double(), t), lambda: ops.token_logprobs(x.t(), t),
                 lambda: ops.token_logprobs(x, t[:3]), lambda: ops.token_logprobs(x, t.float()),
                 lambda: ops.token_logprobs(x, t, top=33), lambda: ops.token_logprobs(x, t, top=-1),
                 lambda: ops.token_logprobs(x[:, :5], t, top=6), lambda: ops.token_logprobs(x[:, :0], t),
                 lambda: ops.token_logprobs(x[0].expand(4, 64), t)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("kind", list(TYPES))
def test_many_long_rows(kind):
    """Enough rows that each is one CTA's: random, tied, rising, masked and bad ones among them, at an odd pitch."""
    from lcgemm import ops

    m, v, top = 604, 17001, 20
    g = torch.Generator().manual_seed(3)
    big = (torch.randn((m, v + 2), generator=g) * 3).to(TYPES[kind])
    big[1] = 0.0
    big[2] = torch.arange(v + 2).float() / v * 20
    big[3, v // 3:] = -math.inf
    big[4, 1:] = torch.finfo(TYPES[kind]).min
    big[5] = (torch.arange(v + 2) // 7 % 3).float()
    tokens = torch.randint(0, v, (m,), generator=g)
    dev = big.cuda()
    got = check(big[:, 1:1 + v], tokens, top, dev[:, 1:1 + v])
    view = dev[:, 1:1 + v]
    dev[7, 100], dev[8] = math.nan, -math.inf
    bad = ops.token_logprobs(view, tokens.cuda(), top=top)
    assert bool(bad.logprob[7:9].isnan().all()) and bool(bad.top_logprobs[7:9].isnan().all())
    keep = [i for i in range(m) if i not in (7, 8)]
    assert all(torch.equal(a[keep], b[keep]) for a, b in zip(bad, got))
