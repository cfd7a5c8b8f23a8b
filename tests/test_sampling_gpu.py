"""Tokens drawn by given random numbers against the definition in 64 bits: every filter alone and with others, short
and long lists, sets of thousands, ties at every border, odd sizes and strides, infinities and NaN. Tokens are equal; the
kernel's sums are within vocab * 2^-45 of the largest weight and the reference's within vocab * 2^-53, so that no random
number here may lie nearer than 1e-7 to a border of the sums (checked for each row that decides). The logarithm of the
probability is one fp32 rounding (2^-24 of it) and that of the sums (below 1e-8)."""
import math

import pytest
import torch

from tests.sampling_reference import sample

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")
    from starter_b200 import ops as ops_mod
    return ops_mod


def rows_of(rows, vocab, dtype, seed, sharp=None):
    g = torch.Generator().manual_seed(seed)
    s = (0.2 + 2.3 * torch.rand((rows, 1), generator=g)) if sharp is None else sharp
    rank = torch.rand((rows, vocab), generator=g).argsort(1).float() + 1
    x = 9 - s * rank.log() + 0.3 * torch.randn((rows, vocab), generator=g)
    return x.to(dtype), torch.rand(rows, generator=g)


def check(ops, x, u, device_x=None, **settings):
    dev = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in settings.items()}
    tokens, logprobs = ops.sample_tokens(x.cuda() if device_x is None else device_x, u.cuda(), **dev)
    again = ops.sample_tokens(x.cuda() if device_x is None else device_x, u.cuda(), **dev)
    assert torch.equal(tokens, again[0]) and torch.equal(logprobs, again[1])
    tokens, logprobs = tokens.cpu(), logprobs.cpu()
    for r in range(x.shape[0]):
        one = {k: v[r].item() if isinstance(v, torch.Tensor) else v for k, v in settings.items()}
        token, logprob, border = sample(x[r], u[r].item(), **one)
        if 0 < u[r] < 1 and border < 1e-7:
            continue                        # either side of the border is right
        assert tokens[r].item() == token, (r, one, u[r].item(), border)
        if math.isinf(logprob):
            assert logprobs[r].item() == logprob
        else:
            assert abs(logprobs[r].item() - logprob) <= 2.0 ** -24 * abs(logprob) + 1e-7, (r, logprobs[r].item(), logprob)


FILTERS = [dict(), dict(top_k=1), dict(top_k=50), dict(top_k=1000), dict(top_k=5000), dict(top_p=0.9), dict(top_p=0.999),
           dict(top_p=0.01), dict(top_p=0.0), dict(min_p=0.05), dict(min_p=1e-6), dict(min_p=1.0), dict(top_k=40, top_p=0.95),
           dict(top_k=20, min_p=0.1), dict(top_p=0.8, min_p=0.01), dict(top_k=3000, top_p=0.7, min_p=1e-5), dict(temperature=0.0),
           dict(temperature=0.3, top_p=0.9), dict(temperature=2.5, top_p=0.9), dict(temperature=100.0, top_p=0.5)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(5, 20011), (3, 151936), (40, 9000)])
@pytest.mark.parametrize("settings", FILTERS, ids=str)
def test_filters(ops, dtype, rows, vocab, settings):
    x, u = rows_of(rows, vocab, dtype, rows + vocab)
    check(ops, x, u, **settings)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 3, 7, 8, 9, 31, 32, 33, 255, 1000, 1023, 1024, 1025, 4097, 8191, 8192, 16385])
@pytest.mark.parametrize("settings", [dict(), dict(top_k=5), dict(top_p=0.6), dict(min_p=0.2), dict(top_k=700, top_p=0.9)], ids=str)
def test_sizes(ops, dtype, vocab, settings):
    """Rows of odd length begin anywhere in a 16-byte vector."""
    x, u = rows_of(9, vocab, dtype, vocab)
    check(ops, x, u, **settings)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 17, 18, 37, 38, 74, 75, 148, 149, 300])
def test_row_counts(ops, dtype, rows):
    """From eight CTAs a row to one."""
    x, u = rows_of(rows, 33000, dtype, rows)
    check(ops, x, u, top_p=0.9)


@pytest.mark.parametrize("dtype,vocab", [(torch.bfloat16, 524288), (torch.float32, 524288), (torch.float32, 400001)])
@pytest.mark.parametrize("settings", [dict(top_k=50, top_p=0.9), dict(top_p=0.9), dict(), dict(top_k=20000)], ids=str)
def test_the_longest_rows(ops, dtype, vocab, settings):
    """More than eight CTAs can keep: every pass reads the row again."""
    x, u = rows_of(2, vocab, dtype, 5)
    check(ops, x, u, **settings)


def test_one_setting_per_row(ops):
    rows = 60
    x, u = rows_of(rows, 50001, torch.float32, 8)
    g = torch.Generator().manual_seed(9)
    r = lambda: torch.rand(rows, generator=g)  # noqa: E731
    which = torch.arange(rows)
    check(ops, x, u, temperature=torch.where(which % 7 == 0, 0.0, 0.3 + 2 * r()),
          top_k=torch.where(which % 3 == 0, 0, (3000 * r() ** 3).int()).int(),
          top_p=torch.where(which % 4 == 1, 1.0, r()), min_p=torch.where(which % 5 == 2, 0.0, 0.3 * r() ** 2))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("levels", [1, 2, 3, 40])
@pytest.mark.parametrize("settings", [dict(), dict(top_k=7), dict(top_k=1500), dict(top_p=0.3), dict(top_p=0.9), dict(min_p=0.3),
                                      dict(top_k=2500, top_p=0.5)], ids=str)
def test_ties_go_by_index(ops, dtype, levels, settings):
    """A row of few values: every border of a filter lies among equal ones."""
    g = torch.Generator().manual_seed(levels)
    x = (torch.randint(0, levels, (6, 12007), generator=g).float() / 4).to(dtype)
    u = torch.rand(6, generator=g)
    check(ops, x, u, **settings)


@pytest.mark.parametrize("settings", [dict(), dict(top_k=3), dict(top_p=0.9), dict(min_p=0.1), dict(temperature=0.0)], ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_infinities_nan_and_rows_without_a_token(ops, dtype, settings):
    x, u = rows_of(9, 5003, dtype, 77)
    x[0] = -math.inf
    x[1] = math.nan
    x[2, 1:] = -math.inf
    x[3, ::2] = -math.inf
    x[4, 100:200] = math.nan
    x[5, [17, 900, 4000]] = math.inf
    x[6, 5002] = math.inf
    x[7, :5000] = -math.inf
    x[8] = -0.0
    x[8, 100:] = 0.0
    check(ops, x, u, **settings)


@pytest.mark.parametrize("settings", [dict(), dict(top_k=40), dict(top_p=0.9), dict(top_k=3000)], ids=str)
def test_random_numbers_at_the_ends(ops, settings):
    x, _ = rows_of(8, 9001, torch.float32, 3)
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, 2.0, -1.0, math.nan, math.inf, 2.0 ** -149])
    check(ops, x, u, **settings)


@pytest.mark.parametrize("scale", [1e-30, 1e30])
@pytest.mark.parametrize("settings", [dict(), dict(top_p=0.9), dict(top_k=2000, top_p=0.5)], ids=str)
def test_extreme_logits(ops, scale, settings):
    x, u = rows_of(4, 6001, torch.float32, 21)
    check(ops, x * scale, u, **settings)
    check(ops, x, u, temperature=scale, **settings)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("settings", [dict(), dict(top_k=40), dict(top_k=2000), dict(top_p=0.9), dict(min_p=0.01)], ids=str)
def test_masks_of_the_lowest_value(ops, dtype, settings):
    """Banned by the type's lowest number instead of -inf: of no weight, though they count as logits."""
    x, u = rows_of(5, 7001, dtype, 61)
    x[:, ::3] = torch.finfo(dtype).min
    x[4, 10:] = torch.finfo(dtype).min
    check(ops, x, u, **settings)


@pytest.mark.parametrize("settings", [dict(), dict(top_k=40), dict(top_p=0.5), dict(min_p=0.5), dict(min_p=1.0)], ids=str)
def test_infinite_temperature(ops, settings):
    """Every logit that is not -inf weighs the same."""
    x, _ = rows_of(3, 3000, torch.float32, 62)
    x[1, :100] = -math.inf
    u = torch.tensor([0.1234567, 0.5, 0.987654])
    tokens, logprobs = ops.sample_tokens(x.cuda(), u.cuda(), temperature=math.inf, **settings)
    for r in range(3):
        order = torch.sort(x[r], descending=True, stable=True)[1]
        order = order[x[r][order] > -math.inf]
        n = settings.get("top_k", len(order))
        n = math.ceil(n * settings.get("top_p", 1.0))
        kept = order[:n].sort()[0]
        assert tokens[r].item() == kept[int(u[r].double() * n)].item()
        assert abs(logprobs[r].item() + math.log(n)) <= 1e-6


def test_strides(ops):
    x, u = rows_of(6, 5001, torch.bfloat16, 30)
    wide = torch.full((6, 5555), math.nan, dtype=torch.bfloat16, device="cuda")
    for offset in (0, 1, 7, 8, 13):
        view = wide[:, offset:offset + 5001]
        view.copy_(x)
        check(ops, x, u, device_x=view, top_p=0.9)
        check(ops, x, u, device_x=view)
    # several draws from one row
    same = x[:1].cuda().expand(6, -1)
    check(ops, x[:1].expand(6, -1), u, device_x=same, top_p=0.95)


def test_frequencies(ops):
    """Evenly spaced numbers draw every token in proportion to its weight: each one's share of n draws is off by
    less than 1 / n at either end of its piece of the sums."""
    n = 4000
    x, _ = rows_of(1, 300, torch.float32, 4)
    u = (torch.arange(n) + 0.5) / n
    tokens, _ = ops.sample_tokens(x.cuda().expand(n, -1), u.cuda(), temperature=0.7)
    share = torch.bincount(tokens.cpu(), minlength=300).double() / n
    want = torch.softmax(x[0].double() / 0.7, 0)
    assert (share - want).abs().max().item() <= 1.0 / n + 1e-6


def test_captured_and_on_another_stream(ops):
    x, u = rows_of(5, 30001, torch.bfloat16, 12)
    xd, ud = x.cuda(), u.cuda()
    want = ops.sample_tokens(xd, ud, top_p=0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.sample_tokens(xd, ud, top_p=0.9)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.sample_tokens(xd, ud, top_p=0.9)
    ud.fill_(0.123)
    graph.replay()
    torch.cuda.synchronize()
    want = ops.sample_tokens(xd, ud, top_p=0.9)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
