"""Attention under a sliding window with sinks, token form: every head layout and row count, windows from one key to
more than the context, windows and sinks that end inside a page or meet in one, positions of their own for each
sequence, and NaN in every place that nobody sees - also in whole pages behind table entries nobody may read."""
import pytest
import torch

from tests.attention_reference import assert_close, attend, window_visible

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")
    from starter_b200 import ops as ops_mod
    return ops_mod


def make(ops, B, nq, nkv, T, positions, window, sinks, capacity, seed=0):
    """Query, cache (NaN wherever no row of the sequence sees, the table's unneeded entries on a page of NaN), and
    the rows and bounds that are wanted."""
    g = torch.Generator().manual_seed(1000 + seed)
    G = nq // nkv
    q = torch.randn((B * T, nq, 128), generator=g).to(torch.bfloat16)
    k = torch.randn((B, nkv, capacity, 128), generator=g).to(torch.bfloat16)
    v = torch.randn((B, nkv, capacity, 128), generator=g).to(torch.bfloat16)
    want = torch.zeros((B, T, nq, 128), dtype=torch.float64)
    bound = torch.zeros_like(want)
    pages = -(-capacity // 64)
    order = torch.randperm(B * pages, generator=g).to(torch.int32).view(B, pages)
    cache = ops.PagedKV(B, nkv, capacity, "cuda", block_table=order.cuda(),
                        pools=tuple(torch.full((B * pages + 1, nkv, 64, 128), float("nan"), dtype=torch.bfloat16,
                                               device="cuda") for _ in range(2)))
    for b in range(B):
        visible = window_visible([positions[b] + t for t in range(T)], capacity, window, sinks)
        seen = visible.any(0)
        k[b][:, ~seen] = float("nan")
        v[b][:, ~seen] = float("nan")
        for h in range(nkv):
            rows = q.view(B, T, nq, 128)[b, :, h * G:(h + 1) * G].reshape(T * G, 128)
            o, e = attend(rows, k[b, h], v[b, h], visible.repeat_interleave(G, 0), SCALE)
            want[b, :, h * G:(h + 1) * G], bound[b, :, h * G:(h + 1) * G] = o.view(T, G, 128), e.view(T, G, 128)
    cache.scatter(k.cuda(), v.cuda(), 0)
    for b in range(B):
        seen = window_visible([positions[b] + t for t in range(T)], pages * 64, window, sinks).any(0)
        dead = ~seen.view(pages, 64).any(1)
        cache.block_table[b, dead.cuda()] = B * pages
    return q.cuda(), cache, want.view(B * T, -1), bound.view(B * T, -1)


def check(ops, B, nq, nkv, T, positions, window, sinks, capacity, seed=0, shared_position=False):
    q, cache, want, bound = make(ops, B, nq, nkv, T, positions, window, sinks, capacity, seed)
    attn = ops.WindowAttention(B, nq, nkv, capacity, "cuda", window, sinks, T)
    position = torch.tensor(positions[:1] if shared_position else positions, dtype=torch.int32, device="cuda")
    got = attn.run(q, cache, position, SCALE)
    assert ops.device_status()[0] == 0
    assert_close(got.cpu(), want, bound)
    assert torch.equal(got, attn.run(q, cache, position, SCALE))          # the parts are joined in one order


@pytest.mark.parametrize("nq,nkv,T", [(32, 8, 1), (8, 8, 1), (8, 1, 1), (6, 2, 1), (28, 4, 1), (40, 8, 1), (16, 1, 1),
                                      (32, 1, 1), (32, 8, 2), (32, 8, 4), (32, 8, 8), (6, 2, 3), (28, 4, 4), (9, 1, 3),
                                      (5, 5, 8), (2, 2, 32), (40, 8, 6)])
@pytest.mark.parametrize("window,sinks", [(100, 4), (1, 0), (1000, 70)])
def test_heads_and_tokens(ops, nq, nkv, T, window, sinks):
    check(ops, 2, nq, nkv, T, [333 - T, 128 - T + 33], window, sinks, 340)


@pytest.mark.parametrize("position", [0, 1, 62, 63, 64, 65, 127, 128, 200, 639])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 0), (16, 0), (63, 5), (64, 64), (65, 65), (130, 0),
                                          (70, 129), (5, 1000), (640, 0)])
def test_where_window_and_sinks_end(ops, position, window, sinks):
    check(ops, 1, 4, 2, 1, [position], window, sinks, 640, seed=position)


@pytest.mark.parametrize("T", [2, 4])
@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 2), (64, 4), (200, 17)])
def test_several_tokens(ops, T, window, sinks):
    check(ops, 4, 8, 2, T, [0, 61, 64, 298], window, sinks, 305)


@pytest.mark.parametrize("B,nq,nkv,window,capacity", [(1, 32, 8, 1024, 8192), (1, 32, 8, 8000, 8192), (37, 32, 8, 300, 700),
                                                      (40, 8, 8, 2000, 2100), (1, 16, 2, 30000, 30100), (5, 28, 4, 700, 900)])
def test_batches_and_long_windows(ops, B, nq, nkv, window, capacity):
    positions = [capacity - 1 - (i * 37) % (capacity // 2) for i in range(B)]
    check(ops, B, nq, nkv, 1, positions, window, 4, capacity)
    if B > 1:
        check(ops, B, nq, nkv, 1, positions[:1] * B, window, 4, capacity, shared_position=True)


def test_rows_that_see_nothing_are_zero(ops):
    """A sequence that has not begun (position -1), and a block of tokens of which the first lie before it."""
    check(ops, 3, 8, 2, 1, [-1, 5, -1], 4, 2, 100)
    check(ops, 2, 8, 2, 3, [-2, -3], 4, 2, 100)


def test_a_position_past_the_pages_reads_nothing_outside_the_table(ops):
    """It sees the keys that its window still holds: none, but for the sinks."""
    q, cache, _, _ = make(ops, 1, 4, 1, 1, [127], 128, 0, 128)
    attn = ops.WindowAttention(1, 4, 1, 128, "cuda", 10, 0)
    for p in (128 + 40, 2 ** 31 - 1):
        out = attn.run(q, cache, torch.tensor([p], dtype=torch.int32, device="cuda"), SCALE)
        assert torch.isfinite(out.float()).all() and ops.device_status()[0] == 0


def test_scores_that_grow_and_masked_infinities(ops):
    """A maximum that moves in every tile, and infinities where nobody looks."""
    q, cache, _, _ = make(ops, 1, 8, 2, 1, [499], 300, 4, 500)
    g = torch.Generator().manual_seed(5)
    k = (torch.randn((1, 2, 500, 128), generator=g) * torch.linspace(0.05, 4, 500)[None, None, :, None]).to(torch.bfloat16)
    v = torch.randn((1, 2, 500, 128), generator=g).to(torch.bfloat16)
    visible = window_visible([499], 500, 300, 4)
    k[:, :, ~visible[0]] = float("inf")
    v[:, :, ~visible[0]] = float("-inf")
    cache.block_table.copy_(torch.arange(cache.pages_per_seq)[None])
    cache.scatter(k.cuda(), v.cuda(), 0)
    got = ops.WindowAttention(1, 8, 2, 500, "cuda", 300, 4).run(q, cache, torch.tensor([499], dtype=torch.int32, device="cuda"), SCALE)
    for h in range(2):
        want, bound = attend(q.cpu()[0, 4 * h:4 * h + 4], k[0, h], v[0, h], visible.expand(4, -1), SCALE)
        # (keys of up to 4 times the size: the scores' fp32 error is up to 4 times as large)
        assert_close(got.cpu().view(8, 128)[4 * h:4 * h + 4], want, 1.15 * bound)


def test_captured_and_on_another_stream(ops):
    q, cache, want, bound = make(ops, 3, 8, 2, 1, [250, 100, 3], 90, 4, 260)
    attn = ops.WindowAttention(3, 8, 2, 260, "cuda", 90, 4)
    position = torch.tensor([250, 100, 3], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = attn.run(q, cache, position, SCALE)
    side.synchronize()
    assert_close(got.cpu(), want, bound)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attn.run(q, cache, position, SCALE)
    position.fill_(-1)
    graph.replay()
    torch.cuda.synchronize()
    assert out.float().abs().max().item() == 0
    position.copy_(torch.tensor([250, 100, 3], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, got)


def test_shapes_of_every_split_count_one_after_the_other(ops):
    """The first call of a split count asks how many clusters are resident; that must not take shared memory from a
    shape that has run before."""
    shapes = [(1, 32, 8, 1000), (2, 16, 8, 700), (5, 32, 8, 500), (20, 32, 8, 300), (40, 32, 8, 200), (70, 32, 8, 100), (3, 32, 8, 5000)]
    made = []
    for again in range(2):
        for B, nq, nkv, capacity in shapes:
            attn = ops.WindowAttention(B, nq, nkv, capacity, "cuda", 400, 4)
            cache = ops.PagedKV(B, nkv, capacity, "cuda")
            q = torch.ones((B, nq, 128), dtype=torch.bfloat16, device="cuda")
            cache.v.fill_(2.0)
            made.append(attn.run(q, cache, torch.full((1,), capacity - 1, dtype=torch.int32, device="cuda"), SCALE))
    torch.cuda.synchronize()
    assert all(bool((x == 2.0).all()) for x in made)
