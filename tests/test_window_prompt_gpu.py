"""Windowed attention over whole prompts: head layouts that fill a tile of 128 rows and such that do not, one and two
query tiles per CTA, windows and sinks that end anywhere in a key tile, chunks behind earlier tokens, NaN wherever
nobody sees."""
import pytest
import torch

from tests.attention_reference import assert_close, attend, window_visible
from tests.test_window_attention_gpu import SCALE, make, ops  # noqa: F401

pytestmark = pytest.mark.gpu


def check(ops, B, nq, nkv, T, positions, window, sinks, capacity, seed=0, shared_position=False):  # noqa: F811
    q, cache, want, bound = make(ops, B, nq, nkv, T, positions, window, sinks, capacity, seed)
    position = torch.tensor(positions[:1] if shared_position else positions, dtype=torch.int32, device="cuda")
    got = ops.window_prompt_attention(q, cache, position, T, SCALE, window, sinks)
    assert ops.device_status()[0] == 0
    assert_close(got.cpu(), want, bound)
    assert torch.equal(got, ops.window_prompt_attention(q, cache, position, T, SCALE, window, sinks))


@pytest.mark.parametrize("nq,nkv", [(32, 8), (8, 8), (16, 8), (8, 1), (6, 2), (28, 4), (40, 8), (9, 1), (32, 1), (13, 1)])
@pytest.mark.parametrize("T,window,sinks", [(77, 20, 3), (300, 130, 0)])
def test_heads(ops, nq, nkv, T, window, sinks):  # noqa: F811
    check(ops, 2, nq, nkv, T, [0, 41], window, sinks, T + 50)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 0), (15, 4), (16, 16), (17, 17), (64, 64), (100, 0), (127, 1),
                                          (128, 128), (129, 129), (200, 77), (5, 300), (1000, 0), (320, 1000)])
@pytest.mark.parametrize("T,before", [(1, 0), (1, 259), (130, 0), (333, 100)])
def test_where_window_and_sinks_end(ops, T, before, window, sinks):  # noqa: F811
    check(ops, 1, 4, 1, T, [before], window, sinks, before + T, seed=T)


@pytest.mark.parametrize("B,nq,nkv,T,before,window,sinks", [
    (1, 32, 8, 1184, 0, 500, 4), (1, 32, 8, 1185, 0, 500, 4), (3, 32, 8, 701, 600, 512, 64), (9, 16, 8, 130, 7, 64, 0),
    (1, 28, 4, 2500, 0, 33, 1), (4, 40, 8, 400, 0, 4000, 0)])
def test_sizes(ops, B, nq, nkv, T, before, window, sinks):  # noqa: F811
    positions = [before + 3 * (i % 2) for i in range(B)]
    check(ops, B, nq, nkv, T, positions, window, sinks, before + T + 10)
    if B > 1:
        check(ops, B, nq, nkv, T, positions[:1] * B, window, sinks, before + T + 10, shared_position=True)


def test_equal_to_the_token_form(ops):  # noqa: F811
    """The same rows, a prompt at a time and four tokens at a time: each rounds P and the result to bf16."""
    B, nq, nkv, T = 2, 8, 2, 4
    q, cache, want, bound = make(ops, B, nq, nkv, T, [700, 90], 128, 5, 710)
    position = torch.tensor([700, 90], dtype=torch.int32, device="cuda")
    a = ops.window_prompt_attention(q, cache, position, T, SCALE, 128, 5).cpu()
    b = ops.WindowAttention(B, nq, nkv, 710, "cuda", 128, 5, T).run(q, cache, position, SCALE).cpu()
    assert_close(a, b.double(), 2 * bound)


@pytest.mark.parametrize("scale", [0.0, -0.05])
def test_scale_that_is_not_positive(ops, scale):  # noqa: F811
    q, cache, _, _ = make(ops, 1, 8, 2, 200, [10], 50, 4, 210)
    k, v = (x.cpu() for x in cache.gather(210))
    got = ops.window_prompt_attention(q, cache, torch.tensor([10], dtype=torch.int32, device="cuda"), 200, scale, 50, 4).cpu()
    visible = window_visible(range(10, 210), 210, 50, 4)
    for h in range(2):
        rows = q.cpu()[:, 4 * h:4 * h + 4].reshape(800, 128)
        want, bound = attend(rows, k[0, h], v[0, h], visible.repeat_interleave(4, 0), scale)
        assert_close(got.view(200, 8, 128)[:, 4 * h:4 * h + 4].reshape(800, 128), want, bound)


def test_growing_scores(ops):  # noqa: F811
    """Every key tile moves the rows' maximum."""
    q, cache, _, _ = make(ops, 1, 8, 2, 500, [0], 300, 4, 500)
    g = torch.Generator().manual_seed(6)
    k = (torch.randn((1, 2, 500, 128), generator=g) * torch.linspace(0.05, 4, 500)[None, None, :, None]).to(torch.bfloat16)
    v = torch.randn((1, 2, 500, 128), generator=g).to(torch.bfloat16)
    cache.scatter(k.cuda(), v.cuda(), 0)
    got = ops.window_prompt_attention(q, cache, torch.zeros(1, dtype=torch.int32, device="cuda"), 500, SCALE, 300, 4).cpu()
    visible = window_visible(range(500), 500, 300, 4)
    for h in range(2):
        rows = q.cpu()[:, 4 * h:4 * h + 4].reshape(2000, 128)
        want, bound = attend(rows, k[0, h], v[0, h], visible.repeat_interleave(4, 0), SCALE)
        # (keys of up to 4 times the size: the scores' fp32 error is up to 4 times as large)
        assert_close(got.view(500, 8, 128)[:, 4 * h:4 * h + 4].reshape(2000, 128), want, 1.15 * bound)


def test_positions_outside_the_pages_read_nothing_outside_the_table(ops):  # noqa: F811
    q, cache, _, _ = make(ops, 1, 4, 1, 40, [0], 128, 0, 128)
    for p in (-5, 100, 128, 2 ** 31 - 1):
        ops.window_prompt_attention(q, cache, torch.tensor([p], dtype=torch.int32, device="cuda"), 40, SCALE, 10, 0)
        assert ops.device_status()[0] == 0


def test_captured(ops):  # noqa: F811
    q, cache, want, bound = make(ops, 2, 8, 2, 150, [100, 3], 90, 4, 260)
    position = torch.tensor([100, 3], dtype=torch.int32, device="cuda")
    ops.window_prompt_attention(q, cache, position, 150, SCALE, 90, 4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.window_prompt_attention(q, cache, position, 150, SCALE, 90, 4)
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert_close(out.cpu(), want, bound)
