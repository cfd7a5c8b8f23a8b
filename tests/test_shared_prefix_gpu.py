"""Attention of a batch over one shared prefix: few rows per kv head and many, every head layout, prefixes from nothing
to many splits, own keys from none on, prefix and sequences in the same pools, NaN wherever nobody sees."""
import pytest
import torch

from tests.attention_reference import assert_close, attend

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")
    from starter_b200 import ops as ops_mod
    return ops_mod


def make(ops, B, nq, nkv, T, prefix, positions, prefix_capacity, capacity, seed=0, growth=False):
    """Prefix and sequences in one pool of pages handed out at random; NaN past the prefix and past the sequences."""
    g = torch.Generator().manual_seed(3000 + seed)
    G = nq // nkv
    q = torch.randn((B * T, nq, 128), generator=g).to(torch.bfloat16)
    pk, pv = (torch.randn((1, nkv, prefix_capacity, 128), generator=g) for _ in range(2))
    if growth:
        pk = pk * torch.linspace(0.05, 4, prefix_capacity)[None, None, :, None]
    k, v = (torch.randn((B, nkv, capacity, 128), generator=g) for _ in range(2))
    pk, pv, k, v = (x.to(torch.bfloat16) for x in (pk, pv, k, v))
    pk[:, :, prefix:] = pv[:, :, prefix:] = float("nan")
    for b in range(B):
        k[b][:, max(0, positions[b] + T):] = v[b][:, max(0, positions[b] + T):] = float("nan")
    pp, sp = -(-prefix_capacity // 64), -(-capacity // 64)
    pools = tuple(torch.full((pp + B * sp, nkv, 64, 128), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    order = torch.randperm(pp + B * sp, generator=g).to(torch.int32).cuda()
    before = ops.PagedKV(1, nkv, prefix_capacity, "cuda", block_table=order[:pp].view(1, pp).contiguous(), pools=pools)
    cache = ops.PagedKV(B, nkv, capacity, "cuda", block_table=order[pp:].view(B, sp).contiguous(), pools=pools)
    before.scatter(pk.cuda(), pv.cuda(), 0)
    cache.scatter(k.cuda(), v.cuda(), 0)
    want = torch.zeros((B, T, nq, 128), dtype=torch.float64)
    bound = torch.zeros_like(want)
    for b in range(B):
        at = torch.tensor([positions[b] + t for t in range(T)])[:, None]
        visible = torch.cat([(torch.arange(prefix_capacity) < prefix)[None].expand(T, -1), torch.arange(capacity)[None] <= at], 1)
        for h in range(nkv):
            rows = q.view(B, T, nq, 128)[b, :, h * G:(h + 1) * G].reshape(T * G, 128)
            o, e = attend(rows, torch.cat([pk[0, h], k[b, h]]), torch.cat([pv[0, h], v[b, h]]),
                          visible.repeat_interleave(G, 0), SCALE)
            want[b, :, h * G:(h + 1) * G], bound[b, :, h * G:(h + 1) * G] = o.view(T, G, 128), e.view(T, G, 128)
    return q.cuda(), before, cache, want.view(B * T, -1), bound.view(B * T, -1)


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def check(ops, B, nq, nkv, T, prefix, positions, prefix_capacity=None, capacity=None, seed=0, growth=False, slack=1.0):
    prefix_capacity = prefix_capacity or max(1, prefix)
    capacity = capacity or max(1, max(positions) + T)
    q, before, cache, want, bound = make(ops, B, nq, nkv, T, prefix, positions, prefix_capacity, capacity, seed, growth)
    attn = ops.SharedPrefixAttention(B, nq, nkv, prefix_capacity, capacity, "cuda", T)
    got = attn.run(q, before, int32([prefix]), cache, int32(positions), SCALE)
    assert ops.device_status()[0] == 0
    assert_close(got.cpu(), want, slack * bound)
    assert torch.equal(got, attn.run(q, before, int32([prefix]), cache, int32(positions), SCALE))


@pytest.mark.parametrize("nq,nkv,T", [(32, 8, 1), (8, 8, 1), (8, 1, 1), (6, 2, 1), (28, 4, 1), (40, 8, 1), (32, 1, 1), (32, 8, 2),
                                      (32, 8, 8), (6, 2, 3), (28, 4, 4), (9, 1, 3)])
@pytest.mark.parametrize("B", [1, 3, 11, 40])
def test_heads_tokens_and_batches(ops, nq, nkv, T, B):
    check(ops, B, nq, nkv, T, 700, [(17 * i) % 90 for i in range(B)])


@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 63, 64, 65, 127, 128, 129, 1000, 5000])
@pytest.mark.parametrize("B", [2, 12, 70])
def test_prefix_lengths(ops, prefix, B):
    check(ops, B, 8, 2, 1, prefix, [i % 70 for i in range(B)], seed=prefix)


@pytest.mark.parametrize("prefix", [0, 1, 100, 129, 2000, 6000])
@pytest.mark.parametrize("B", [2, 12, 70])
def test_a_prefix_that_fills_part_of_its_pages(ops, prefix, B):
    """The splits are planned for the capacity; with fewer tiles some have nothing to do."""
    check(ops, B, 8, 2, 1, prefix, [i % 70 for i in range(B)], prefix_capacity=6000, capacity=128, seed=prefix)


@pytest.mark.parametrize("B", [2, 40])
def test_rows_without_own_keys_and_rows_without_any(ops, B):
    """Position -1: nothing behind the prefix yet; with an empty prefix the row sees nothing and is zero."""
    check(ops, B, 8, 2, 1, 300, [-1 if i % 2 else 20 for i in range(B)], capacity=64)
    check(ops, B, 8, 2, 1, 0, [-1 if i % 2 else 20 for i in range(B)], capacity=64)
    check(ops, B, 8, 2, 2, 0, [-2 if i % 2 else -1 for i in range(B)], capacity=64)


@pytest.mark.parametrize("B,nq,nkv,T,prefix,own", [(64, 32, 8, 2, 9000, 300), (130, 32, 8, 1, 3001, 40), (5, 16, 8, 1, 30000, 10),
                                                   (32, 8, 8, 1, 12345, 600), (300, 8, 1, 1, 1111, 70), (3, 32, 8, 1, 200, 5000)])
def test_sizes(ops, B, nq, nkv, T, prefix, own):
    check(ops, B, nq, nkv, T, prefix, [own - (11 * i) % own // 2 for i in range(B)])


@pytest.mark.parametrize("B", [3, 30])
def test_growing_scores(ops, B):
    # (keys of up to 4 times the size: the scores' fp32 error is up to 4 times as large)
    check(ops, B, 8, 2, 1, 1500, [30] * B, growth=True, slack=1.15)


def test_one_position_for_all_sequences_and_lengths_past_the_pages(ops):
    q, before, cache, want, bound = make(ops, 4, 8, 2, 1, 256, [63] * 4, 256, 64)
    attn = ops.SharedPrefixAttention(4, 8, 2, 256, 64, "cuda")
    assert_close(attn.run(q, before, int32([256]), cache, int32([63]), SCALE).cpu(), want, bound)
    # beyond the pages both are cut to them
    assert_close(attn.run(q, before, int32([2 ** 31 - 1]), cache, int32([63]), SCALE).cpu(), want, bound)
    got = attn.run(q, before, int32([-7]), cache, int32([-1]), SCALE)
    assert got.float().abs().max().item() == 0 and ops.device_status()[0] == 0


@pytest.mark.parametrize("B", [4, 40])
def test_captured_and_on_another_stream(ops, B):
    positions = [i % 50 for i in range(B)]
    q, before, cache, want, bound = make(ops, B, 8, 2, 1, 900, positions, 1000, 64)
    attn = ops.SharedPrefixAttention(B, 8, 2, 1000, 64, "cuda")
    length, position = int32([900]), int32(positions)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = attn.run(q, before, length, cache, position, SCALE)
    side.synchronize()
    assert_close(got.cpu(), want, bound)
    graphs = []
    for _ in range(2):                       # two graphs of one instance, replayed on two streams at once
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = attn.run(q, before, length, cache, position, SCALE)
        graphs.append((graph, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for (graph, out), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert torch.equal(out, got)


@pytest.mark.parametrize("B", [4, 40])
def test_inputs_written_by_the_launch_before(ops, B):
    """Query, keys, positions and lengths come from kernels right before the call, back to back with other calls."""
    positions = [i % 50 for i in range(B)]
    q, before, cache, want, bound = make(ops, B, 8, 2, 1, 900, positions, 1000, 64)
    attn = ops.SharedPrefixAttention(B, 8, 2, 1000, 64, "cuda")
    length, position = int32([900]), int32(positions)
    good = [t.clone() for t in (q, length, position, before.k, before.v)]
    got = []
    for _ in range(10):
        q.zero_(); length.fill_(3); position.fill_(-1); before.k.zero_(); before.v.zero_()
        attn.run(q, before, length, cache, position, SCALE)
        for t, s in zip((q, length, position, before.k, before.v), good):
            t.copy_(s)
        got.append(attn.run(q, before, length, cache, position, SCALE))
    for x in got:
        assert torch.equal(x, got[0])
    assert_close(got[0].cpu(), want, bound)
