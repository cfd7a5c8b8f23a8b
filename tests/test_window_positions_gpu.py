"""Windowed attention of rows at the end of the pages and behind it. The block table is a slice of a larger tensor whose
other entries name a page of NaN, as do its own entries of pages that nobody sees: a stray read of the table, or of such a
page, shows in the result (in bounds of the pools, whatever is read). Rows behind the pages see what their window still
holds of them, and the sinks."""
import pytest
import torch

from tests.attention_reference import assert_close, attend, window_visible

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5
FAR = 2 ** 31 - 1


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")
    from starter_b200 import ops as ops_mod
    return ops_mod


def check(ops, run, B, nq, nkv, T, positions, window, sinks, capacity, begins=-2 ** 31):
    """run(query, cache, position) against the definition; rows see keys below their position, at most the pages'.
    begins: positions below it count as it."""
    g = torch.Generator().manual_seed(B + T + window)
    G, pages = nq // nkv, capacity // 64
    q = torch.randn((B * T, nq, 128), generator=g).to(torch.bfloat16)
    k, v = (torch.randn((B, nkv, capacity, 128), generator=g).to(torch.bfloat16) for _ in range(2))
    bad = B * pages                                          # the page of NaN
    wide = torch.full((B + 2, pages), bad, dtype=torch.int32, device="cuda")
    wide[1:B + 1] = torch.randperm(bad, generator=g).to(torch.int32).view(B, pages).cuda()
    cache = ops.PagedKV(B, nkv, capacity, "cuda", block_table=wide[1:B + 1],
                        pools=tuple(torch.full((bad + 1, nkv, 64, 128), float("nan"), dtype=torch.bfloat16, device="cuda")
                                    for _ in range(2)))
    want, bound = (torch.zeros((B, T, nq, 128), dtype=torch.float64) for _ in range(2))
    dead = torch.zeros((B, pages), dtype=torch.bool)
    for b in range(B):
        visible = window_visible([max(positions[b], begins) + t for t in range(T)], capacity, window, sinks)
        seen = visible.any(0)
        dead[b] = ~seen.view(pages, 64).any(1)
        k[b][:, ~seen] = float("nan")
        v[b][:, ~seen] = float("nan")
        for h in range(nkv):
            rows = q.view(B, T, nq, 128)[b, :, h * G:(h + 1) * G].reshape(T * G, 128)
            o, e = attend(rows, k[b, h], v[b, h], visible.repeat_interleave(G, 0), SCALE)
            want[b, :, h * G:(h + 1) * G], bound[b, :, h * G:(h + 1) * G] = o.view(T, G, 128), e.view(T, G, 128)
    cache.scatter(k.cuda(), v.cuda(), 0)
    wide[1:B + 1][dead.cuda()] = bad
    got = run(q.cuda(), cache, torch.tensor(positions, dtype=torch.int32, device="cuda"))
    assert ops.device_status()[0] == 0
    assert_close(got.cpu(), want.view(B * T, -1), bound.view(B * T, -1))


@pytest.mark.parametrize("nq,nkv,T", [(4, 1, 1), (32, 8, 1), (8, 2, 4), (28, 4, 4), (4, 4, 32)])
@pytest.mark.parametrize("window,sinks", [(10, 0), (64, 0), (70, 5), (1000, 0), (1, 64), (FAR, 0)])
def test_a_few_rows(ops, nq, nkv, T, window, sinks):
    def run(q, cache, position):
        return ops.WindowAttention(len(positions), nq, nkv, 192, "cuda", window, sinks, T).run(q, cache, position, SCALE)
    positions = [192 - T, 190, 191, 192, 193, 200, 250, 192 + 64, 1191, 2 ** 20, 2 ** 30 + 7, FAR, 0, -T, -2 ** 31]
    if window == FAR:                                        # (counted up to 2^31 - 65, positions as well)
        positions = positions[:11]
    check(ops, run, len(positions), nq, nkv, T, positions, window, sinks, 192)


@pytest.mark.parametrize("nq,nkv,T", [(4, 1, 40), (32, 8, 1), (8, 2, 129), (28, 4, 200), (32, 8, 500)])
@pytest.mark.parametrize("window,sinks", [(10, 0), (64, 0), (70, 5), (300, 0), (1, 200), (FAR, 0)])
def test_prompts(ops, nq, nkv, T, window, sinks):
    """One query tile for a block and (the last shape) two; blocks that begin before the pages' end and end behind it."""
    def run(q, cache, position):
        return ops.window_prompt_attention(q, cache, position, T, SCALE, window, sinks)
    positions = [384 - T // 2, 320, 383, 384, 1000, 0, -5, 2 ** 20, 2 ** 30]
    if window != FAR:                                        # (counted up to 2^31 - 512 - T, positions as well)
        positions += [FAR]
    check(ops, run, len(positions), nq, nkv, T, positions, window, sinks, 384, begins=0)


def test_prompts_wholly_behind_the_pages(ops):
    """No row sees anything, and the first item of a block has nothing to read."""
    for T in (1, 40, 300):
        def run(q, cache, position):
            return ops.window_prompt_attention(q, cache, position, T, SCALE, 50, 0)
        check(ops, run, 3, 8, 2, T, [192 + 50, 500, 2 ** 30], 50, 0, 192, begins=0)


@pytest.mark.parametrize("batch", [2, 40])
def test_own_keys_of_a_shared_prefix(ops, batch):
    """A position behind the own pages sees all that they hold."""
    g = torch.Generator().manual_seed(batch)
    nkv, G, T = 2, 4, 4
    prefix, cache = ops.PagedKV(1, nkv, 100, "cuda"), ops.PagedKV(batch, nkv, 64, "cuda")
    k0, v0 = (torch.randn((1, nkv, 100, 128), generator=g).to(torch.bfloat16) for _ in range(2))
    k, v = (torch.randn((batch, nkv, 64, 128), generator=g).to(torch.bfloat16) for _ in range(2))
    prefix.scatter(k0.cuda(), v0.cuda(), 0)
    cache.scatter(k.cuda(), v.cuda(), 0)
    q = torch.randn((batch * T, nkv * G, 128), generator=g).to(torch.bfloat16)
    attn = ops.SharedPrefixAttention(batch, nkv * G, nkv, 100, 64, "cuda", T)
    positions = [FAR, 64] + [2 ** 20] * (batch - 2)
    got = attn.run(q.cuda(), prefix, torch.tensor([100], dtype=torch.int32, device="cuda"), cache,
                   torch.tensor(positions, dtype=torch.int32, device="cuda"), SCALE).cpu().view(batch, T, nkv * G, 128)
    for b in {0, 1, batch - 1}:
        for h in range(nkv):
            keys, values = torch.cat([k0[0, h], k[b, h]]), torch.cat([v0[0, h], v[b, h]])
            rows = q.view(batch, T, nkv * G, 128)[b, :, h * G:(h + 1) * G].reshape(T * G, 128)
            want, bound = attend(rows, keys, values, torch.ones((T * G, 164), dtype=torch.bool), SCALE)
            assert_close(got[b, :, h * G:(h + 1) * G].reshape(T * G, 128), want, bound)
