"""Calls of the windowed and shared-prefix attention and of the sampler at their limits: pages and rows whose offsets pass
32 bits, calls from several threads at once, captured calls that live beside one another."""
import threading

import pytest
import torch

from tests.attention_reference import assert_close, attend, window_visible
from tests.sampling_reference import sample

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")
    from starter_b200 import ops as ops_mod
    return ops_mod


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def test_pages_far_into_a_large_pool(ops):
    """Pages behind the first 2^31 numbers of a pool (and 4 GB): each form of attention over them."""
    nkv, group, tokens = 8, 2, 200
    g = torch.Generator().manual_seed(5)
    pools = tuple(torch.empty((33000, nkv, 64, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    assert pools[0].numel() > 2 ** 31
    table = int32([32999, 7, 32990, 32780]).view(1, 4)
    pages = ops.PagedKV(1, nkv, tokens, "cuda", block_table=table, pools=pools)
    k, v = (torch.randn((1, nkv, tokens, 128), generator=g).to(torch.bfloat16) for _ in range(2))
    pages.scatter(k.cuda(), v.cuda(), 0)
    own_table = int32([[32998], [8], [32777]] * 8)          # (several sequences may share a page)
    own = ops.PagedKV(24, nkv, 64, "cuda", block_table=own_table, pools=pools)
    own.k[own_table[:3, 0].long()] = 0
    own.v[own_table[:3, 0].long()] = 0
    q = torch.randn((tokens, nkv * group, 128), generator=g).to(torch.bfloat16)

    def check(got, rows, visible, keys, values):
        for h in range(nkv):
            part = q[rows, h * group:(h + 1) * group].reshape(-1, 128)
            want, bound = attend(part, keys[h], values[h], visible.repeat_interleave(group, 0), SCALE)
            assert_close(got.view(-1, nkv * group, 128)[:, h * group:(h + 1) * group].reshape(-1, 128).cpu(), want, bound)

    last = slice(tokens - 1, tokens)
    one = ops.WindowAttention(1, nkv * group, nkv, tokens, "cuda", 150, 3)
    check(one.run(q[last].cuda(), pages, int32([tokens - 1]), SCALE), last, window_visible([tokens - 1], tokens, 150, 3), k[0], v[0])
    check(ops.window_prompt_attention(q.cuda(), pages, int32([0]), tokens, SCALE, 150, 3), slice(0, tokens),
          window_visible(range(tokens), tokens, 150, 3), k[0], v[0])
    for batch in (2, 24):                                   # rows of one kv head: 4 and 48
        cache = ops.PagedKV(batch, nkv, 64, "cuda", block_table=own_table[:batch].contiguous(), pools=pools)
        attn = ops.SharedPrefixAttention(batch, nkv * group, nkv, tokens, 64, "cuda")
        got = attn.run(q[:batch].cuda(), pages, int32([tokens]), cache, int32([0]), SCALE)
        zero = torch.zeros((nkv, 1, 128), dtype=torch.bfloat16)
        check(got, slice(0, batch), torch.ones((batch, tokens + 1), dtype=torch.bool), torch.cat([k[0], zero], 1), torch.cat([v[0], zero], 1))
    assert ops.device_status() == [0, 0, 0, 0]


@pytest.mark.parametrize("settings", [dict(), dict(top_k=30, top_p=0.9), dict(top_p=0.8)], ids=str)
def test_rows_far_apart(ops, settings):
    """Rows whose numbers lie 2^30 and more apart."""
    g = torch.Generator().manual_seed(6)
    x, u = 2 * torch.randn((3, 9001), generator=g).to(torch.bfloat16), torch.rand(3, generator=g)
    stride = 2 ** 30 + 5
    far = torch.empty(2 * stride + 9001, dtype=torch.bfloat16, device="cuda").as_strided((3, 9001), (stride, 1))
    far.copy_(x)
    tokens, logprobs = ops.sample_tokens(far, u.cuda(), **settings)
    for r in range(3):
        token, logprob, border = sample(x[r], u[r].item(), **settings)
        assert border > 1e-7 and tokens[r].item() == token
        assert abs(logprobs[r].item() - logprob) <= 2.0 ** -24 * abs(logprob) + 1e-7


@pytest.mark.parametrize("dtype,vocab", [(torch.bfloat16, v) for v in (80000, 88000, 89500, 91000, 92160, 95000)] +
                         [(torch.float32, v) for v in (41000, 44400, 45500, 46080, 47000)])
def test_rows_that_just_fit_a_block(ops, dtype, vocab):
    """Many rows, a block to each: up to its shared memory's end and beyond."""
    g = torch.Generator().manual_seed(8)
    x, u = (2 * torch.randn((160, vocab), generator=g)).to(dtype), torch.rand(160, generator=g)
    tokens, _ = ops.sample_tokens(x.cuda(), u.cuda(), top_k=50)
    for r in (0, 80, 159):
        token, _, border = sample(x[r], u[r].item(), top_k=50)
        assert border > 1e-7 and tokens[r].item() == token


def calls(ops):
    """Operators of several shapes on fixed inputs: [a function that gives a tensor]."""
    g = torch.Generator().manual_seed(7)
    made = []

    def normal(*shape):
        return torch.randn(shape, generator=g).to(torch.bfloat16).cuda()

    def cache(batch, nkv, capacity):
        c = ops.PagedKV(batch, nkv, capacity, "cuda")
        c.k.copy_(normal(*c.k.shape))
        c.v.copy_(normal(*c.v.shape))
        return c

    for B, nq, nkv, capacity in [(1, 32, 8, 3000), (3, 16, 8, 700), (40, 32, 8, 200), (6, 32, 4, 500)]:
        c, q, attn = cache(B, nkv, capacity), normal(B, nq, 128), ops.WindowAttention(B, nq, nkv, capacity, "cuda", 400, 4)
        made.append(lambda c=c, q=q, a=attn, p=int32([capacity - 1]): a.run(q, c, p, SCALE))
    # one instance of the shared form, prefixes of different page counts
    attn = ops.SharedPrefixAttention(12, 16, 4, 100, 70, "cuda")
    own, q, at, start = cache(12, 4, 70), normal(12, 16, 128), int32([69]), int32([0])
    for capacity in (100, 6000):
        made.append(lambda pre=cache(1, 4, capacity), n=int32([capacity]): attn.run(q, pre, n, own, at, SCALE))
    c, prompt = cache(1, 2, 333), normal(333, 8, 128)
    made.append(lambda: ops.window_prompt_attention(prompt, c, start, 333, SCALE, 90, 4))
    for rows, vocab in [(1, 60000), (5, 9000), (70, 20000)]:
        x, u = 3 * normal(rows, vocab), torch.rand(rows, generator=g).cuda()
        made.append(lambda x=x, u=u: ops.sample_tokens(x, u, top_p=0.9)[1])
        made.append(lambda x=x.float(), u=u: ops.sample_tokens(x, u, top_k=20)[1])
    return made


def test_threads_with_streams_of_their_own(ops):
    made = calls(ops)
    want = [f() for f in made]
    torch.cuda.synchronize()
    wrong = []

    def work(n):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for again in range(8):
                    for i in range(len(made)):
                        at = (i * (2 * n + 1) + n) % len(made)
                        if not torch.equal(made[at](), want[at]):
                            wrong.append((n, at))
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(n,)) for n in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_graphs_beside_one_another(ops):
    """All of them captured twice into graphs that live at once, replayed in turn on two streams."""
    made = calls(ops)
    want = [f() for f in made]
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = [f() for f in made]
        graphs.append((graph, out, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for again in range(4):
        for graph, out, stream in graphs:
            with torch.cuda.stream(stream):
                for x in out:
                    x.zero_()
                graph.replay()
    torch.cuda.synchronize()
    for graph, out, stream in graphs:
        assert all(torch.equal(x, w) for x, w in zip(out, want))
    assert ops.device_status() == [0, 0, 0, 0]
