"""The operators together, as a server would run them: a long prompt under a window, its pages shared by several
sequences, tokens drawn by given random numbers, then tails of their own under a window. Every stage is compared with
its definition on the very values that it was given."""
import pytest
import torch

from tests.attention_reference import assert_close, attend, window_visible
from tests.sampling_reference import sample

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5
NQ, NKV, G, HIDDEN, VOCAB = 8, 2, 4, 256, 700


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")
    from starter_b200 import ops as ops_mod
    return ops_mod


class Toy:
    """Embedding, one attention layer, tied head: enough for every operator to feed the next."""

    def __init__(self):
        g = torch.Generator().manual_seed(1)
        w = lambda *s: (torch.randn(s, generator=g) * s[0] ** -0.5).to(torch.bfloat16).cuda()  # noqa: E731
        self.embed = torch.randn((VOCAB, HIDDEN), generator=g).to(torch.bfloat16).cuda()
        self.q, self.k, self.v, self.o = w(HIDDEN, NQ * 128), w(HIDDEN, NKV * 128), w(HIDDEN, NKV * 128), w(NQ * 128, HIDDEN)

    def project(self, tokens):
        """tokens [B, T] -> query [B*T, NQ, 128], key and value [B, NKV, T, 128]."""
        x = self.embed[tokens]
        B, T = tokens.shape
        kv = [(x @ w).view(B, T, NKV, 128).transpose(1, 2).contiguous() for w in (self.k, self.v)]
        return (x @ self.q).view(B * T, NQ, 128).contiguous(), *kv

    def logits(self, attended):
        return 4 * (attended @ self.o) @ self.embed.T


def check_rows(got, q, keys, values, visible):
    """One sequence: got [T, NQ*128], q [T, NQ, 128], keys/values [NKV, n, 128], visible [T, n]."""
    for h in range(NKV):
        rows = q[:, h * G:(h + 1) * G].reshape(-1, 128)
        want, bound = attend(rows.cpu(), keys[h].cpu(), values[h].cpu(), visible.repeat_interleave(G, 0), SCALE)
        # (queries and keys of up to 3 times unit size: the scores' fp32 error is that much larger)
        assert_close(got.view(-1, NQ, 128)[:, h * G:(h + 1) * G].reshape(-1, 128).cpu(), want, 1.2 * bound)


def test_prompt_prefix_samples_and_tails(ops):
    toy, g = Toy(), torch.Generator().manual_seed(2)
    P, B, STEPS, WINDOW, SINKS = 301, 6, 5, 100, 4
    prompt = torch.randint(0, VOCAB, (1, P), generator=g).cuda()
    prefix = ops.PagedKV(1, NKV, 320, "cuda", poison=float("nan"))
    q, k, v = toy.project(prompt)
    prefix.scatter(k, v, 0)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    attended = ops.window_prompt_attention(q, prefix, zero, P, SCALE, WINDOW, SINKS)
    pk, pv = prefix.gather(P)
    check_rows(attended, q, pk[0], pv[0], window_visible(range(P), P, WINDOW, SINKS))

    # the first tokens: several draws from the prompt's last logits
    settings = dict(temperature=0.8, top_k=60, top_p=0.95)
    u = torch.rand((STEPS + 1, B), generator=g)
    logits = toy.logits(attended[-1:]).expand(B, -1)
    tokens, logprobs = ops.sample_tokens(logits, u[0].cuda(), **settings)
    drawn = [tokens]

    def check_draw(logits, u, tokens, logprobs):
        for b in range(B):
            token, logprob, border = sample(logits[b].cpu(), u[b].item(), **settings)
            assert border > 1e-7 and tokens[b].item() == token
            assert abs(logprobs[b].item() - logprob) <= 1e-6 * max(1.0, abs(logprob))

    check_draw(logits, u[0], tokens, logprobs)
    cache = ops.PagedKV(B, NKV, 70, "cuda", poison=float("nan"))
    shared = ops.SharedPrefixAttention(B, NQ, NKV, 320, 70, "cuda")
    tail = ops.WindowAttention(B, NQ, NKV, 70, "cuda", 3, 1)
    length = torch.tensor([P], dtype=torch.int32, device="cuda")
    position = torch.zeros(B, dtype=torch.int32, device="cuda")
    for step in range(STEPS):
        q, k, v = toy.project(tokens[:, None])
        cache.scatter(k, v, step)
        attended = shared.run(q, prefix, length, cache, position, SCALE)
        ck, cv = cache.gather(step + 1)
        every = torch.ones((1, P + step + 1), dtype=torch.bool)
        for b in range(B):
            check_rows(attended[b:b + 1], q[b:b + 1], torch.cat([pk[0], ck[b]], 1), torch.cat([pv[0], cv[b]], 1), every)
        near = tail.run(q, cache, position, SCALE)
        for b in range(B):
            check_rows(near[b:b + 1], q[b:b + 1], ck[b], cv[b], window_visible([step], step + 1, 3, 1))
        logits = toy.logits(attended + near)
        tokens, logprobs = ops.sample_tokens(logits, u[step + 1].cuda(), **settings)
        check_draw(logits, u[step + 1], tokens, logprobs)
        drawn.append(tokens)
        position += 1
    assert len({tuple(row) for row in torch.stack(drawn, 1).tolist()}) > 1           # the continuations part
    assert ops.device_status() == [0, 0, 0, 0]


def test_a_step_in_one_graph(ops):
    """Attention over the shared prefix, logits, draw, and the next position, captured once and replayed: the same
    tokens as call by call."""
    toy, g = Toy(), torch.Generator().manual_seed(3)
    P, B, STEPS = 150, 40, 6
    prefix, cache = (ops.PagedKV(n, NKV, 192, "cuda") for n in (1, B))
    prefix.scatter(*toy.project(torch.randint(0, VOCAB, (1, P), generator=g).cuda())[1:], 0)
    keys = toy.project(torch.randint(0, VOCAB, (B, 192), generator=g).cuda())[1:]
    cache.scatter(*keys, 0)                                # (what later positions will see)
    shared = ops.SharedPrefixAttention(B, NQ, NKV, 192, 192, "cuda")
    length = torch.tensor([P], dtype=torch.int32, device="cuda")
    start = torch.randint(0, VOCAB, (B,), generator=g).cuda()
    us = torch.rand((STEPS, B), generator=g).cuda()
    tokens, position, u = start.clone(), torch.full((B,), 20, dtype=torch.int32, device="cuda"), torch.zeros(B, device="cuda")

    def step():
        q = toy.project(tokens[:, None])[0]
        drawn, _ = ops.sample_tokens(toy.logits(shared.run(q, prefix, length, cache, position, SCALE)), u, top_p=0.9)
        tokens.copy_(drawn)
        position.add_(1)

    def run(do):
        tokens.copy_(start)
        position.fill_(20)
        out = []
        for i in range(STEPS):
            u.copy_(us[i])
            do()
            out.append(tokens.clone())
        return torch.stack(out)

    want = run(step)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    assert torch.equal(run(graph.replay), want)


def test_over_an_engines_pages(ops, golden_dir):
    """A view of an engine's layer: its pages after a prompt, seen through a window as wide as the context, give what
    the decode path's attention gives."""
    from starter_b200 import Engine
    engine = Engine(str(golden_dir / "tiny_qwen3"), device="cuda:0")
    list(engine.generate([[3, 5, 7, 11, 13, 17, 19]] * 2, 2))
    state = engine.decode_state
    cache = ops.PagedKV(2, state.w.local_kv_heads, state.capacity, "cuda", block_table=state.block_table,
                        pools=(state.kpools[0], state.vpools[0]))
    nq = state.w.local_q_heads
    q = torch.randn((2, nq, 128), generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
    position = torch.tensor([6], dtype=torch.int32, device="cuda")
    want = ops.SmallQueryAttention(2, nq, state.w.local_kv_heads, state.capacity, "cuda").run(q, cache, position, SCALE)
    got = ops.WindowAttention(2, nq, state.w.local_kv_heads, state.capacity, "cuda", 1000).run(q, cache, position, SCALE)
    k, v = cache.gather(7)
    group = nq // cache.n_kv
    for b in range(2):
        for h in range(cache.n_kv):
            rows = slice(h * group, (h + 1) * group)
            _, bound = attend(q[b, rows].cpu(), k[b, h].cpu(), v[b, h].cpu(), torch.ones((group, 7), dtype=torch.bool), SCALE)
            a, c = (x.view(2, nq, 128)[b, rows].cpu().double() for x in (got, want))
            assert ((a - c).abs() <= 2 * bound).all()      # each of the two is within the bound of the exact rows
