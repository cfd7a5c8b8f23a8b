"""Refusals of the windowed, shared-prefix and sampling operators: all on the host, before any launch."""
import ctypes as C

import pytest
import torch

A = 4096          # a made-up, aligned address: nothing is launched


def layout(nkv=2, pages=3, k=A, v=A, table=A):
    from starter_b200._lib import KVLayout
    return KVLayout(k, v, table, pages, nkv)


def refused(rc, text=None):
    from starter_b200 import _lib
    message = (_lib.lib.q_last_error() or b"").decode()
    assert rc == -1, message
    if text:
        assert text in message, message


def test_window_attention_refuses_bad_arguments():
    from starter_b200._lib import lib
    kv = layout()

    def call(q=A, kv=kv, pos=A, out=A, batch=1, T=1, nq=8, window=5, sinks=0):
        return lib.q_attention_window(q, C.byref(kv) if kv else None, pos, 0, out, batch, T, nq, window, sinks, 0.1, None)
    refused(call(q=None), "null")
    refused(call(kv=None), "null")
    refused(call(pos=None), "null")
    refused(call(out=None), "null")
    refused(call(q=A + 8), "aligned")
    refused(call(kv=layout(k=A + 8)), "aligned")
    refused(call(pos=A + 2), "aligned")
    refused(call(kv=layout(pages=0)), "incomplete")
    refused(call(batch=0))
    refused(call(T=0))
    refused(call(nq=7))
    refused(call(nq=2, T=33), "32 query rows")
    refused(call(window=0), "window")
    refused(call(sinks=-1), "sinks")
    refused(call(batch=40000), "too many")


def test_window_attention_class_refuses_before_a_launch():
    from starter_b200 import ops
    for bad in (dict(window=0), dict(window=5, sinks=-1), dict(window=5, tokens_per_seq=9), dict(window=2 ** 31)):
        with pytest.raises(ValueError):
            ops.WindowAttention(1, 32, 8, 100, "cuda", **bad)
    with pytest.raises(ValueError):
        ops.WindowAttention(1, 32, 8, 100, "cpu", 5)
    attn = ops.WindowAttention(1, 8, 2, 100, "cuda", 5)
    cache = ops.PagedKV(1, 2, 100, "cpu")
    with pytest.raises(ValueError):
        attn.run(torch.zeros((1, 8, 128), dtype=torch.bfloat16), cache, torch.zeros(1, dtype=torch.int32), 0.1)


def test_caches_over_given_pages():
    from starter_b200 import ops
    k, v = (torch.zeros((6, 2, 64, 128), dtype=torch.bfloat16) for _ in range(2))
    cache = ops.PagedKV(2, 2, 150, "cpu", pools=(k, v))
    assert cache.k is k and cache.v is v and cache.layout.d_kpool == k.data_ptr()
    table = torch.tensor([[5, 0]], dtype=torch.int32)
    assert ops.PagedKV(1, 2, 100, "cpu", block_table=table, pools=(k, v)).block_table is table
    for bad in (dict(pools=(k[:5], v[:5])), dict(pools=(k, v[:5])), dict(pools=(k.float(), v.float())),
                dict(pools=(k, v), poison=1.0), dict(pools=(k[:, :1], v[:, :1]))):
        with pytest.raises(ValueError):
            ops.PagedKV(2, 2, 150, "cpu", **bad)


def test_window_prompt_refuses_bad_arguments():
    from starter_b200._lib import lib
    kv = layout()

    def call(q=A, kv=kv, pos=A, out=A, batch=1, T=1, nq=8, window=5, sinks=0):
        return lib.q_attention_window_prefill(q, C.byref(kv) if kv else None, pos, 0, out, batch, T, nq, window, sinks, 0.1, None)
    refused(call(q=None), "null")
    refused(call(kv=None), "null")
    refused(call(out=None), "null")
    refused(call(q=A + 8), "aligned")
    refused(call(out=A + 2), "aligned")
    refused(call(pos=A + 2), "aligned")
    refused(call(kv=layout(pages=0)), "incomplete")
    refused(call(T=0))
    refused(call(nq=7))
    refused(call(nq=66), "exceed 32")
    refused(call(window=0), "window")
    refused(call(sinks=-1), "sinks")


def test_shared_prefix_refuses_bad_arguments():
    from starter_b200._lib import lib
    kv = layout()

    def call(q=A, prefix=kv, length=A, kv=kv, pos=A, scratch=A, out=A, batch=2, T=1, nq=8):
        return lib.q_attention_shared(q, C.byref(prefix) if prefix else None, length, C.byref(kv) if kv else None, pos, 0,
                                      scratch, out, batch, T, nq, 0.1, None)
    for name in ("q", "prefix", "length", "kv", "pos", "scratch", "out"):
        refused(call(**{name: None}), "null")
    refused(call(q=A + 8), "aligned")
    refused(call(scratch=A + 8), "aligned")
    refused(call(length=A + 1), "aligned")
    refused(call(prefix=layout(k=A + 8)), "aligned")
    refused(call(prefix=layout(nkv=4)), "different kv heads")
    refused(call(prefix=layout(v=None)), "incomplete")
    refused(call(prefix=layout(pages=0)), "too many")
    refused(call(nq=2, T=33), "32 query rows")
    refused(call(batch=0))
    assert lib.q_attention_shared_scratch_bytes(2, 1, 8, 2, 10) > 0
    for bad in ((0, 1, 8, 2, 10), (2, 0, 8, 2, 10), (2, 1, 7, 2, 10), (2, 1, 8, 0, 10), (2, 9, 8, 2, 10), (2, 1, 8, 2, 0)):
        assert lib.q_attention_shared_scratch_bytes(*bad) == 0


def test_shared_prefix_class_refuses_before_a_launch():
    from starter_b200 import ops
    with pytest.raises(ValueError):
        ops.SharedPrefixAttention(1, 32, 8, 0, 100, "cuda")
    with pytest.raises(ValueError):
        ops.SharedPrefixAttention(1, 32, 8, 100, 100, "cpu")
    with pytest.raises(ValueError):
        ops.SharedPrefixAttention(1, 32, 8, 100, 100, "cuda", 9)


def test_sampling_refuses_bad_arguments():
    from starter_b200._lib import Sampling, lib

    def call(x=A, u=A, s=Sampling(1.0, 0, 1.0, 0.0), tokens=A, logprobs=A, rows=2, vocab=10, stride=10, fp32=1):
        return lib.q_sample_tokens(x, fp32, stride, u, C.byref(s) if s else None, tokens, logprobs, rows, vocab, None)
    for name in ("x", "u", "s", "tokens", "logprobs"):
        refused(call(**{name: None}), "null")
    refused(call(rows=0))
    refused(call(vocab=0))
    refused(call(vocab=2 ** 19 + 1))
    refused(call(stride=-1), "stride")
    refused(call(s=Sampling(-0.5, 0, 1.0, 0.0)), "temperature")
    refused(call(s=Sampling(float("nan"), 0, 1.0, 0.0)), "temperature")
    refused(call(s=Sampling(1.0, 0, float("nan"), 0.0)), "NaN")
    refused(call(s=Sampling(1.0, 0, 1.0, float("nan"))), "NaN")
    refused(call(x=A + 2), "aligned")
    refused(call(x=A + 1, fp32=0), "aligned")
    refused(call(tokens=A + 4), "aligned")
    refused(call(s=Sampling(1.0, 0, 1.0, 0.0, None, A + 2)), "aligned")


def test_sampling_operator_refuses_before_a_launch():
    from starter_b200 import ops
    with pytest.raises(ValueError):
        ops.sample_tokens(torch.zeros((2, 5)), torch.zeros(2))


def test_sampling_reference():
    """Known answers of the definition that the GPU tests compare with."""
    from tests.sampling_reference import sample
    x = torch.tensor([1.0, 3.0, 2.0, 3.0])
    assert sample(x, 0.9, temperature=0.0)[0] == 1
    assert sample(x, 0.9, top_k=1)[0] == 1 and sample(x, 0.6, top_k=2)[0] == 3
    p = torch.softmax(x.double(), 0)
    for u in (0.0, 0.03, 0.5, 0.7, 0.999):
        assert sample(x, u)[0] == int((p.cumsum(0) <= u).sum())
    # weights 0.135, 1, 0.368, 1 of 2.503: the first of the set has 0.3995
    assert sample(x, 0.99, top_p=0.5)[0] == 3 and sample(x, 0.99, top_p=0.39)[0] == 1
    assert sample(x, 0.99, min_p=0.5)[0] == 3 and sample(x, 0.99, min_p=0.3)[0] == 3
    assert sample(x, 0.45, min_p=0.3)[0] == 2                  # of ids 1, 2, 3 with weights 1, 0.37, 1
    assert sample(torch.full((3,), -torch.inf), 0.5)[0] == -1
