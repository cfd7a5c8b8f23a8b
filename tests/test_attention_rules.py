"""Rules of the windowed and shared-prefix attention that their sources show, and refusals on the host."""
import ctypes as C

from starter_b200._lib import lib
from tests.test_bounded_ops_cpu import A, layout, refused


def test_windowed_prompts_refuse_more_tokens_than_positions_count():
    def call(T, window=5):
        return lib.q_attention_window_prefill(A, C.byref(layout()), A, 0, A, 1, T, 8, window, 0, 0.1, None)
    refused(call(2 ** 30 + 1), "tokens")
    refused(call(2 ** 31 - 1), "tokens")
    refused(call(0), "bad batch/T/heads")
    refused(call(-5), "bad batch/T/heads")
