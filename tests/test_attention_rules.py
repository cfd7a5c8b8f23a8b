"""Rules of the windowed and shared-prefix attention that their sources show, and refusals on the host."""
import ctypes as C
import re

from starter_b200._lib import lib
from tests.test_bounded_ops_cpu import A, layout, refused
from tests.test_kernel_waits import between, source


def test_windowed_prompts_refuse_more_tokens_than_positions_count():
    def call(T, window=5):
        return lib.q_attention_window_prefill(A, C.byref(layout()), A, 0, A, 1, T, 8, window, 0, 0.1, None)
    refused(call(2 ** 30 + 1), "tokens")
    refused(call(2 ** 31 - 1), "tokens")
    refused(call(0), "bad batch/T/heads")
    refused(call(-5), "bad batch/T/heads")


def flat(text):
    return re.sub(r"\s+", " ", text)


def test_few_row_attention_reads_nothing_before_its_dependency_wait():
    """Position, table, queries and keys may be what the launch right before writes; and dependents that read early may
    start only when whatever came before this launch is complete."""
    kernel = between(source("attn_rows.cu"), "k_attn_rows(RowsArgs a, int* status) {", "\nstruct RowsPlan")
    wait = kernel.index("if (!a.early) pdl_wait();")
    assert not re.search(r"seen_of\(|__ldcg\(|a\.pos\b|a\.table\b|a\.q\b|copy_rows\(", kernel[:wait])
    assert kernel.index("pdl_launch_dependents();") > wait and kernel.count("pdl_launch_dependents();") == 1


def test_the_join_waits_for_the_prefix_before_it_reads_or_writes_results():
    """q_attention_shared's second launch reads its own keys under the first one's tail: it may, since the first one has
    passed its own wait before it releases its dependents. What the first one writes, and the result, come behind the
    second wait."""
    text = source("attn_rows.cu")
    kernel = between(text, "k_attn_rows(RowsArgs a, int* status) {", "\nstruct RowsPlan")
    wait = kernel.index("if (a.early) pdl_wait();")
    assert not re.search(r"a\.parts|a\.out|parts_used", kernel[:wait])
    shared = between(text, 'extern "C" int q_attention_shared(', "\n}\n")
    first, second = shared.split("a.early = true;")
    assert "early" not in first and "rows_launch(s.plan" in first and "q_attention_parts_tc(" in first
    assert "rows_launch(p, a," in second and text.count("a.early = true;") == 1
    prompt = source("attn_prompt.cu")
    kernel = prompt[prompt.index("__global__"):]
    after = kernel[kernel.index("pdl_wait();"):]
    assert after.index("if (FORM != CAUSAL) pdl_launch_dependents();") < after.index("int pos = ")
    assert "if (FORM == CAUSAL) pdl_launch_dependents();" in kernel[:kernel.index("pdl_wait();")]


def test_no_cta_writes_into_another_before_it_runs():
    """Stores into the shared memory of a cluster's other CTAs come behind the barrier that says that they have begun."""
    rows = between(source("attn_rows.cu"), "k_attn_rows(RowsArgs a, int* status) {", "\nstruct RowsPlan")
    consumers = rows[rows.index("const int g = lane >> 2"):]
    assert consumers.index("barrier.cluster.wait.acquire") < consumers.index("remote_addr(")
    assert "remote_addr(" not in rows[:rows.index("const int g = lane >> 2")]
    sample = between(source("sampling.cu"), "k_sample(const SampleArgs a) {", "\ncudaError_t sample_room")
    begun = sample.index("barrier.cluster.wait.acquire")
    assert begun < min(sample.index("put32("), sample.index("put64("), sample.index("get32("), sample.index("at_rank("))


def test_few_row_attention_leaves_no_copy_in_flight():
    """Also where a wait ran out: every copy that was asked for is waited for before the CTA may leave, with a limit."""
    kernel = between(source("attn_rows.cu"), "k_attn_rows(RowsArgs a, int* status) {", "\nstruct RowsPlan")
    producer = between(kernel, "if (warp == DC) {", "} else {\n")
    loop, drain = producer.split("for (int j = max(0, it - NS); j < it; ++j)")
    assert "copy_rows(" in loop and "copy_rows(" not in drain and "mbar_wait_plain(" in drain
    assert drain.index("mbar_wait_plain(") < drain.index("barrier.cluster.wait.acquire")
    assert not re.search(r"\bwhile \(!?mbar_try|mbar_try\(", kernel)


def test_three_groups_of_warps_keep_to_their_stages():
    """A stage is a group's own, so that the group can track its parity."""
    text = source("attn_rows.cu")
    assert "if (p.dg == 3) p.stages = 3;" in text and "for (int it = tg; it < ntiles; it += DG)" in text
    sizes = between(text, "void rows_sizes(", "\n}\n")
    assert sizes.index("if (each < p.stages)") < sizes.index("if (p.dg == 3) p.stages = 3;")


def test_the_deep_form_commits_nothing_that_nobody_waits_for():
    """After the last products of a CTA only B_OF is committed, which the softmax warps wait for: an arrival after that
    could come into shared memory that is another CTA's by then."""
    deep = flat(between(source("attn_prompt.cu"), "auto ahead = [&]() {", "int r = 0;"))
    products = deep[deep.index("while (ok && v.more)"):]
    advance, guard = products.index("v.next(sh, items, pos, pos_ptr);"), products.index("if (v.more) {")
    assert advance < guard
    assert products[guard:].startswith("if (v.more) { tc_commit(bar(B_VE, buf)); tc_commit(bar(B_PV, 0)); } if (last) tc_commit(bar(B_OF, 0));")
    assert products.count("tc_commit(") == 3


def test_the_sampler_reads_nothing_before_its_dependency_wait():
    kernel = between(source("sampling.cu"), "k_sample(const SampleArgs a) {", "\ncudaError_t sample_room")
    wait = kernel.index("pdl_wait();")
    assert not re.search(r"__ldcg\(|raw\(|a\.x\b|a\.u\b|a\.tokens|a\.logprobs", kernel[:wait])
    assert kernel.index("pdl_launch_dependents();") > wait and kernel.count("pdl_launch_dependents();") == 1
