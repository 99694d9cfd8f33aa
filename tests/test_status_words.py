"""Status words: what clears one has run when the call that told it returns.  Read from the source, since no timing on the GPU shows it for certain."""

import pytest

from kiln_b200 import _cabi


def body(name, entry):
    text = (_cabi.CSRC_DIR / name).read_text()
    at = text.index(f"KB200_EXPORT int {entry}(")
    return text[at:text.index("\n}\n", at)]


@pytest.mark.parametrize("name, entry", [("cache.cu", "kb200_cache_status"), ("plan.cu", "kb200_plan_status")])
def test_a_status_word_is_cleared_before_it_is_told(name, entry):
    """A memset or a kernel on the legacy stream is not waited for by non-blocking streams such as torch's: without a wait, what the next call there says
    could be erased."""
    text = body(name, entry)
    clear = max(text.rfind("cudaMemset("), text.rfind("<<<"), text.rfind("attention_reset_arrivals("))
    assert clear > 0 and text.index("cudaStreamSynchronize(cudaStreamLegacy)", clear) < text.index("return fail(", clear)


def test_a_cache_clears_what_it_told_and_nothing_else():
    """Calls on other streams may be under way, and set bits between the look and the clearing."""
    text = body("cache.cu", "kb200_cache_status")
    assert "cudaMemset" not in text and "told_kernel<<<1, 1, 0, cudaStreamLegacy>>>(c.view.status, word)" in text
