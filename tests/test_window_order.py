"""CPU: rows of values that the windowed attention blanks in shared memory are written by ordinary stores, and read or written
again by the asynchronous proxy: by a product in the one kernel, by the copy that refills the stage in the other.  Only a proxy
fence ahead of the hand-over orders the two; without it zeros could land over fresh values, now and then.  So the order is looked up in the sources."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bytetransformer_b200", "csrc")


def _body(start):
    src = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, "window_mha.cu")).read())
    at = src.index(start)
    return src[at:src.index("\n}\n", at)]


BLANK = "= make_uint4(0u, 0u, 0u, 0u);"


def test_the_block_kernel_fences_between_blanking_and_the_product():
    body = _body("window_mha_kernel(const")
    assert body.count(BLANK) == 1
    blank = body.index(BLANK)
    assert blank < body.index("fence_proxy_async_smem();", blank) < body.index("mbar_arrive(&p_full[g])", blank)


def test_the_few_query_kernel_fences_between_blanking_and_the_next_copy():
    body = _body("window_few_kernel(const")
    assert body.count(BLANK) == 1
    blank = body.index(BLANK)
    fence = body.index("fence_proxy_async_smem();", blank)
    refill = body.index("fetch(step + kFewStages * kFewWarps, stage)", blank)
    # every lane that stored fences, and the warp meets before one of its lanes asks for the copy
    assert blank < fence < body.index("__syncwarp();", fence) < refill
