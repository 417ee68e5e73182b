"""Orders that kernels have to keep and no run shows: read off the sources."""

import pytest

from simple_inference_autoresearch_b200.kernels import build


def body_of(unit, kernel):
    """The text of a kernel from its name to the end of its braces."""
    text = (build.CSRC / f"{unit}.cu").read_text()
    at = text.index("{", text.index(f"\n{kernel}("))
    depth, i = 1, at + 1
    while depth:
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        i += 1
    return text[at:i]


@pytest.mark.parametrize("unit,kernel", [("attention_quant", "attn_quant_kernel"), ("attention_quant_tc", "attn_quant_tc_kernel")])
def test_loads_of_what_kernels_in_front_stored_follow_a_fence(unit, kernel):
    """Rows, queries and tiles are written by ordinary stores of the kernel in front and read here through the asynchronous
    proxy: behind the wait for that kernel, in front of the first load, the two have to be ordered."""
    body = body_of(unit, kernel)
    wait, fence = body.index("pdl_wait();"), body.index("fence.proxy.async.global;")
    loads = [body.index(w) for w in ("tma_load_2d(", "tma_load_3d(", "bulk_load(") if w in body]
    assert wait < fence < min(loads)


def test_tensor_memory_is_taken_between_the_wait_and_the_next_kernels_start():
    """Two blocks of 256 columns fill an SM's 512.  Products take columns in front of their wait for the kernel in front;
    one that starts beside a block of this kernel that has none yet would leave the two waiting for each other.  And in
    front of this kernel's own wait a product may still be about to take its columns."""
    body = body_of("attention_quant_tc", "attn_quant_tc_kernel")
    assert body.index("pdl_wait();") < body.index("tmem_alloc(") < body.index("__syncthreads();") < body.index("pdl_launch_dependents();")
    assert body.count("pdl_launch_dependents();") == 1 and body.count("tmem_alloc(") == 1


@pytest.mark.parametrize("unit,kernel", [("attention_tc", "attn_prefill_tc_kernel"), ("attention_quant_tc", "attn_quant_tc_kernel")])
def test_the_loading_thread_waits_for_its_last_copies_on_every_way_out(unit, kernel):
    """Another warp may give up after the last load was issued: the copies have to land before the block leaves all the same."""
    body = body_of(unit, kernel)
    at = body.index("for (int i = max(0, issued_k - kStages); i < issued_k; ++i) mbar_wait(&k_full")
    loop_end = body.rindex("issued_v = i + 1;", 0, at)
    between = body[loop_end:at]
    assert "if (" not in between.replace("if (bad_page)", "") and "mbar_wait(&q_full, 0);" in between
