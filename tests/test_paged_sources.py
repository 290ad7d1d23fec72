"""How the many-rows attention kernel ends when a wait runs out.  No such end can be brought about on a shared GPU, so what it rests on is
read from the source: every wait is bounded and decided by the warp as one, and warps meet only where a limit holds."""
import os
import re

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "relax_b200", "csrc", "paged_attn_prompt.cu")


def code():
    with open(SOURCE) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def test_warps_of_a_tile_meet_within_a_limit():
    """A named barrier of the four warps would never be complete once one of them has left its loop."""
    text = code()
    assert "bar_sync(" not in text and "bar.sync" not in text and "__syncthreads_" not in text
    body = text[text.index("paged_prompt_kernel(const __grid_constant__"):text.index("int launch_paged_prompt")]
    loops = body[body.index("if (warp < 4)"):body.index("if (*abort_flag) {")]
    assert "__syncthreads()" not in loops
    meeting = re.findall(r"[^\n]*tile_barrier\(\)[^\n]*;", loops)
    assert len(meeting) == 3 and all("if (!tile_barrier()) break;" in line for line in meeting)


def test_the_lanes_of_a_warp_give_up_together():
    """Tensor memory is read by whole warps: a lane that saw a barrier complete must not go on where another one gave up."""
    text = code()
    waits = text[text.index("bool wait_long("):text.index("void exp2_poly(")] if "bool wait_long(" in text else ""
    assert waits and text.count("mbar_try_wait(") == waits.count("__all_sync(0xffffffffu, mbar_try_wait(bar, parity))") == 3
    assert not re.search(r"\bmbar_wait", text)
    assert "__any_sync(0xffffffffu, *abort_flag" in waits and "kWaitNs" in waits


def test_the_few_rows_kernel_ends_whatever_the_lengths_do():
    """A warp reads the lengths more than once.  Where they change in between (a caller that writes them on another stream, which gives no
    result), its walk over the sequences stays inside the batch, and a sequence without work does not keep it where it is."""
    with open(SOURCE.replace("paged_attn_prompt", "paged_attn_decode")) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    walk = text[text.index("int pieces = 0;"):text.index("__syncthreads();", text.index("int pieces = 0;"))]
    assert "while (at < end && per_tile > 0) {" in walk
    assert re.findall(r"units_of\([^)]*\)", walk) == ["units_of(b, per_tile)"] and "b < p.c.batch ? units_of(b, per_tile) : 0" in walk
    assert "while (seq_units == 0 && b < p.c.batch);" in walk
