"""CPU checks of the generation kernels' sources and C entry points: what must not be found out on a device."""
import os
import re
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _kernel(source, name):
    """The text of a __global__ function without comments."""
    text = open(os.path.join(ROOT, "turbot5_b200", "csrc", source)).read()
    text = re.sub(r"//[^\n]*", "", text)
    at = text.index("{", re.search(r"\b%s\(const __grid_constant__" % name, text).start())
    depth = 0
    for i in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[at:i + 1]


def _depth(text, at):
    return text[:at].count("{") - text[:at].count("}")


def test_step_writes_to_the_first_block_only_once_it_has_started():
    """A block may write another's shared memory once that block has started: every thread arrives at the beginning and
    waits before the first access through `lead`.  What is written there the first block does not set itself: nothing would
    order the two."""
    body = _kernel("beam_search.cu", "step_kernel")
    arrive, wait, exchange = body.index("cluster_arrive()"), body.index("cluster_wait()"), body.index("cluster.sync()")
    first = min(m.start() for m in re.finditer(r"lead->|map_shared_rank\(&sm, (?!0\))", body))
    assert arrive < wait < first < exchange
    # by every thread of every block that stays: on the function's own level, with no way out between the two
    assert _depth(body, arrive) == _depth(body, wait) == 1 and "return" not in body[arrive:wait]
    written = set(re.findall(r"lead->(\w+)", body))
    assert written == {"umax", "usum", "reached", "found", "counts"}
    own = set(re.findall(r"\bsm\.(\w+)", body[:exchange]))
    assert not written & own, written & own
    # counts: of the blocks that there are only
    assert re.search(r"= r < C \? sm\.counts\[r\] : 0;", body)


def test_warps_of_the_step_leave_a_loop_together():
    """Other warps add to the number of candidates while a warp reads it: were it read by every lane for itself, some could
    leave the loop and others wait for them at its end.  Between the lanes' reads and the way out stands a broadcast."""
    body = _kernel("beam_search.cu", "step_kernel")
    pushes = body[body.index("cluster_wait()"):body.index("cluster.sync()")]
    ways_out = [line for line in pushes.splitlines() if "break" in line]
    assert len(ways_out) == 1 and re.search(r"if \(__shfl_sync\(0xffffffffu, [^;]*found_here, 0\) > share\) break;", ways_out[0])


def _status(call):
    """The status of a C entry point, asked in a process of its own: what ends it ends no test."""
    code = "import ctypes\nfrom tests.test_cpu_host_side import _c_struct\nfrom turbot5_b200 import _native as nat\nL = nat.lib()\n" \
           "ptr = lambda a: ctypes.cast(ctypes.byref(a), ctypes.c_void_p)\nprint('status', " + call + ")"
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.returncode, r.stderr[-500:])
    return int(r.stdout.split()[-1])


def test_scales_are_reordered_with_their_caches_only():
    """Without caches there is nothing to share blocks by."""
    assert _status("L.t5b_beam_cache_reorder(ptr(_c_struct('t5b_cache_reorder_args')(n_caches=0, n_scales=1, outer=2, B=1, num_beams=4, H=2, "
                   "capacity=64, token_bytes=64, parents=16, scales=(ctypes.c_void_p * 64)(16))), None)") == 5


def test_numbers_of_tokens_near_the_largest_number_are_refused():
    """The number of blocks that they fill is not computed beyond 2^31."""
    full = ", ".join("%s=16" % n for n in ("k", "v", "k_cache", "v_cache", "k_scale", "v_scale", "start_ptr"))
    for m in ((1 << 31) - 1, (1 << 31) - 62, 65534 * 64 + 2):
        assert _status("L.t5b_cache_quantize(ptr(_c_struct('t5b_cache_quantize_args')(dtype=nat.F16, B=1, H=1, M=%d, D=16, capacity=64, %s)), None)"
                       % (m, full)) == 2


def test_cache_lengths_near_the_largest_number_are_refused():
    """Rounding up to whole items must not pass 2^31."""
    full = ", ".join("%s=16" % n for n in ("q", "k", "v", "k_scale", "v_scale", "out"))
    for n in ((1 << 31) - 1, (1 << 31) - 63):
        assert _status("L.t5b_decode_quantized_fwd(ptr(_c_struct('t5b_decode_quantized_args')(dtype=nat.F16, B=1, H=1, M=1, N=%d, D=16, %s)), None)"
                       % (n, full)) == 2


def test_no_exception_of_an_allocation_leaves_a_c_entry_point():
    for name in os.listdir(os.path.join(ROOT, "turbot5_b200", "csrc")):
        if name.endswith((".cu", ".cuh")):
            text = re.sub(r"//[^\n]*|/\*.*?\*/", "", open(os.path.join(ROOT, "turbot5_b200", "csrc", name)).read(), flags=re.S)
            assert not re.search(r"\bnew\s+\w|std::(vector|string|map|unordered_map)\b", text), name
