"""What a kernel does after a bounded wait ran out, read on the CPU: it waits for what is still under way, each copy by the phase of its barrier that it
completes (csrc/ring.h), before shared or tensor memory goes to something else. On a GPU a wait would have to run out for it."""
import re
import subprocess
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "sapient_b200" / "csrc"
PROGRAM = r"""
#include "ring.h"
#include <cstdio>
#include <vector>

// A barrier: phases completed so far. A wait for a parity is over at once if the phase under way has the other one.
struct Barrier { int completed = 0, requested = 0; };

int main() {
    for (int stages = 2; stages <= 5; ++stages)
        for (int steps = 1; steps <= 23; ++steps)
            for (int failed = 0; failed < steps; ++failed) {
                std::vector<Barrier> bar(stages);
                auto request = [&](int k) {
                    const sp::RingAt at = sp::ring_at(k, stages);
                    if (bar[at.stage].requested != bar[at.stage].completed) { std::printf("stage of step %d is in use\n", k); return false; }
                    ++bar[at.stage].requested;
                    return true;
                };
                for (int k = 0; k < stages - 1 && k < steps; ++k)
                    if (!request(k)) return 1;
                for (int i = 0;; ++i) {  // as the kernel's loop: the copies of step i + stages - 1, then the wait for step i
                    if (i + stages - 1 < steps && !request(i + stages - 1)) return 1;
                    if (i == failed) break;
                    Barrier& b = bar[sp::ring_at(i, stages).stage];
                    if ((b.completed & 1) != (int)sp::ring_at(i, stages).parity) { std::printf("step %d waits for another phase\n", i); return 1; }
                    ++b.completed;
                }
                std::vector<bool> waited(stages);
                for (int k = failed; k < sp::ring_requested(failed, stages, steps); ++k) {
                    const sp::RingAt at = sp::ring_at(k, stages);
                    if ((bar[at.stage].completed & 1) != (int)at.parity) { std::printf("%d stages, %d steps, %d failed: the wait for step %d is over at once\n", stages, steps, failed, k); return 1; }
                    waited[at.stage] = true;
                }
                for (int s = 0; s < stages; ++s)
                    if (waited[s] != (bar[s].requested != bar[s].completed)) { std::printf("%d stages, %d steps, %d failed: stage %d\n", stages, steps, failed, s); return 1; }
            }
    return 0;
}
"""


def test_each_copy_under_way_is_waited_for(tmp_path):
    src, exe = tmp_path / "ring.cpp", tmp_path / "ring"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", str(CSRC), str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout


def test_attention_rows_wait_for_them():
    text = (CSRC / "attention_fp8.cu").read_text()
    after = text[text.index("if (!ok && lane == 0)"):]
    assert re.search(r"for \(int k = i; k < ring_requested\(i, STAGES, steps\); \+\+k\) tc5_wait\(&full\[warp\]\[ring_at\(k, STAGES\)\.stage\], ring_at\(k, STAGES\)\.parity\)",
                     after[: after.index("__syncwarp")])


def test_attention_tiles_wait_for_products_before_tensor_memory_is_freed():
    text = (CSRC / "attention_fp8_tile.cu").read_text()
    commit, free = text.index("tc5_commit(&o_full)"), text.index("tcgen05.dealloc")
    line = text[text.rfind("\n", 0, commit): commit]
    assert "ok" not in line, "the products are committed whether or not a wait ran out"
    wait = re.search(r"tc5_wait\(&o_full, 0\) && ok", text[commit:free])
    assert wait, "the wait for them is made whether or not another ran out"
