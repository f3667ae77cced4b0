"""csrc/dev_mat_i4_plan.cuh on the host: what mat_mat_i4's kernel for more rows reads of its shared memory lies in what its launch allocates."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "llama-gguf_b200", "csrc")
PROGRAM = r"""
#include <cstdio>
#include "dev_mat_i4_plan.cuh"
using namespace dev;
int main() {
    const int scales[] = {2, 4}, groups[] = {32, 64, 128}, experts[] = {0, 1, 8, 64, 1024};
    for (int s : scales)
        for (int g : groups)
            for (int e : experts)
                for (int rows = 17; rows <= 2 * I4_PAIRS; rows++) {
                    const I4ManyPlan p = i4_many_plan(s, g, rows, e);
                    const int lists = e ? (int)i4_list_bytes(e, rows < I4_PAIRS ? rows : I4_PAIRS) : 0;
                    auto bad = [&](const char* what, long a, long b) { return printf("scales of %d bytes, groups of %d, %d experts, %d rows: %s: %ld, %ld\n", s, g, e, rows, what, a, b), 1; };
                    if (p.ring < 2 || p.ring > I4_MANY_RING) return bad("ring", p.ring, 0);
                    if ((long)p.smem + lists > I4_MANY_MOST || I4_MANY_MOST + I4_MANY_OWN > 227 * 1024) return bad("too much", (long)p.smem + lists, I4_MANY_MOST);
                    const long slot = i4_many_slot(s, g, p.most), team = p.ring * slot;
                    if ((long)p.smem != I4_TEAMS * team) return bad("not the teams' rings", (long)p.smem, I4_TEAMS * team);
                    // a unit has up to 64 rows; a launch's (an expert's) last unit any number of them
                    for (int many = 1; many <= (rows < I4_MANY_ROWS ? rows : I4_MANY_ROWS); many++) {
                        const int have = (many + 7) / 8, computed = i4_many_blocks(have);
                        if (computed < have) return bad("columns without a block", have, computed);
                        // the weights and scales of eight tiles, then eight rows of 128 channels for each block, which belong to the same step
                        const long read = I4_TEAM_TILES * i4_slot(s, g, 2) + computed * 8 * 128;
                        if (read > slot) return bad("a step is read behind its end", read, slot);
                        if (I4_TEAMS * team - slot + read > (long)p.smem) return bad("shared memory is read behind its end", I4_TEAMS * team - slot + read, (long)p.smem);
                        // the sums, in the ring's place: 16 bytes a lane for each tile and block
                        if ((long)I4_TEAM_TILES * (p.most / 8) * 512 > team || have > p.most / 8) return bad("sums", (long)I4_TEAM_TILES * (p.most / 8) * 512, team);
                    }
                }
    puts("ok");
    return 0;
}
"""


def test_steps_are_read_within_what_a_launch_allocates(tmp_path):
    (tmp_path / "t.cpp").write_text(PROGRAM)
    exe = str(tmp_path / "t")
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", CSRC, "-o", exe, str(tmp_path / "t.cpp")], check=True)
    assert subprocess.run([exe], capture_output=True, text=True).stdout == "ok\n"
