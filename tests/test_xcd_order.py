"""The order of an attention's shares over the XCDs (csrc/xcd_order.h), on the host."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_shares_are_spread(tmp_path):
    """Every share has one workgroup, and no XCD has more than its eighth and two small chunks, or an eighth of a round's heads: one long
    prompt among short ones, prompts of few key heads, single tokens of few requests with many heads."""
    source, binary = tmp_path / "order.cpp", tmp_path / "order"
    source.write_text('''#include <cstdio>
#include <vector>
#include "xcd_order.h"
using namespace afhip;
int main() {
    // requests, of which `full` have all row tiles and the others one
    const struct { uint32_t requests, full, row_tiles, heads; } cases[] = {
        {1, 1, 500, 8}, {1, 1, 500, 1}, {1, 1, 63, 3}, {1, 1, 10, 10}, {16, 1, 500, 8}, {16, 2, 500, 4}, {1, 1, 1, 64}, {4, 4, 1, 32}, {64, 64, 1, 8},
        {1, 1, 1, 8}, {9, 9, 25, 8}, {3, 3, 63, 2}, {20, 20, 3, 8}, {70, 70, 1, 40}, {33, 1, 125, 8}, {2, 1, 1000, 5}};
    for (const auto& c : cases) {
        const uint32_t part = c.row_tiles * c.heads, total = c.requests * part, chunk = static_cast<uint32_t>(xcd_chunk(c.row_tiles, c.heads, total));
        const uint32_t groups = (total + 8 * chunk - 1) / (8 * chunk) * (8 * chunk);
        std::vector<int> had(groups, 0);
        uint32_t on[8] = {}, busy = 0;
        for (uint32_t g = 0; g < groups; ++g) {
            const uint32_t share = xcd_share(g, chunk);
            if (share >= groups || had[share]++) return std::printf("workgroup %u: share %u of %u\\n", g, share, groups), 1;
            const bool works = share < total && (share / part < c.full || share % c.row_tiles == 0);
            on[g % 8] += works;
            busy += works;
        }
        for (uint32_t most : on)
            if (most > busy / 8 + busy / 16 + 32) return std::printf("%u requests, %u row tiles, %u heads: %u of %u on one XCD\\n", c.requests, c.row_tiles, c.heads, most, busy), 1;
    }
    return 0;
}
''')
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "antfly_amd", "csrc"), str(source), "-o", str(binary)], check=True)
    done = subprocess.run([str(binary)], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stdout
