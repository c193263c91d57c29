"""How the typed products cut their work, on the CPU: the host side of
csrc/typed.cuh, compiled as it is, over offsets that are right, leave rows out
or overlap.  What the counts bound is memory that kernels write."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>
#include "typed.cuh"
using namespace tg;

static int bad = 0;
#define CHECK(c) do { if (!(c)) { if (bad++ < 5) std::printf("line %d: %s (M %lld, types %d, per %d, longest %d)\n", __LINE__, #c, (long long)M, types, per, longest); } } while (0)

int main() {
    std::mt19937_64 rng(1);
    const auto below = [&](int64_t n) { return static_cast<int64_t>(rng() % static_cast<uint64_t>(n)); };
    int cut = 0, overlapping = 0;
    for (int trial = 0; trial < 40000; ++trial) {
        const int64_t M = 9 + (trial % 3 == 0 ? below(2000) : (trial % 3 == 1 ? below(300000) : below(INT32_MAX - 9)));
        const int types = 1 + static_cast<int>(below(std::min<int64_t>(trial % 2 ? 1024 : 40, M - 1)));
        const int per = 1 + static_cast<int>(below(trial % 5 ? 200 : 4));
        const int longest = trial % 4 ? 1 << 30 : 64, slots = 148;
        // offsets, clamped as the kernels clamp them
        std::vector<int> o(types + 1);
        const int kind = trial % 7;
        for (int t = 0; t <= types; ++t)
            o[t] = kind == 0 ? static_cast<int>(t % 2 ? M : 0) : static_cast<int>(below(M + 1));
        if (kind > 2) std::sort(o.begin(), o.end());
        if (kind > 4) o[0] = 0, o[types] = static_cast<int>(M);
        std::vector<int> n(types);
        int64_t owned = 0, steps = 0;
        for (int t = 0; t < types; ++t) {
            n[t] = std::max(0, o[t + 1] - o[t]);
            owned += n[t];
            steps += (n[t] + kStep - 1) / kStep;
        }
        overlapping += owned > M;
        // weight gradients: items of max_pieces() pieces, partial sums of max_slots()
        const int64_t limit = piece_limit(steps, M, types, per, slots, longest);
        const int64_t least = piece_limit(M / kStep, M, types, per, slots, longest);
        int64_t pieces = 0, kept = 0;
        for (int t = 0; t < types; ++t) {
            const int count = piece_count(n[t], limit);
            pieces += count;
            cut += count > 1;
            kept += count > 1 ? count : 0;
            CHECK(count <= 1 || n[t] > least);  // the join looks at no shorter type
            if (count > 1) {
                const int64_t len = piece_rows(n[t], count);
                CHECK(len % kStep == 0 && len <= limit && len * count >= n[t] && len * (count - 1) < n[t]);
            }
        }
        CHECK(pieces <= max_pieces(M, types, per, slots, longest));
        CHECK(kept <= max_slots(M, types, per, slots, longest));
        // bias gradients: partial sums of M / kBiasChunk + types chunks
        const int64_t rows = bias_chunk(owned, M);
        int64_t chunks = 0;
        for (int t = 0; t < types; ++t) chunks += (n[t] + rows - 1) / rows;
        CHECK(chunks <= M / kBiasChunk + types);
        CHECK(owned > M || rows == kBiasChunk);
        // counts of pieces never wrap around
        int sum = 0;
        int64_t exact = 0;
        for (int t = 0; t < types; ++t) {
            const int before = sum, c = static_cast<int>((n[t] + 127LL) / 128);
            sum = add_pieces(sum, c);
            exact += c;
            CHECK(sum >= before && sum - before <= c && sum == std::min<int64_t>(exact, INT_MAX));
        }
    }
    std::printf("cut %d, overlapping %d, bad %d\n", cut, overlapping, bad);
    return bad || !cut || !overlapping;
}
"""


def test_partial_sums_stay_within_their_buffers(tmp_path):
    if not (os.path.exists(NVCC) or shutil.which("nvcc")):
        pytest.skip("no nvcc")
    src = tmp_path / "plan.cu"
    src.write_text(PROGRAM)
    csrc, inc = os.path.join(ROOT, "tinygnn_b200", "csrc"), os.path.join(ROOT, "include")
    exe = str(tmp_path / "plan")
    subprocess.run([NVCC if os.path.exists(NVCC) else "nvcc", "-std=c++17", "-O1", "-gencode", "arch=compute_100a,code=sm_100a",
                    "--expt-relaxed-constexpr", "-I", csrc, "-I", inc, str(src), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
