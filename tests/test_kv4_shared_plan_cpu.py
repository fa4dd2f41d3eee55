"""The plan of the attention over shared pages (csrc/soi_kv4_shared_plan.h), built for the host: a unit's stages are those of 128-bit
arithmetic, around 2^32 too, and no lengths need more units or states than the workspace is sized for.

The lengths live on the device, so only these bounds keep the planning kernel inside its workspace.
"""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "sparse-offload-infer_amd" / "csrc"

HARNESS = r"""
#include <cstdio>
#include <random>
#include <vector>
#include "soi_kv4_shared_plan.h"
using namespace soi;

static long cases = 0;

static bool quotient(uint64_t total, int want, int of) {
    const unsigned __int128 d = static_cast<unsigned __int128>(want) * of, n = (total + d - 1) / d;
    const unsigned __int128 spec = n < 1 ? 1 : n > kShMostStages ? kShMostStages : n;
    ++cases;
    const int got = sh_per_unit(total, want, of);
    if (got == static_cast<int>(spec)) return true;
    printf("FAIL total=%llu want=%d of=%d: %d, not %d\n", (unsigned long long)total, want, of, got, static_cast<int>(spec));
    return false;
}

int main() {
    std::mt19937_64 rng(1);
    auto upto = [&](int64_t n) { return static_cast<int64_t>(rng() % static_cast<uint64_t>(n + 1)); };
    if (!quotient(4294967200ull, 512, sh_cost(1))) return 1;  // 55925
    for (int want = 1; want <= 512; want += want < 8 ? 1 : 7)
        for (int cw = 1; cw <= 4; cw *= 2) {
            const uint64_t d = static_cast<uint64_t>(want) * sh_cost(cw);
            for (uint64_t i = 0; i <= 3 * d; i += 1 + i / 50)
                if (!quotient((1ull << 32) - 2 * d + i, want, sh_cost(cw)) || !quotient(i, want, sh_cost(cw))) return 1;
            for (int i = 0; i < 200; ++i)
                if (!quotient(rng() >> (12 + upto(50)), want, sh_cost(cw))) return 1;
        }
    for (int trial = 0; trial < 40000; ++trial) {
        const int64_t B = 1 + upto(trial % 3 ? 40 : 2047), NKV = 1ll << upto(6), rep = 1 + upto(trial % 5 ? 8 : 70), hd = 64ll << upto(2);
        const int64_t most = 1ll << upto(30);
        std::vector<int64_t> cu{0};
        while (cu.back() < B && static_cast<int64_t>(cu.size()) < 2048) cu.push_back(std::min<int64_t>(B, cu.back() + upto(1ll << upto(11))));
        if (trial % 7 == 0) cu = {0, B};
        if (trial % 11 == 0) cu = {0};
        const int64_t G = static_cast<int64_t>(cu.size()) - 1;
        std::vector<int64_t> len(B), start(B, 0), keys(G, 0);
        int64_t max_len = 0, max_shared = 0;
        const bool full = trial % 2;
        for (auto& l : len) max_len = std::max(max_len, l = full ? most : upto(most));
        for (int64_t g = 0; g < G; ++g) {
            if (cu[g + 1] == cu[g]) continue;
            int64_t k = most;
            for (int64_t b = cu[g]; b < cu[g + 1]; ++b) k = std::min(k, len[b]);
            keys[g] = (full && trial % 4 == 1 ? k : upto(k)) / 64 * 64;
            for (int64_t b = cu[g]; b < cu[g + 1]; ++b) start[b] = upto(5) ? keys[g] : 0;  // (some of a group share nothing)
            max_shared = std::max(max_shared, keys[g]);
        }
        const ShSizes sz(B, G, NKV * rep, NKV, hd, max_len, max_shared);
        const int cw = static_cast<int>(sz.cw), want = static_cast<int>(sz.want);
        const int64_t own_tiles = (rep + 31) / 32;
        auto tiles = [&](int64_t g) { return ((cu[g + 1] - cu[g]) * rep + 32 * cw - 1) / (32 * cw); };
        int64_t total = 0, units = 0, states = 0;
        for (int64_t g = 0; g < G; ++g) total += tiles(g) * sh_stages(static_cast<int>(keys[g])) * sh_cost(cw);
        for (int64_t b = 0; b < B; ++b) total += own_tiles * sh_stages(static_cast<int>(len[b] - start[b])) * sh_cost(1);
        const int pre_per = sh_per_unit(total, want, sh_cost(cw)), own_per = sh_per_unit(total, want, sh_cost(1));
        for (int64_t g = 0; g < G; ++g) {
            const int64_t ns = sh_splits(static_cast<int>(keys[g]), pre_per);
            units += tiles(g) * ns;
            states += (cu[g + 1] - cu[g]) * rep * ns;
            if (ns && ((ns - 1) * pre_per * kShKeys >= keys[g] || ns * pre_per * kShKeys < keys[g])) return printf("FAIL splits\n"), 1;
        }
        for (int64_t b = 0; b < B; ++b) {
            const int64_t ns = sh_splits(static_cast<int>(len[b] - start[b]), own_per);
            units += own_tiles * ns;
            states += rep * ns;
        }
        ++cases;
        if (units > sz.units || states > sz.states) {
            printf("FAIL B=%lld G=%lld NKV=%lld rep=%lld hd=%lld total=%lld: %lld units of %lld, %lld states of %lld\n", (long long)B,
                   (long long)G, (long long)NKV, (long long)rep, (long long)hd, (long long)total, (long long)units, (long long)sz.units,
                   (long long)states, (long long)sz.states);
            return 1;
        }
    }
    printf("%ld cases\n", cases);
    return 0;
}
"""


def test_units_and_states_fit(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    src, exe = tmp_path / "plan.cpp", tmp_path / "plan"
    src.write_text(HARNESS)
    subprocess.run([gxx, "-O2", "-std=c++17", "-D__host__=", "-D__device__=", "-D__forceinline__=inline", f"-I{CSRC}", "-o", str(exe),
                    str(src)], check=True, capture_output=True, text=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert int(r.stdout.split()[0]) > 100_000
