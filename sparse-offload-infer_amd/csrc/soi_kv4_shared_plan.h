// How the attention of sequences that share pages (kv4_shared.hip) is cut into units, and the most units and states that there can
// be: evaluated on the host (grid, workspace) and by the planning kernel. Kept apart from the kernels so that a host-only build
// can check one against the other.
#pragma once

#include <stdint.h>

namespace soi {

constexpr int kShKeys = 64;               // tokens of a stage
constexpr int kShMostStages = 1 << 24;    // of a context: contexts hold up to 2^30 tokens

// What a stage costs a wave, roughly (in units of ten cycles): unpacking its part, and cw rounds of 32 tokens.
__host__ __device__ __forceinline__ int sh_cost(int cw) { return 60 + 90 * (cw == 4 ? 2 : 1); }

__host__ __device__ __forceinline__ int sh_stages(int keys) { return (keys + kShKeys - 1) / kShKeys; }

// Stages of a unit, each of cost `of`, where `want` units share `total`: ceil(total / (want of)), from 1 up to all of a context.
// (by a 32-bit division where the sum in front of it has 32 bits)
__host__ __device__ __forceinline__ int sh_per_unit(uint64_t total, int want, int of) {
    const uint64_t d = static_cast<uint64_t>(want) * static_cast<uint64_t>(of), t = total + d - 1;
    const uint64_t n = t >> 32 ? t / d : static_cast<uint32_t>(t) / static_cast<uint32_t>(d);
    return n < 1 ? 1 : n > kShMostStages ? kShMostStages : static_cast<int>(n);
}

// units of `keys` tokens side by side, `per` stages each
__host__ __device__ __forceinline__ int sh_splits(int keys, int per) { return (sh_stages(keys) + per - 1) / per; }

// Units aimed at: two workgroups to a CU (one for heads of 256). 64 sequences of up to 512 tokens behind 8192 shared ones, 32 /
// 8 heads of 128, with 1 / 2 / 4 / 8: 55 / 37 / 45 / 45 us for the units and 6 / 8 / 14 / 26 us to add up their states
// (weights in one binary16 number then; 42 us now at 2).
// The most units and states there can be. Each of the plan's splits but a tile's last costs at least a unit's share, so there
// are at most `want` units more than tiles, and as many states as columns and those units' (full tiles for all of the units: 217
// MB instead of 79 for 2048 sequences in 1024 groups, 32 / 8 heads of 128).
struct ShSizes {
    int64_t cw, want, units, states;
    ShSizes(int64_t B, int64_t G, int64_t NQ, int64_t NKV, int64_t hd, int64_t max_len, int64_t max_shared) {
        auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
        const int64_t rep = NQ / NKV, per_group = up(B * rep, G < 1 ? 1 : G);
        cw = per_group > 64 ? 4 : per_group > 32 ? 2 : 1;
        want = up(256 * (hd == 256 ? 1 : 2), NKV);
        const int64_t pre_tiles = B * rep / (32 * cw) + G, own_tiles = B * up(rep, 32);
        auto units_of = [&](int64_t tiles, int64_t keys) {
            const int64_t most = tiles * up(keys, kShKeys);
            return want + tiles < most ? want + tiles : most;
        };
        const int64_t pre = units_of(pre_tiles, max_shared), own = units_of(own_tiles, max_len);
        units = pre + own;
        auto states_of = [&](int64_t all, int64_t wide) {
            const int64_t most = B * rep + want * wide;
            return all * wide < most ? all * wide : most;
        };
        states = states_of(pre, 32 * cw) + states_of(own, rep < 32 ? rep : 32);
    }
};

}  // namespace soi
