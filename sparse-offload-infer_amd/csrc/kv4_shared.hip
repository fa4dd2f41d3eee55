// One query token per sequence over the paged 4-bit KV cache (soi_kv4.h) where sequences come in groups that begin with the
// same pages, gfx950: a group's shared tokens are read, unpacked and multiplied once for all its sequences.
//
//   out[b, h] = sum_t softmax_t(scale q[b, h] . k_t) v_t over the tokens t < lens[b], as kv4_attention.hip
//
// Work is cut into units: a range of tokens of one page table row against up to 32 cw columns, a column being one (sequence,
// query head) of the KV head. A group's shared tokens are units with its sequences' heads as columns, the tokens behind them
// units of one sequence. A first launch of one workgroup lists the units from the lengths (about `want` of equal cost for each
// KV head), a second one runs them, a third adds up each (sequence, head)'s states.
//
// A unit is taken in stages of 128 tokens. The workgroup's four waves unpack a stage's K and V codes into LDS as binary16
// integers (exact), the next stage's bytes on their way into registers meanwhile. Then each wave takes 32 columns
// (v_mfma_f32_32x32x16_f16, lanes n = lane & 31, h = lane >> 5), cw of them side by side, 4 / cw waves sharing the stage's
// tokens:
//   * S^T = K Q^T: lane (n, h) ends with the scores of column n and tokens 8 (r >> 2) + 4 h + (r & 3), r < 16; a scale group's
//     sums are multiplied by its scale in binary32;
//   * O^T = V^T P^T takes these, exponentiated, as its B operand as they lie, times V's scale, rounded to binary16 once: a set
//     of weights for each scale group. V is kept as V^T [dimension][token], tokens in the order that this operand's k slots
//     want (16 j + 4 h + 0 .. 3, + 8 .. 11 side by side: one 16-byte read). The cache's V units hold four tokens of one
//     dimension, so unpacking writes such rows without a transposition;
//   * the base of the exponents follows weight times the stage's largest V scale, so the products fill binary16's range
//     whatever V's size: rounded by 2^-11 of themselves down to 2^-26 of the largest weight times the largest scale that meets
//     it, 0 below 2^-37 of it. (K and V rounded to binary16 values in LDS would save a third of the vector work, but their
//     rounding triples the output's error.)
// 16-byte chunks are XOR-swizzled so that operand reads and the unpacked rows' writes spread over the banks.
#include "soi_host.h"
#include "soi_kv4.h"
#include "soi_attn.h"

#include <type_traits>

namespace soi {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kShWaves = 4, kShThreads = kShWaves * kWave, kShKeys = 128;
constexpr int kShRound = 64;                     // shared tokens end on a multiple of this
constexpr int kShMost = 2048;                    // sequences of a call
constexpr float kShLow = 12.0f, kShHigh = 15.0f;  // a column's largest weight times V scale is between 2^kShLow and 2^kShHigh
constexpr int sh_per_cu(int hd) { return hd == 64 ? 3 : hd == 128 ? 2 : 1; }  // workgroups that a CU holds

struct ShUnit {
    int row, key0, key1;    // tokens key0 .. key1 - 1 of page table row `row`
    int seq0, col0, ncols;  // columns col0 .. col0 + ncols - 1 of the sequences from seq0 on
    int state, step;        // state of its first column, the next wave's share of the tokens `step` further
    int cw, pad[3];         // waves side by side
};
struct ShSeq {                    // the states of a sequence's head r of a KV head:
    int pre, pre_step, pre_n;     // pre + i pre_step + r, i < pre_n, over the shared tokens
    int own, own_n, pad[3];       // own + i rep + r, i < own_n, over the others
};
struct ShHead {
    int units, pad[3];
};

struct ShArgs {
    const uint16_t* q;
    int64_t q_stride;
    uint16_t* out;
    const int32_t *cu, *shared;
    ShHead* head;
    ShUnit* units;
    ShSeq* seqs;
    float* part;  // [NKV][states][hd + 4]: sums, base, weight
    int NQ, rep, G, max_len, max_shared;
    int cw, want, most_units, states;
    float scale_log2;
};

// What a stage costs a wave, roughly (in units of ten cycles): unpacking its part, and cw rounds of 32 tokens.
__device__ __forceinline__ int sh_cost(int cw) { return 110 + 80 * cw; }

constexpr int kShPlan = 1024;  // threads of the plan
template <class N>
__device__ __forceinline__ N sh_scan(N v, N* s_part, N& all) {  // exclusive over the threads, and the sum
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    N x = v;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const N y = __shfl_up(x, o);
        x += lane >= o ? y : 0;
    }
    if (lane == 63) s_part[wave] = x;
    __syncthreads();
    N base = 0;
    all = 0;
    for (int w = 0; w < kShPlan / kWave; ++w) {
        base += w < wave ? s_part[w] : 0;
        all += s_part[w];
    }
    __syncthreads();
    return base + x - v;
}

// The units of a call, and where each sequence's states are. A group shares what all its sequences that share anything have
// in common, so that a unit's columns all see all its tokens; sequences outside every group share nothing.
__global__ __launch_bounds__(kShPlan) void kv4_shared_plan_kernel(const ShArgs a, const Kv4Cache c) {
    // of each group: first sequence, shared tokens, the first sequence that shares them, its first unit and state
    __shared__ int s_cu[kShMost + 1], s_keys[kShMost], s_row[kShMost], s_unit[kShMost], s_state[kShMost];
    __shared__ int s_part[kShPlan / kWave];
    __shared__ int64_t s_part64[kShPlan / kWave];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, B = c.B, rep = a.rep;
    for (int g = tid; g <= a.G; g += kShPlan) s_cu[g] = ldg(a.cu + g);
    for (int g = tid; g < a.G; g += kShPlan) s_keys[g] = s_row[g] = 0x7fffffff;
    __syncthreads();
    int bad = 0;
    for (int g = tid; g <= a.G; g += kShPlan) bad |= s_cu[g] < (g ? s_cu[g - 1] : 0) || s_cu[g] > B;
    const int G = __syncthreads_or(bad) ? 0 : a.G;  // offsets that are none: nobody shares anything
    auto length = [&](int b) {
        const int L = ldg(c.lens + b);
        return L < 0 ? 0 : L < a.max_len ? L : a.max_len;
    };
    auto group_of = [&](int b) {  // -1: none
        int lo = 0, hi = G;       // the last g < G with cu[g] <= b
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s_cu[mid] <= b) lo = mid;
            else hi = mid;
        }
        return G > 0 && s_cu[lo] <= b && b < s_cu[lo + 1] ? lo : -1;
    };
    auto shares = [&](int b, int L) {
        int n = ldg(a.shared + b);
        n = n < a.max_shared ? n : a.max_shared;
        n = n < L ? n : L;
        return n < kShRound ? 0 : n / kShRound * kShRound;
    };
    for (int b = tid; b < B; b += kShPlan) {
        const int g = group_of(b), n = shares(b, length(b));
        if (g >= 0 && n > 0) {
            atomicMin(&s_keys[g], n);
            atomicMin(&s_row[g], b);
        }
    }
    __syncthreads();
    const int width = 32 * a.cw, own_tiles = (rep + 31) / 32, pre_kw = kShWaves / a.cw;
    auto stages = [](int keys) { return (keys + kShKeys - 1) / kShKeys; };
    auto keys_of = [&](int g) { return s_row[g] == 0x7fffffff ? 0 : s_keys[g]; };
    auto columns = [&](int g) { return (s_cu[g + 1] - s_cu[g]) * rep; };
    auto tiles = [&](int g) { return (columns(g) + width - 1) / width; };
    int64_t cost = 0, total;
    for (int g = tid; g < G; g += kShPlan) cost += static_cast<int64_t>(tiles(g)) * stages(keys_of(g)) * sh_cost(a.cw);
    for (int b = tid; b < B; b += kShPlan) {
        const int L = length(b), g = group_of(b);
        cost += static_cast<int64_t>(own_tiles) * stages(L - (g >= 0 && shares(b, L) > 0 ? keys_of(g) : 0)) * sh_cost(1);
    }
    sh_scan(cost, s_part64, total);
    auto per_unit = [&](int of) {  // stages of a unit, each of cost `of`
        const int64_t d = static_cast<int64_t>(a.want) * of, n = (total + d - 1) / d;
        return static_cast<int>(n < 1 ? 1 : n);
    };
    const int pre_per = per_unit(sh_cost(a.cw)), own_per = per_unit(sh_cost(1));
    auto splits = [&](int keys, int per) { return (stages(keys) + per - 1) / per; };
    int unit0 = 0, state0 = 0;
    for (int g0 = 0; g0 < G; g0 += kShPlan) {
        const int g = g0 + tid, ns = g < G ? splits(keys_of(g), pre_per) : 0;
        int units, states;
        const int u = unit0 + sh_scan(ns ? tiles(g) * ns : 0, s_part, units);
        const int s = state0 + sh_scan(ns ? columns(g) * ns * pre_kw : 0, s_part, states);
        if (g < G) {
            s_unit[g] = u;
            s_state[g] = s;
        }
        unit0 += units;
        state0 += states;
    }
    __syncthreads();
    for (int g = wave; g < G; g += kShPlan / kWave) {  // a wave lists a group's units
        const int keys = keys_of(g), ns = splits(keys, pre_per), cols = columns(g), n = ns ? tiles(g) * ns : 0;
        for (int i = lane; i < n; i += kWave) {
            const int t = i / ns, k = i - t * ns, k0 = k * pre_per * kShKeys, k1 = k0 + pre_per * kShKeys;
            const int left = cols - t * width;
            if (s_unit[g] + i < a.most_units)
                a.units[s_unit[g] + i] = ShUnit{s_row[g], k0, k1 < keys ? k1 : keys, s_cu[g], t * width, left < width ? left : width,
                                                s_state[g] + k * pre_kw * cols + t * width, cols, a.cw, {0, 0, 0}};
        }
    }
    for (int b0 = 0; b0 < B; b0 += kShPlan) {
        const int b = b0 + tid, L = b < B ? length(b) : 0, g = b < B ? group_of(b) : -1;
        const int start = g >= 0 && shares(b, L) > 0 ? keys_of(g) : 0, ns = splits(L - start, own_per);
        int units, states;
        int u = unit0 + sh_scan(ns * own_tiles, s_part, units);
        const int s = state0 + sh_scan(ns * kShWaves * rep, s_part, states);
        unit0 += units;
        state0 += states;
        if (b >= B) continue;
        for (int t = 0; t < own_tiles; ++t)
            for (int k = 0; k < ns; ++k, ++u) {
                const int k0 = start + k * own_per * kShKeys, k1 = k0 + own_per * kShKeys, left = rep - 32 * t;
                if (u < a.most_units)
                    a.units[u] = ShUnit{b, k0, k1 < L ? k1 : L, b, 32 * t, left < 32 ? left : 32,
                                        s + k * kShWaves * rep + 32 * t, rep, 1, {0, 0, 0}};
            }
        const int cols = start ? columns(g) : 0;
        a.seqs[b] = ShSeq{start ? s_state[g] + (b - s_cu[g]) * rep : 0, cols, start ? splits(start, pre_per) * pre_kw : 0,
                          s, ns * kShWaves, {0, 0, 0}};
    }
    if (tid == 0) a.head->units = unit0 < a.most_units ? unit0 : a.most_units;
}

// the waves' LDS writes are done, and all reads before; loads into registers stay in flight
__device__ __forceinline__ void sh_meet() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// physical 16-byte chunk of chunk c of a K row (HD / 8 chunks), and of a V row (16 chunks: the stage's tokens)
template <int HD>
__device__ __forceinline__ int sh_swz_k(int key) {
    return HD == 64 ? (key >> 1) & 7 : key & 15;
}

template <int HD, int GS>
__global__ __launch_bounds__(kShThreads, sh_per_cu(HD)) void kv4_shared_kernel(const ShArgs a, const Kv4Cache c) {
    constexpr int W = HD / 32, U = HD / 64, G = HD / GS, KK = HD / 16, DT = HD / 32, ROWB = 2 * HD, VROWB = 2 * kShKeys;
    // K: a thread unpacks KT pieces of 16 bytes, of PK that a token has; V: VT times eight tokens of UU dimension blocks
    constexpr int PK = HD / 32, KT = kShKeys * PK / kShThreads, UU = U < 2 ? U : 2, VT = U / UU;
    static_assert(G <= PK && 2 * G <= 16, "a piece of K, and a lane m of V, for each scale");
    __shared__ __attribute__((aligned(1024))) uint8_t s_k[kShKeys * ROWB], s_v[HD * VROWB];
    __shared__ __attribute__((aligned(16))) uint16_t s_ks[G][kShKeys], s_vs[G][kShKeys];  // scales, zeros for tokens that are not there
    __shared__ uint64_t s_valid;   // a byte for each 16 tokens of the stage: they have a page
    __shared__ uint32_t s_top[2];  // bits of the largest finite V scale, of this stage and the next
    if (static_cast<int>(blockIdx.y) >= ldg(&a.head->units)) return;
    const ShUnit un = a.units[blockIdx.y];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n = lane & 31, hh = lane >> 5;
    const int kvh = blockIdx.x, cwave = wave % un.cw, kwave = wave / un.cw, kw = kShWaves / un.cw;
    const int wcols = un.ncols - 32 * cwave;  // columns of this wave
    const int col = un.col0 + 32 * cwave + (n < wcols ? n : 0);

    f16x8 qf[KK];
    if (wcols > 0) {
        const int seq = un.seq0 + col / a.rep, r = col % a.rep;
        const uint16_t* qr = a.q + seq * a.q_stride + static_cast<int64_t>(kvh * a.rep + r) * HD;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) qf[kk] = __builtin_bit_cast(f16x8, ldg_any(qr + 16 * kk + 8 * hh));
    }

    // The stage's bytes in registers. K piece t: token k_key(t), words 4 k_p .. + 3. V: tokens 16 j + 4 vh + 0 .. 3 and + 8 .. 11,
    // dimensions 16 x + m.
    auto k_key = [&](int t) { return (tid + kShThreads * t) / PK; };
    const int k_p = tid % PK, m = tid & 15, vh = (tid >> 4) & 1, j = tid >> 5;
    u32x4 kraw[KT];
    uint16_t ksc[KT];  // the token's scale of group k_p, if there is one
    u32x2 vraw[VT][2][UU], vsc;  // lanes m < 2 G: the scales of four tokens, + 8 (m & 1), of group m >> 1
    int kid[KT], vid;
    auto pages = [&](int key0, int (&ki)[KT], int& vi) {
#pragma unroll
        for (int t = 0; t < KT; ++t) ki[t] = key0 < un.key1 ? kv4_page(c, un.row, key0 + k_key(t)) : -1;
        vi = key0 < un.key1 ? kv4_page(c, un.row, key0 + 16 * j) : -1;
    };
    auto head_of = [&](int id) { return static_cast<int64_t>(id < 0 ? 0 : id) * c.NKV + kvh; };
    auto fetch = [&](int key0) {
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            const int slot = (key0 + k_key(t)) & (c.page - 1);
            const int64_t h = head_of(kid[t]);
            kraw[t] = ldg(reinterpret_cast<const u32x4*>(c.k_pages + (h * c.page + slot) * (HD / 2) + 16 * k_p));
            ksc[t] = ldg(c.k_scale + (h * G + (k_p < G ? k_p : 0)) * c.page + slot);
        }
        const int slot = (key0 + 16 * j + 4 * vh) & (c.page - 1);
        const int64_t h = head_of(vid);
        const uint8_t* vp = c.v_pages + h * c.page * (HD / 2) + (slot >> 2) * (16 * U * 8) + m * (U * 8);
        vsc = ldg(reinterpret_cast<const u32x2*>(c.v_scale + (h * G + (m < 2 * G ? m >> 1 : 0)) * c.page + slot + 8 * (m & 1)));
#pragma unroll
        for (int t = 0; t < VT; ++t)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                if constexpr (UU == 1) {
                    vraw[t][x][0] = ldg(reinterpret_cast<const u32x2*>(vp + x * 2 * (16 * U * 8)));
                } else {
                    const u32x4 r = ldg(reinterpret_cast<const u32x4*>(vp + x * 2 * (16 * U * 8) + 16 * t));
                    vraw[t][x][0] = u32x2{r.x, r.y};
                    vraw[t][x][1] = u32x2{r.z, r.w};
                }
            }
    };
    // Tokens that are not there (past the unit, or without a page) get scales 0: theirs may be anything.
    auto unpack = [&](int key0, int odd) {
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            const int key = k_key(t);
            const bool live = kid[t] >= 0 && key0 + key < un.key1;
            if (k_p < G) s_ks[k_p][key] = live ? ksc[t] : 0;
            uint8_t* row = s_k + key * ROWB;
            const uint32_t word[4] = {kraw[t].x, kraw[t].y, kraw[t].z, kraw[t].w};
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int w = 4 * k_p + x, i = HD == 256 ? 4 * (k_p & 1) + x : w % W, g = w / W;  // word W g + i: chunk 4 i + g
                f16x2 v[4];
                dequant_int4x8_bitfield(word[x], v);
                const f16x8 o = {v[0].x, v[0].y, v[1].x, v[1].y, v[2].x, v[2].y, v[3].x, v[3].y};
                *reinterpret_cast<f16x8*>(row + (((4 * i + g) ^ sh_swz_k<HD>(key)) << 4)) = o;
            }
        }
        const int left = vid < 0 ? 0 : un.key1 - key0 - 16 * j - 4 * vh;  // live tokens from the thread's first on
        if ((tid & 31) == 0) reinterpret_cast<uint8_t*>(&s_valid)[j] = vid >= 0;
        if (m < 2 * G) {
            uint32_t w[2] = {vsc.x, vsc.y}, most = 0;
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const int there = left - 8 * (m & 1) - 2 * y;
                w[y] = there > 1 ? w[y] : there == 1 ? w[y] & 0xffffu : 0u;
                const uint32_t lo = w[y] & 0x7fffu, hi = w[y] >> 16 & 0x7fffu;
                most = lo < 0x7c00u && lo > most ? lo : most;
                most = hi < 0x7c00u && hi > most ? hi : most;
            }
            *reinterpret_cast<u32x2*>(&s_vs[m >> 1][16 * j + 4 * vh + 8 * (m & 1)]) = u32x2{w[0], w[1]};
            atomicMax(&s_top[odd], most);
        }
#pragma unroll
        for (int t = 0; t < VT; ++t)
#pragma unroll
            for (int u = 0; u < UU; ++u)
#pragma unroll
                for (int k = 0; k < 4; ++k) {  // dimension 64 (UU t + u) + 16 k + m
                    const int dim = 64 * (UU * t + u) + 16 * k + m;
                    f16x2 v[2][2];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t w[2] = {vraw[t][x][u].x, vraw[t][x][u].y};  // tokens (0, 1), (2, 3)
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            const f16x2 bias = {(f16)-1032.0f, (f16)-1032.0f}, bias16 = {(f16)-72.0f, (f16)-72.0f};
                            const f16x2 sixteenth = {(f16)0.0625f, (f16)0.0625f};
                            const uint32_t y8 = k < 2 ? w[y] : w[y] >> 8;
                            v[x][y] = k & 1 ? __builtin_elementwise_fma(as_f16x2(and_xor(y8, 0x00f000f0u, 0x64806480u)), sixteenth,
                                                                        bias16)
                                            : as_f16x2(and_xor(y8, 0x000f000fu, 0x64086408u)) + bias;
                        }
                    }
                    const f16x8 o = {v[0][0].x, v[0][0].y, v[0][1].x, v[0][1].y, v[1][0].x, v[1][0].y, v[1][1].x, v[1][1].y};
                    *reinterpret_cast<f16x8*>(s_v + dim * VROWB + (((2 * j + vh) ^ (dim & 15)) << 4)) = o;
                }
    };

    f32x16 acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] = 0.0f;
    float base = kNegBig, l = 0.0f;
    // scale_top: binades from the stage's largest V scale up to 1
    auto products = [&](int key0, int sub, bool whole, uint64_t valid, float scale_top) {
        const int at = 32 * sub + 4 * hh;  // the lane's first token, the others 8 (r >> 2) + (r & 3) further
        float z[16];
        const uint8_t* row = s_k + (32 * sub + n) * ROWB;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            f32x16 sum;
#pragma unroll
            for (int r = 0; r < 16; ++r) sum[r] = 0.0f;
#pragma unroll
            for (int kk = g * (GS / 16); kk < (g + 1) * (GS / 16); ++kk) {
                const f16x8 kf = *reinterpret_cast<const f16x8*>(row + (((2 * kk + hh) ^ sh_swz_k<HD>(n)) << 4));
                sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[kk], sum, 0, 0, 0);
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const u32x2 sc = *reinterpret_cast<const u32x2*>(&s_ks[g][at + 8 * x]);
                const f16x2 lo = as_f16x2(sc.x), hi = as_f16x2(sc.y);
                const f16 s4[4] = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    z[4 * x + e] = fmaf(sum[4 * x + e], static_cast<float>(s4[e]), g ? z[4 * x + e] : 0.0f);
            }
            if (HD == 256) __builtin_amdgcn_sched_barrier(0);  // (all groups at once would spill)
        }
        if (!whole) {
            const int left = un.key1 - key0 - at;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const bool live = 8 * (r >> 2) + (r & 3) < left && ((valid >> (16 * sub + 8 * (r >> 3))) & 1);
                z[r] = live ? z[r] : -__builtin_inff();
            }
        }
        float top = z[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, z[r]);
        top = fmaf(fmaxf(top, xor_lanes<32>(top)), a.scale_log2, -scale_top);
        // the base rises only where a product would pass 2^kShHigh, to where the largest is 2^kShLow; a column does not depend
        // on its neighbours
        if (ballot(top > base + kShHigh)) {
            const float up = top > base + kShHigh ? top - kShLow : base, w = fast_exp2(base - up);
            base = up;
            l *= w;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[d][r] *= w;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            z[r] = fast_exp2(fmaf(z[r], a.scale_log2, -base));
            l += z[r];
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            f16x8 pb[2];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const u32x2 sc = *reinterpret_cast<const u32x2*>(&s_vs[g][at + 8 * x]);
                const f16x2 lo = as_f16x2(sc.x), hi = as_f16x2(sc.y);
                const f16 s4[4] = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
                for (int e = 0; e < 4; ++e)  // (fma, not a product: one mixed-precision instruction)
                    pb[x >> 1][4 * (x & 1) + e] = static_cast<f16>(fmaf(z[4 * x + e], static_cast<float>(s4[e]), 0.0f));
            }
#pragma unroll
            for (int d = g * (GS / 32); d < (g + 1) * (GS / 32); ++d) {
                const uint8_t* vrow = s_v + (32 * d + n) * VROWB;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const f16x8 vf = *reinterpret_cast<const f16x8*>(vrow + (((4 * sub + 2 * x + hh) ^ (n & 15)) << 4));
                    acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pb[x], acc[d], 0, 0, 0);
                }
            }
            if (HD == 256) __builtin_amdgcn_sched_barrier(0);
        }
    };

    pages(un.key0, kid, vid);
    fetch(un.key0);
    if (tid < 2) s_top[tid] = 0;
    sh_meet();
    int odd = 0;
    for (int key0 = un.key0; key0 < un.key1; key0 += kShKeys, odd ^= 1) {
        int next_kid[KT], next_vid;
        pages(key0 + kShKeys, next_kid, next_vid);
        if (key0 > un.key0) sh_meet();  // the stage before is read
        unpack(key0, odd);
        if (tid == 0) s_top[odd ^ 1] = 0;
#pragma unroll
        for (int t = 0; t < KT; ++t) kid[t] = next_kid[t];
        vid = next_vid;
        if (key0 + kShKeys < un.key1) fetch(key0 + kShKeys);
        sh_meet();
        const uint64_t valid = s_valid;
        const bool whole = key0 + kShKeys <= un.key1 && valid == 0x0101010101010101ull;
        const float scale_top = 14.0f - static_cast<float>(s_top[odd] >> 10);  // (the exponent's bits: scales below 2^(bits - 14))
        if (wcols > 0)
            for (int sub = kwave; sub < kShKeys / 32; sub += kw)
                if (key0 + 32 * sub < un.key1) products(key0, sub, whole, valid, scale_top);
    }
    if (n >= wcols) return;  // (no barrier from here on)
    l += xor_lanes<32>(l);
    float* st = a.part + (static_cast<int64_t>(kvh) * a.states + un.state + kwave * un.step + 32 * cwave + n) * (HD + 4);
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int x = 0; x < 4; ++x)
            stg(reinterpret_cast<f32x4*>(st + 32 * d + 8 * x + 4 * hh),
                f32x4{acc[d][4 * x], acc[d][4 * x + 1], acc[d][4 * x + 2], acc[d][4 * x + 3]});
    if (hh == 0) stg(reinterpret_cast<f32x2*>(st + HD), f32x2{base, l});
}

// The states of a (sequence, head), in a fixed order: a wave each.
template <int HD>
__global__ __launch_bounds__(256) void kv4_shared_combine_kernel(const ShArgs a) {
    constexpr int E = HD / 64;
    const int lane = threadIdx.x & 63, h = static_cast<int>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = blockIdx.y;
    if (h >= a.NQ) return;
    const ShSeq s = a.seqs[b];
    const int kvh = h / a.rep, r = h - kvh * a.rep, ns = s.pre_n + s.own_n;
    const float* part = a.part + static_cast<int64_t>(kvh) * a.states * (HD + 4);
    auto state = [&](int i) {
        const int at = i < s.pre_n ? s.pre + i * s.pre_step + r : s.own + (i - s.pre_n) * a.rep + r;
        return part + static_cast<int64_t>(at) * (HD + 4);
    };
    float M = kNegBig;
    for (int i = lane; i < ns; i += kWave) M = fmaxf(M, ldg(state(i) + HD));
    M = wave_max_bcast(M);
    float l = 0.0f, v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = 0.0f;
    for (int i0 = 0; i0 < ns; i0 += kWave) {
        f32x2 ml = {kNegBig, 0.0f};
        if (i0 + lane < ns) ml = ldg(reinterpret_cast<const f32x2*>(state(i0 + lane) + HD));
        const float w = fast_exp2(ml.x - M);
        l = fmaf(ml.y, w, l);
        const int here = ns - i0 < kWave ? ns - i0 : kWave;
        for (int i = 0; i < here; i += 4) {
            float x[4][E];
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int e = 0; e < E; ++e) x[k][e] = ldg(state(i0 + (i + k < here ? i + k : i)) + 64 * e + lane);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (i + k >= here) break;
                const float wk = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), i + k));
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = fmaf(x[k][e], wk, v[e]);
            }
        }
    }
    l = wave_sum_bcast(l);
#pragma unroll
    for (int e = 0; e < E; ++e)
        stg(a.out + (static_cast<int64_t>(b) * a.NQ + h) * HD + 64 * e + lane, f32_to_f16_bits(l == 0.0f ? 0.0f : v[e] / l));
}

// The most units and states there can be. Each of the plan's splits but a tile's last costs at least a unit's share, so there
// are at most `want` units more than tiles.
struct ShSizes {
    int64_t cw, want, units, states;
    ShSizes(int64_t B, int64_t G, int64_t NQ, int64_t NKV, int64_t hd, int64_t max_len, int64_t max_shared) {
        const int64_t rep = NQ / NKV, per_group = ceil_div64(B * rep, G < 1 ? 1 : G);
        cw = per_group > 64 ? 4 : per_group > 32 ? 2 : 1;
        want = ceil_div64(256 * sh_per_cu(static_cast<int>(hd)), NKV);
        const int64_t pre_tiles = B * rep / (32 * cw) + G, own_tiles = B * ceil_div64(rep, 32);
        auto units_of = [&](int64_t tiles, int64_t keys) {
            const int64_t most = tiles * ceil_div64(keys, kShKeys);
            return want + tiles < most ? want + tiles : most;
        };
        const int64_t pre = units_of(pre_tiles, max_shared), own = units_of(own_tiles, max_len);
        units = pre + own;
        states = pre * 32 * kShWaves + own * kShWaves * (rep < 32 ? rep : 32);
    }
    size_t bytes(int64_t B, int64_t NKV, int64_t hd) const {
        return sizeof(ShHead) + units * sizeof(ShUnit) + B * sizeof(ShSeq) + static_cast<size_t>(NKV) * states * (hd + 4) * 4;
    }
};

static bool sh_sizes_fit(int64_t B, int64_t G, int64_t NQ, int64_t NKV, int64_t hd, int64_t max_len, int64_t max_shared) {
    return B >= 1 && B <= kShMost && G >= 0 && G <= kShMost && NKV >= 1 && NQ >= NKV && NQ <= 65535 && NQ % NKV == 0 && hd >= 1 && max_len >= 0 &&
           max_len <= (int64_t(1) << 30) && max_shared >= 0 && max_shared <= max_len;
}

}  // namespace soi

using namespace soi;

extern "C" size_t soi_kv4_shared_attention_workspace_bytes(int64_t batch, int64_t groups, int64_t num_q_heads,
                                                           int64_t num_kv_heads, int64_t head_dim, int64_t max_len,
                                                           int64_t max_shared) {
    if (!sh_sizes_fit(batch, groups, num_q_heads, num_kv_heads, head_dim, max_len, max_shared)) return 0;
    return ShSizes(batch, groups, num_q_heads, num_kv_heads, head_dim, max_len, max_shared).bytes(batch, num_kv_heads, head_dim);
}

extern "C" int soi_kv4_shared_attention(const soi_kv4_cache* cache, const uint16_t* q, int64_t q_stride, int64_t num_q_heads,
                                        const int32_t* cu_groups, int64_t groups, const int32_t* shared_lens, int64_t max_len,
                                        int64_t max_shared, uint16_t* out, float scale, void* workspace, size_t workspace_bytes,
                                        void* stream) {
    const char* what = "soi_kv4_shared_attention";
    int st = kv4_check(cache, what);
    if (st) return st;
    const int64_t hd = cache->head_dim, gs = cache->group_size, B = cache->batch, NKV = cache->num_kv_heads;
    SOI_REQUIRE(num_q_heads >= 1 && num_q_heads <= 65535 && num_q_heads % NKV == 0,
                "%s: num_q_heads must be a multiple of num_kv_heads up to 65535", what);
    SOI_REQUIRE(B <= kShMost, "%s: at most %d sequences, got %lld", what, kShMost, (long long)B);
    SOI_REQUIRE(groups >= 0 && groups <= kShMost, "%s: the number of groups must be in [0, %d], got %lld", what, kShMost,
                (long long)groups);
    SOI_REQUIRE(q_stride >= num_q_heads * hd || B == 1, "%s: q rows overlap: stride %lld below %lld", what,
                (long long)q_stride, (long long)(num_q_heads * hd));
    SOI_REQUIRE(max_len >= 0 && max_len <= cache->max_blocks * cache->page_size,
                "%s: max_len must be in [0, max_blocks * page_size]", what);
    SOI_REQUIRE(max_shared >= 0 && max_shared <= max_len, "%s: max_shared must be in [0, max_len]", what);
    SOI_REQUIRE(scale > 0.0f && scale < __builtin_inff(), "%s: scale must be positive and finite", what);
    SOI_REQUIRE(q && out && q != out && cu_groups && shared_lens, "%s: null pointer or out = q", what);
    const ShSizes sz(B, groups, num_q_heads, NKV, hd, max_len, max_shared);
    SOI_REQUIRE(sz.units <= 65535 && sz.states < (int64_t(1) << 31), "%s: too many sequences and heads", what);
    const size_t need = sz.bytes(B, NKV, hd);
    if (!workspace || workspace_bytes < need || !aligned16(workspace)) {
        set_last_error("%s: workspace of %zu bytes (16-byte aligned) needed, got %zu", what, need, workspace_bytes);
        return SOI_ERR_WORKSPACE;
    }
    ShArgs a;
    a.q = q;
    a.q_stride = q_stride;
    a.out = out;
    a.cu = cu_groups;
    a.shared = shared_lens;
    a.head = static_cast<ShHead*>(workspace);
    a.units = reinterpret_cast<ShUnit*>(a.head + 1);
    a.seqs = reinterpret_cast<ShSeq*>(a.units + sz.units);
    a.part = reinterpret_cast<float*>(a.seqs + B);
    a.NQ = static_cast<int>(num_q_heads);
    a.rep = static_cast<int>(num_q_heads / NKV);
    a.G = static_cast<int>(groups);
    a.max_len = static_cast<int>(max_len);
    a.max_shared = static_cast<int>(max_shared);
    a.cw = static_cast<int>(sz.cw);
    a.want = static_cast<int>(sz.want);
    a.most_units = static_cast<int>(sz.units);
    a.states = static_cast<int>(sz.states);
    a.scale_log2 = scale * kLog2e;
    const Kv4Cache c = kv4_device(cache);
    hipStream_t s = as_stream(stream);
    hipLaunchKernelGGL(kv4_shared_plan_kernel, dim3(1), dim3(kShPlan), 0, s, a, c);
    if (sz.units > 0) {
        const dim3 grid(static_cast<unsigned>(NKV), static_cast<unsigned>(sz.units));
#define SOI_X(H, G) hipLaunchKernelGGL((kv4_shared_kernel<H, G>), grid, dim3(kShThreads), 0, s, a, c)
        SOI_KV4_SHAPES(SOI_X);
#undef SOI_X
    }
    const dim3 cgrid(static_cast<unsigned>(ceil_div64(num_q_heads, 4)), static_cast<unsigned>(B));
    if (hd == 64) hipLaunchKernelGGL(kv4_shared_combine_kernel<64>, cgrid, dim3(256), 0, s, a);
    else if (hd == 128) hipLaunchKernelGGL(kv4_shared_combine_kernel<128>, cgrid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(kv4_shared_combine_kernel<256>, cgrid, dim3(256), 0, s, a);
    return launch_status(what);
}
