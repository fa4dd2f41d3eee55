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
// A unit is taken in stages of 64 tokens. The workgroup's four waves unpack a stage's K and V codes into LDS as binary16
// integers (exact), the next stage's bytes on their way into registers meanwhile. Then each wave takes 32 columns
// (v_mfma_f32_32x32x16_f16, lanes n = lane & 31, h = lane >> 5), cw of them side by side, two sharing the stage's tokens where
// cw < 4 (cw 1 leaves two waves that only unpack):
//   * S^T = K Q^T: lane (n, h) ends with the scores of column n and tokens 8 (r >> 2) + 4 h + (r & 3), r < 16; a scale group's
//     sums are multiplied by its scale in binary32;
//   * O^T = V^T P^T takes these, exponentiated, as its B operand as they lie, times V's scale: a set of weights for each scale
//     group, each in two binary16 numbers, the product rounded and what that left, with a matrix instruction for either. V is
//     kept as V^T [dimension][token], tokens in the order that this operand's k slots want (16 j + 4 h + 0 .. 3, + 8 .. 11 side by
//     side: one 16-byte read). The cache's V units hold four tokens of one dimension, so unpacking writes such rows without a
//     transposition;
//   * the base of the exponents follows weight times the stage's largest V scale, so the products fill binary16's range
//     whatever V's size: off by 2^-22 of themselves, or by 2^-25 where the unit's largest product so far is at least 2^11: 2^-36
//     of it. (One binary16 number a weight is off by 2^-11: 45 instead of 49 us for the 64 sequences below, and outputs that
//     differ by 2e-4 from the formula's in 32 bits, where those of two numbers differ by 1e-5 to 4e-5. K and V rounded to binary16
//     values in LDS would save a third of the vector work, with such a rounding each.)
// 16-byte chunks are XOR-swizzled so that operand reads and the unpacked rows' writes spread over the banks.
//
// 64 sequences behind 8192 shared tokens (up to 512 of their own; 32 / 8 heads of 128): plan 5.8, units 42, states added 5.8 us;
// kv4_attention.hip, which reads the prompt 64 times, takes 113 us, but is faster where less is shared: a token behind the shared
// ones costs it a quarter. Bound by the launches' latency and, in a unit, by vector instructions: unpacking, and scales,
// exponentials and conversions of every score, beside 8.9 GFLOP of products (7 us at a library product's rate; half as much
// again for the weights' second numbers). With one number a weight, stages of 128 tokens (two workgroups to a CU instead of three)
// took 57 us in all and those of 64 took 45; page table lookups with branches, and addresses kept in registers until they spilled,
// cost a third of the units' time.
#include "soi_host.h"
#include "soi_kv4.h"
#include "soi_kv4_shared_plan.h"
#include "soi_attn.h"

#include <type_traits>

namespace soi {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

constexpr int kShWaves = 4, kShThreads = kShWaves * kWave;
constexpr int kShRound = 64;                     // shared tokens end on a multiple of this
constexpr int kShMost = 2048;                    // sequences of a call
constexpr float kShLow = 12.0f, kShHigh = 15.0f;  // a column's largest weight times V scale is between 2^kShLow and 2^kShHigh
// workgroups that a CU's registers hold
constexpr int sh_per_cu(int hd, int gs) { return hd == 64 ? 4 : hd == 256 ? 1 : gs == 32 ? 2 : 3; }

struct ShUnit {
    int row, key0, key1;    // tokens key0 .. key1 - 1 of page table row `row`
    int seq0, col0, ncols;  // columns col0 .. col0 + ncols - 1 of the sequences from seq0 on
    int state, cw;          // state of its first column; waves side by side
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

template <int NT>
__device__ __forceinline__ int64_t sh_scan(int64_t v, int64_t* s_part, int64_t& all) {  // exclusive over the threads, and the sum
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t x = v;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const int64_t y = __shfl_up(x, o);
        x += lane >= o ? y : 0;
    }
    if (lane == 63) s_part[wave] = x;
    __syncthreads();
    int64_t base = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < NT / kWave; ++w) {
        base += w < wave ? s_part[w] : 0;
        all += s_part[w];
    }
    __syncthreads();
    return base + x - v;
}

// The units of a call, and where each sequence's states are. A group shares what all its sequences that share anything have
// in common, so that a unit's columns all see all its tokens; sequences outside every group share nothing. NT: a thread for
// each sequence and group, where 1024 are enough.
template <int NT>
__global__ __launch_bounds__(NT) void kv4_shared_plan_kernel(const ShArgs a, const Kv4Cache c) {
    // of each group: first sequence, shared tokens, the first sequence that shares them, its first unit and state; of each
    // sequence: its length, its group (none: kNone) if it shares anything
    constexpr int kMost = NT < 1024 ? NT : kShMost, kNone = 0xffff;
    __shared__ int s_cu[kMost + 1], s_keys[kMost], s_row[kMost], s_unit[kMost], s_state[kMost], s_len[kMost];
    __shared__ uint16_t s_group[kMost];
    __shared__ int64_t s_part[NT / kWave];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, B = c.B, rep = a.rep;
    for (int g = tid; g <= a.G; g += NT) s_cu[g] = ldg(a.cu + g);
    for (int g = tid; g < a.G; g += NT) s_keys[g] = s_row[g] = 0x7fffffff;
    int shared[kMost / NT];
#pragma unroll
    for (int i = 0; i < kMost / NT; ++i) {
        const int b = tid + i * NT;
        if (b < B) {
            int L = ldg(c.lens + b), n = ldg(a.shared + b);
            L = L < 0 ? 0 : L < a.max_len ? L : a.max_len;
            n = n < a.max_shared ? n : a.max_shared;
            n = n < L ? n : L;
            shared[i] = n < kShRound ? 0 : n / kShRound * kShRound;
            s_len[b] = L;
        }
    }
    __syncthreads();
    int bad = 0;
    for (int g = tid; g <= a.G; g += NT) bad |= s_cu[g] < (g ? s_cu[g - 1] : 0) || s_cu[g] > B;
    const int G = __syncthreads_or(bad) ? 0 : a.G;  // offsets that are none: nobody shares anything
#pragma unroll
    for (int i = 0; i < kMost / NT; ++i) {
        const int b = tid + i * NT;
        if (b >= B) continue;
        int lo = 0, hi = G;  // the last g < G with cu[g] <= b
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s_cu[mid] <= b) lo = mid;
            else hi = mid;
        }
        const bool in = G > 0 && s_cu[lo] <= b && b < s_cu[lo + 1] && shared[i] > 0;
        s_group[b] = static_cast<uint16_t>(in ? lo : kNone);
        if (in) {
            atomicMin(&s_keys[lo], shared[i]);
            atomicMin(&s_row[lo], b);
        }
    }
    __syncthreads();
    const int width = 32 * a.cw, own_tiles = (rep + 31) / 32;
    auto keys_of = [&](int g) { return s_row[g] == 0x7fffffff ? 0 : s_keys[g]; };
    auto columns = [&](int g) { return (s_cu[g + 1] - s_cu[g]) * rep; };
    auto tiles = [&](int g) { return (columns(g) + width - 1) / width; };
    auto start_of = [&](int b) { return s_group[b] == kNone ? 0 : keys_of(s_group[b]); };
    int64_t cost = 0, total;
    for (int g = tid; g < G; g += NT) cost += static_cast<int64_t>(tiles(g)) * sh_stages(keys_of(g)) * sh_cost(a.cw);
    for (int b = tid; b < B; b += NT) cost += static_cast<int64_t>(own_tiles) * sh_stages(s_len[b] - start_of(b)) * sh_cost(1);
    sh_scan<NT>(cost, s_part, total);
    const int pre_per = sh_per_unit(total, a.want, sh_cost(a.cw)), own_per = sh_per_unit(total, a.want, sh_cost(1));
    auto both = [](int units, int64_t states) { return states << 24 | units; };  // (at most 65535 units, 2^31 states)
    int64_t at = 0;
    for (int g0 = 0; g0 < G; g0 += NT) {
        const int g = g0 + tid, ns = g < G ? sh_splits(keys_of(g), pre_per) : 0;
        int64_t all;
        const int64_t x = at + sh_scan<NT>(ns ? both(tiles(g) * ns, static_cast<int64_t>(columns(g)) * ns) : 0, s_part, all);
        if (g < G) {
            s_unit[g] = static_cast<int>(x & 0xffffff);
            s_state[g] = static_cast<int>(x >> 24);
        }
        at += all;
    }
    __syncthreads();
    for (int g = wave; g < G; g += NT / kWave) {  // a wave lists a group's units
        const int keys = keys_of(g), ns = sh_splits(keys, pre_per), cols = columns(g), n = ns ? tiles(g) * ns : 0;
        for (int i = lane; i < n; i += kWave) {
            const int t = i / ns, k = i - t * ns, k0 = k * pre_per * kShKeys, k1 = k0 + pre_per * kShKeys;
            const int left = cols - t * width;
            if (s_unit[g] + i < a.most_units)
                a.units[s_unit[g] + i] = ShUnit{s_row[g], k0, k1 < keys ? k1 : keys, s_cu[g], t * width, left < width ? left : width,
                                                s_state[g] + k * cols + t * width, a.cw};
        }
    }
    for (int b0 = 0; b0 < B; b0 += NT) {
        const int b = b0 + tid, L = b < B ? s_len[b] : 0, start = b < B ? start_of(b) : 0, ns = sh_splits(L - start, own_per);
        int64_t all;
        const int64_t x = at + sh_scan<NT>(both(ns * own_tiles, static_cast<int64_t>(ns) * rep), s_part, all);
        at += all;
        if (b >= B) continue;
        int u = static_cast<int>(x & 0xffffff);
        const int s = static_cast<int>(x >> 24);
        for (int t = 0; t < own_tiles; ++t)
            for (int k = 0; k < ns; ++k, ++u) {
                const int k0 = start + k * own_per * kShKeys, k1 = k0 + own_per * kShKeys, left = rep - 32 * t;
                if (u < a.most_units)
                    a.units[u] = ShUnit{b, k0, k1 < L ? k1 : L, b, 32 * t, left < 32 ? left : 32, s + k * rep + 32 * t, 1};
            }
        const int g = start ? s_group[b] : 0, cols = start ? columns(g) : 0, ps = start ? s_state[g] : 0;
        const int pn = start ? sh_splits(start, pre_per) : 0;
        // (none where states would lie past the workspace, which ShSizes says they do not)
        const bool pre_fits = ps + static_cast<int64_t>(pn) * cols <= a.states, own_fits = s + static_cast<int64_t>(ns) * rep <= a.states;
        a.seqs[b] = ShSeq{start ? ps + (b - s_cu[g]) * rep : 0, cols, pre_fits ? pn : 0, s, own_fits ? ns : 0, {0, 0, 0}};
    }
    if (tid == 0) {
        const int units = static_cast<int>(at & 0xffffff);
        a.head->units = units < a.most_units ? units : a.most_units;
    }
}

// an index that the compiler does not compute ahead of the loop and keep (addresses that differ in a few bits would take more
// registers than there are)
__device__ __forceinline__ int sh_here(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

// the waves' LDS writes are done, and all reads before; loads into registers stay in flight
__device__ __forceinline__ void sh_meet() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// (a lo(s), b hi(s)) as binary16, each product rounded once; less the same products in `from`
__device__ __forceinline__ uint32_t times_f16(float a, float b, uint32_t s, uint32_t from = 0) {
    const f16x2 w = as_f16x2(s), f = as_f16x2(from);  // (fma, not a product: one mixed-precision instruction)
    return __builtin_bit_cast(uint32_t, f16x2{static_cast<f16>(fmaf(a, static_cast<float>(w.x), -static_cast<float>(f.x))),
                                              static_cast<f16>(fmaf(b, static_cast<float>(w.y), -static_cast<float>(f.y)))});
}

// physical 16-byte chunk of chunk c: c ^ swizzle, of a K row (HD / 8 chunks) and of a V row (8 chunks: the stage's tokens)
template <int HD>
__device__ __forceinline__ int sh_swz_k(int key) {
    return HD == 64 ? (key >> 1) & 7 : (key & 3) << 2 | ((key >> 2) & 3);
}
__device__ __forceinline__ int sh_swz_v(int dim) { return (dim >> 1) & 7; }

// BIG: pages of at least a stage, so a stage lies in one page, and its addresses are wave-uniform but for the lane's offset.
template <int HD, int GS, bool BIG>
__global__ __launch_bounds__(kShThreads, sh_per_cu(HD, GS)) void kv4_shared_kernel(const ShArgs a, const Kv4Cache c) {
    constexpr int W = HD / 32, U = HD / 64, G = HD / GS, KK = HD / 16, DT = HD / 32, ROWB = 2 * HD, VROWB = 2 * kShKeys;
    // K: KT pieces of 16 bytes, of PK that a token has, a thread; V: eight tokens of UU blocks of 64 dimensions a thread. Heads
    // of 64 have enough for half the threads: the first half unpacks V, the second K.
    constexpr int PK = HD / 32, KT = HD == 256 ? 2 : 1, UU = HD == 256 ? 2 : 1;
    static_assert(G <= PK && 2 * G <= 16, "a piece of K, and a lane m of V, for each scale");
    __shared__ __attribute__((aligned(1024))) uint8_t s_kv[kShKeys * ROWB + HD * VROWB];
    uint8_t *const s_k = s_kv, *const s_v = s_kv + kShKeys * ROWB;
    // scales, zeros for tokens that are not there; K's times scale_log2
    __shared__ __attribute__((aligned(16))) float s_ks[G][kShKeys];
    __shared__ __attribute__((aligned(16))) uint16_t s_vs[G][kShKeys];
    __shared__ uint32_t s_valid;   // a byte for each 16 tokens of the stage: they have a page
    __shared__ __attribute__((aligned(8))) float s_top[2][2];  // bits of the largest finite V scale, by two waves, two stages
    __shared__ f32x2 s_state[2][32];  // (base, weight) of a wave's columns
    const int units = ldg(&a.head->units);
    const ShUnit un = a.units[blockIdx.y];  // (read whether there is one or not: one round trip)
    if (static_cast<int>(blockIdx.y) >= units) return;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n = lane & 31, hh = lane >> 5;
    const int kvh = blockIdx.x, cwave = wave % un.cw, kwave = wave / un.cw;
    const int kw = un.cw == 4 ? 1 : 2;  // waves that share a stage's tokens (cw 1 leaves two that only unpack)
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
    // dimensions 64 (v_u + u) + 16 k + m.
    const bool has_k = HD > 64 || tid >= kShThreads / 2, has_v = HD > 64 || tid < kShThreads / 2;  // (the same for a wave)
    struct Part {
        uint32_t id, k_p, m, vh, j, v_u;
        __device__ __forceinline__ Part()
            : id(static_cast<uint32_t>(sh_here(static_cast<int>(threadIdx.x)))), k_p(id % PK), m(id & 15), vh((id >> 4) & 1), j((id >> 5) & 3),
              v_u(HD > 64 ? UU * (id >> 7) : 0) {}
        __device__ __forceinline__ int k_key(int t) const {
            return ((HD > 64 ? id : id & (kShThreads / 2 - 1)) + kShThreads * t) / PK;
        }
    };
    u32x4 kraw[KT];
    uint16_t ksc[KT];  // the token's scale of group k_p, if there is one
    u32x2 vraw[2][UU], vsc;  // lanes m < 2 G: the scales of four tokens, + 8 (m & 1), of group m >> 1
    constexpr int NID = BIG ? 1 : KT + 1;  // page table entries of a stage: its one page, or the K pieces' and V's
    int ids[NID];                          // pages, -1: none
    // The entries as the table has them, without a branch: nothing waits for them here.
    const int32_t* table = c.table + static_cast<int64_t>(un.row) * c.max_blocks;
    auto entry = [&](int pos) {
        const int blk = pos >> c.page_shift;
        return ldg(table + (blk < c.max_blocks ? blk : 0));
    };
    auto page = [&](int pos, int id) { return pos >> c.page_shift < c.max_blocks && id >= 0 && id < c.P ? id : -1; };
    auto pages = [&](int key0, int (&e)[NID]) {
        if constexpr (BIG) {
            e[0] = entry(key0);
        } else {
            const Part p;
#pragma unroll
            for (int t = 0; t < KT; ++t) e[t] = entry(key0 + p.k_key(t));
            e[KT] = entry(key0 + 16 * p.j);
        }
    };
    auto check = [&](int key0, const int (&e)[NID]) {
        if constexpr (BIG) {
            ids[0] = page(key0, __builtin_amdgcn_readfirstlane(e[0]));
        } else {
            const Part p;
#pragma unroll
            for (int t = 0; t < KT; ++t) ids[t] = page(key0 + p.k_key(t), e[t]);
            ids[KT] = page(key0 + 16 * p.j, e[KT]);
        }
    };
    // (page, head) of an entry; every one of them takes 256 bytes or more, so their number has 31 bits
    auto head_of = [&](int id) { return static_cast<uint32_t>(id < 0 ? 0 : id) * static_cast<uint32_t>(c.NKV) + kvh; };
    const uint32_t page_bytes = c.page * (HD / 2), scale_count = G * c.page;
    auto fetch = [&](int key0) {
        const Part p;
        const int lead = key0 & (c.page - 1);  // BIG: the stage's first slot
        if (has_k) {
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                const uint64_t h = head_of(ids[BIG ? 0 : t]);
                const uint32_t slot = BIG ? p.k_key(t) : (key0 + p.k_key(t)) & (c.page - 1), g = p.k_p < G ? p.k_p : 0;
                const uint8_t* kp = c.k_pages + (h * page_bytes + (BIG ? lead * (HD / 2) : 0));
                const uint16_t* sp = c.k_scale + (h * scale_count + (BIG ? lead : 0));
                kraw[t] = ldg(reinterpret_cast<const u32x4*>(kp + (slot * (HD / 2) + 16 * p.k_p)));
                ksc[t] = ldg(sp + (g * c.page + slot));
            }
        }
        if (has_v) {
            const uint64_t h = head_of(ids[NID - 1]);
            const uint32_t first = 16 * p.j + 4 * p.vh, slot = BIG ? first : (key0 + first) & (c.page - 1);
            const uint8_t* vp = c.v_pages + (h * page_bytes + (BIG ? lead * (HD / 2) : 0));
            const uint16_t* sp = c.v_scale + (h * scale_count + (BIG ? lead : 0));
            const uint32_t off = (slot >> 2) * (16 * U * 8) + (p.m * U + p.v_u) * 8;
            vsc = ldg(reinterpret_cast<const u32x2*>(sp + ((p.m < 2 * G ? p.m >> 1 : 0) * c.page + slot + 8 * (p.m & 1))));
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                if constexpr (UU == 1) {
                    vraw[x][0] = ldg(reinterpret_cast<const u32x2*>(vp + (off + x * 2 * (16 * U * 8))));
                } else {
                    const u32x4 r = ldg(reinterpret_cast<const u32x4*>(vp + (off + x * 2 * (16 * U * 8))));
                    vraw[x][0] = u32x2{r.x, r.y};
                    vraw[x][1] = u32x2{r.z, r.w};
                }
            }
        }
    };
    // Tokens that are not there (past the unit, or without a page) get scales 0: theirs may be anything.
    auto unpack_k = [&](int key0, bool whole) {
        const Part p;
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            const int key = p.k_key(t);
            float ks = f16_bits_to_f32(ksc[t]) * a.scale_log2;
            if (!whole) ks = ids[BIG ? 0 : t] >= 0 && key0 + key < un.key1 ? ks : 0.0f;
            if (p.k_p < G) s_ks[p.k_p][key] = ks;
            const int row = sh_here(key * ROWB);
            const uint32_t word[4] = {kraw[t].x, kraw[t].y, kraw[t].z, kraw[t].w};
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int w = 4 * p.k_p + x, i = HD == 256 ? 4 * (p.k_p & 1) + x : w % W, g = w / W;  // word W g + i: chunk 4 i + g
                f16x2 v[4];
                dequant_int4x8_bitfield(word[x], v);
                const f16x8 o = {v[0].x, v[0].y, v[1].x, v[1].y, v[2].x, v[2].y, v[3].x, v[3].y};
                *reinterpret_cast<f16x8*>(s_k + row + (((4 * i + g) ^ sh_swz_k<HD>(key)) << 4)) = o;
            }
        }
    };
    auto unpack_v = [&](int key0, int odd, bool whole) {
        const Part p;
        const int m = p.m, vh = p.vh, j = p.j, v_u = p.v_u;
        if (!BIG && (tid & 31) == 0) reinterpret_cast<uint8_t*>(&s_valid)[j] = ids[NID - 1] >= 0;
        if (wave < 2) {  // (waves of v_u 0: the scales are theirs)
            uint32_t w[2] = {vsc.x, vsc.y};
            if (!whole) {
                const int left = ids[NID - 1] < 0 ? 0 : un.key1 - key0 - 16 * j - 4 * vh - 8 * (m & 1);  // tokens that are there
                w[0] = left > 1 ? w[0] : left == 1 ? w[0] & 0xffffu : 0u;
                w[1] = left > 3 ? w[1] : left == 3 ? w[1] & 0xffffu : 0u;
            }
            if (m < 2 * G) *reinterpret_cast<u32x2*>(&s_vs[m >> 1][16 * j + 4 * vh + 8 * (m & 1)]) = u32x2{w[0], w[1]};
            // (lanes past 2 G repeat group 0's first scales)
            u16x2 t[2];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const u16x2 v = __builtin_bit_cast(u16x2, w[y] & 0x7fff7fffu);
                t[y] = v & (v < (uint16_t)0x7c00);
            }
            const u16x2 most = __builtin_elementwise_max(t[0], t[1]);
            const float wave_top = wave_max_bcast(static_cast<float>(max(most.x, most.y)));
            if (lane == 0) s_top[odd][wave] = wave_top;
        }
#pragma unroll
        for (int u = 0; u < UU; ++u)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int dim = 64 * (v_u + u) + 16 * k + m;
                f16x2 v[2][2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const uint32_t w[2] = {vraw[x][u].x, vraw[x][u].y};  // tokens (0, 1), (2, 3)
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
                *reinterpret_cast<f16x8*>(s_v + dim * VROWB + (((2 * j + vh) ^ sh_swz_v(dim)) << 4)) = o;
            }
    };

    f32x16 acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] = 0.0f;
    float base = 0.0f, l = 0.0f;
    bool fresh = true;  // no token yet
    // scale_top: binades from the stage's largest V scale up to 1
    auto products = [&](int key0, int sub, bool whole, uint32_t valid, float scale_top) {
        const int at = sh_here(32 * sub + 4 * hh);  // the lane's first token, the others 8 (r >> 2) + (r & 3) further
        float z[16];                                // score in binades, less the base
        const int k_at = sh_here((32 * sub + n) * ROWB + ((hh ^ sh_swz_k<HD>(n)) << 4));  // K's chunk hh, 2 kk + hh: bits flipped
#pragma unroll
        for (int g = 0; g < G; ++g) {
            f32x16 sum;
#pragma unroll
            for (int r = 0; r < 16; ++r) sum[r] = 0.0f;
#pragma unroll
            for (int kk = g * (GS / 16); kk < (g + 1) * (GS / 16); ++kk) {
                const f16x8 kf = *reinterpret_cast<const f16x8*>(s_k + (k_at ^ (kk << 5)));
                sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[kk], sum, 0, 0, 0);
                if ((kk & 3) == 3) __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const f32x4 sc = *reinterpret_cast<const f32x4*>(&s_ks[g][at + 8 * x]);
#pragma unroll
                for (int e = 0; e < 4; ++e) z[4 * x + e] = fmaf(sum[4 * x + e], sc[e], g ? z[4 * x + e] : -base);
            }
            __builtin_amdgcn_sched_barrier(0);  // (all groups at once would spill)
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
        top = fmaxf(top, xor_lanes<32>(top)) - scale_top;
        // the base rises only where a product would pass 2^kShHigh, to where the largest is 2^kShLow (and is set so by the first
        // token that is there); a column does not depend on its neighbours
        const bool raise = top > kShHigh || (fresh && top > -__builtin_inff());
        if (ballot(raise)) {
            const float by = raise ? top - kShLow : 0.0f, w = fresh ? 0.0f : fast_exp2(-by);
            fresh = fresh && !raise;
            base += by;
            l *= w;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[d][r] *= w;
#pragma unroll
            for (int r = 0; r < 16; ++r) z[r] -= by;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            z[r] = fast_exp2(z[r]);
            l += z[r];
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            u32x4 pb[2], rest[2];  // the products rounded, and what the rounding left
            const int v_at = sh_here(n * VROWB + (((4 * sub + hh) ^ sh_swz_v(n)) << 4));
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const u32x2 sc = *reinterpret_cast<const u32x2*>(&s_vs[g][at + 8 * x]);
                const uint32_t w[2] = {sc.x, sc.y};
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const float p0 = z[4 * x + 2 * y], p1 = z[4 * x + 2 * y + 1];
                    uint32_t top = times_f16(p0, p1, w[y]);
                    asm("" : "+v"(top));  // (one value: it came in two roundings where the compiler made it twice)
                    pb[x >> 1][2 * (x & 1) + y] = top;
                    rest[x >> 1][2 * (x & 1) + y] = times_f16(p0, p1, w[y], top);
                }
            }
#pragma unroll
            for (int d = g * (GS / 32); d < (g + 1) * (GS / 32); ++d) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const f16x8 vf = *reinterpret_cast<const f16x8*>(s_v + (v_at ^ (x << 5)) + 32 * d * VROWB);
                    acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, __builtin_bit_cast(f16x8, pb[x]), acc[d], 0, 0, 0);
                    acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, __builtin_bit_cast(f16x8, rest[x]), acc[d], 0, 0, 0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    int next[NID];
    pages(un.key0, next);
    check(un.key0, next);
    pages(un.key0 + kShKeys, next);
    fetch(un.key0);
    int odd = 0;
    for (int key0 = un.key0; key0 < un.key1; key0 += kShKeys, odd ^= 1) {
        if (key0 > un.key0) sh_meet();  // the stage before is read
        const bool inside = key0 + kShKeys <= un.key1, there = BIG && ids[0] >= 0;
        if (has_k) unpack_k(key0, inside && there);
        if (has_v) unpack_v(key0, odd, inside && there);
        if (key0 + kShKeys < un.key1) {
            check(key0 + kShKeys, next);
            fetch(key0 + kShKeys);
            pages(key0 + 2 * kShKeys, next);
        }
        sh_meet();
        const uint32_t valid = BIG ? (there ? 0x01010101u : 0u) : s_valid;
        const bool whole = inside && valid == 0x01010101u;
        const f32x2 tops = *reinterpret_cast<const f32x2*>(s_top[odd]);
        const int top_bits = static_cast<int>(fmaxf(tops.x, tops.y));
        const float scale_top = 14.0f - static_cast<float>(top_bits >> 10);  // (the exponent's bits: scales below 2^(bits - 14))
        if (wcols <= 0 || kwave >= kw) continue;
        const int subs = min(kShKeys / 32, (un.key1 - key0 + 31) >> 5);
        for (int sub = kwave; sub < subs; sub += kw) products(key0, sub, whole, valid, scale_top);
    }
    if (fresh) base = kNegBig;
    l += xor_lanes<32>(l);
    // the second of two waves that share the unit's tokens hands its state to the first through LDS, where K and V were
    if (kw > 1) {
        static_assert(2 * 32 * HD * 4 <= kShKeys * ROWB + HD * VROWB, "room for two waves' states");
        uint8_t* st = s_kv + (cwave * 32 + n) * HD * 4;
        sh_meet();
        if (kwave == 1) {
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    *reinterpret_cast<f32x4*>(st + (((8 * d + 2 * x + hh) ^ (n & 15)) << 4)) =
                        f32x4{acc[d][4 * x], acc[d][4 * x + 1], acc[d][4 * x + 2], acc[d][4 * x + 3]};
            if (hh == 0) s_state[cwave][n] = f32x2{base, l};
        }
        sh_meet();
        if (kwave > 0) return;
        const f32x2 bl = s_state[cwave][n];
        const float top = fmaxf(base, bl.x), w0 = fast_exp2(base - top), w1 = fast_exp2(bl.x - top);
        base = top;
        l = fmaf(l, w0, bl.y * w1);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const f32x4 v = *reinterpret_cast<const f32x4*>(st + (((8 * d + 2 * x + hh) ^ (n & 15)) << 4));
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[d][4 * x + e] = fmaf(acc[d][4 * x + e], w0, v[e] * w1);
            }
    }
    if (n >= wcols) return;
    float* st = a.part + (static_cast<int64_t>(kvh) * a.states + un.state + 32 * cwave + n) * (HD + 4);
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
    // the first states' sums are requested with the (base, weight) pairs: up to kFirst states are two round trips
    constexpr int kFirst = 16;
    auto pair = [&](int i) { return i < ns ? ldg(reinterpret_cast<const f32x2*>(state(i) + HD)) : f32x2{kNegBig, 0.0f}; };
    float x[kFirst][E];
    auto load = [&](int i0) {
#pragma unroll
        for (int k = 0; k < kFirst; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e) x[k][e] = i0 + k < ns ? ldg(state(i0 + k) + 64 * e + lane) : 0.0f;
    };
    const f32x2 first = pair(lane);
    load(0);
    float M = first.x;
    for (int i = lane + kWave; i < ns; i += kWave) M = fmaxf(M, ldg(state(i) + HD));
    M = wave_max_bcast(M);
    float l = 0.0f, v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = 0.0f;
    for (int i0 = 0; i0 < ns; i0 += kWave) {
        const f32x2 ml = i0 ? pair(i0 + lane) : first;
        const float w = fast_exp2(ml.x - M);
        l = fmaf(ml.y, w, l);
        for (int i = i0; i < ns && i < i0 + kWave; i += kFirst) {
            if (i) load(i);
#pragma unroll
            for (int k = 0; k < kFirst; ++k) {
                if (i + k >= ns) break;
                const float wk = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), i - i0 + k));
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

static size_t sh_bytes(const ShSizes& sz, int64_t B, int64_t NKV, int64_t hd) {
    return sizeof(ShHead) + sz.units * sizeof(ShUnit) + B * sizeof(ShSeq) + static_cast<size_t>(NKV) * sz.states * (hd + 4) * 4;
}

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
    return sh_bytes(ShSizes(batch, groups, num_q_heads, num_kv_heads, head_dim, max_len, max_shared), batch, num_kv_heads, head_dim);
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
    const size_t need = sh_bytes(sz, B, NKV, hd);
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
    if (B <= 256 && groups <= 256) hipLaunchKernelGGL(kv4_shared_plan_kernel<256>, dim3(1), dim3(256), 0, s, a, c);
    else hipLaunchKernelGGL(kv4_shared_plan_kernel<1024>, dim3(1), dim3(1024), 0, s, a, c);
    if (sz.units > 0) {
        const dim3 grid(static_cast<unsigned>(NKV), static_cast<unsigned>(sz.units));
#define SOI_X(H, G)                                                                                              \
    do {                                                                                                         \
        if (cache->page_size >= kShKeys)                                                                         \
            hipLaunchKernelGGL((kv4_shared_kernel<H, G, true>), grid, dim3(kShThreads), 0, s, a, c);             \
        else                                                                                                     \
            hipLaunchKernelGGL((kv4_shared_kernel<H, G, false>), grid, dim3(kShThreads), 0, s, a, c);            \
    } while (0)
        SOI_KV4_SHAPES(SOI_X);
#undef SOI_X
    }
    const dim3 cgrid(static_cast<unsigned>(ceil_div64(num_q_heads, 4)), static_cast<unsigned>(B));
    if (hd == 64) hipLaunchKernelGGL(kv4_shared_combine_kernel<64>, cgrid, dim3(256), 0, s, a);
    else if (hd == 128) hipLaunchKernelGGL(kv4_shared_combine_kernel<128>, cgrid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(kv4_shared_combine_kernel<256>, cgrid, dim3(256), 0, s, a);
    return launch_status(what);
}
