// One query token per sequence over the paged 4-bit KV cache (soi_kv4.h), gfx950.
//
// out[b, h] = sum_t softmax_t(scale q[b, h] . k_t) v_t over the tokens t < lens[b] of KV head h / (NQ / NKV), as the
// reference's decode_attention (csrc/kernels/decode_attention.cu:17-55) for every sequence of a batch.
//
// Bound by reading the cache, 2 (hd / 2 + 2 hd / gs) bytes per token and KV head. The dot products have rep = NQ / NKV
// rows for each of those bytes, too many for v_dot2 at rep 8, so they run on the matrix cores with the heads as one
// 16-column operand (v_mfma_f32_16x16x32_f16, lanes c = lane & 15, g = lane >> 4):
//   * a wave takes blocks of 64 tokens. Row m of score tile i < 4 is token 16 (m >> 2) + 4 i + (m & 3) of the block, so
//     that lane (c, g) ends with the scores of head c and tokens 16 g .. 16 g + 15: one 16-token piece of a page, whose
//     scales are 32 consecutive bytes, and which is where the V operand's k slots want them;
//   * S^T = K Q^T: the A operand of step i is word i of the lane's W words of its token, the nibbles as exact binary16
//     integers; a step covers 32 dimensions, inside one quantization group, so the binary16 scale multiplies the
//     step's binary32 sum;
//   * O^T = V^T P^T: the lane's own scores are its B operand (k slots (g, 0 .. 7) of half a block: tokens 16 g + 8 half
//     + 0 .. 7); the A operand of 16 dimensions is a nibble of its V units. V's scale enters with p, in binary32,
//     before the one rounding to binary16 that the matrix cores need; the sum of p is taken unrounded;
//   * p = 2^(score - base), where the base keeps the largest p times the wave's largest V scale so far in [2^14, 2^15): the
//     products fill binary16's range whatever V's size, are rounded by 2^-11 of their own value down to 2^-28 of the
//     largest, and end in 0 below 2^-40 of it (V scales below 2^-14 count as 2^-14 here);
//   * the base is one per head and wave (two lane swaps a block), sums are rescaled only in a block that raises one of them.
// No operand is reordered between lanes. The scales of a block pass through LDS (a wave's own part: each lane loads 16
// bytes of them, and reads back the 32 bytes it needs of each group), K and V go straight to registers, a block ahead.
//
// Work is split evenly whatever the lengths: the blocks of all sequences, in order, are cut into splits of `bps` blocks,
// none across two sequences, bps following from the sum of the lengths on the device. Workgroup (head, y) finds split y
// by a scan over the sequences. A sequence of one split is written at once; the states of more are combined in split
// order by a second launch.
//
// Measured: 4 contexts of up to 131072 tokens (386002 in all), 64 / 8 heads of 128, groups of 64 (420 MB): 84 us, 5.0 TB/s,
// what a large copy reaches on this card (a pure read can reach 7). 48 contexts of 1870 tokens on average, 32 / 8 heads,
// groups of 32, pages of 16 (104 MB): 35 to 36 us, 31.4 of them the first launch (3.3 TB/s: a page is 1 KB of K here, each
// wave waits for its table entries, and the nibbles' arithmetic is most of a block's time; 1.3 us of it came with the base
// that follows V's scales, most of that in a wave's first block); one context of 2000: 8.5 us, two dependent launches of
// 5.4 and 3.4 us. Heads of 256: 8 contexts, 251773 tokens, 16 / 2 heads, groups of 64 (137 MB): 36 us, 3.8 TB/s.
// Registers, not LDS, set the workgroups of a CU (4 / 3 / 2 for 64 / 128 / 256 dimensions); K and V registers are loaded
// again as soon as their products are issued, so that a block's loads are in flight during the rest of the block before.
#include "soi_host.h"
#include "soi_kv4.h"
#include "soi_attn.h"

#include <type_traits>

namespace soi {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

constexpr int kKv4Waves = 4;
constexpr int kKv4Block = 64;  // tokens a wave takes at a time
constexpr int kv4_per_cu(int hd) { return hd == 64 ? 4 : hd == 128 ? 3 : 2; }  // workgroups that a CU's registers hold

struct Kv4AttnArgs {
    const uint16_t* q;
    int64_t q_stride;
    uint16_t* out;
    float* part;  // [splits][NQ][HD + 2]: m, l, acc
    int NQ, rep, htiles, want, max_len;
    float scale_log2;
};

__device__ __forceinline__ int kv4_len(const Kv4Cache& c, int b, int max_len) {
    const int L = ldg(c.lens + b);
    return L < 0 ? 0 : L < max_len ? L : max_len;
}

// blocks of a context; an empty one has a block too, whose workgroup writes the zeros
__device__ __forceinline__ int kv4_blocks(int L) { return L <= kKv4Block ? 1 : (L + kKv4Block - 1) / kKv4Block; }

__device__ __forceinline__ int wave_scan(int v) {  // inclusive sum over the lanes
    auto up = [](int x, auto ctrl, auto rows) {
        return __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
    };
    using std::integral_constant;
    v += up(v, integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});
    v += up(v, integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
    v += up(v, integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
    v += up(v, integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
    v += up(v, integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});
    v += up(v, integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});
    return v;
}

// Where split y lies (FIND_SPLIT), or where the splits of sequence `at` begin: blocks per split `bps` (about `want` splits of
// all sequences' blocks together, whole rounds of a workgroup's waves), the sequence b (-1: there is no split y) with its
// length L, the split within it, and the index y0 of its first split. Every wave runs the same scan; up to 64 sequences are
// one load.
struct Kv4Place {
    int bps, b, L, split, y0;
};
template <bool FIND_SPLIT>
__device__ __forceinline__ Kv4Place kv4_place(const Kv4AttnArgs& a, const Kv4Cache& c, int lane, int at) {
    auto len_of = [&](int s) { return s + lane < c.B ? kv4_len(c, s + lane, a.max_len) : -1; };
    auto blocks_of = [](int L) { return L < 0 ? 0 : kv4_blocks(L); };
    const int len0 = len_of(0);
    int total = blocks_of(len0);
    for (int s = kWave; s < c.B; s += kWave) total += blocks_of(len_of(s));
    total = __builtin_amdgcn_readlane(wave_scan(total), 63);
    Kv4Place p{0, -1, 0, 0, 0};
    p.bps = ((total + a.want - 1) / a.want + kKv4Waves - 1) / kKv4Waves * kKv4Waves;
    for (int s = 0; s < c.B; s += kWave) {
        const int len = s ? len_of(s) : len0;
        const int ns = (blocks_of(len) + p.bps - 1) / p.bps;
        const int incl = wave_scan(ns), all = __builtin_amdgcn_readlane(incl, 63);
        if (FIND_SPLIT ? at < p.y0 + all : at < s + kWave) {
            const int i = FIND_SPLIT ? __builtin_ctzll(ballot(p.y0 + incl > at)) : at - s;
            p.b = s + i;
            p.L = __builtin_amdgcn_readlane(len, i);
            p.y0 += i ? __builtin_amdgcn_readlane(incl, i - 1) : 0;
            p.split = at - p.y0;
            return p;
        }
        p.y0 += all;
    }
    return p;
}

template <int HD, int GS>
struct Kv4Block {
    static constexpr int W = HD / 32, U = HD / 64, G = HD / GS, SC = G <= 4 ? 1 : 2;
    uint32_t k[4][W];  // tile i: W words of the lane's token
    u32x2 v[4][U];     // quad i: units of tokens 4 i .. 4 i + 3 (of 16 g ..)
    u32x4 s[SC];       // 16 bytes of the block's scales
};

// BIG: pages of at least a block, so a block lies in one page and its addresses are wave-uniform but for the lane's offset.
template <int HD, int GS, bool BIG>
__global__ __launch_bounds__(kKv4Waves * kWave, kv4_per_cu(HD)) void kv4_attn_kernel(const Kv4AttnArgs a, const Kv4Cache c) {
    constexpr int W = HD / 32, U = HD / 64, G = HD / GS, DT = HD / 16, SC = Kv4Block<HD, GS>::SC;
    __shared__ float s_state[kKv4Waves][16][HD + 2];
    __shared__ __attribute__((aligned(16))) uint16_t s_scale[kKv4Waves][2][G][4][16];  // K, V; group; piece; token
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int col = lane & 15, g = lane >> 4;
    const int kvh = static_cast<int>(blockIdx.x) / a.htiles, ht = static_cast<int>(blockIdx.x) % a.htiles;
    const int y = blockIdx.y;
    const Kv4Place at = kv4_place<true>(a, c, lane, y);
    if (at.b < 0) return;
    const int b = at.b, L = at.L, split = at.split, bps = at.bps;
    const int nb = kv4_blocks(L);
    const int b1 = min(nb, (split + 1) * bps);
    const int h0 = kvh * a.rep + ht * 16, nh = min(16, a.rep - ht * 16);  // the query heads of this workgroup

    f16x8 qf[W];
    {
        const uint16_t* qr = a.q + b * a.q_stride + static_cast<int64_t>(h0 + (col < nh ? col : 0)) * HD;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            u32x4 r = ldg_any(qr + 8 * (4 * i + g));
            if (col >= nh) r = u32x4{0, 0, 0, 0};
            qf[i] = __builtin_bit_cast(f16x8, r);
        }
    }

    // The page of piece lane & 3 of a block, read one block before its operands are.
    auto pages_of = [&](int blk) { return blk < b1 ? kv4_page(c, b, blk * kKv4Block + (BIG ? 0 : 16 * (lane & 3))) : -1; };
    auto piece_page = [&](int ids, int piece) {
        if constexpr (BIG) return __builtin_amdgcn_readfirstlane(ids);
        const int p0 = __builtin_amdgcn_readlane(ids, 0), p1 = __builtin_amdgcn_readlane(ids, 1);
        const int p2 = __builtin_amdgcn_readlane(ids, 2), p3 = __builtin_amdgcn_readlane(ids, 3);
        return piece < 2 ? (piece < 1 ? p0 : p1) : (piece < 3 ? p2 : p3);
    };
    // A block's operands: the lane's K token in piece col >> 2, its V tokens in piece g, its scales in piece
    // (lane >> 1) & 3: 16-byte chunk (lane >> 1 is piece + 4 (group + G kv)), half lane & 1.
    auto slot_of = [&](int blk, int piece) {  // of the piece's first token, from the block's (BIG) or the page's first slot
        return BIG ? 16 * piece : (blk * kKv4Block + 16 * piece) & (c.page - 1);
    };
    auto lead_of = [&](int blk) { return BIG ? (blk * kKv4Block) & (c.page - 1) : 0; };
    auto head_of = [&](int id) { return static_cast<int64_t>(id < 0 ? 0 : id) * c.NKV + kvh; };
    Kv4Block<HD, GS> x;
    auto load_k = [&](int blk, int ids) {
        const int kid = piece_page(ids, col >> 2), sid = piece_page(ids, (lane >> 1) & 3), lead = lead_of(blk);
        const uint8_t* kp = c.k_pages + (head_of(kid) * c.page + lead) * (HD / 2) +
                            (slot_of(blk, col >> 2) + (col & 3)) * (HD / 2) + 4 * W * g;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (W == 2) {
                const u32x2 r = ldg(reinterpret_cast<const u32x2*>(kp + 4 * i * (HD / 2)));
                x.k[i][0] = r.x;
                x.k[i][1] = r.y;
            } else {
#pragma unroll
                for (int j = 0; j < W; j += 4) {
                    const u32x4 r = ldg(reinterpret_cast<const u32x4*>(kp + 4 * i * (HD / 2) + 4 * j));
                    x.k[i][j] = r.x;
                    x.k[i][j + 1] = r.y;
                    x.k[i][j + 2] = r.z;
                    x.k[i][j + 3] = r.w;
                }
            }
        }
        const int st = slot_of(blk, (lane >> 1) & 3) + 8 * (lane & 1);
#pragma unroll
        for (int e = 0; e < SC; ++e) {
            const int gk = (lane >> 3) + 8 * e, grp = gk % G;  // lanes past 2 G repeat V's
            const uint16_t* sp = gk < G ? c.k_scale : c.v_scale;
            x.s[e] = ldg(reinterpret_cast<const u32x4*>(sp + head_of(sid) * G * c.page + lead + grp * c.page + st));
        }
    };
    auto load_v = [&](int blk, int ids) {
        const int vid = piece_page(ids, g);
        const uint8_t* vp = c.v_pages + (head_of(vid) * c.page + lead_of(blk)) * (HD / 2) + slot_of(blk, g) * (HD / 2) +
                            col * (U * 8);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (U == 1) {
                x.v[i][0] = ldg(reinterpret_cast<const u32x2*>(vp + i * 16 * U * 8));
            } else {
#pragma unroll
                for (int j = 0; j < U; j += 2) {
                    const u32x4 r = ldg(reinterpret_cast<const u32x4*>(vp + i * 16 * U * 8 + 8 * j));
                    x.v[i][j] = u32x2{r.x, r.y};
                    x.v[i][j + 1] = u32x2{r.z, r.w};
                }
            }
        }
    };

    f32x4 acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = f32x4{0, 0, 0, 0};
    float m = kNegBig, l = 0.0f;  // m: the base of the exponents, the running maximum less `lift`
    // the wave's V scales so far are below 2^(15 - lift), whose bits are `cap` (but for those that are not finite, whose
    // products are infinite or NaN whatever the base)
    float lift = 29.0f;
    uint32_t cap = 1u << 10;

    // One set of operand registers: K's are loaded again as soon as the scores are done, V's after the products, so each
    // load has about half a block's work in front of it; page ids are a block further ahead.
    int blk = split * bps + wave;
    int ids = pages_of(blk), next_ids = pages_of(blk + kKv4Waves);
    if (blk < b1) {
        load_k(blk, ids);
        load_v(blk, ids);
    }
    auto step = [&](auto MORE) {  // MORE: another block of this wave follows
        const int vid = piece_page(ids, g);
        // live: how many of the lane's tokens 16 g + 0 .. 15 there are
        const int left = L - blk * kKv4Block - 16 * g;
        const int live = vid < 0 ? 0 : left < 0 ? 0 : left < 16 ? left : 16;
        const bool whole = ballot(live < 16) == 0;
        u32x4 vs;  // 8 of the block's V scales, in the lanes kVLanes
        constexpr uint64_t kVLanes = SC == 2 ? ~0ull : ~0ull << (8 * G % 64);
        {
            u32x4* dst = reinterpret_cast<u32x4*>(&s_scale[wave][0][0][0][0]);
#pragma unroll
            for (int e = 0; e < SC; ++e) {
                u32x4 w = x.s[e];
                if (!whole) {  // scales of slots without a token are whatever was there: zeros, so that 0 weights stay 0
                    const int n = __shfl(live, 16 * ((lane >> 1) & 3)) - 8 * (lane & 1);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        w[k] = 2 * k + 1 < n ? w[k] : 2 * k < n ? w[k] & 0xffffu : 0u;
                }
                if (lane + 64 * e < 16 * G) dst[lane + 64 * e] = w;
                vs = w;
            }
            __builtin_amdgcn_wave_barrier();
        }
        float up = 0.0f;  // binades by which the base moves for the block's V scales
        auto most_of = [](const u32x4& w) {
            const u16x2 a = __builtin_elementwise_max(__builtin_bit_cast(u16x2, w.x), __builtin_bit_cast(u16x2, w.y));
            const u16x2 b = __builtin_elementwise_max(__builtin_bit_cast(u16x2, w.z), __builtin_bit_cast(u16x2, w.w));
            const u16x2 c = __builtin_elementwise_max(a, b);
            return static_cast<uint32_t>(max(c.x, c.y));
        };
        if (ballot(most_of(vs) >= cap) & kVLanes) {  // (wave-uniform): a larger scale than any before, or not a finite one
            u32x4 w = vs & 0x7fff7fffu;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const u16x2 b = __builtin_bit_cast(u16x2, w[k]);
                w[k] = __builtin_bit_cast(uint32_t, b & (b < (uint16_t)0x7c00));
            }
            const float top = wave_max_bcast(kVLanes >> lane & 1 ? static_cast<float>(most_of(w)) : 0.0f);
            const int field = static_cast<int>(top) >> 10;  // the exponent's bits
            if (((field + 1) << 10) > static_cast<int>(cap)) {
                up = lift - (29 - field);
                lift = 29 - field;
                cap = (field + 1) << 10;
            }
        }

        float s[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float t[4] = {0, 0, 0, 0};
#pragma unroll
            for (int r = 0; r < G; ++r) {
                f32x4 sum = {0, 0, 0, 0};
#pragma unroll
                for (int j = r * (GS / 32); j < (r + 1) * (GS / 32); ++j) {
                    f16x2 v[4];
                    dequant_int4x8_bitfield(x.k[i][j], v);
                    const f16x8 ka = {v[0].x, v[0].y, v[1].x, v[1].y, v[2].x, v[2].y, v[3].x, v[3].y};
                    sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qf[j], sum, 0, 0, 0);
                }
                const u32x2 sc = *reinterpret_cast<const u32x2*>(&s_scale[wave][0][r][g][4 * i]);
                const f16x2 lo = as_f16x2(sc.x), hi = as_f16x2(sc.y);
                t[0] = fmaf(sum[0], static_cast<float>(lo.x), t[0]);
                t[1] = fmaf(sum[1], static_cast<float>(lo.y), t[1]);
                t[2] = fmaf(sum[2], static_cast<float>(hi.x), t[2]);
                t[3] = fmaf(sum[3], static_cast<float>(hi.y), t[3]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[4 * i + e] = t[e];
                asm volatile("" : "+v"(s[4 * i + e]));  // (the compiler would keep all products and sum them up later)
            }
            if (i & 1) __builtin_amdgcn_sched_barrier(0);  // (and unpack all tiles at once)
        }
        const int ids2 = pages_of(blk + 2 * kKv4Waves);
        if constexpr (MORE) load_k(blk + kKv4Waves, next_ids);
        __builtin_amdgcn_sched_barrier(0);
        if (!whole) {
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = e < live ? s[e] : -__builtin_inff();
        }
        float top = s[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top = fmaxf(top, s[e]);
        top = fmaxf(top, xor_lanes<16>(top));
        top = fmaf(fmaxf(top, xor_lanes<32>(top)), a.scale_log2, -lift);
        const float from = m + up;
        if (ballot(top > from) || up > 0.0f) {
            const float mn = fmaxf(from, top), w = fast_exp2(m - mn);
            m = mn;
            l *= w;
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[d] *= w;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            s[e] = fast_exp2(fmaf(s[e], a.scale_log2, -m));
            l += s[e];
        }
        // per half block (8 tokens a lane) and scale group: P^T, then the group's dimension tiles
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int r = 0; r < G; ++r) {
                const u32x4 sc = *reinterpret_cast<const u32x4*>(&s_scale[wave][1][r][g][8 * half]);
                f16x8 pb;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const f16x2 w = as_f16x2(sc[e >> 1]);  // (fma, not a product: one mixed-precision instruction)
                    pb[e] = static_cast<f16>(fmaf(s[8 * half + e], static_cast<float>(w[e & 1]), 0.0f));
                }
#pragma unroll
                for (int d = r * (GS / 16); d < (r + 1) * (GS / 16); ++d) {
                    const int u = d >> 2, n = d & 3;
                    const uint32_t w[4] = {x.v[2 * half][u].x, x.v[2 * half][u].y, x.v[2 * half + 1][u].x,
                                           x.v[2 * half + 1][u].y};  // tokens (0, 1), (2, 3), (4, 5), (6, 7)
                    const f16x2 bias = {(f16)-1032.0f, (f16)-1032.0f}, bias16 = {(f16)-72.0f, (f16)-72.0f};
                    const f16x2 sixteenth = {(f16)0.0625f, (f16)0.0625f};
                    f16x2 v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t y8 = n < 2 ? w[e] : w[e] >> 8;
                        v[e] = n & 1 ? __builtin_elementwise_fma(as_f16x2(and_xor(y8, 0x00f000f0u, 0x64806480u)), sixteenth,
                                                                 bias16)
                                     : as_f16x2(and_xor(y8, 0x000f000fu, 0x64086408u)) + bias;
                    }
                    const f16x8 va = {v[0].x, v[0].y, v[1].x, v[1].y, v[2].x, v[2].y, v[3].x, v[3].y};
                    acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pb, acc[d], 0, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);  // (all groups at once would spill)
            }
        }
        if constexpr (MORE) load_v(blk + kKv4Waves, next_ids);
        ids = next_ids;
        next_ids = ids2;
    };
    for (; blk + kKv4Waves < b1; blk += kKv4Waves) step(std::true_type{});  // (wave-uniform)
    if (blk < b1) step(std::false_type{});

    // lane (c, g): dimensions 16 d + 4 g + 0 .. 3 of head c
    l += xor_lanes<16>(l);
    l += xor_lanes<32>(l);
    float* st = s_state[wave][col];
    if (g == 0) {
        st[0] = m;
        st[1] = l;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) st[2 + 16 * d + 4 * g + e] = acc[d][e];
    __syncthreads();
    for (int x = tid; x < nh * HD; x += kKv4Waves * kWave) {
        const int h = x / HD, d = x % HD;
        float M = kNegBig, lsum = 0.0f, v = 0.0f;
#pragma unroll
        for (int w = 0; w < kKv4Waves; ++w) M = fmaxf(M, s_state[w][h][0]);
#pragma unroll
        for (int w = 0; w < kKv4Waves; ++w) {
            const float e = fast_exp2(s_state[w][h][0] - M);
            lsum = fmaf(s_state[w][h][1], e, lsum);
            v = fmaf(s_state[w][h][2 + d], e, v);
        }
        if (nb <= bps) {
            stg(a.out + (static_cast<int64_t>(b) * a.NQ + h0 + h) * HD + d, f32_to_f16_bits(lsum == 0.0f ? 0.0f : v / lsum));
        } else {
            float* p = a.part + (static_cast<int64_t>(y) * a.NQ + h0 + h) * (HD + 2);
            stg(p + 2 + d, v);
            if (d == 0) {
                stg(p, M);
                stg(p + 1, lsum);
            }
        }
    }
}

// The states of split contexts, summed in a fixed order: a workgroup per (sequence, query head), whose four waves take
// eight states each of every 32. The first 32 states' sums are requested with the (m, l) pairs, so a context of up to 32
// splits is two round trips: the lengths, then all states.
constexpr int kKv4MostSplits = 1032;  // of one sequence: want + 1 at most, want <= 1024

template <int HD>
__global__ __launch_bounds__(kKv4Waves * kWave) void kv4_combine_kernel(const Kv4AttnArgs a, const Kv4Cache c) {
    constexpr int E = HD / 64, N = 8;
    __shared__ float s_w[kKv4MostSplits], s_v[kKv4Waves][HD];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = blockIdx.x;
    const Kv4Place at = kv4_place<false>(a, c, lane, blockIdx.y);
    const int b = at.b, ns = (kv4_blocks(at.L) + at.bps - 1) / at.bps;
    if (ns == 1) return;  // written by its one split
    const int64_t stride = static_cast<int64_t>(a.NQ) * (HD + 2);
    const float* p = a.part + at.y0 * stride + static_cast<int64_t>(h) * (HD + 2);
    float x[N][E];
    auto load = [&](int s) {
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e) x[k][e] = ldg(p + (s + k < ns ? s + k : 0) * stride + 2 + 64 * e + lane);
    };
    float m0 = kNegBig, l0 = 0.0f;
    if (lane < ns) {
        m0 = ldg(p + lane * stride);
        l0 = ldg(p + lane * stride + 1);
    }
    load(wave * N);
    float M = m0;
    for (int s = lane + kWave; s < ns; s += kWave) M = fmaxf(M, ldg(p + s * stride));
    M = wave_max_bcast(M);
    float lsum = 0.0f;
    for (int s = lane; s < ns; s += kWave) {
        const float e = fast_exp2((s < kWave ? m0 : ldg(p + s * stride)) - M);
        if (wave == 0) s_w[s] = e;
        lsum = fmaf(s < kWave ? l0 : ldg(p + s * stride + 1), e, lsum);
    }
    lsum = wave_sum_bcast(lsum);
    __syncthreads();  // the weights
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = 0.0f;
    for (int s = wave * N; s < ns; s += kKv4Waves * N) {
        if (s >= kKv4Waves * N) load(s);
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (s + k >= ns) break;
            const float w = s_w[s + k];
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = fmaf(x[k][e], w, v[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) s_v[wave][64 * e + lane] = v[e];
    __syncthreads();  // the waves' sums
    const int d = threadIdx.x;
    if (d >= HD) return;
    const float sum = (s_v[0][d] + s_v[1][d]) + (s_v[2][d] + s_v[3][d]);
    stg(a.out + (static_cast<int64_t>(b) * a.NQ + h) * HD + d, f32_to_f16_bits(lsum == 0.0f ? 0.0f : sum / lsum));
}

// Splits aimed at (over all sequences) so that the workgroups fill the 256 CUs once, and the most there can be of them.
struct Kv4Plan {
    int64_t want, splits;
    bool combine;
    Kv4Plan(int64_t B, int64_t NKV, int64_t rep, int64_t hd, int64_t max_len) {
        const int64_t kKv4Target = 256 * kv4_per_cu(static_cast<int>(hd));
        const int64_t units = NKV * ceil_div64(rep, 16), nb = max_len < 1 ? 1 : ceil_div64(max_len, kKv4Block);
        want = kKv4Target / units < 1 ? 1 : kKv4Target / units;
        const int64_t most = B * ceil_div64(nb, kKv4Waves);  // a split has at least a block for every wave
        splits = want + B < most ? want + B : most;
        combine = nb > kKv4Waves;
    }
};

}  // namespace soi

using namespace soi;

extern "C" size_t soi_kv4_decode_attention_workspace_bytes(int64_t batch, int64_t num_q_heads, int64_t num_kv_heads,
                                                           int64_t head_dim, int64_t max_len) {
    if (batch < 1 || num_kv_heads < 1 || num_q_heads < num_kv_heads || num_q_heads % num_kv_heads || head_dim < 1 ||
        max_len < 0 || max_len > (int64_t(1) << 30))
        return 0;
    const Kv4Plan p(batch, num_kv_heads, num_q_heads / num_kv_heads, head_dim, max_len);
    return p.combine ? static_cast<size_t>(p.splits) * num_q_heads * (head_dim + 2) * sizeof(float) : 0;
}

extern "C" int soi_kv4_decode_attention(const soi_kv4_cache* cache, const uint16_t* q, int64_t q_stride,
                                        int64_t num_q_heads, int64_t max_len, uint16_t* out, float scale, void* workspace,
                                        size_t workspace_bytes, void* stream) {
    const char* what = "soi_kv4_decode_attention";
    int st = kv4_check(cache, what);
    if (st) return st;
    const int64_t hd = cache->head_dim, gs = cache->group_size, B = cache->batch, NKV = cache->num_kv_heads;
    SOI_REQUIRE(num_q_heads >= 1 && num_q_heads <= 65535 && num_q_heads % NKV == 0,
                "%s: num_q_heads must be a multiple of num_kv_heads up to 65535", what);
    SOI_REQUIRE(q_stride >= num_q_heads * hd || B == 1, "%s: q rows overlap: stride %lld below %lld", what,
                (long long)q_stride, (long long)(num_q_heads * hd));
    SOI_REQUIRE(max_len >= 0 && max_len <= cache->max_blocks * cache->page_size,
                "%s: max_len must be in [0, max_blocks * page_size]", what);
    // the sum of the sequences' 64-token blocks is held in 32 bits
    SOI_REQUIRE(ceil_div64(max_len, kKv4Block) * B < (int64_t(1) << 31), "%s: batch * max_len out of range", what);
    SOI_REQUIRE(scale > 0.0f && scale < __builtin_inff(), "%s: scale must be positive and finite", what);
    SOI_REQUIRE(q && out && q != out, "%s: null pointer or out = q", what);
    const int64_t rep = num_q_heads / NKV;
    const Kv4Plan plan(B, NKV, rep, hd, max_len);
    SOI_REQUIRE(plan.splits <= 65535, "%s: too many sequences", what);
    const size_t need = soi_kv4_decode_attention_workspace_bytes(B, num_q_heads, NKV, hd, max_len);
    if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 3))) {
        set_last_error("%s: workspace of %zu bytes (4-byte aligned) needed, got %zu", what, need, workspace_bytes);
        return SOI_ERR_WORKSPACE;
    }
    const int64_t htiles = ceil_div64(rep, 16);
    const Kv4AttnArgs a{q, q_stride, out, static_cast<float*>(workspace), static_cast<int>(num_q_heads),
                        static_cast<int>(rep), static_cast<int>(htiles), static_cast<int>(plan.want),
                        static_cast<int>(max_len), scale * kLog2e};
    const Kv4Cache c = kv4_device(cache);
    const dim3 grid(static_cast<unsigned>(NKV * htiles), static_cast<unsigned>(plan.splits));
    hipStream_t s = as_stream(stream);
#define SOI_X(H, G)                                                                                         \
    do {                                                                                                    \
        if (cache->page_size >= kKv4Block)                                                                  \
            hipLaunchKernelGGL((kv4_attn_kernel<H, G, true>), grid, dim3(kKv4Waves * kWave), 0, s, a, c);   \
        else                                                                                                \
            hipLaunchKernelGGL((kv4_attn_kernel<H, G, false>), grid, dim3(kKv4Waves * kWave), 0, s, a, c);  \
    } while (0)
    SOI_KV4_SHAPES(SOI_X);
#undef SOI_X
    st = launch_status(what);
    if (st || !plan.combine) return st;
    const dim3 cgrid(static_cast<unsigned>(num_q_heads), static_cast<unsigned>(B));
#define SOI_C(H) hipLaunchKernelGGL((kv4_combine_kernel<H>), cgrid, dim3(kKv4Waves * kWave), 0, s, a, c)
    if (hd == 64) SOI_C(64);
    else if (hd == 128) SOI_C(128);
    else SOI_C(256);
#undef SOI_C
    return launch_status(what);
}
