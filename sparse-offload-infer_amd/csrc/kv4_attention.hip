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
//   * the running maximum is one per head and wave (two lane swaps a block), sums are rescaled only in a block that
//     raises one of them.
// No operand is reordered between lanes. The scales of a block pass through LDS (a wave's own part: each lane loads 16
// bytes of them, and reads back the 32 bytes it needs of each group), K and V go straight to registers, a block ahead.
//
// Work is split evenly whatever the lengths: the blocks of all sequences, in order, are cut into splits of `bps` blocks,
// none across two sequences, bps following from the sum of the lengths on the device. Workgroup (head, y) finds split y
// by a scan over the sequences. A sequence of one split is written at once; the states of more are combined in split
// order by a second launch.
#include "soi_host.h"
#include "soi_kv4.h"
#include "soi_attn.h"

#include <type_traits>

namespace soi {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kKv4Waves = 4;
constexpr int kKv4Block = 64;  // tokens a wave takes at a time

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

// Blocks per split, about `want` splits of all sequences' blocks together: whole rounds of a workgroup's waves.
__device__ __forceinline__ int kv4_bps(const Kv4AttnArgs& a, const Kv4Cache& c, int lane) {
    int total = 0;
    for (int s = 0; s < c.B; s += kWave) total += s + lane < c.B ? kv4_blocks(kv4_len(c, s + lane, a.max_len)) : 0;
    total = __builtin_amdgcn_readlane(wave_scan(total), 63);
    const int n = (total + a.want - 1) / a.want;
    return (n + kKv4Waves - 1) / kKv4Waves * kKv4Waves;
}

// Splits before sequence `upto`, and for `y`, where it is not negative, the sequence and its split that hold split y
// (b = -1: none). One of the two questions a call.
__device__ __forceinline__ int kv4_find(const Kv4AttnArgs& a, const Kv4Cache& c, int bps, int lane, int upto, int y, int& b,
                                        int& split) {
    int base = 0;
    b = -1;
    split = 0;
    for (int s = 0; s < upto; s += kWave) {
        const int ns = s + lane < upto ? (kv4_blocks(kv4_len(c, s + lane, a.max_len)) + bps - 1) / bps : 0;
        const int incl = wave_scan(ns);
        const int all = __builtin_amdgcn_readlane(incl, 63);
        if (y >= 0 && y < base + all) {
            const int at = __builtin_ctzll(ballot(base + incl > y));
            b = s + at;
            split = y - base - (at ? __builtin_amdgcn_readlane(incl, at - 1) : 0);
            return base;
        }
        base += all;
    }
    return base;
}

template <int HD, int GS>
struct Kv4Block {
    static constexpr int W = HD / 32, U = HD / 64, G = HD / GS, SC = G <= 4 ? 1 : 2;
    uint32_t k[4][W];  // tile i: W words of the lane's token
    u32x2 v[4][U];     // quad i: units of tokens 4 i .. 4 i + 3 (of 16 g ..)
    u32x4 s[SC];       // 16 bytes of the block's scales
};

template <int HD, int GS>
__global__ __launch_bounds__(kKv4Waves * kWave, HD == 256 ? 1 : 3) void kv4_attn_kernel(const Kv4AttnArgs a, const Kv4Cache c) {
    constexpr int W = HD / 32, U = HD / 64, G = HD / GS, DT = HD / 16, SC = Kv4Block<HD, GS>::SC;
    __shared__ float s_state[kKv4Waves][16][HD + 2];
    __shared__ __attribute__((aligned(16))) uint16_t s_scale[kKv4Waves][2][G][4][16];  // K, V; group; piece; token
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int col = lane & 15, g = lane >> 4;
    const int kvh = static_cast<int>(blockIdx.x) / a.htiles, ht = static_cast<int>(blockIdx.x) % a.htiles;
    const int y = blockIdx.y;
    const int bps = kv4_bps(a, c, lane);
    int b, split;
    kv4_find(a, c, bps, lane, c.B, y, b, split);
    if (b < 0) return;
    const int L = __builtin_amdgcn_readfirstlane(kv4_len(c, b, a.max_len));
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

    // A block's operands: page ids by 16-token piece, the lane's K token in piece col >> 2, its V tokens in piece g, its
    // scales in piece (lane >> 1) & 3: chunk (lane >> 1 is piece + 4 (group + G kv)), half lane & 1.
    auto page_of = [&](int blk, int piece) { return kv4_page(c, b, blk * kKv4Block + 16 * piece); };
    auto load = [&](Kv4Block<HD, GS>& x, int blk, int vid) {
        const int kid = page_of(blk, col >> 2);
        const int kt = (blk * kKv4Block + 16 * (col >> 2) + (col & 3)) & (c.page - 1);
        const int vt = (blk * kKv4Block + 16 * g) & (c.page - 1);
        const uint8_t* kp = c.k_pages + ((static_cast<int64_t>(kid < 0 ? 0 : kid) * c.NKV + kvh) * c.page + kt) * (HD / 2) +
                            4 * W * g;
        const int64_t vhead = static_cast<int64_t>(vid < 0 ? 0 : vid) * c.NKV + kvh;
        const uint8_t* vp = c.v_pages + (vhead * c.page + vt) * (HD / 2) + col * (U * 8);
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
        {
            const int piece = (lane >> 1) & 3, sid = page_of(blk, piece);
            const int st = (blk * kKv4Block + 16 * piece + 8 * (lane & 1)) & (c.page - 1);
            const int64_t head = static_cast<int64_t>(sid < 0 ? 0 : sid) * c.NKV + kvh;
#pragma unroll
            for (int e = 0; e < SC; ++e) {
                const int gk = (lane >> 3) + 8 * e, kv = gk / G < 1 ? 0 : 1, grp = gk % G;  // lanes past 2 G repeat V's
                x.s[e] = ldg(reinterpret_cast<const u32x4*>((kv ? c.v_scale : c.k_scale) + (head * G + grp) * c.page + st));
            }
        }
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
    float m = kNegBig, l = 0.0f;

    int blk = split * bps + wave;
    Kv4Block<HD, GS> cur;
    int vid = -1;
    if (blk < b1) {
        vid = page_of(blk, g);
        load(cur, blk, vid);
    }
    for (; blk < b1; blk += kKv4Waves) {
        Kv4Block<HD, GS> nxt;
        int nvid = -1;
        if (blk + kKv4Waves < b1) {  // wave-uniform; the next block's operands are in flight during this one's products
            nvid = page_of(blk + kKv4Waves, g);
            load(nxt, blk + kKv4Waves, nvid);
        }
        __builtin_amdgcn_sched_barrier(0);
        // live: how many of the lane's tokens 16 g + 0 .. 15 there are
        const int left = L - blk * kKv4Block - 16 * g;
        const int live = vid < 0 ? 0 : left < 0 ? 0 : left < 16 ? left : 16;
        const bool whole = ballot(live < 16) == 0;
        {
            u32x4* dst = reinterpret_cast<u32x4*>(&s_scale[wave][0][0][0][0]);
#pragma unroll
            for (int e = 0; e < SC; ++e) {
                u32x4 w = cur.s[e];
                if (!whole) {  // scales of slots without a token are whatever was there: zeros, so that 0 weights stay 0
                    const int n = __shfl(live, 16 * ((lane >> 1) & 3)) - 8 * (lane & 1);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        w[k] = 2 * k + 1 < n ? w[k] : 2 * k < n ? w[k] & 0xffffu : 0u;
                }
                if (lane + 64 * e < 16 * G) dst[lane + 64 * e] = w;
            }
            __builtin_amdgcn_wave_barrier();
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
                    dequant_int4x8_bitfield(cur.k[i][j], v);
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
            for (int e = 0; e < 4; ++e) s[4 * i + e] = t[e];
        }
        if (!whole) {
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = e < live ? s[e] : -__builtin_inff();
        }
        float top = s[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top = fmaxf(top, s[e]);
        top = fmaxf(top, xor_lanes<16>(top));
        top = fmaxf(top, xor_lanes<32>(top)) * a.scale_log2;
        if (ballot(top > m)) {
            const float mn = fmaxf(m, top), w = fast_exp2(m - mn);
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
        // per half block (8 tokens a lane): P^T of each scale group, then its dimension tiles
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            f16x8 pb[G];
#pragma unroll
            for (int r = 0; r < G; ++r) {
                const u32x4 sc = *reinterpret_cast<const u32x4*>(&s_scale[wave][1][r][g][8 * half]);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const f16x2 w = as_f16x2(sc[e >> 1]);
                    pb[r][e] = static_cast<f16>(s[8 * half + e] * static_cast<float>(w[e & 1]));
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t w[4] = {cur.v[2 * half][u].x, cur.v[2 * half][u].y, cur.v[2 * half + 1][u].x,
                                       cur.v[2 * half + 1][u].y};  // tokens (0, 1), (2, 3), (4, 5), (6, 7)
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const f16x2 bias = {(f16)-1032.0f, (f16)-1032.0f}, bias16 = {(f16)-72.0f, (f16)-72.0f};
                    const f16x2 sixteenth = {(f16)0.0625f, (f16)0.0625f};
                    f16x2 v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t x = n < 2 ? w[e] : w[e] >> 8;
                        v[e] = n & 1 ? __builtin_elementwise_fma(as_f16x2(and_xor(x, 0x00f000f0u, 0x64806480u)), sixteenth,
                                                                 bias16)
                                     : as_f16x2(and_xor(x, 0x000f000fu, 0x64086408u)) + bias;
                    }
                    const f16x8 va = {v[0].x, v[0].y, v[1].x, v[1].y, v[2].x, v[2].y, v[3].x, v[3].y};
                    const int d = 4 * u + n;
                    acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pb[16 * d / GS], acc[d], 0, 0, 0);
                }
            }
        }
        cur = nxt;
        vid = nvid;
    }

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

// The states of split contexts, in split order: a wave per (sequence, query head).
constexpr int kKv4MostSplits = 1032;  // of one sequence: want + 1 at most, want <= kKv4Target

template <int HD>
__global__ __launch_bounds__(kKv4Waves * kWave) void kv4_combine_kernel(const Kv4AttnArgs a, const Kv4Cache c) {
    constexpr int E = HD / 64;
    __shared__ float s_w[kKv4Waves][kKv4MostSplits];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int h = static_cast<int>(blockIdx.x) * kKv4Waves + wave, b = blockIdx.y;
    const int bps = kv4_bps(a, c, lane);
    const int ns = (kv4_blocks(__builtin_amdgcn_readfirstlane(kv4_len(c, b, a.max_len))) + bps - 1) / bps;
    if (ns == 1 || h >= a.NQ) return;  // written by its one split
    int unused_b, unused_s;
    const int y0 = kv4_find(a, c, bps, lane, b, -1, unused_b, unused_s);
    const int64_t stride = static_cast<int64_t>(a.NQ) * (HD + 2);
    const float* p = a.part + y0 * stride + static_cast<int64_t>(h) * (HD + 2);
    float* sw = s_w[wave];
    float M = kNegBig;
    for (int s = lane; s < ns; s += kWave) {
        const float ms = ldg(p + s * stride);
        sw[s] = ms;
        M = fmaxf(M, ms);
    }
    M = wave_max_bcast(M);
    float lsum = 0.0f;
    for (int s = lane; s < ns; s += kWave) {
        const float e = fast_exp2(sw[s] - M);
        sw[s] = e;
        lsum = fmaf(ldg(p + s * stride + 1), e, lsum);
    }
    lsum = wave_sum_bcast(lsum);
    __builtin_amdgcn_wave_barrier();
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = 0.0f;
    for (int s = 0; s < ns; s += 8) {
        float x[8][E];
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e) x[k][e] = ldg(p + (s + k < ns ? s + k : s) * stride + 2 + 64 * e + lane);
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = s + k < ns ? fmaf(x[k][e], sw[s + k], v[e]) : v[e];
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
        stg(a.out + (static_cast<int64_t>(b) * a.NQ + h) * HD + 64 * e + lane,
            f32_to_f16_bits(lsum == 0.0f ? 0.0f : v[e] / lsum));
}

// Splits aimed at (over all sequences) so that the workgroups are about kKv4Target, and the most there can be of them.
constexpr int64_t kKv4Target = 768;
struct Kv4Plan {
    int64_t want, splits;
    bool combine;
    Kv4Plan(int64_t B, int64_t NKV, int64_t rep, int64_t max_len) {
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
    const Kv4Plan p(batch, num_kv_heads, num_q_heads / num_kv_heads, max_len);
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
    const Kv4Plan plan(B, NKV, rep, max_len);
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
#define SOI_X(H, G) hipLaunchKernelGGL((kv4_attn_kernel<H, G>), grid, dim3(kKv4Waves * kWave), 0, s, a, c)
    SOI_KV4_SHAPES(SOI_X);
#undef SOI_X
    st = launch_status(what);
    if (st || !plan.combine) return st;
    const dim3 cgrid(static_cast<unsigned>(ceil_div64(num_q_heads, kKv4Waves)), static_cast<unsigned>(B));
#define SOI_C(H) hipLaunchKernelGGL((kv4_combine_kernel<H>), cgrid, dim3(kKv4Waves * kWave), 0, s, a, c)
    if (hd == 64) SOI_C(64);
    else if (hd == 128) SOI_C(128);
    else SOI_C(256);
#undef SOI_C
    return launch_status(what);
}
