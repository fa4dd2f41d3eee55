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
// No operand is reordered between lanes and nothing passes through LDS before the four waves of a workgroup merge.
// Long contexts are split over workgroups (`bps` blocks each), whose states a second launch combines in split order.
#include "soi_host.h"
#include "soi_kv4.h"
#include "soi_attn.h"

namespace soi {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kKv4Waves = 4;
constexpr int kKv4Block = 64;  // tokens a wave takes at a time

struct Kv4AttnArgs {
    const uint16_t* q;
    int64_t q_stride;
    uint16_t* out;
    float* part;  // [B, NQ, nsplit][HD + 2]: m, l, acc
    int NQ, rep, htiles, nsplit, bps;
    float scale_log2;
};

// Splits of a context of L tokens: at least one, which writes the zeros of an empty context.
__device__ __forceinline__ int kv4_splits(int L, int bps) {
    const int nb = (L + kKv4Block - 1) / kKv4Block;
    const int ns = (nb + bps - 1) / bps;
    return ns < 1 ? 1 : ns;
}

__device__ __forceinline__ int kv4_len(const Kv4Cache& c, int b, int max_len) {
    const int L = ldg(c.lens + b);
    return L < 0 ? 0 : L < max_len ? L : max_len;
}

template <int HD, int GS>
struct Kv4Block {
    static constexpr int W = HD / 32, U = HD / 64, G = HD / GS;
    uint32_t k[4][W];      // tile i: W words of the lane's token
    u32x2 v[4][U];         // quad i: units of tokens 4 i .. 4 i + 3 (of 16 g ..)
    u32x4 ks[G][2], vs[G][2];  // scales of tokens 16 g .. + 15
};

template <int HD, int GS>
__global__ __launch_bounds__(kKv4Waves * kWave) void kv4_attn_kernel(const Kv4AttnArgs a, const Kv4Cache c, int max_len) {
    constexpr int W = HD / 32, U = HD / 64, G = HD / GS, DT = HD / 16;
    __shared__ float s_state[kKv4Waves][16][HD + 2];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int col = lane & 15, g = lane >> 4;
    const int kvh = static_cast<int>(blockIdx.x) / a.htiles, ht = static_cast<int>(blockIdx.x) % a.htiles;
    const int split = blockIdx.y, b = blockIdx.z;
    const int L = kv4_len(c, b, max_len);
    const int ns = kv4_splits(L, a.bps);
    if (split >= ns) return;
    const int nb = (L + kKv4Block - 1) / kKv4Block;
    const int b1 = min(nb, (split + 1) * a.bps);
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

    // a block's operands; the page ids of the lane's K token (piece col >> 2) and of its V tokens (piece g)
    auto page_of = [&](int blk, int piece) { return kv4_page(c, b, blk * kKv4Block + 16 * piece); };
    auto load = [&](Kv4Block<HD, GS>& x, int blk, int kid, int vid) {
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
#pragma unroll
        for (int r = 0; r < G; ++r) {
            const u32x4* ks = reinterpret_cast<const u32x4*>(c.k_scale + (vhead * G + r) * c.page + vt);
            const u32x4* vs = reinterpret_cast<const u32x4*>(c.v_scale + (vhead * G + r) * c.page + vt);
            x.ks[r][0] = ldg(ks);
            x.ks[r][1] = ldg(ks + 1);
            x.vs[r][0] = ldg(vs);
            x.vs[r][1] = ldg(vs + 1);
        }
    };
    auto scale_at = [](const u32x4 (&s)[2], int t) {  // token t < 16, a constant after unrolling
        const uint32_t w = s[t >> 3][(t >> 1) & 3];
        return f16_bits_to_f32(static_cast<uint16_t>(t & 1 ? w >> 16 : w & 0xffffu));
    };

    f32x4 acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = f32x4{0, 0, 0, 0};
    float m = kNegBig, l = 0.0f;

    int blk = split * a.bps + wave;
    Kv4Block<HD, GS> cur;
    int vid = -1;
    if (blk < b1) {
        vid = page_of(blk, g);
        load(cur, blk, page_of(blk, col >> 2), vid);
    }
    for (; blk < b1; blk += kKv4Waves) {
        Kv4Block<HD, GS> nxt;
        int nvid = -1;
        if (blk + kKv4Waves < b1) {  // wave-uniform; the next block's operands are in flight during this one's products
            nvid = page_of(blk + kKv4Waves, g);
            load(nxt, blk + kKv4Waves, page_of(blk + kKv4Waves, col >> 2), nvid);
        }
        __builtin_amdgcn_sched_barrier(0);

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
#pragma unroll
                for (int e = 0; e < 4; ++e) t[e] = fmaf(sum[e], scale_at(cur.ks[r], 4 * i + e), t[e]);
            }
            const int tok = blk * kKv4Block + 16 * g + 4 * i;
#pragma unroll
            for (int e = 0; e < 4; ++e) s[4 * i + e] = vid >= 0 && tok + e < L ? t[e] * a.scale_log2 : -__builtin_inff();
        }
        float top = s[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top = fmaxf(top, s[e]);
        top = fmaxf(top, xor_lanes<16>(top));
        top = fmaxf(top, xor_lanes<32>(top));
        if (ballot(top > m)) {
            const float mn = fmaxf(m, top), w = fast_exp2(m - mn);
            m = mn;
            l *= w;
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[d] *= w;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const bool live = vid >= 0 && blk * kKv4Block + 16 * g + e < L;
            s[e] = live ? fast_exp2(s[e] - m) : 0.0f;
            l += s[e];
        }
        // per half block (8 tokens a lane): P^T of each scale group, then its dimension tiles
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            f16x8 pb[G];
#pragma unroll
            for (int r = 0; r < G; ++r) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const bool live = vid >= 0 && blk * kKv4Block + 16 * g + 8 * half + e < L;
                    const float p = s[8 * half + e] * scale_at(cur.vs[r], 8 * half + e);
                    pb[r][e] = static_cast<f16>(live ? p : 0.0f);
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
        const int64_t row = static_cast<int64_t>(b) * a.NQ + h0 + h;
        if (ns == 1) {
            stg(a.out + row * HD + d, f32_to_f16_bits(lsum == 0.0f ? 0.0f : v / lsum));
        } else {
            float* p = a.part + (row * a.nsplit + split) * (HD + 2);
            stg(p + 2 + d, v);
            if (d == 0) {
                stg(p, M);
                stg(p + 1, lsum);
            }
        }
    }
}

// The states of a split context, in split order; one workgroup per (sequence, query head), one thread per dimension.
template <int HD>
__global__ __launch_bounds__(HD) void kv4_combine_kernel(const Kv4AttnArgs a, const Kv4Cache c, int max_len) {
    const int h = blockIdx.x, b = blockIdx.y, d = threadIdx.x;
    const int ns = kv4_splits(kv4_len(c, b, max_len), a.bps);
    if (ns == 1) return;  // written by its one split
    const int64_t row = static_cast<int64_t>(b) * a.NQ + h;
    const float* p = a.part + row * a.nsplit * (HD + 2);
    float M = kNegBig, lsum = 0.0f, v = 0.0f;
    for (int s = 0; s < ns; ++s) M = fmaxf(M, ldg(p + s * (HD + 2)));
    for (int s = 0; s < ns; ++s) {
        const float e = fast_exp2(ldg(p + s * (HD + 2)) - M);
        lsum = fmaf(ldg(p + s * (HD + 2) + 1), e, lsum);
        v = fmaf(ldg(p + s * (HD + 2) + 2 + d), e, v);
    }
    stg(a.out + row * HD + d, f32_to_f16_bits(lsum == 0.0f ? 0.0f : v / lsum));
}

// Blocks per split and splits of the longest context: workgroups for about three to a CU, whole rounds of the four waves.
static void kv4_plan(int64_t B, int64_t NKV, int64_t htiles, int64_t max_len, int64_t& bps, int64_t& nsplit) {
    const int64_t nb = max_len < 1 ? 1 : ceil_div64(max_len, kKv4Block);
    int64_t want = ceil_div64(768, B * NKV * htiles);
    bps = ceil_div64(ceil_div64(nb, want), kKv4Waves) * kKv4Waves;
    nsplit = ceil_div64(nb, bps);
    if (nsplit > 65535) {
        bps = ceil_div64(ceil_div64(nb, 65535), kKv4Waves) * kKv4Waves;
        nsplit = ceil_div64(nb, bps);
    }
}

}  // namespace soi

using namespace soi;

extern "C" size_t soi_kv4_decode_attention_workspace_bytes(int64_t batch, int64_t num_q_heads, int64_t num_kv_heads,
                                                           int64_t head_dim, int64_t max_len) {
    if (batch < 1 || num_kv_heads < 1 || num_q_heads < num_kv_heads || num_q_heads % num_kv_heads || head_dim < 1 ||
        max_len < 0 || max_len > (int64_t(1) << 30))
        return 0;
    int64_t bps, nsplit;
    kv4_plan(batch, num_kv_heads, ceil_div64(num_q_heads / num_kv_heads, 16), max_len, bps, nsplit);
    return nsplit == 1 ? 0 : static_cast<size_t>(batch) * num_q_heads * nsplit * (head_dim + 2) * sizeof(float);
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
    SOI_REQUIRE(scale > 0.0f && scale < __builtin_inff(), "%s: scale must be positive and finite", what);
    SOI_REQUIRE(q && out && q != out, "%s: null pointer or out = q", what);
    const int64_t rep = num_q_heads / NKV, htiles = ceil_div64(rep, 16);
    int64_t bps, nsplit;
    kv4_plan(B, NKV, htiles, max_len, bps, nsplit);
    const size_t need = soi_kv4_decode_attention_workspace_bytes(B, num_q_heads, NKV, hd, max_len);
    if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 3))) {
        set_last_error("%s: workspace of %zu bytes (4-byte aligned) needed, got %zu", what, need, workspace_bytes);
        return SOI_ERR_WORKSPACE;
    }
    const Kv4AttnArgs a{q, q_stride, out, static_cast<float*>(workspace), static_cast<int>(num_q_heads),
                        static_cast<int>(rep), static_cast<int>(htiles), static_cast<int>(nsplit),
                        static_cast<int>(bps), scale * kLog2e};
    const Kv4Cache c = kv4_device(cache);
    const dim3 grid(static_cast<unsigned>(NKV * htiles), static_cast<unsigned>(nsplit), static_cast<unsigned>(B));
    const int ml = static_cast<int>(max_len);
    hipStream_t s = as_stream(stream);
#define SOI_X(H, G) hipLaunchKernelGGL((kv4_attn_kernel<H, G>), grid, dim3(kKv4Waves * kWave), 0, s, a, c, ml)
    SOI_KV4_SHAPES(SOI_X);
#undef SOI_X
    st = launch_status(what);
    if (st || nsplit == 1) return st;
    const dim3 cgrid(static_cast<unsigned>(num_q_heads), static_cast<unsigned>(B));
#define SOI_C(H) hipLaunchKernelGGL((kv4_combine_kernel<H>), cgrid, dim3(H), 0, s, a, c, ml)
    if (hd == 64) SOI_C(64);
    else if (hd == 128) SOI_C(128);
    else SOI_C(256);
#undef SOI_C
    return launch_status(what);
}
