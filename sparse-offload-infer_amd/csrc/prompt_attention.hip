// Causal attention of packed prompts over binary16 q, k, v on the matrix cores (gfx950).
//
// Sequence b owns query rows cu_q[b] .. cu_q[b + 1] - 1 and key rows cu_k[b] .. cu_k[b + 1] - 1. Query i of nq sees keys
// j <= i + nk - nq of nk (the last query sees every key; nk > nq continues a context), and
//   out[i, h] = sum_j softmax_j(scale q[i, h] . k[j, h / rep]) v[j, h / rep];
// a query that sees no key gives zeros. The framework's other prompt attention (prompt.hip) takes one sequence over a
// contiguous cache in the decode step's order of sums, on v_dot2; this one takes the tile order the matrix cores want.
//
// A workgroup of NW waves owns 32 NW queries of one head; a wave owns 32 of them (v_mfma_f32_32x32x16_f16, lane
// n = lane & 31 is a query, h = lane >> 5):
//   * S^T = K Q^T: lane (n, h) ends with the scores of query n and keys 8 (r >> 2) + 4 h + (r & 3), r < 16, of each
//     32-key tile: a row's maximum is a lane's own but for one swap with lane + 32;
//   * O^T = V^T P^T takes these scores, exponentiated, as its B operand as they lie. The k slots of V are then
//     tokens 16 j + 4 h + 0 .. 3 and + 8 .. 11, four tokens of one dimension a lane, which ds_read_b64_tr_b16 reads
//     straight from the row-major V tile;
//   * the output's rescaling is lane-wise too (a lane's accumulators are all of its own query).
// K and V tiles of 64 keys go from memory into LDS without passing through registers (global_load_lds), two buffers,
// the next tile's loads in flight during a tile's products; 16-byte chunks are XOR-swizzled on the way so that the
// operand reads spread over the banks.
#include "soi_host.h"
#include "soi_device.h"
#include "soi_attn.h"

namespace soi {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint8_t lds_u8;

constexpr int kPaKeys = 64;  // keys per LDS tile
// m is the base of the exponents, raised only where a score would pass it by more than this (in powers of two): weights
// then reach 2^kPaSlack, well inside binary16, and most tiles of a row rescale nothing
constexpr float kPaSlack = 8.0f;

struct PaArgs {
    const uint16_t *q, *k, *v;
    uint16_t* out;
    int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, o_ts, o_hs;  // token and head strides, in elements
    const int32_t *cu_q, *cu_k;
    int Tq, Tk, NQ, NKV, hd;
    float scale_log2;
};

// physical 16-byte chunk of logical chunk c: c ^ swizzle(row)
template <int HD>
__device__ __forceinline__ int pa_swz_k(int row) {
    return HD == 64 ? (row >> 1) & 7 : row & 15;
}
template <int HD>
__device__ __forceinline__ int pa_swz_v(int row) {
    return HD == 64 ? ((row >> 1) & 1) << 2 | ((row >> 2) & 3) : (row & 3) << 2 | ((row >> 2) & 3);
}

// A wave's 1 KB pieces of a tile into LDS: lane offsets `off` from `base`, zeros from `bytes` on. The load is written in
// asm because the compiler, which cannot tell the two buffers apart, would let every LDS read wait for the loads in
// flight (the kernel waits for them itself, at the barrier; no register is written). m0 holds the LDS address.
template <int LOADS>
__device__ __forceinline__ void pa_load(const uint16_t* base, int64_t bytes, const uint32_t (&off)[LOADS], uint32_t lds) {
    const uint64_t p = reinterpret_cast<uint64_t>(base);
    const u32x4 r = {static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(p))),
                     static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(p >> 32))) & 0xffffu,
                     static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(bytes))), 0x00027000u};
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds + i * 1024),
                     "v"(off[i]), "s"(r)
                     : "memory");
}

template <int HD, int NW>
__global__ __launch_bounds__(NW * kWave, HD == 256 ? 1 : 2) void prompt_attention_kernel(const PaArgs a) {
    constexpr int CPR = HD / 8, ROWB = HD * 2, TILEB = kPaKeys * ROWB;  // chunks and bytes of a row, bytes of a tile
    constexpr int KK = HD / 16, DT = HD / 32, NT = kPaKeys / 32, NJ = kPaKeys / 16;
    constexpr int LOADS = TILEB / 1024 / NW;  // 1 KB loads per wave and tile
    static_assert(TILEB % (1024 * NW) == 0, "whole loads per wave");
    __shared__ __attribute__((aligned(1024))) uint8_t s_kv[2][2][TILEB];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, hh = lane >> 5;
    // heads of one KV head lie NKV apart in x: with NKV a multiple of 8 they run on one XCD and share its L2
    const int kvh = static_cast<int>(blockIdx.x) % a.NKV, rep = a.NQ / a.NKV;
    const int head = kvh * rep + static_cast<int>(blockIdx.x) / a.NKV;
    const int b = blockIdx.y;
    auto clamp = [](int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; };
    auto uniform = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
    const int q_lo = clamp(uniform(ldg(a.cu_q + b)), 0, a.Tq), q_hi = clamp(uniform(ldg(a.cu_q + b + 1)), q_lo, a.Tq);
    const int k_lo = clamp(uniform(ldg(a.cu_k + b)), 0, a.Tk), k_hi = clamp(uniform(ldg(a.cu_k + b + 1)), k_lo, a.Tk);
    const int nq = q_hi - q_lo, nk = k_hi - k_lo, off = nk - nq;
    const int qt = static_cast<int>(gridDim.z - 1 - blockIdx.z);  // the longest rows of all sequences first
    const int q0 = qt * (32 * NW);
    if (q0 >= nq) return;
    const int wq0 = q0 + 32 * wave;
    // keys seen by the workgroup's and by the wave's last query
    const int keys = clamp(min(q0 + 32 * NW, nq) + off, 0, nk);
    const int wkeys = wq0 < nq ? clamp(min(wq0 + 32, nq) + off, 0, nk) : 0;
    const int tiles = (keys + kPaKeys - 1) / kPaKeys;
    const int row = wq0 + n;  // the lane's query
    const int last = row + off;  // the last key it sees

    f16x8 qf[KK];
    {
        const uint16_t* qr = a.q + static_cast<int64_t>(q_lo + min(row, nq - 1)) * a.q_ts + head * a.q_hs;
#pragma unroll
        for (int i = 0; i < KK; ++i) {
            const int d = 16 * i + 8 * hh;
            qf[i] = __builtin_bit_cast(f16x8, ldg_any(d < a.hd ? static_cast<const void*>(qr + d) : g_zero16));
        }
    }
    // Tile loads: the buffer descriptor starts at the tile's first key and ends with the sequence's last one, so rows past
    // the end arrive as zeros, and so do the chunks between hd and HD (their offset is past any end). The lanes' offsets
    // are the same for every tile.
    uint32_t ko[LOADS], vof[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int id = (wave * LOADS + i) * 64 + lane, r = id / CPR, p = id % CPR;
        const int ck = p ^ pa_swz_k<HD>(r), cv = p ^ pa_swz_v<HD>(r);
        ko[i] = 8 * ck < a.hd ? static_cast<uint32_t>(r * a.k_ts + 8 * ck) * 2 : 0xfffffff0u;
        vof[i] = 8 * cv < a.hd ? static_cast<uint32_t>(r * a.v_ts + 8 * cv) * 2 : 0xfffffff0u;
    }
    const uint16_t* kb = a.k + k_lo * a.k_ts + kvh * a.k_hs;
    const uint16_t* vb = a.v + k_lo * a.v_ts + kvh * a.v_hs;
    const uint32_t lds = __builtin_amdgcn_readfirstlane(
        static_cast<int>(reinterpret_cast<uintptr_t>((lds_u8*)&s_kv[0][0][0])) + wave * LOADS * 1024);
    auto load = [&](int tile, int buf) {
        const int key = tile * kPaKeys, rows = min(nk - key, kPaKeys);
        pa_load<LOADS>(kb + key * a.k_ts, ((rows - 1) * a.k_ts + a.hd) * 2, ko, lds + (2 * buf) * TILEB);
        pa_load<LOADS>(vb + key * a.v_ts, ((rows - 1) * a.v_ts + a.hd) * 2, vof, lds + (2 * buf + 1) * TILEB);
    };

    f32x16 acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] = 0.0f;
    float m = kNegBig, l = 0.0f;

    const int krow = n * ROWB, kx = hh ^ pa_swz_k<HD>(n);  // K operand: key n of a 32-key tile, chunk 2 kk + hh
    const int vr = 4 * hh + ((lane & 15) >> 2);             // V operand: token vr (+ 8 s + 16 j)
    const int vc = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), vo = 8 * (lane & 1);

    if (tiles > 0) load(0, 0);
    for (int t = 0; t < tiles; ++t) {
        // this wave's part of tile t has landed and its reads of tile t - 1 are done; after the barrier everyone's
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const int buf = t & 1;
        if (t + 1 < tiles) load(t + 1, buf ^ 1);
        const int k0 = t * kPaKeys;
        if (k0 >= wkeys) continue;  // wave-uniform: nothing of this tile is seen here
        const lds_u8* kt = (const lds_u8*)&s_kv[buf][0][0];
        const lds_u8* vt = (const lds_u8*)&s_kv[buf][1][0];

        f32x16 s[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[i][r] = 0.0f;
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                const f16x8 ka = *(const __attribute__((address_space(3))) f16x8*)(kt + i * 32 * ROWB + krow +
                                                                                   (((2 * kk) ^ kx) << 4));
                s[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka, qf[kk], s[i], 0, 0, 0);
            }
        }
        if (k0 + kPaKeys - 1 > wq0 + off) {  // some query of the wave does not see some key of the tile
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int key = k0 + 32 * i + 8 * (r >> 2) + 4 * hh + (r & 3);
                    s[i][r] = key <= last ? s[i][r] : -__builtin_inff();
                }
        }
        float top = s[0][0];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, s[i][r]);
        top = fmaxf(top, xor_lanes<32>(top)) * a.scale_log2;
        if (ballot(top > m + kPaSlack)) {
            const float mn = fmaxf(m, top), w = fast_exp2(m - mn);
            m = mn;
            l *= w;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[d][r] *= w;
        }
        f16x8 pb[NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float p = fast_exp2(fmaf(s[j >> 1][8 * (j & 1) + e], a.scale_log2, -m));
                pb[j][e] = static_cast<f16>(p);
            }
        // the sum is that of the weights the products use: rounded p, added in binary32
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 8; e += 2) l = dot2(f16x2{pb[j][e], pb[j][e + 1]}, f16x2{(f16)1.0f, (f16)1.0f}, l);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                s16x4 w[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int r = vr + 8 * x;  // + 16 j, which leaves the swizzle alone
                    w[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (__attribute__((address_space(3))) s16x4*)(vt + (16 * j + r) * ROWB +
                                                                   (((4 * d + vc) ^ pa_swz_v<HD>(r)) << 4) + vo));
                }
                const f16x8 va = __builtin_bit_cast(
                    f16x8, __builtin_shufflevector(w[0], w[1], 0, 1, 2, 3, 4, 5, 6, 7));
                acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, pb[j], acc[d], 0, 0, 0);
            }
    }
    l += xor_lanes<32>(l);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (row >= nq) return;
    uint16_t* orow = a.out + static_cast<int64_t>(q_lo + row) * a.o_ts + head * a.o_hs;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int dim = 32 * d + 8 * x + 4 * hh;
            if (dim >= a.hd) continue;
            const u32x2 o = {pack_f16x2(acc[d][4 * x] * inv, acc[d][4 * x + 1] * inv),
                             pack_f16x2(acc[d][4 * x + 2] * inv, acc[d][4 * x + 3] * inv)};
            stg(reinterpret_cast<u32x2*>(orow + dim), o);
        }
}

}  // namespace soi

using namespace soi;

extern "C" int soi_prompt_attention(const uint16_t* q, int64_t q_token_stride, int64_t q_head_stride, const uint16_t* k,
                                    int64_t k_token_stride, int64_t k_head_stride, const uint16_t* v,
                                    int64_t v_token_stride, int64_t v_head_stride, const int32_t* cu_q,
                                    const int32_t* cu_k, int64_t batch, int64_t Tq, int64_t Tk, int64_t max_q,
                                    int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim, uint16_t* out,
                                    int64_t out_token_stride, int64_t out_head_stride, float scale, void* stream) {
    const char* what = "soi_prompt_attention";
    SOI_REQUIRE(head_dim >= 8 && head_dim % 8 == 0 && head_dim <= 256, "%s: head_dim must be a multiple of 8 up to 256, got %lld",
                what, (long long)head_dim);
    SOI_REQUIRE(num_kv_heads >= 1 && num_q_heads >= 1 && num_q_heads <= 65535 && num_q_heads % num_kv_heads == 0,
                "%s: num_q_heads must be a multiple of num_kv_heads", what);
    SOI_REQUIRE(batch >= 1 && batch <= 65535, "%s: the number of sequences must be in [1, 65535]", what);
    SOI_REQUIRE(Tq >= 0 && Tk >= 0 && Tq < (int64_t(1) << 30) && Tk < (int64_t(1) << 30), "%s: token counts out of range", what);
    SOI_REQUIRE(max_q >= 0 && max_q <= 8 * 65535, "%s: max_q must be in [0, 524280]", what);
    SOI_REQUIRE(scale > 0.0f && scale < __builtin_inff(), "%s: scale must be positive and finite", what);
    if (Tq == 0 || max_q == 0) return SOI_OK;
    SOI_REQUIRE(q && out && cu_q && cu_k && (Tk == 0 || (k && v)), "%s: null pointer", what);
    SOI_REQUIRE(k_token_stride >= 0 && k_token_stride < (int64_t(1) << 24) && v_token_stride >= 0 &&
                    v_token_stride < (int64_t(1) << 24),
                "%s: key and value rows must be less than 2^24 elements apart", what);
    SOI_REQUIRE(aligned16(k) && aligned16(v) && k_token_stride % 8 == 0 && k_head_stride % 8 == 0 &&
                    v_token_stride % 8 == 0 && v_head_stride % 8 == 0,
                "%s: k and v must be 16-byte aligned with strides of whole 16 bytes", what);
    SOI_REQUIRE((reinterpret_cast<uintptr_t>(out) & 7u) == 0 && out_token_stride % 4 == 0 && out_head_stride % 4 == 0,
                "%s: out must be 8-byte aligned with strides of whole 8 bytes", what);
    const PaArgs a{q, k, v, out, q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride,
                   v_head_stride, out_token_stride, out_head_stride, cu_q, cu_k, static_cast<int>(Tq),
                   static_cast<int>(Tk), static_cast<int>(num_q_heads), static_cast<int>(num_kv_heads),
                   static_cast<int>(head_dim), scale * kLog2e};
    constexpr int NW = 4;
    const dim3 grid(static_cast<unsigned>(num_q_heads), static_cast<unsigned>(batch),
                    static_cast<unsigned>(ceil_div64(max_q, 32 * NW)));
#define SOI_P(H) hipLaunchKernelGGL((prompt_attention_kernel<H, NW>), grid, dim3(NW * kWave), 0, as_stream(stream), a)
    if (head_dim <= 64) SOI_P(64);
    else if (head_dim <= 128) SOI_P(128);
    else SOI_P(256);
#undef SOI_P
    return launch_status(what);
}
