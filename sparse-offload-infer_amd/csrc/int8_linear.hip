// Products of 8-bit rows with 8-bit weights (gfx950):
//
//   linear    y[t, n] = fp16(sx[t] sw[n] sum_k x[t, k] w[n, k] (+ r[t, n]))
//   gate_up   y[t, n] = fp16(silu(g) u), g and u such products of the same rows with two matrices
//
// The sums are 32-bit integers and exact (K < 131072), so neither the tile nor a split of K changes a result; the scales, the
// residual and silu are binary32, rounded once.
//
// Both operands have their K values side by side in memory, and the matrix cores (v_mfma_i32_*_i8) take 16 of a row from a
// lane: A is 16 or 32 weight rows, B as many activation rows, so a lane ends with four neighbouring outputs of one token.
#include "soi_host.h"
#include "soi_device.h"

#include <type_traits>

namespace soi {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;

struct I8Args {
    const int8_t *x, *w, *w2;
    const float *sx, *sw, *sw2;
    const uint16_t* res;
    uint16_t* y;
    int T, N, K;
    int ks;    // few rows: the waves of a workgroup that share a row of weights
    int quad;  // the outputs of four neighbouring n, and what is read with them, lie on whole 8 or 16 bytes
};

// Output n .. n + 3 of token t from their sums (g, and u where GATED).
template <bool GATED>
__device__ __forceinline__ void i8_values(const I8Args& a, int t, int n, const i32x4& g, const i32x4& u, float (&v)[4]) {
    const float sx = ldg(a.sx + t);
    float sg[4], su[4];
    if (a.quad) {
        const f32x4 s = ldg(reinterpret_cast<const f32x4*>(a.sw + n));
#pragma unroll
        for (int e = 0; e < 4; ++e) sg[e] = s[e];
        if constexpr (GATED) {
            const f32x4 r = ldg(reinterpret_cast<const f32x4*>(a.sw2 + n));
#pragma unroll
            for (int e = 0; e < 4; ++e) su[e] = r[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = n + e < a.N ? n + e : a.N - 1;
            sg[e] = ldg(a.sw + i);
            if constexpr (GATED) su[e] = ldg(a.sw2 + i);
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[e] = static_cast<float>(g[e]) * sg[e] * sx;
        if constexpr (GATED) v[e] = silu_f32(v[e]) * (static_cast<float>(u[e]) * su[e] * sx);
    }
}

// stores them, the residual added
__device__ __forceinline__ void i8_store(const I8Args& a, int t, int n, float (&v)[4]) {
    const int64_t at = static_cast<int64_t>(t) * a.N + n;
    if (a.quad) {
        if (a.res) {
            const u32x2 r = ldg(reinterpret_cast<const u32x2*>(a.res + at));
            const f16x2 lo = as_f16x2(r.x), hi = as_f16x2(r.y);
            v[0] += static_cast<float>(lo.x);
            v[1] += static_cast<float>(lo.y);
            v[2] += static_cast<float>(hi.x);
            v[3] += static_cast<float>(hi.y);
        }
        stg(reinterpret_cast<u32x2*>(a.y + at), u32x2{pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3])});
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (n + e < a.N) stg(a.y + at + e, f32_to_f16_bits(a.res ? v[e] + f16_bits_to_f32(ldg(a.res + at + e)) : v[e]));
}

// ---------------------------------------------------------------------------
// Few rows: the weights' bytes bound it, so they go straight from memory to the matrix cores, each once. A wave has R tiles
// of 16 weight rows (GATED: half of them of either matrix) against C tiles of 16 activation rows, whose bytes come from the
// caches; `ks` waves of a workgroup split K and add their sums up through LDS.
// ---------------------------------------------------------------------------
constexpr int kFewWaves = 8;

template <int R, int C, bool GATED>
__global__ __launch_bounds__(kFewWaves * kWave) void int8_few_kernel(const I8Args a) {
    constexpr int U = 4, RN = GATED ? R / 2 : R;  // 64-byte steps in flight; tiles of n
    __shared__ i32x4 s_sum[kFewWaves][R * C][kWave];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int part = wave % a.ks, team = wave / a.ks, teams = kFewWaves / a.ks;
    const int n0 = (static_cast<int>(blockIdx.x) * teams + team) * 16 * RN, t0 = static_cast<int>(blockIdx.y) * 16 * C;
    const int8_t *wp[R], *xp[C];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int n = n0 + 16 * (GATED ? r >> 1 : r) + col;
        const int8_t* base = GATED && (r & 1) ? a.w2 : a.w;
        wp[r] = base + static_cast<int64_t>(n < a.N ? n : a.N - 1) * a.K + 16 * g;
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int t = t0 + 16 * c + col;
        xp[c] = a.x + static_cast<int64_t>(t < a.T ? t : a.T - 1) * a.K + 16 * g;
    }
    i32x4 acc[R][C];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < C; ++c) acc[r][c] = i32x4{0, 0, 0, 0};
    auto step = [&](int k, auto WHOLE) {
        u32x4 w[R][U], x[C][U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool in = WHOLE || k + 64 * u + 16 * g < a.K;
            const auto* zero = reinterpret_cast<const int8_t*>(g_zero16);
#pragma unroll
            for (int r = 0; r < R; ++r)
                w[r][u] = ldg_stream(reinterpret_cast<const u32x4*>(in ? wp[r] + k + 64 * u : zero));
#pragma unroll
            for (int c = 0; c < C; ++c) x[c][u] = ldg(reinterpret_cast<const u32x4*>(in ? xp[c] + k + 64 * u : zero));
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int c = 0; c < C; ++c)
                    acc[r][c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, w[r][u]),
                                                                      __builtin_bit_cast(i32x4, x[c][u]), acc[r][c], 0, 0, 0);
    };
    if (n0 < a.N)
        for (int k = part * 64 * U; k < a.K; k += a.ks * 64 * U) {
            if (k + 64 * U <= a.K) step(k, std::true_type{});
            else step(k, std::false_type{});
        }
    // tile (r, c) of a lane: token 16 c + col, outputs 16 r + 4 g + 0 .. 3
    auto finish = [&](int tile, const i32x4& s0, const i32x4& s1) {  // tile: of n and t
        const int t = t0 + 16 * (tile % C) + col, n = n0 + 16 * (tile / C) + 4 * g;
        if (t < a.T && n < a.N) {
            float v[4];
            i8_values<GATED>(a, t, n, s0, s1, v);
            i8_store(a, t, n, v);
        }
    };
    if (a.ks == 1) {
#pragma unroll
        for (int r = 0; r < RN; ++r)
#pragma unroll
            for (int c = 0; c < C; ++c) finish(r * C + c, acc[GATED ? 2 * r : r][c], acc[GATED ? 2 * r + 1 : r][c]);
        return;
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < C; ++c) s_sum[wave][r * C + c][lane] = acc[r][c];
    __syncthreads();
    auto total = [&](int i) {
        i32x4 s = s_sum[team * a.ks][i][lane];
        for (int k = 1; k < a.ks; ++k) s += s_sum[team * a.ks + k][i][lane];
        return s;
    };
    for (int tile = part; tile < RN * C; tile += a.ks) {
        if constexpr (GATED) finish(tile, total(2 * (tile / C) * C + tile % C), total((2 * (tile / C) + 1) * C + tile % C));
        else finish(tile, total(tile), i32x4{0, 0, 0, 0});
    }
}

// ---------------------------------------------------------------------------
// Many rows: tiles of BN weight rows x BT activation rows, kI8Step bytes of K a stage, two stages in LDS. A stage goes from
// memory into LDS without passing through registers, during the products of the stage before; 16-byte chunks are XOR-swizzled
// on the way, so that the operand reads of 32 rows spread over the banks.
// ---------------------------------------------------------------------------
constexpr int kI8Step = 128;

__device__ __forceinline__ int i8_swz(int row) { return (row >> 1) & 7; }

// 1 KB pieces (8 rows of a stage) into LDS: lane offsets `off` from `base`, zeros from `bytes` on. In asm because the compiler
// would let every LDS read wait for the loads in flight (the kernel waits for them itself, at the barrier). m0 holds the LDS
// address; with the s_nop the load is 5 wait states behind whatever wrote the descriptor's registers.
template <int LOADS>
__device__ __forceinline__ void i8_load(const int8_t* base, int bytes, const uint32_t (&off)[LOADS], uint32_t lds) {
    const uint64_t p = reinterpret_cast<uint64_t>(base);
    const u32x4 r = {static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(p))),
                     static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(p >> 32))) & 0xffffu,
                     static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(bytes)), 0x00027000u};
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds + i * 1024),
                     "v"(off[i]), "s"(r)
                     : "memory", "m0");
}

// WN x WT waves, each with NI x TI tiles of 32 x 32. GATED: odd 32-row strips of the weights' tile are the second matrix's.
template <int WN, int WT, int NI, int TI, bool GATED, int OCC>
__global__ __launch_bounds__(WN * WT * kWave, OCC) void int8_many_kernel(const I8Args a, int ntiles, int ttiles) {
    constexpr int NW = WN * WT, BN = 32 * WN * NI, BT = 32 * WT * TI, STAGE = (BN + BT) * kI8Step;
    constexpr int WL = BN / 8 / NW, XL = BT / 8 / NW;  // 1 KB loads of a wave and stage
    static_assert(BN % (8 * NW) == 0 && BT % (8 * NW) == 0, "whole loads per wave");
    __shared__ __attribute__((aligned(1024))) uint8_t s_tile[2][STAGE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wn = wave % WN, wt = wave / WN, m = lane & 31, hh = lane >> 5;
    // Workgroups go to the XCDs in turn: each XCD takes a contiguous part of the tiles, and walks it in blocks of 4 token tiles
    // by all n, so that the rows in its L2 are used again.
    int tile;
    {
        const int all = ntiles * ttiles, per = (all + 7) >> 3, full = all & 7 ? all & 7 : 8;
        const int xcd = blockIdx.x & 7, i = static_cast<int>(blockIdx.x) >> 3;
        tile = xcd < full ? xcd * per + i : full * per + (xcd - full) * (per - 1) + i;
    }
    constexpr int GT = 4;
    const int band = tile / (GT * ntiles), in = tile - band * GT * ntiles;
    const int high = min(GT, ttiles - band * GT);
    const int n0 = (in / high) * (GATED ? BN / 2 : BN), t0 = (band * GT + in % high) * BT;

    // The lane's chunk of each load: row 8 i + lane / 8 of the wave's part, physical chunk lane % 8. Rows past the matrix are
    // past the descriptor's end; GATED: a wave's loads of a strip stay inside one matrix.
    uint32_t wo[WL], xo[XL];
    const int c8 = lane & 7;
#pragma unroll
    for (int i = 0; i < WL; ++i) {
        const int r = (wave * WL + i) * 8 + (lane >> 3);
        const int row = GATED ? (r >> 6) * 32 + (r & 31) : r;
        wo[i] = static_cast<uint32_t>(row) * a.K + 16 * (c8 ^ i8_swz(r));
    }
#pragma unroll
    for (int i = 0; i < XL; ++i) {
        const int r = (wave * XL + i) * 8 + (lane >> 3);
        xo[i] = static_cast<uint32_t>(r) * a.K + 16 * (c8 ^ i8_swz(r));
    }
    static_assert(!GATED || WL == 4 || WL % 8 == 0, "a wave's loads of weights are whole strips");
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_u8*)&s_tile[0][0]));
    const int64_t wrows = min(a.N - n0, GATED ? BN / 2 : BN), xrows = min(a.T - t0, BT);
    const int8_t* wb = a.w + static_cast<int64_t>(n0) * a.K;
    const int8_t* wb2 = GATED ? a.w2 + static_cast<int64_t>(n0) * a.K : nullptr;
    const int8_t* xb = a.x + static_cast<int64_t>(t0) * a.K;
    const int wend = static_cast<int>(wrows * a.K), xend = static_cast<int>(xrows * a.K);
    auto load = [&](int k0, uint32_t lds) {
        const int left = a.K - k0;
        uint32_t w[WL], x[XL];
        const bool tail = left < kI8Step;  // chunks past the row's end would be the next row's
#pragma unroll
        for (int i = 0; i < WL; ++i) {
            const int r = (wave * WL + i) * 8 + (lane >> 3);
            w[i] = tail && 16 * (c8 ^ i8_swz(r)) >= left ? 0xfffffff0u : wo[i];
        }
#pragma unroll
        for (int i = 0; i < XL; ++i) {
            const int r = (wave * XL + i) * 8 + (lane >> 3);
            x[i] = tail && 16 * (c8 ^ i8_swz(r)) >= left ? 0xfffffff0u : xo[i];
        }
        if constexpr (GATED && WL == 4) {
            i8_load<WL>((wave & 1 ? wb2 : wb) + k0, wend - k0, w, lds + wave * WL * 1024);
        } else if constexpr (GATED) {
#pragma unroll
            for (int i = 0; i < WL; i += 4) {
                const uint32_t o[4] = {w[i], w[i + 1], w[i + 2], w[i + 3]};
                i8_load<4>((i & 4 ? wb2 : wb) + k0, wend - k0, o, lds + (wave * WL + i) * 1024);
            }
        } else {
            i8_load<WL>(wb + k0, wend - k0, w, lds + wave * WL * 1024);
        }
        i8_load<XL>(xb + k0, xend - k0, x, lds + BN * kI8Step + wave * XL * 1024);
    };

    i32x16 acc[NI][TI];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < TI; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
    const uint32_t w_at = lds0 + (wn * NI * 32 + m) * kI8Step + ((hh ^ i8_swz(m)) << 4);
    const uint32_t x_at = lds0 + BN * kI8Step + (wt * TI * 32 + m) * kI8Step + ((hh ^ i8_swz(m)) << 4);
    load(0, lds0);
    uint32_t cur = 0;
    for (int k0 = 0; k0 < a.K; k0 += kI8Step) {
        // every wave's loads of this stage have landed, and its reads of the other buffer are done
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0070);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (k0 + kI8Step < a.K) load(k0 + kI8Step, lds0 + (cur ^ STAGE));
#pragma unroll
        for (int kk = 0; kk < kI8Step / 32; ++kk) {
            i32x4 wf[NI], xf[TI];
#pragma unroll
            for (int i = 0; i < NI; ++i)
                wf[i] = __builtin_bit_cast(
                    i32x4, *(const lds_u32x4*)((lds_u8*)((w_at ^ (kk << 5)) + cur) + i * 32 * kI8Step));
#pragma unroll
            for (int j = 0; j < TI; ++j)
                xf[j] = __builtin_bit_cast(
                    i32x4, *(const lds_u32x4*)((lds_u8*)((x_at ^ (kk << 5)) + cur) + j * 32 * kI8Step));
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int j = 0; j < TI; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[i], xf[j], acc[i][j], 0, 0, 0);
        }
        cur ^= STAGE;
    }
    // lane (m, hh): token m of a tile, outputs 8 q + 4 hh + 0 .. 3 of its 32
    constexpr int NO = GATED ? NI / 2 : NI;
#pragma unroll
    for (int i = 0; i < NO; ++i)
#pragma unroll
        for (int j = 0; j < TI; ++j) {
            const int t = t0 + (wt * TI + j) * 32 + m;
            if (t >= a.T) continue;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int n = n0 + (wn * NO + i) * 32 + 8 * q + 4 * hh;
                if (n >= a.N) continue;
                const i32x16 &x0 = acc[GATED ? 2 * i : i][j], &x1 = acc[GATED ? 2 * i + 1 : i][j];
                float v[4];
                i8_values<GATED>(a, t, n, i32x4{x0[4 * q], x0[4 * q + 1], x0[4 * q + 2], x0[4 * q + 3]},
                                 i32x4{x1[4 * q], x1[4 * q + 1], x1[4 * q + 2], x1[4 * q + 3]}, v);
                i8_store(a, t, n, v);
            }
        }
}

template <bool GATED>
static void int8_launch(I8Args a, hipStream_t st) {
    const int64_t T = a.T, N = a.N;
    if (T <= 64) {
        // as many waves share a row of weights as keep the CUs in waves
#define SOI_F(R, C)                                                                                                     \
    do {                                                                                                                \
        const int64_t tiles = ceil_div64(N, 16 * (GATED ? R / 2 : R));                                                  \
        a.ks = tiles >= 4096 ? 1 : tiles >= 2048 ? 2 : tiles >= 1024 ? 4 : 8;                                           \
        const unsigned gx = static_cast<unsigned>(ceil_div64(tiles, kFewWaves / a.ks));                                 \
        hipLaunchKernelGGL((int8_few_kernel<R, C, GATED>), dim3(gx, static_cast<unsigned>(ceil_div64(T, 16 * C))),      \
                           dim3(kFewWaves * kWave), 0, st, a);                                                          \
    } while (0)
        if (T <= 16) SOI_F(2, 1);
        else if (T <= 32) SOI_F(2, 2);
        else if (T <= 48) SOI_F(2, 3);
        else SOI_F(2, 4);
#undef SOI_F
        return;
    }
#define SOI_M(WN, WT, NI, TI, OCC)                                                                                           \
    do {                                                                                                                     \
        const int64_t bn = 32 * WN * NI / (GATED ? 2 : 1), bt = 32 * WT * TI;                                                \
        const int64_t nt = ceil_div64(N, bn), tt = ceil_div64(T, bt);                                                        \
        hipLaunchKernelGGL((int8_many_kernel<WN, WT, NI, TI, GATED, OCC>), dim3(static_cast<unsigned>(nt * tt)),             \
                           dim3(WN * WT * kWave), 0, st, a, static_cast<int>(nt), static_cast<int>(tt));                     \
    } while (0)
    const int64_t n_all = GATED ? 2 * N : N;
    if (ceil_div64(n_all, 256) * ceil_div64(T, 256) >= 256) SOI_M(2, 4, 4, 2, 2);
    else SOI_M(2, 2, 2, 2, 2);
#undef SOI_M
}

static int int8_check(const char* what, const int8_t* x, const float* x_scale, const int8_t* w, const float* w_scale,
                      const uint16_t* out, int64_t T, int64_t N, int64_t K) {
    SOI_REQUIRE(K >= 16 && K % 16 == 0 && K < 131072, "%s: K must be a multiple of 16 below 131072, got %lld", what, (long long)K);
    SOI_REQUIRE(T >= 0 && N >= 1 && T < (int64_t(1) << 22) && N < (int64_t(1) << 22),
                "%s: rows and outputs must be fewer than 2^22, got %lld and %lld", what, (long long)T, (long long)N);
    if (T == 0) return SOI_OK;
    SOI_REQUIRE(x && x_scale && w && w_scale && out, "%s: null pointer", what);
    SOI_REQUIRE(aligned16(x) && aligned16(w), "%s: x and the weights must be 16-byte aligned", what);
    return SOI_OK;
}

}  // namespace soi

using namespace soi;

extern "C" int soi_int8_linear(const int8_t* x, const float* x_scale, const int8_t* Wq, const float* w_scale,
                               const uint16_t* residual, uint16_t* y, int64_t T, int64_t N, int64_t K, void* stream) {
    const char* what = "soi_int8_linear";
    const int st = int8_check(what, x, x_scale, Wq, w_scale, y, T, N, K);
    if (st || T == 0) return st;
    const bool quad = N % 4 == 0 && aligned16(w_scale) && ((reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(residual)) & 7) == 0;
    const I8Args a{x, Wq, nullptr, x_scale, w_scale, nullptr, residual, y, static_cast<int>(T), static_cast<int>(N),
                   static_cast<int>(K), 1, quad};
    int8_launch<false>(a, as_stream(stream));
    return launch_status(what);
}

extern "C" int soi_int8_gate_up(const int8_t* x, const float* x_scale, const int8_t* gate_Wq, const float* gate_scale,
                                const int8_t* up_Wq, const float* up_scale, uint16_t* h, int64_t T, int64_t N, int64_t K,
                                void* stream) {
    const char* what = "soi_int8_gate_up";
    int st = int8_check(what, x, x_scale, gate_Wq, gate_scale, h, T, N, K);
    if (st || T == 0) return st;
    st = int8_check(what, x, x_scale, up_Wq, up_scale, h, T, N, K);
    if (st) return st;
    const bool quad = N % 4 == 0 && aligned16(gate_scale) && aligned16(up_scale) && (reinterpret_cast<uintptr_t>(h) & 7) == 0;
    const I8Args a{x, gate_Wq, up_Wq, x_scale, gate_scale, up_scale, nullptr, h, static_cast<int>(T), static_cast<int>(N),
                   static_cast<int>(K), 1, quad};
    int8_launch<true>(a, as_stream(stream));
    return launch_status(what);
}
