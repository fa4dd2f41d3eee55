// Products of 8-bit rows with 8-bit weights (gfx950):
//
//   linear    y[t, n] = fp16(sx[t] sw[n] sum_k x[t, k] w[n, k] (+ r[t, n]))
//   gate_up   y[t, n] = fp16(silu(g) u), g and u such products of the same rows with two matrices
//
// The sums are 32-bit integers and exact (K < 131072), so neither the tile nor a split of K changes a result; the scales, the
// residual and silu are binary32, rounded once.
//
// Both operands have their K values side by side in memory, and the matrix cores (v_mfma_i32_*_i8) take 16 of a row from a
// lane: A is 32 weight rows, B as many activation rows, so a lane ends with four neighbouring outputs of one token.
//
// Few rows are bound by the weights' bytes, or by latency: 5 rows 2048 -> 4096 3.8 us, 48 rows 2048 -> 151936 62 us (5.2 TB/s).
// Many are bound by the operands' way through LDS, the power limit and gate_up's epilogue: 4096 rows 6144 -> 2048 with residual
// 56 us (1.84 POP/s; a library product without the epilogue 61 us), 8192 rows 2048 -> 2 x 6144 225 us (1.83 POP/s; library 244).
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
    int wide;  // 1: the outputs of four neighbouring n, and what is read with them, lie on whole 8 or 16 bytes; 2: eight outputs on 16
};

// silu with the hardware's exponential and reciprocal (2^-22 each, next to a rounding to 2^-11): the library's exponential and
// an exact quotient took a third of gate_up's time at 8192 rows.
__device__ __forceinline__ float i8_silu(float g) {
    return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.4426950408889634f));
}

// The weights' scales of outputs n .. n + 3.
template <bool GATED>
struct I8Scales {
    float g[4], u[GATED ? 4 : 1];
};
template <bool GATED>
__device__ __forceinline__ I8Scales<GATED> i8_scales(const I8Args& a, int n) {
    I8Scales<GATED> s;
    auto four = [&](const float* p, float* o) {
        if (a.wide) {
            const f32x4 v = ldg(reinterpret_cast<const f32x4*>(p + n));
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = v[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = ldg(p + (n + e < a.N ? n + e : a.N - 1));
        }
    };
    four(a.sw, s.g);
    if constexpr (GATED) four(a.sw2, s.u);
    return s;
}

// Four outputs of a token with scale sx from their sums (g, and u where GATED).
template <bool GATED>
__device__ __forceinline__ void i8_values(float sx, const I8Scales<GATED>& s, const i32x4& g, const i32x4& u, float (&v)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[e] = static_cast<float>(g[e]) * s.g[e] * sx;
        if constexpr (GATED) v[e] = i8_silu(v[e]) * (static_cast<float>(u[e]) * s.u[e] * sx);
    }
}

// two outputs; rounded to binary32 first in every kernel, so that a row's bits do not follow from the tile it is in
__device__ __forceinline__ float i8_pack(float a, float b) {
    asm("" : "+v"(a), "+v"(b));
    return __builtin_bit_cast(float, f16x2{static_cast<f16>(a), static_cast<f16>(b)});
}

// the residual of outputs n .. n + 3, where they are wide
__device__ __forceinline__ void i8_add(const I8Args& a, int t, int n, float (&v)[4]) {
    const u32x2 r = ldg(reinterpret_cast<const u32x2*>(a.res + static_cast<int64_t>(t) * a.N + n));
    const f16x2 lo = as_f16x2(r.x), hi = as_f16x2(r.y);
    v[0] += static_cast<float>(lo.x);
    v[1] += static_cast<float>(lo.y);
    v[2] += static_cast<float>(hi.x);
    v[3] += static_cast<float>(hi.y);
}

// the residual added, and the outputs stored
__device__ __forceinline__ void i8_finish(const I8Args& a, int t, int n, float (&v)[4]) {
    const int64_t at = static_cast<int64_t>(t) * a.N + n;
    if (a.wide) {
        if (a.res) i8_add(a, t, n, v);
        stg(reinterpret_cast<u32x2*>(a.y + at), u32x2{pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3])});
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (n + e < a.N) stg(a.y + at + e, f32_to_f16_bits(a.res ? v[e] + f16_bits_to_f32(ldg(a.res + at + e)) : v[e]));
}

// ---------------------------------------------------------------------------
// Many rows: tiles of BN weight rows x BT activation rows, STEP bytes of K a stage, NBUF stages in LDS. A stage goes from
// memory into LDS without passing through registers, NBUF - 1 stages ahead; 16-byte chunks are XOR-swizzled on the way, so that
// the operand reads of 32 rows spread over the banks.
// ---------------------------------------------------------------------------
template <int STEP>
__device__ __forceinline__ int i8_swz(int row) {
    return STEP == 128 ? (row >> 1) & 7 : (row >> 2) & 3;
}

// 1 KB pieces of a stage into LDS: lane offsets `off` from `base`, zeros from `bytes` on. In asm because the compiler would
// let every LDS read wait for the loads in flight (the kernel waits for them itself, at the barrier). m0 holds the LDS
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
template <int WN, int WT, int NI, int TI, int STEP, int NBUF, bool GATED, int OCC>
__global__ __launch_bounds__(WN * WT * kWave, OCC) void int8_many_kernel(const I8Args a, int ntiles, int ttiles) {
    constexpr int NW = WN * WT, BN = 32 * WN * NI, BT = 32 * WT * TI, STAGE = (BN + BT) * STEP, CH = STEP / 16, RL = 1024 / STEP;
    constexpr int WL = BN / RL / NW, XL = BT / RL / NW;  // 1 KB loads of a wave and stage, RL rows each
    static_assert(BN % (RL * NW) == 0 && BT % (RL * NW) == 0, "whole loads per wave");
    constexpr int SL = 32 / RL;  // loads of a strip
    static_assert(!GATED || NI % 2 == 0, "a wave has strips of both matrices");
    static_assert(!GATED || SL % WL == 0 || WL % (2 * SL) == 0, "a wave's loads of weights are parts of a strip, or pairs of them");
    __shared__ __attribute__((aligned(1024))) uint8_t s_tile[NBUF * STAGE];
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

    // The lane's chunk of each load: row RL i + lane / CH of the wave's part, physical chunk lane % CH. Rows past the matrix are
    // past the descriptor's end.
    uint32_t wo[WL], xo[XL];
    auto chunk = [&](int r) { return 16 * ((lane & (CH - 1)) ^ i8_swz<STEP>(r)); };
    auto row_of = [&](int i) { return i * RL + lane / CH; };
#pragma unroll
    for (int i = 0; i < WL; ++i) {
        const int r = row_of(wave * WL + i);
        wo[i] = static_cast<uint32_t>(GATED ? (r >> 6) * 32 + (r & 31) : r) * a.K + chunk(r);
    }
#pragma unroll
    for (int i = 0; i < XL; ++i) {
        const int r = row_of(wave * XL + i);
        xo[i] = static_cast<uint32_t>(r) * a.K + chunk(r);
    }
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_u8*)&s_tile[0]));
    const int64_t wrows = min(a.N - n0, GATED ? BN / 2 : BN), xrows = min(a.T - t0, BT);
    const int8_t* wb = a.w + static_cast<int64_t>(n0) * a.K;
    const int8_t* wb2 = GATED ? a.w2 + static_cast<int64_t>(n0) * a.K : nullptr;
    const int8_t* xb = a.x + static_cast<int64_t>(t0) * a.K;
    const int wend = static_cast<int>(wrows * a.K), xend = static_cast<int>(xrows * a.K);
    int at = 0;         // the next stage's first byte of a row
    uint32_t into = 0;  // and its place in LDS
    auto load = [&] {
        const int left = a.K - at;
        const int wbytes = left > 0 ? wend - at : 0, xbytes = left > 0 ? xend - at : 0;  // (nothing past the last stage)
        const uint32_t lds = lds0 + into;
        auto issue = [&](const uint32_t (&w)[WL], const uint32_t (&x)[XL]) {
            if constexpr (!GATED || WL <= SL) {
                const bool second = GATED && (wave * WL / SL) & 1;
                i8_load<WL>((second ? wb2 : wb) + at, wbytes, w, lds + wave * WL * 1024);
            } else {
#pragma unroll
                for (int i = 0; i < WL; i += SL) {
                    uint32_t o[SL];
#pragma unroll
                    for (int e = 0; e < SL; ++e) o[e] = w[i + e];
                    i8_load<SL>((i / SL & 1 ? wb2 : wb) + at, wbytes, o, lds + (wave * WL + i) * 1024);
                }
            }
            i8_load<XL>(xb + at, xbytes, x, lds + BN * STEP + wave * XL * 1024);
        };
        if (left >= STEP || left <= 0) {
            issue(wo, xo);
        } else {  // chunks past the row's end would be the next row's
            uint32_t w[WL], x[XL];
#pragma unroll
            for (int i = 0; i < WL; ++i) w[i] = chunk(row_of(wave * WL + i)) >= left ? 0xfffffff0u : wo[i];
#pragma unroll
            for (int i = 0; i < XL; ++i) x[i] = chunk(row_of(wave * XL + i)) >= left ? 0xfffffff0u : xo[i];
            issue(w, x);
        }
        at += STEP;
        into = into == (NBUF - 1) * STAGE ? 0 : into + STAGE;
    };

    i32x16 acc[NI][TI];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < TI; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
    const uint32_t w_at = lds0 + (wn * NI * 32 + m) * STEP + ((hh ^ i8_swz<STEP>(m)) << 4);
    const uint32_t x_at = lds0 + BN * STEP + (wt * TI * 32 + m) * STEP + ((hh ^ i8_swz<STEP>(m)) << 4);
    // Operands of a 32-byte step are read while the step before is multiplied. The barrier between two stages lies in front of
    // the last products of the first one, which hide it, and the reads behind it.
    constexpr int KK = STEP / 32, kFlight = (NBUF - 2) * (WL + XL);
    i32x4 wf[2][NI], xf[2][TI];
    auto read = [&](int kk, uint32_t cur) {
#pragma unroll
        for (int i = 0; i < NI; ++i)
            wf[kk & 1][i] = __builtin_bit_cast(i32x4, *(const lds_u32x4*)((lds_u8*)((w_at ^ (kk << 5)) + cur) + i * 32 * STEP));
#pragma unroll
        for (int j = 0; j < TI; ++j)
            xf[kk & 1][j] = __builtin_bit_cast(i32x4, *(const lds_u32x4*)((lds_u8*)((x_at ^ (kk << 5)) + cur) + j * 32 * STEP));
    };
    auto multiply = [&](int kk) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < TI; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[kk & 1][i], xf[kk & 1][j], acc[i][j], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    // this wave's loads of the next stage have landed, and its reads are done; after the barrier everyone's
    auto meet = [] {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0070 | (kFlight & 15) | (kFlight >> 4) << 14);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < NBUF - 1; ++i) load();
    uint32_t cur = 0;
    meet();
    load();  // (into the last buffer, which nothing has used)
    read(0, cur);
    for (int k0 = 0; k0 < a.K; k0 += STEP) {
#pragma unroll
        for (int kk = 0; kk < KK - 1; ++kk) {
            read(kk + 1, cur);
            multiply(kk);
        }
        meet();
        load();  // into this stage's buffer
        cur = cur == (NBUF - 1) * STAGE ? 0 : cur + STAGE;
        read(0, cur);
        multiply(KK - 1);
    }
    // lane (m, hh): token m of a tile, outputs 8 q + 4 hh + 0 .. 3 of its 32
    constexpr int NO = GATED ? NI / 2 : NI;
    float sx[TI];
#pragma unroll
    for (int j = 0; j < TI; ++j) {
        const int t = t0 + (wt * TI + j) * 32 + m;
        sx[j] = ldg(a.sx + (t < a.T ? t : a.T - 1));
    }
    auto quad = [](const i32x16& s, int q) { return i32x4{s[4 * q], s[4 * q + 1], s[4 * q + 2], s[4 * q + 3]}; };
    if (a.wide == 2) {
        // Lanes m and m + 32 change a quad for a quad, so that each stores eight outputs side by side (N is a multiple of 8: what
        // is past it is never stored).
#pragma unroll
        for (int i = 0; i < NO; ++i)
#pragma unroll
            for (int q = 0; q < 4; q += 2) {
                const int n = n0 + (wn * NO + i) * 32 + 8 * q;
                __builtin_amdgcn_sched_barrier(0);  // (all outputs at once would spill)
                if (n >= a.N) continue;
                I8Scales<GATED> sc[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) sc[x] = i8_scales<GATED>(a, min(n + 8 * x, a.N - 8) + 4 * hh);
#pragma unroll
                for (int j = 0; j < TI; ++j) {
                    const int t = t0 + (wt * TI + j) * 32 + m;
                    if (t >= a.T) continue;  // (lanes m and m + 32 alike)
                    float o[4];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        float v[4];
                        i8_values<GATED>(sx[j], sc[x], quad(acc[GATED ? 2 * i : i][j], q + x), quad(acc[GATED ? 2 * i + 1 : i][j], q + x), v);
                        if (!GATED && a.res && n + 8 * x < a.N) i8_add(a, t, n + 8 * x + 4 * hh, v);
                        o[2 * x] = i8_pack(v[0], v[1]);
                        o[2 * x + 1] = i8_pack(v[2], v[3]);
                    }
                    swap32(o[0], o[2]);  // the lower lanes have quad q of 8 q + 0 .. 7 now, the upper ones quad q + 1
                    swap32(o[1], o[3]);
                    const u32x4 w = {__builtin_bit_cast(uint32_t, o[0]), __builtin_bit_cast(uint32_t, o[1]),
                                     __builtin_bit_cast(uint32_t, o[2]), __builtin_bit_cast(uint32_t, o[3])};
                    if (n + 8 * hh < a.N) stg(reinterpret_cast<u32x4*>(a.y + static_cast<int64_t>(t) * a.N + n + 8 * hh), w);
                }
            }
        return;
    }
#pragma unroll
    for (int i = 0; i < NO; ++i)
#pragma unroll
        for (int j = 0; j < TI; ++j) {
            const int t = t0 + (wt * TI + j) * 32 + m;
            __builtin_amdgcn_sched_barrier(0);
            if (t >= a.T) continue;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int n = n0 + (wn * NO + i) * 32 + 8 * q + 4 * hh;
                if (n >= a.N) continue;
                float v[4];
                i8_values<GATED>(sx[j], i8_scales<GATED>(a, n), quad(acc[GATED ? 2 * i : i][j], q), quad(acc[GATED ? 2 * i + 1 : i][j], q), v);
                i8_finish(a, t, n, v);
            }
        }
}

// ---------------------------------------------------------------------------
// Few tiles (few rows, or few outputs): a tile of 32 NI weight rows (GATED: half of them of either matrix) x 32 TI activation
// rows is a workgroup's whose eight waves share K, 64 bytes at a time in turn. A wave stages its own slices in LDS, the next one
// on its way during a slice's products, and waits for nobody until the waves' sums are added up.
// ---------------------------------------------------------------------------
constexpr int kFewWaves = 8;

template <int NI, int TI, bool GATED>
__global__ __launch_bounds__(kFewWaves * kWave, 2) void int8_few_kernel(const I8Args a) {
    constexpr int STEP = 64, WR = 32 * NI, XR = 32 * TI, STAGE = (WR + XR) * STEP, WL = 2 * NI, XL = 2 * TI, BN = GATED ? WR / 2 : WR;
    __shared__ __attribute__((aligned(1024))) uint8_t s_tile[kFewWaves * 2 * STAGE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 31, hh = lane >> 5;
    const int n0 = static_cast<int>(blockIdx.x) * BN, t0 = static_cast<int>(blockIdx.y) * XR;
    // the lane's row and chunk of each 1 KB load of 16 rows
    auto chunk = [&](int i) { return 16 * ((lane & 3) ^ i8_swz<STEP>(16 * i + (lane >> 2))); };
    uint32_t wo[WL], xo[XL];
#pragma unroll
    for (int i = 0; i < WL; ++i) wo[i] = static_cast<uint32_t>((16 * i + (lane >> 2)) % BN) * a.K + chunk(i);
#pragma unroll
    for (int i = 0; i < XL; ++i) xo[i] = static_cast<uint32_t>(16 * i + (lane >> 2)) * a.K + chunk(i);
    const int wend = min(a.N - n0, BN) * a.K, xend = min(a.T - t0, XR) * a.K;
    const int8_t* wb = a.w + static_cast<int64_t>(n0) * a.K;
    const int8_t* wb2 = GATED ? a.w2 + static_cast<int64_t>(n0) * a.K : wb;
    const int8_t* xb = a.x + static_cast<int64_t>(t0) * a.K;
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_u8*)&s_tile[0])) + wave * 2 * STAGE;
    auto load = [&](int k, uint32_t lds) {  // the slice from byte k on; nothing past the rows' end, which would be the next row's
        const int left = a.K - k, at = left > 0 ? k : 0;
        uint32_t w[2][WL / 2], x[XL];
#pragma unroll
        for (int i = 0; i < WL; ++i) w[i / (WL / 2)][i % (WL / 2)] = chunk(i) < left ? wo[i] : 0xfffffff0u;
#pragma unroll
        for (int i = 0; i < XL; ++i) x[i] = chunk(i) < left ? xo[i] : 0xfffffff0u;
        i8_load<WL / 2>(wb + at, wend - at, w[0], lds);
        i8_load<WL / 2>(wb2 + at, wend - at, w[1], lds + WL / 2 * 1024);
        i8_load<XL>(xb + at, xend - at, x, lds + WR * STEP);
    };
    i32x16 acc[NI][TI];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < TI; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
    const uint32_t w_at = lds0 + m * STEP + ((hh ^ i8_swz<STEP>(m)) << 4), x_at = w_at + WR * STEP;
    load(wave * STEP, lds0);
    uint32_t cur = 0;
    for (int k = wave * STEP; k < a.K; k += kFewWaves * STEP) {
        load(k + kFewWaves * STEP, lds0 + (cur ? 0 : STAGE));
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0f70 | (WL + XL));  // this slice has landed; the next one's loads are in flight
        asm volatile("" ::: "memory");
#pragma unroll
        for (int kk = 0; kk < STEP / 32; ++kk) {
            i32x4 wf[NI], xf[TI];
#pragma unroll
            for (int i = 0; i < NI; ++i)
                wf[i] = __builtin_bit_cast(i32x4, *(const lds_u32x4*)((lds_u8*)((w_at ^ (kk << 5)) + cur) + i * 32 * STEP));
#pragma unroll
            for (int j = 0; j < TI; ++j)
                xf[j] = __builtin_bit_cast(i32x4, *(const lds_u32x4*)((lds_u8*)((x_at ^ (kk << 5)) + cur) + j * 32 * STEP));
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int j = 0; j < TI; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[i], xf[j], acc[i][j], 0, 0, 0);
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0xc07f);  // the slice is read before its place is loaded again
        asm volatile("" ::: "memory");
        cur = cur ? 0 : STAGE;
    }
    // The waves' sums, [wave][token][four outputs] with a token's quads swizzled, in the same LDS once no load is in flight.
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    constexpr int Q = WR / 4;  // quads of a token
    static_assert(kFewWaves * XR * Q * 16 <= sizeof(s_tile), "room for the sums");
    i32x4* sums = reinterpret_cast<i32x4*>(s_tile);
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < TI; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                sums[(wave * XR + 32 * j + m) * Q + ((8 * i + 2 * q + hh) ^ (m & (Q - 1)))] =
                    i32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    __syncthreads();
    for (int x = threadIdx.x; x < XR * BN / 4; x += kFewWaves * kWave) {
        const int row = x / (BN / 4), c = x % (BN / 4), t = t0 + row, n = n0 + 4 * c;
        if (t >= a.T || n >= a.N) continue;
        auto total = [&](int quad) {
            i32x4 s = sums[row * Q + (quad ^ (row & (Q - 1)))];
#pragma unroll
            for (int k = 1; k < kFewWaves; ++k) s += sums[(k * XR + row) * Q + (quad ^ (row & (Q - 1)))];
            return s;
        };
        float v[4];
        i8_values<GATED>(ldg(a.sx + t), i8_scales<GATED>(a, n), total(c), GATED ? total(BN / 4 + c) : i32x4{0, 0, 0, 0}, v);
        i8_finish(a, t, n, v);
    }
}

template <bool GATED>
static void int8_launch(I8Args a, hipStream_t st) {
    const int64_t T = a.T, N = a.N;
#define SOI_M(WN, WT, NI, TI, STEP, NBUF, OCC)                                                                               \
    do {                                                                                                                     \
        const int64_t bn = 32 * WN * NI / (GATED ? 2 : 1), bt = 32 * WT * TI;                                                \
        const int64_t nt = ceil_div64(N, bn), tt = ceil_div64(T, bt);                                                        \
        hipLaunchKernelGGL((int8_many_kernel<WN, WT, NI, TI, STEP, NBUF, GATED, OCC>), dim3(static_cast<unsigned>(nt * tt)), \
                           dim3(WN * WT * kWave), 0, st, a, static_cast<int>(nt), static_cast<int>(tt));                     \
    } while (0)
#define SOI_F(NI, TI)                                                                                                \
    hipLaunchKernelGGL((int8_few_kernel<NI, TI, GATED>),                                                             \
                       dim3(static_cast<unsigned>(ceil_div64(N, 32 * NI / (GATED ? 2 : 1))),                         \
                            static_cast<unsigned>(ceil_div64(T, 32 * TI))),                                          \
                       dim3(kFewWaves * kWave), 0, st, a)
    const int64_t n_all = GATED ? 2 * N : N;
    auto tiles = [&](int64_t n, int64_t t) { return ceil_div64(n_all, n) * ceil_div64(T, t); };
    // Where few tiles keep the CUs short of work, workgroups share K among their waves, of the smallest tiles while these fit the
    // CUs once: 32 x 32, 64 x 32, 64 x 64 weight rows x tokens. Then workgroups keep K to themselves, three stages in LDS: 128 x
    // 64, two to a CU, where one tile has all rows (bound by the weights' bytes) or those fit the CUs once, then 128 x 128 of eight
    // waves up to one a CU. More work than that hides its own loads: 128 x 128 of four waves and two stages, two to a CU, and 256 x
    // 256 where those fill their last round.
    // us at 2048 -> 4096 (linear, 64 / 128 / 256 / 400 / 1000 rows): 32 x 32 5.5 / 6.1 / 9.7 / 14.8 / -, 64 x 32 5.6 / 5.7 / 9.3 /
    // 16.1 / -, 64 x 64 5.2 / 5.9 / 7.3 / 12.3 / 23.4, 128 x 64 8.9 / 8.6 / 9.0 / 10.0 / 16.2, 128 x 128 of eight waves 10.5 / 10.6 /
    // 10.8 / 11.7 / 13.9, of four 14.2 / 14.5 / 14.6 / 14.6 / 16.2. 2048 -> 16384, 1 / 32 / 64 / 128 / 256 rows: 64 x 32 8.0 / 7.7 / - / -
    // / -, 64 x 64 - / - / 9.1 / 15.2 / 17.3, 128 x 64 8.9 / 9.3 / 10.3 / 10.5 / 15.6, eight waves - / - / 11.4 / 12.1 / 14.4. 2048 ->
    // 151936, 1 / 32 / 48 rows: 32 x 32 51 / 68 / 125, 128 x 64 51 / 56 / 61, 128 x 128 of four waves 60 / 66 / 73. gate_up, 2048 ->
    // 2 x 6144, 128 / 256 / 512 / 2048 / 8192 rows: 64 x 64 13.1 / - / - / - / -, 128 x 64 9.2 / 13.0 / 20 / 78 / -, eight waves 10.9 /
    // 11.6 / 22 / 67 / -, four 14 / 14.6 / 18 / 58 / 240, 256 x 256 26 / 28 / 30 / 65 / 227; linear 6144 -> 8192, 8192 rows: 443, 407.
    const int64_t big = tiles(256, 256), rounds = ceil_div64(big, 256);
    if (tiles(32, 32) <= 256) SOI_F(1, 1);
    else if (tiles(64, 32) <= 256) SOI_F(2, 1);
    else if (tiles(64, 64) <= 256) SOI_F(2, 2);
    else if (T <= 64 || tiles(128, 64) <= 256) SOI_M(2, 2, 2, 1, 128, 3, 2);
    else if (tiles(128, 128) <= 256) SOI_M(2, 4, 2, 1, 128, 3, 2);
    else if (big < 256 || 5 * big < 4 * 256 * rounds) SOI_M(2, 2, 2, 2, 128, 2, 2);
    else if constexpr (GATED) SOI_M(4, 2, 2, 4, 64, 4, 2);
    else SOI_M(2, 4, 4, 2, 64, 4, 2);
#undef SOI_F
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

static int int8_wide(int64_t N, const float* s0, const float* s1, const uint16_t* y, const uint16_t* res) {
    if (N % 4 || !aligned16(s0) || !aligned16(s1) || ((reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(res)) & 7))
        return 0;
    return N % 8 == 0 && aligned16(y) ? 2 : 1;
}

}  // namespace soi

using namespace soi;

extern "C" int soi_int8_linear(const int8_t* x, const float* x_scale, const int8_t* Wq, const float* w_scale,
                               const uint16_t* residual, uint16_t* y, int64_t T, int64_t N, int64_t K, void* stream) {
    const char* what = "soi_int8_linear";
    const int st = int8_check(what, x, x_scale, Wq, w_scale, y, T, N, K);
    if (st || T == 0) return st;
    const int wide = int8_wide(N, w_scale, w_scale, y, residual);
    const I8Args a{x, Wq, nullptr, x_scale, w_scale, nullptr, residual, y, static_cast<int>(T), static_cast<int>(N),
                   static_cast<int>(K), wide};
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
    const int wide = int8_wide(N, gate_scale, up_scale, h, nullptr);
    const I8Args a{x, gate_Wq, up_Wq, x_scale, gate_scale, up_scale, nullptr, h, static_cast<int>(T), static_cast<int>(N),
                   static_cast<int>(K), wide};
    int8_launch<true>(a, as_stream(stream));
    return launch_status(what);
}
