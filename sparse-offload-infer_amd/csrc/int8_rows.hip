// Activation rows in 8-bit integers with a scale for each token, for the integer products of int8_linear.hip (gfx950):
// the rows themselves, or their RMSNorm, or RMSNorm of a residual sum that is returned too.
//
//   h = fp16(x + r),  n = h w / sqrt(mean h^2 + eps),  s = fp32(max|n| / 127),  q = rint(n / s) (ties to even)
//
// The norm is not rounded before it is quantized. A row that holds a value that is not finite gets a scale that is not
// finite with codes 0, so it reads back as NaN; a row of zeros has scale 0.
//
// A code flips where n / s is next to a border, so n / s is taken in binary64: h w is a product of two binary16 numbers
// and exact in binary32, where the maximum is taken too; 1 / sqrt and 1 / s are one number a row, and an element costs one
// binary64 product (full rate here, and hidden behind the loads). Without a norm n / s can be a tie exactly (s a short
// number): the quotient is refined by its exact remainder once, which makes it correctly rounded.
//
// Bound by memory: 2 bytes an element read and 1 written, with a residual 4 and 3. A row is a wave's (up to 2048 values), so
// nothing waits at a barrier, or a workgroup's of 4 or 16 waves; it stays in registers between the passes. RMSNorm of a residual
// sum, 2048 wide: 1 row 3.3 us (launch and one round trip), 4096 rows 14.2 us = 4.1 TB/s where a large copy takes 11.4.
#include "soi_host.h"
#include "soi_device.h"

namespace soi {

struct RowsArgs {
    const uint16_t *x, *res, *weight;
    int64_t x_stride, res_stride;
    int8_t* q;
    float* scale;
    uint16_t* sum;
    double eps;
    int T, H;
};

template <int MASK>
__device__ __forceinline__ double xor_f64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_bit_cast(uint32_t, xor_lanes<MASK>(__builtin_bit_cast(float, static_cast<uint32_t>(u))));
    const uint32_t hi = __builtin_bit_cast(uint32_t, xor_lanes<MASK>(__builtin_bit_cast(float, static_cast<uint32_t>(u >> 32))));
    return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}

__device__ __forceinline__ double wave_sum_f64(double v) {  // every lane, fixed order
    v += xor_f64<1>(v);
    v += xor_f64<2>(v);
    v += xor_f64<4>(v);
    v += xor_f64<8>(v);
    v += xor_f64<16>(v);
    v += xor_f64<32>(v);
    return v;
}

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    auto step = [&](auto get) {
        const uint32_t o = __builtin_bit_cast(uint32_t, get(__builtin_bit_cast(float, v)));
        v = v > o ? v : o;
    };
    step([](float f) { return xor_lanes<1>(f); });
    step([](float f) { return xor_lanes<2>(f); });
    step([](float f) { return xor_lanes<4>(f); });
    step([](float f) { return xor_lanes<8>(f); });
    step([](float f) { return xor_lanes<16>(f); });
    step([](float f) { return xor_lanes<32>(f); });
    return v;
}

// NW waves a row, C pieces of 8 values a lane. One-wave rows come four to a workgroup.
template <int NW, int C, bool NORM, bool RES>
__global__ __launch_bounds__(NW == 1 ? 256 : NW * kWave) void int8_rows_kernel(const RowsArgs a) {
    constexpr int kLanes = NW * kWave;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int row = NW == 1 ? static_cast<int>(blockIdx.x) * 4 + wave : static_cast<int>(blockIdx.x);
    if (NW == 1 && row >= a.T) return;  // (no barriers in a one-wave row)
    const int i0 = NW == 1 ? lane : static_cast<int>(threadIdx.x), pieces = a.H >> 3;
    const uint16_t* x = a.x + row * a.x_stride;
    u32x4 h[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int i = i0 + c * kLanes;
        h[c] = i < pieces ? ldg_any(x + 8 * i) : u32x4{0, 0, 0, 0};
    }
    if constexpr (RES) {
        const uint16_t* r = a.res + row * a.res_stride;
        u32x4 d[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int i = i0 + c * kLanes;
            d[c] = i < pieces ? ldg_any(r + 8 * i) : u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int i = i0 + c * kLanes;
#pragma unroll
            for (int e = 0; e < 4; ++e) h[c][e] = add_f16x2(h[c][e], d[c][e]);
            if (i < pieces) stg(reinterpret_cast<u32x4*>(a.sum + static_cast<int64_t>(row) * a.H + 8 * i), h[c]);
        }
    }
    u32x4 w[NORM ? C : 1];
    if constexpr (NORM) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int i = i0 + c * kLanes;
            w[c] = i < pieces ? ldg_any(a.weight + 8 * i) : u32x4{0, 0, 0, 0};
        }
    }
    // h w, exact in binary32
    auto value = [&](int c, int e) {
        const float v = f16_bits_to_f32(static_cast<uint16_t>(h[c][e >> 1] >> (16 * (e & 1))));
        if constexpr (!NORM) return v;
        return v * f16_bits_to_f32(static_cast<uint16_t>(w[NORM ? c : 0][e >> 1] >> (16 * (e & 1))));
    };
    uint32_t top = 0;  // max|h w|: on the bit patterns, where infinity and NaN come out on top
    double sum = 0.0;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t m = __builtin_bit_cast(uint32_t, value(c, e)) & 0x7fffffffu;
            top = top > m ? top : m;
            if constexpr (NORM) {
                const float v = f16_bits_to_f32(static_cast<uint16_t>(h[c][e >> 1] >> (16 * (e & 1))));
                sum += static_cast<double>(v * v);  // (the square is exact)
            }
        }
    top = wave_max_u32(top);
    if constexpr (NORM) sum = wave_sum_f64(sum);
    if constexpr (NW > 1) {
        __shared__ double s_sum[NW];
        __shared__ uint32_t s_top[NW];
        if (lane == 0) {
            s_sum[wave] = sum;
            s_top[wave] = top;
        }
        __syncthreads();
        sum = 0.0;
#pragma unroll
        for (int k = 0; k < NW; ++k) {
            sum += s_sum[k];
            top = top > s_top[k] ? top : s_top[k];
        }
    }
    double inv = 1.0;
    if constexpr (NORM) inv = rsqrt_f64(sum / a.H + a.eps);
    const float s = static_cast<float>(static_cast<double>(__builtin_bit_cast(float, top)) * inv / 127.0);
    const bool live = s > 0.0f && s < __builtin_inff();
    const double sd = static_cast<double>(s), rec = live ? 1.0 / sd : 0.0, mul = live ? inv * rec : 0.0;
    int8_t* q = a.q + static_cast<int64_t>(row) * a.H;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int i = i0 + c * kLanes;
        u32x2 out = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const double v = static_cast<double>(live ? value(c, e) : 0.0f);
            double t = v * mul;
            if constexpr (!NORM) t = fma(fma(-t, sd, v), rec, t);
            int k = static_cast<int>(__builtin_rint(t));
            k = k > 127 ? 127 : k < -127 ? -127 : k;
            out[e >> 2] |= (static_cast<uint32_t>(k) & 255u) << (8 * (e & 3));
        }
        if (i < pieces) stg(reinterpret_cast<u32x2*>(q + 8 * i), out);
    }
    if (i0 == 0) stg(a.scale + row, s);
}

template <bool NORM, bool RES>
static void int8_rows_launch(const RowsArgs& a, hipStream_t st) {
    const unsigned T = static_cast<unsigned>(a.T), T4 = (T + 3) / 4;
#define SOI_R(NW, C) \
    hipLaunchKernelGGL((int8_rows_kernel<NW, C, NORM, RES>), dim3(NW == 1 ? T4 : T), dim3(NW == 1 ? 256 : NW * kWave), 0, st, a)
    if (a.H <= 512) SOI_R(1, 1);
    else if (a.H <= 1024) SOI_R(1, 2);
    else if (a.H <= 2048) SOI_R(1, 4);
    else if (a.H <= 4096) SOI_R(4, 2);
    else if (a.H <= 8192) SOI_R(4, 4);
    else if (a.H <= 16384) SOI_R(4, 8);
    else if (a.H <= 32768) SOI_R(16, 4);
    else SOI_R(16, 8);
#undef SOI_R
}

}  // namespace soi

using namespace soi;

extern "C" int soi_int8_rows(const uint16_t* x, int64_t x_stride, const uint16_t* residual, int64_t residual_stride,
                             const uint16_t* weight, double eps, int64_t T, int64_t H, int8_t* q, float* scale, uint16_t* sum,
                             void* stream) {
    const char* what = "soi_int8_rows";
    SOI_REQUIRE(H >= 16 && H % 16 == 0 && H <= 65536, "%s: rows must hold a multiple of 16 values up to 65536, got %lld", what,
                (long long)H);
    SOI_REQUIRE(T >= 0 && T < (int64_t(1) << 30) / 256, "%s: the number of rows must be in [0, 2^22), got %lld", what,
                (long long)T);
    SOI_REQUIRE((residual == nullptr) == (sum == nullptr), "%s: residual and sum come together", what);
    SOI_REQUIRE(!residual || weight, "%s: a residual sum needs a norm weight", what);
    SOI_REQUIRE(eps >= 0.0 && eps < __builtin_inf(), "%s: eps must be finite and not negative", what);
    if (T == 0) return SOI_OK;
    SOI_REQUIRE(x && q && scale, "%s: null pointer", what);
    SOI_REQUIRE((x_stride >= H || T == 1) && (!residual || residual_stride >= H || T == 1), "%s: rows overlap", what);
    SOI_REQUIRE(aligned16(q) && aligned16(sum) && (reinterpret_cast<uintptr_t>(scale) & 3) == 0,
                "%s: q and sum must be 16-byte aligned", what);
    const RowsArgs a{x, residual, weight, x_stride, residual_stride, q, scale, sum, eps, static_cast<int>(T), static_cast<int>(H)};
    hipStream_t st = as_stream(stream);
    if (residual) int8_rows_launch<true, true>(a, st);
    else if (weight) int8_rows_launch<true, false>(a, st);
    else int8_rows_launch<false, false>(a, st);
    return launch_status(what);
}
