// Writing and reading the paged 4-bit KV cache (soi_kv4.h) for packed tokens of several sequences (gfx950).
//
// Reference: the per-token glue around its attention, qk_norm / apply_rope / kv_cache_append
// (python/soinfer/ops.py:222-250), one sequence and a binary16 cache.
//
// Packed tokens: sequence b's new tokens are rows cu[b] .. cu[b + 1] - 1, and its last one is at position
// lens[b] - 1. A decode step is cu = 0, 1, .. B.
//
// Both are bound by memory: an append reads 2 (NQ + 2 NKV) hd bytes a token and writes 2 NQ hd, 2 NKV hd if k is kept and
// the token's 2 NKV (hd / 2 + 2 hd / gs) of cache; a read reads these and writes 4 NKV hd. Measured at 16 / 8 heads of 128,
// groups of 64: 24 prompts of 15420 tokens appended in 57 us (246 MB, 4.3 TB/s; a large copy reaches 5.0), 65728 tokens
// of 16 sequences read in 54 us (341 MB, 6.3 TB/s); one token 4.6 and 3.1 us, a launch and three dependent loads.
#include "soi_host.h"
#include "soi_kv4.h"

namespace soi {

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// The sequence and position of packed token t, for TPW consecutive tokens t0 .. of a wave (lane's own: t). Returns
// false for a token behind the last sequence (or where cu is not ascending: no token is then taken twice, and no
// index leaves the arrays).
//
// A decode step has one token per sequence, so sequence t is tried first: its two ends and its length come in one
// round trip. Otherwise the wave counts the ends that are <= t, 64 of them a load.
template <int TPW>
__device__ __forceinline__ bool kv4_locate(const int32_t* cu, const int32_t* lens, int B, int t0, int i, int lane, int& b,
                                           int& pos) {
    const int t = t0 + i;
    b = t < B ? t : B - 1;
    int lo = ldg(cu + b), hi = ldg(cu + b + 1);
    int len = ldg(lens + b);
    bool found = lo <= t && t < hi;
    if (ballot(!found)) {  // wave-uniform
        int n = 0;
        for (int c = 0; c < B; c += kWave) {
            const int e = c + lane < B ? ldg(cu + 1 + c + lane) : 0x7fffffff;
            int mine = 0;
#pragma unroll
            for (int j = 0; j < TPW; ++j) {
                const int m = __popcll(ballot(e <= t0 + j));
                mine = i == j ? m : mine;
            }
            n += mine;
        }
        b = n < B ? n : B - 1;
        lo = ldg(cu + b);
        hi = ldg(cu + b + 1);
        len = ldg(lens + b);
        found = lo <= t && t < hi;
    }
    pos = len - (hi - t);
    return found;
}

// The token group of a workgroup: workgroups go to the eight XCDs in turn, so an XCD gets one contiguous eighth of the
// groups, and the lines that neighbouring tokens share (64 tokens' scales of a group, two tokens' K words) meet in one L2.
__device__ __forceinline__ int kv4_token_group() {
    const int n = gridDim.x, per = (n + 7) >> 3, full = n & 7 ? n & 7 : 8;  // the first `full` XCDs have `per` workgroups
    const int x = blockIdx.x & 7, i = static_cast<int>(blockIdx.x) >> 3;
    return x < full ? x * per + i : full * per + (x - full) * (per - 1) + i;
}

// Sum over the LPT lanes of a token (8, 16 or 32 neighbours), in every one of them.
template <int LPT>
__device__ __forceinline__ double token_sum(double v) {
    auto step = [&](auto get) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = __builtin_bit_cast(uint32_t, get(__builtin_bit_cast(float, static_cast<uint32_t>(u))));
        const uint32_t hi = __builtin_bit_cast(uint32_t, get(__builtin_bit_cast(float, static_cast<uint32_t>(u >> 32))));
        v += __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
    };
    step([](float x) { return dpp_f<0xb1>(x); });
    step([](float x) { return dpp_f<0x4e>(x); });
    step([](float x) { return dpp_f<0x141>(x); });  // the other quad of the 8 lanes, whose lanes agree by now
    if (LPT >= 16) step([](float x) { return dpp_f<0x128>(x); });
    if (LPT >= 32) step([](float x) { return xor_lanes<16>(x); });
    return v;
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, false));
}

template <int MASK>
__device__ __forceinline__ uint32_t xor_u(uint32_t v) {
    return __builtin_bit_cast(uint32_t, xor_lanes<MASK>(__builtin_bit_cast(float, v)));
}

// Lane o of a token's hd / 8 holds eight dimensions in two quads, 4 o + 0 .. 3 (x) and hd / 2 + 4 o + 0 .. 3 (y): the pairs
// of the rotation are one lane's, so an element is widened once for both its products, and a lane needs the cos and sin
// of four angles only.
struct Quads {
    u32x2 x, y;
};

// Scale bits of x's and y's group (low and high half of the result) and the codes, 0 .. 15 each: x's four in the low
// nibbles of the bytes, y's in the high ones. max|x| is taken on the bit patterns, where infinity and NaN come out on top.
// max / 7 is never a binary16 tie nor within 2^-15 of one, so the product with 1 / 7 rounds as the quotient would. A
// quotient x / s of two binary16 numbers is a tie exactly or further than 2^-13 of its size from one, so one refined
// reciprocal decides every rounding as the exact quotient would.
template <int HD, int GS>
__device__ __forceinline__ uint32_t kv4_quantize(const Quads& v, uint32_t& codes) {
    const uint32_t w[4] = {v.x.x, v.x.y, v.y.x, v.y.y};
    u16x2 m[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu);
    const u16x2 mx = __builtin_elementwise_max(m[0], m[1]), my = __builtin_elementwise_max(m[2], m[3]);
    u16x2 top = {mx.x > mx.y ? mx.x : mx.y, my.x > my.y ? my.x : my.y};  // x's, y's
    auto take = [&](uint32_t o) { top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, o)); };
    auto bits = [&] { return __builtin_bit_cast(uint32_t, top); };
    take(dpp_u<0xb1>(bits()));  // eight lanes: 32 dimensions
    take(dpp_u<0x4e>(bits()));
    take(dpp_u<0x141>(bits()));
    if (GS >= 64 && HD >= 128) take(dpp_u<0x128>(bits()));  // sixteen
    if (GS >= 128 && HD >= 256) take(xor_u<16>(bits()));    // thirty-two
    if (GS > HD / 2) take((bits() << 16) | (bits() >> 16));  // one group for both quads
    uint32_t scales = 0;
    codes = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint16_t s = f32_to_f16_bits(f16_bits_to_f32(h ? top.y : top.x) * (1.0f / 7.0f));
        const float sf = f16_bits_to_f32(s);
        const bool live = s > 0 && s < 0x7c00;
        const float r = live ? __builtin_amdgcn_rcpf(sf) : 0.0f;
        uint32_t c = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float e = static_cast<float>(as_f16x2(w[2 * h + (i >> 1)])[i & 1]);
            float q = e * r;
            q = fmaf(fmaf(-q, sf, e), r, q);
            q = __builtin_amdgcn_fmed3f(rintf(q), -7.0f, 7.0f);
            // (a binary32 integer plus 1.5 x 2^23 has its two's complement in the low bits)
            c |= (__builtin_bit_cast(uint32_t, q + 12582912.0f) & 15u) << (8 * i + 4 * h);
        }
        codes |= live ? c : 0u;
        scales |= static_cast<uint32_t>(s) << (16 * h);
    }
    return scales;
}

// Four nibbles in the low halves of the bytes -> 16 bits.
__device__ __forceinline__ uint32_t squeeze4(uint32_t b) {
    b = (b | (b >> 4)) & 0x00ff00ffu;
    return (b | (b >> 8)) & 0xffffu;
}
__device__ __forceinline__ uint32_t stretch4(uint32_t n) {
    n = (n | (n << 8)) & 0x00ff00ffu;
    return (n | (n << 4)) & 0x0f0f0f0fu;
}

// Two binary32 numbers rounded to binary16 by one instruction. (The empty asm keeps the compiler from making one rounding
// of this one and the conversion from binary64 before it.)
__device__ __forceinline__ uint32_t round_f16x2(float a, float b) {
    asm("" : "+v"(a), "+v"(b));
    return __builtin_bit_cast(uint32_t, f16x2{static_cast<f16>(a), static_cast<f16>(b)});
}

struct Kv4AppendArgs {
    const uint16_t* qkv;
    int64_t qkv_stride;
    const uint16_t* q_norm;  // null: no norm
    const uint16_t* k_norm;
    const float* cos_t;
    const float* sin_t;
    uint16_t* q_out;
    uint16_t* k_out;  // null: the rotated k goes to the cache only
    const int32_t* cu;
    int T, NQ, table_rows, heads_per_wave;
    double eps;
};

// A token's head is hd / 8 lanes of two quads each, so a wave takes 512 / hd consecutive tokens, and `heads_per_wave` heads
// of them one after another with the same cos / sin values in registers, the next head's row on its way.
//
// The norm and the rotation are evaluated in binary64 (binary16 and binary32 operands: the products are exact), then
// rounded to binary32 and to binary16 where qk_norm_rope_append rounds. A cached code is then a function of the inputs
// alone: a binary32 evaluation would now and then fall on the other side of a rounding border, and a code with it. (MI355X
// issues binary64 fma at the rate of single binary32 ones; what it costs is the conversions.)
template <int HD, int GS>
__global__ __launch_bounds__(256) void kv4_append_kernel(const Kv4AppendArgs a, const Kv4Cache c) {
    constexpr int LPT = HD / 8, TPW = kWave / LPT, W = HD / 32, H2 = HD / 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int o = lane % LPT, i = lane / LPT;
    const int t0 = kv4_token_group() * TPW, t = t0 + i;
    const int heads = a.NQ + 2 * c.NKV;
    const int h0 = (static_cast<int>(blockIdx.y) * 4 + wave) * a.heads_per_wave;
    if (h0 >= heads) return;  // wave-uniform
    const int h1 = min(heads, h0 + a.heads_per_wave);
    // the first head's row does not wait for the token's place (a row of the input, whatever sequence it belongs to)
    const uint16_t* src = a.qkv + static_cast<int64_t>(t < a.T ? t : 0) * a.qkv_stride + 4 * o;
    auto row_of = [&](int h) {
        const uint16_t* p = src + static_cast<int64_t>(h) * HD;
        return Quads{ldg_any8(p), ldg_any8(p + H2)};
    };
    Quads next = row_of(h0);
    Quads wq{}, wk{};
    if (a.q_norm) {
        wq = Quads{ldg_any8(a.q_norm + 4 * o), ldg_any8(a.q_norm + H2 + 4 * o)};
        wk = Quads{ldg_any8(a.k_norm + 4 * o), ldg_any8(a.k_norm + H2 + 4 * o)};
    }
    int b, pos;
    const bool found = kv4_locate<TPW>(a.cu, c.lens, c.B, t0, i, lane, b, pos) && t < a.T;
    const int id = found ? kv4_page(c, b, pos) : -1;
    const bool keep = id >= 0 && pos < a.table_rows;  // past the tables nothing is appended, q takes the last row
    const int slot = pos & (c.page - 1);
    const int row = pos < 0 ? 0 : pos < a.table_rows ? pos : a.table_rows - 1;
    double cs[4], sn[4];
    {
        const int64_t at = static_cast<int64_t>(row) * H2 + 4 * o;
        const f32x4 cv = __builtin_bit_cast(f32x4, ldg_any(a.cos_t + at)), sv = __builtin_bit_cast(f32x4, ldg_any(a.sin_t + at));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            cs[j] = cv[j];
            sn[j] = sv[j];
        }
    }
    for (int h = h0; h < h1; ++h) {
        Quads v = next;
        if (h + 1 < h1) next = row_of(h + 1);
        const bool is_q = h < a.NQ, is_v = h >= a.NQ + c.NKV;
        if (!is_v) {
            if (a.q_norm) {
                const Quads g = is_q ? wq : wk;
                const uint32_t e[4] = {v.x.x, v.x.y, v.y.x, v.y.y}, w[4] = {g.x.x, g.x.y, g.y.x, g.y.y};
                double ss = 0.0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float f = static_cast<float>(as_f16x2(e[j >> 1])[j & 1]);
                    ss += static_cast<double>(f * f);  // exact in binary32
                }
                const double inv = rsqrt_f64(token_sum<LPT>(ss) / HD + a.eps);
                uint32_t r[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f16x2 p = as_f16x2(e[j]), q = as_f16x2(w[j]);  // element x weight: exact in binary32
                    const float lo = static_cast<float>(p.x) * static_cast<float>(q.x);
                    const float hi = static_cast<float>(p.y) * static_cast<float>(q.y);
                    r[j] = round_f16x2(static_cast<float>(lo * inv), static_cast<float>(hi * inv));
                }
                v = Quads{u32x2{r[0], r[1]}, u32x2{r[2], r[3]}};
            }
            {
                const uint32_t xa[2] = {v.x.x, v.x.y}, xb[2] = {v.y.x, v.y.y};
                float ra[4], rb[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const double p = static_cast<float>(as_f16x2(xa[j >> 1])[j & 1]);
                    const double q = static_cast<float>(as_f16x2(xb[j >> 1])[j & 1]);
                    ra[j] = static_cast<float>(fma(p, cs[j], -(q * sn[j])));
                    rb[j] = static_cast<float>(fma(q, cs[j], p * sn[j]));
                }
                v = Quads{u32x2{round_f16x2(ra[0], ra[1]), round_f16x2(ra[2], ra[3])},
                          u32x2{round_f16x2(rb[0], rb[1]), round_f16x2(rb[2], rb[3])}};
            }
            uint16_t* out = is_q ? a.q_out + (static_cast<int64_t>(t) * a.NQ + h) * HD
                                 : a.k_out ? a.k_out + (static_cast<int64_t>(t) * c.NKV + h - a.NQ) * HD : nullptr;
            if (out && found) {
                stg(reinterpret_cast<u32x2*>(out + 4 * o), v.x);
                stg(reinterpret_cast<u32x2*>(out + H2 + 4 * o), v.y);
            }
            if (is_q) continue;
        }
        uint32_t codes;
        const uint32_t s = kv4_quantize<HD, GS>(v, codes);
        const int kvh = h - a.NQ - (is_v ? c.NKV : 0);
        const int64_t head = static_cast<int64_t>(keep ? id : 0) * c.NKV + kvh;
        if (!is_v) {
            // a quad in AWQ order is nibbles 0, 4, 1, 5 of the word's bytes 0, 2; an octet's second quad is a byte further.
            // Even lanes take x's octet (their quad and the next lane's), odd lanes y's
            auto awq = [](uint32_t b) { return (b & 0xfu) | (b >> 16 & 0xfu) << 4 | (b >> 8 & 0xfu) << 16 | (b >> 24) << 20; };
            const uint32_t qx = awq(codes & 0x0f0f0f0fu), qy = awq(codes >> 4 & 0x0f0f0f0fu);
            const uint32_t other = dpp_u<0xb1>(o & 1 ? qx : qy);
            const uint32_t word = o & 1 ? other | qy << 8 : qx | other << 8;
            const int oct = (o >> 1) + (o & 1 ? HD / 16 : 0);
            if (keep)
                stg(reinterpret_cast<uint32_t*>(c.k_pages + (head * c.page + slot) * (HD / 2)) + W * (oct & 3) + (oct >> 2),
                    word);
        } else {
            uint32_t va, vb;  // units of 16 bits: two a lane
            int ma, ua, ub;
            if constexpr (HD == 64) {
                // x is nibbles n = 0, 1 (o >> 2), y is n = 2, 3; the lane pair o, o ^ 4 shares units m = 4 (o & 3) + 0 .. 3
                const uint32_t p = xor_u<4>(codes);
                const bool hi = o & 4;
                const uint32_t l0 = hi ? p : codes, l1 = hi ? codes : p;      // from the lanes of n = 0 and 1
                auto unit = [&](int j) {
                    const uint32_t a0 = l0 >> (8 * j), a1 = l1 >> (8 * j);
                    return (a0 & 0xfu) | (a1 & 0xfu) << 4 | (a0 & 0xf0u) << 4 | (a1 & 0xf0u) << 8;
                };
                va = hi ? unit(2) : unit(0);
                vb = hi ? unit(3) : unit(1);
                ma = 4 * (o & 3) + (hi ? 2 : 0);
                ua = 0;
                ub = 0;
            } else {
                // x is nibble n = (o >> 2) & 3 of units m = 4 (o & 3) + j, u = o >> 4, y the same of u + hd / 128: a 4 x 4
                // transpose of the code bytes over the lanes of one o & 3, whose bits 2 and 3 are n
                uint32_t w = codes;
                const uint32_t p = xor_u<4>(w);
                w = (o & 4) ? (w & 0xff00ff00u) | (p >> 8 & 0x00ff00ffu) : (w & 0x00ff00ffu) | (p & 0x00ff00ffu) << 8;
                const uint32_t r = xor_u<8>(w);
                w = (o & 8) ? (w & 0xffff0000u) | r >> 16 : (w & 0x0000ffffu) | r << 16;
                va = squeeze4(w & 0x0f0f0f0fu);
                vb = squeeze4(w >> 4 & 0x0f0f0f0fu);
                ma = 4 * (o & 3) + (o >> 2 & 3);
                ua = o >> 4;
                ub = ua + HD / 128;
            }
            if (keep) {
                uint16_t* units = reinterpret_cast<uint16_t*>(c.v_pages + head * c.page * (HD / 2)) +
                                  static_cast<int64_t>(slot >> 2) * (16 * (HD / 64) * 4) + (slot & 3);
                stg(units + (ma * (HD / 64) + ua) * 4, static_cast<uint16_t>(va));
                stg(units + ((ma + (HD == 64 ? 1 : 0)) * (HD / 64) + ub) * 4, static_cast<uint16_t>(vb));
            }
        }
        // the scales: the first lane of each group of x, and of y where that is another group
        if (keep && o % (GS / 4 < LPT ? GS / 4 : LPT) == 0) {
            uint16_t* sp = (is_v ? c.v_scale : c.k_scale) + head * (HD / GS) * c.page + slot;
            const int gx = 4 * o / GS;
            stg(sp + gx * c.page, static_cast<uint16_t>(s));
            if (GS <= H2) stg(sp + (gx + H2 / GS) * c.page, static_cast<uint16_t>(s >> 16));
        }
    }
}

// The cached rows of packed tokens as binary16, k_out and v_out [T, NKV, hd]. Lane o of a token's hd / 8 takes dimensions
// 8 o .. + 7: one K word, and two V units that the four lanes of one (o & 1, o >> 3) transpose between them. A value is
// one rounding of code x scale. Tokens whose position has no page read as zeros. kHeads heads' loads go out together:
// a head is 12 bytes a lane, too few to cover the latency alone. The rows are stored non-temporally: 65728 tokens of 8
// heads of 128 (341 MB) take 54 us with it (6.3 TB/s), 82 us without.
template <int HD, int GS, int kHeads>
__global__ __launch_bounds__(256) void kv4_read_kernel(const int32_t* __restrict__ cu, const Kv4Cache c,
                                                       uint16_t* __restrict__ k_out, uint16_t* __restrict__ v_out, int T,
                                                       int heads_per_wave) {
    constexpr int LPT = HD / 8, TPW = kWave / LPT, W = HD / 32;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int o = lane % LPT, i = lane / LPT;
    const int t0 = kv4_token_group() * TPW, t = t0 + i;
    const int h0 = (static_cast<int>(blockIdx.y) * 4 + wave) * heads_per_wave;
    if (h0 >= c.NKV) return;  // wave-uniform
    const int h1 = min(c.NKV, h0 + heads_per_wave);
    int b, pos;
    const bool found = kv4_locate<TPW>(cu, c.lens, c.B, t0, i, lane, b, pos) && t < T;
    const int id = found ? kv4_page(c, b, pos) : -1;
    const int slot = id >= 0 ? pos & (c.page - 1) : 0;
    // lane o = 8 u + 2 n + e: units 8 e + n and 8 e + n + 4 of u hold, for n' = 0 .. 3, dimensions 64 u + 16 n' + 8 e + n
    // and + 4, which are lane (u, n', e)'s
    const int e = o & 1, n = o >> 1 & 3, u = o >> 3;
    const int64_t page0 = static_cast<int64_t>(id >= 0 ? id : 0) * c.NKV;
    const int64_t k_at = static_cast<int64_t>(slot) * (HD / 2) + 4 * (W * (o & 3) + (o >> 2));
    const int64_t v_at = static_cast<int64_t>(slot >> 2) * (16 * (HD / 64) * 4) + ((8 * e + n) * (HD / 64) + u) * 4 + (slot & 3);
    const int64_t s_at = static_cast<int64_t>(8 * o / GS) * c.page + slot;
    for (int h = h0; h < h1; h += kHeads) {
        uint32_t kw[kHeads], va[kHeads], vb[kHeads];
        uint16_t ks[kHeads], vs[kHeads];
#pragma unroll
        for (int x = 0; x < kHeads; ++x) {
            const int64_t head = page0 + (h + x < h1 ? h + x : h);
            kw[x] = ldg(reinterpret_cast<const uint32_t*>(c.k_pages + head * c.page * (HD / 2) + k_at));
            const uint16_t* units = reinterpret_cast<const uint16_t*>(c.v_pages + head * c.page * (HD / 2)) + v_at;
            va[x] = ldg(units);
            vb[x] = ldg(units + 4 * (HD / 64) * 4);  // unit m + 4
            ks[x] = ldg(c.k_scale + head * (HD / GS) * c.page + s_at);
            vs[x] = ldg(c.v_scale + head * (HD / GS) * c.page + s_at);
        }
#pragma unroll
        for (int x = 0; x < kHeads; ++x) {
            if (h + x >= h1) break;
            uint32_t w = stretch4(va[x]) | stretch4(vb[x]) << 4;  // byte n': the two codes of lane (u, n', e)
            const uint32_t p = dpp_u<0x4e>(w);                    // lane ^ 2: n ^ 1
            w = (o & 2) ? (w & 0xff00ff00u) | (p >> 8 & 0x00ff00ffu) : (w & 0x00ff00ffu) | (p & 0x00ff00ffu) << 8;
            const uint32_t r = xor_u<4>(w);                       // lane ^ 4: n ^ 2
            w = (o & 4) ? (w & 0xffff0000u) | r >> 16 : (w & 0x0000ffffu) | r << 16;
            // byte j: dimensions j (low nibble) and j + 4; in AWQ order 0, 2, 4, 6, 1, 3, 5, 7
            const uint32_t lo = w & 0x0f0f0f0fu, hi = w >> 4 & 0x0f0f0f0fu;
            const uint32_t vw = (lo & 0xfu) | (lo >> 16 & 0xfu) << 4 | (hi & 0xfu) << 8 | (hi >> 16 & 0xfu) << 12 |
                                (lo >> 8 & 0xfu) << 16 | (lo >> 24) << 20 | (hi >> 8 & 0xfu) << 24 | (hi >> 24) << 28;
            if (!found) continue;
            auto put = [&](uint16_t* out, uint32_t word, uint16_t s) {
                f16x2 v[4];
                dequant_int4x8_bitfield(word, v);
                const f16 sh = __builtin_bit_cast(f16, s);
                u32x4 q;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f16x2 f = v[j] * f16x2{sh, sh};
                    q[j] = id >= 0 ? __builtin_bit_cast(uint32_t, f) : 0u;
                }
                stg_stream(reinterpret_cast<u32x4*>(out + (static_cast<int64_t>(t) * c.NKV + h + x) * HD) + o, q);
            };
            put(k_out, kw[x], ks[x]);
            put(v_out, vw, vs[x]);
        }
    }
}

int kv4_check(const soi_kv4_cache* c, const char* what) {
    SOI_REQUIRE(c, "%s: null cache", what);
    SOI_REQUIRE(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256, "%s: head_dim must be 64, 128 or 256, got %lld",
                what, (long long)c->head_dim);
    SOI_REQUIRE((c->group_size == 32 || c->group_size == 64 || c->group_size == 128) && c->group_size <= c->head_dim,
                "%s: group_size must be 32, 64 or 128 and at most head_dim, got %lld", what, (long long)c->group_size);
    SOI_REQUIRE(c->page_size >= 16 && c->page_size <= (1 << 20) && (c->page_size & (c->page_size - 1)) == 0,
                "%s: page_size must be a power of two from 16 up, got %lld", what, (long long)c->page_size);
    SOI_REQUIRE(c->num_pages >= 1 && c->num_pages < (int64_t(1) << 31), "%s: num_pages out of range", what);
    SOI_REQUIRE(c->num_kv_heads >= 1 && c->num_kv_heads <= 4096, "%s: num_kv_heads out of range", what);
    SOI_REQUIRE(c->batch >= 1 && c->batch <= 65535, "%s: the number of sequences must be in [1, 65535], got %lld", what,
                (long long)c->batch);
    SOI_REQUIRE(c->max_blocks >= 1 && c->max_blocks <= (int64_t(1) << 30) / c->page_size,
                "%s: max_blocks * page_size must be in [page_size, 2^30]", what);
    SOI_REQUIRE(c->k_pages && c->k_scale && c->v_pages && c->v_scale && c->block_table && c->seq_lens, "%s: null pointer",
                what);
    SOI_REQUIRE(aligned16(c->k_pages) && aligned16(c->v_pages) && aligned16(c->k_scale) && aligned16(c->v_scale),
                "%s: pages and scales must be 16-byte aligned", what);
    return SOI_OK;
}

Kv4Cache kv4_device(const soi_kv4_cache* c) {
    Kv4Cache d;
    d.k_pages = c->k_pages;
    d.k_scale = c->k_scale;
    d.v_pages = c->v_pages;
    d.v_scale = c->v_scale;
    d.table = c->block_table;
    d.lens = c->seq_lens;
    d.B = static_cast<int>(c->batch);
    d.max_blocks = static_cast<int>(c->max_blocks);
    d.P = static_cast<int>(c->num_pages);
    d.NKV = static_cast<int>(c->num_kv_heads);
    d.page = static_cast<int>(c->page_size);
    d.page_shift = __builtin_ctz(static_cast<unsigned>(c->page_size));
    return d;
}

// Heads per wave: one while that leaves fewer than about 4 waves per SIMD, then as many as keep that (the cos / sin rows
// and the token's place are read once for them).
static int kv4_heads_per_wave(int64_t token_waves, int64_t heads) {
    const int64_t n = token_waves * heads / 4096;
    return static_cast<int>(n < 1 ? 1 : n > heads ? heads : n > 8 ? 8 : n);
}

// A workgroup takes 512 / hd tokens with 256 threads, and a grid holds fewer than 2^32 threads.
static int64_t kv4_most_tokens(int64_t hd) { return ((int64_t(1) << 24) - 1) * (kWave / (hd / 8)); }

}  // namespace soi

using namespace soi;

extern "C" int soi_kv4_append(const soi_kv4_cache* cache, const uint16_t* qkv, int64_t qkv_stride, const uint16_t* q_norm,
                              const uint16_t* k_norm, const float* cos_table, const float* sin_table, int64_t table_rows,
                              const int32_t* cu_seqlens, int64_t T, int64_t num_q_heads, uint16_t* q_out, uint16_t* k_out,
                              float eps, void* stream) {
    const char* what = "soi_kv4_append";
    int st = kv4_check(cache, what);
    if (st) return st;
    const int64_t hd = cache->head_dim, gs = cache->group_size, heads = num_q_heads + 2 * cache->num_kv_heads;
    SOI_REQUIRE(num_q_heads >= 1 && num_q_heads <= 65535, "%s: num_q_heads out of range", what);
    SOI_REQUIRE(T >= 0 && T <= kv4_most_tokens(hd), "%s: the number of tokens must be in [0, %lld], got %lld", what,
                (long long)kv4_most_tokens(hd), (long long)T);
    SOI_REQUIRE(qkv_stride >= heads * hd || T <= 1, "%s: qkv rows overlap: stride %lld below %lld", what,
                (long long)qkv_stride, (long long)(heads * hd));
    SOI_REQUIRE((q_norm == nullptr) == (k_norm == nullptr), "%s: q_norm and k_norm come together", what);
    SOI_REQUIRE(table_rows >= 1 && table_rows <= (int64_t(1) << 30), "%s: RoPE table rows out of range", what);
    if (T == 0) return SOI_OK;
    SOI_REQUIRE(qkv && cos_table && sin_table && cu_seqlens && q_out, "%s: null pointer", what);
    SOI_REQUIRE(aligned16(q_out) && aligned16(k_out), "%s: q_out and k_out must be 16-byte aligned", what);
    Kv4AppendArgs a{qkv, qkv_stride, q_norm, k_norm, cos_table, sin_table, q_out, k_out, cu_seqlens, static_cast<int>(T),
                    static_cast<int>(num_q_heads), static_cast<int>(table_rows), 1, static_cast<double>(eps)};
    const int64_t tw = ceil_div64(T, kWave / (hd / 8));
    a.heads_per_wave = kv4_heads_per_wave(tw, heads);
    const dim3 grid(static_cast<unsigned>(tw), static_cast<unsigned>(ceil_div64(heads, 4 * a.heads_per_wave)));
    const Kv4Cache c = kv4_device(cache);
#define SOI_X(H, G) hipLaunchKernelGGL((kv4_append_kernel<H, G>), grid, dim3(256), 0, as_stream(stream), a, c)
    SOI_KV4_SHAPES(SOI_X);
#undef SOI_X
    return launch_status(what);
}

extern "C" int soi_kv4_read(const soi_kv4_cache* cache, const int32_t* cu_seqlens, int64_t T, uint16_t* k_out,
                            uint16_t* v_out, void* stream) {
    const char* what = "soi_kv4_read";
    int st = kv4_check(cache, what);
    if (st) return st;
    const int64_t hd = cache->head_dim, gs = cache->group_size;
    SOI_REQUIRE(T >= 0 && T <= kv4_most_tokens(hd), "%s: the number of tokens must be in [0, %lld], got %lld", what,
                (long long)kv4_most_tokens(hd), (long long)T);
    if (T == 0) return SOI_OK;
    SOI_REQUIRE(cu_seqlens && k_out && v_out && k_out != v_out, "%s: null pointer or k_out = v_out", what);
    SOI_REQUIRE(aligned16(k_out) && aligned16(v_out), "%s: k_out and v_out must be 16-byte aligned", what);
    const int64_t tw = ceil_div64(T, kWave / (hd / 8));
    const int hpw = kv4_heads_per_wave(tw, cache->num_kv_heads);
    const dim3 grid(static_cast<unsigned>(tw), static_cast<unsigned>(ceil_div64(cache->num_kv_heads, 4 * hpw)));
    const Kv4Cache c = kv4_device(cache);
#define SOI_X(H, G)                                                                                               \
    hipLaunchKernelGGL((kv4_read_kernel<H, G, 4>), grid, dim3(256), 0, as_stream(stream), cu_seqlens, c, k_out,   \
                       v_out, static_cast<int>(T), hpw)
    SOI_KV4_SHAPES(SOI_X);
#undef SOI_X
    return launch_status(what);
}
