// Writing and reading the paged 4-bit KV cache (soi_kv4.h) for packed tokens of several sequences (gfx950).
//
// Reference: the per-token glue around its attention, qk_norm / apply_rope / kv_cache_append
// (python/soinfer/ops.py:222-250), one sequence and a binary16 cache.
//
// Packed tokens: sequence b's new tokens are rows cu[b] .. cu[b + 1] - 1, and its last one is at position
// lens[b] - 1. A decode step is cu = 0, 1, .. B.
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

// Scale bits and codes (0 .. 15, one a byte of lo / hi) of the lane's eight values, over a group of GS / 8 lanes.
// max|x| is taken on the bit patterns: infinity and NaN come out on top. The quotient x / s of two binary16 numbers is
// either a tie exactly or further than 2^-13 of its size from one, so one refined reciprocal decides every rounding as
// the exact quotient would.
template <int GS>
__device__ __forceinline__ uint16_t kv4_quantize(const u32x4& x, uint32_t q[8]) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    u16x2 m = __builtin_bit_cast(u16x2, w[0] & 0x7fff7fffu);
#pragma unroll
    for (int i = 1; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
    uint32_t top = m.x > m.y ? m.x : m.y;
    auto take = [&](uint32_t o) { top = o > top ? o : top; };
    take(dpp_u<0xb1>(top));
    take(dpp_u<0x4e>(top));
    if (GS >= 64) take(dpp_u<0x141>(top));
    if (GS >= 128) take(dpp_u<0x128>(top));
    const uint16_t s = f32_to_f16_bits(f16_bits_to_f32(static_cast<uint16_t>(top)) / 7.0f);
    const float sf = f16_bits_to_f32(s);
    const bool live = s > 0 && s < 0x7c00;
    const float r = live ? __builtin_amdgcn_rcpf(sf) : 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float v = f16_bits_to_f32(static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1))));
        float y = v * r;
        y = fmaf(fmaf(-y, sf, v), r, y);
        y = fminf(fmaxf(rintf(y), -7.0f), 7.0f);
        q[i] = live ? static_cast<uint32_t>(static_cast<int>(y)) & 15u : 0u;
    }
    return s;
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

// One wave per hd / 8 ... lanes: a token's head is hd / 8 lanes of eight dimensions each, so a wave takes 64 / (hd / 8)
// consecutive tokens, and `heads_per_wave` heads of them one after another with the same cos / sin values in registers.
//
// The norm and the rotation are evaluated in binary64 (binary16 and binary32 operands: the products are exact), then
// rounded to binary16 where qk_norm_rope_append rounds. A cached code is then a function of the inputs alone: a binary32
// evaluation would now and then fall on the other side of a rounding border, and a code with it.
template <int HD, int GS>
__global__ __launch_bounds__(256) void kv4_append_kernel(const Kv4AppendArgs a, const Kv4Cache c) {
    constexpr int LPT = HD / 8, TPW = kWave / LPT, W = HD / 32;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int o = lane % LPT, i = lane / LPT;
    const int t0 = static_cast<int>(blockIdx.x) * TPW, t = t0 + i;
    const int heads = a.NQ + 2 * c.NKV;
    const int h0 = (static_cast<int>(blockIdx.y) * 4 + wave) * a.heads_per_wave;
    if (h0 >= heads) return;  // wave-uniform
    int b, pos;
    const bool found = kv4_locate<TPW>(a.cu, c.lens, c.B, t0, i, lane, b, pos) && t < a.T;
    const int id = found ? kv4_page(c, b, pos) : -1;
    const bool keep = id >= 0 && pos < a.table_rows;  // past the tables nothing is appended, q takes the last row
    const int slot = pos & (c.page - 1);
    const int row = pos < 0 ? 0 : pos < a.table_rows ? pos : a.table_rows - 1;
    float cs[8], sn[8];
    {
        const int64_t at = static_cast<int64_t>(row) * (HD / 2) + 8 * (o % (LPT / 2));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            cs[j] = ldg(a.cos_t + at + j);
            sn[j] = ldg(a.sin_t + at + j);
        }
    }
    const uint16_t* src = a.qkv + (found ? static_cast<int64_t>(t) : 0) * a.qkv_stride + 8 * o;
    const double sign = o < LPT / 2 ? -1.0 : 1.0;
    for (int h = h0; h < h0 + a.heads_per_wave && h < heads; ++h) {
        u32x4 x = ldg_any(src + static_cast<int64_t>(h) * HD);
        const bool is_q = h < a.NQ, is_v = h >= a.NQ + c.NKV;
        if (!is_v) {
            const uint16_t* wn = is_q ? a.q_norm : a.k_norm;
            if (wn) {
                const u32x4 g = ldg_any(wn + 8 * o);
                const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, gw[4] = {g.x, g.y, g.z, g.w};
                double ss = 0.0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const double v = f16_bits_to_f32(static_cast<uint16_t>(xw[j >> 1] >> (16 * (j & 1))));
                    ss = fma(v, v, ss);
                }
                const double inv = 1.0 / sqrt(token_sum<LPT>(ss) / HD + a.eps);
                uint32_t rw[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f16x2 p = as_f16x2(xw[j]), q = as_f16x2(gw[j]);
                    rw[j] = pack_f16x2(
                        static_cast<float>(static_cast<double>(p.x) * inv * static_cast<double>(q.x)),
                        static_cast<float>(static_cast<double>(p.y) * inv * static_cast<double>(q.y)));
                }
                x = u32x4{rw[0], rw[1], rw[2], rw[3]};
            }
            const uint32_t xw[4] = {x.x, x.y, x.z, x.w};
            uint32_t rw[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f16x2 p = as_f16x2(xw[j]), q = as_f16x2(xor_u<LPT / 2>(xw[j]));
                float r[2];
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    r[e] = static_cast<float>(fma(static_cast<double>(p[e]), static_cast<double>(cs[2 * j + e]),
                                                  sign * static_cast<double>(q[e]) * static_cast<double>(sn[2 * j + e])));
                rw[j] = pack_f16x2(r[0], r[1]);
            }
            x = u32x4{rw[0], rw[1], rw[2], rw[3]};
            if (is_q) {
                if (found)
                    stg(reinterpret_cast<u32x4*>(a.q_out + (static_cast<int64_t>(t) * a.NQ + h) * HD) + o, x);
                continue;
            }
            if (a.k_out && found)
                stg(reinterpret_cast<u32x4*>(a.k_out + (static_cast<int64_t>(t) * c.NKV + h - a.NQ) * HD) + o, x);
        }
        uint32_t q[8];
        const uint16_t s = kv4_quantize<GS>(x, q);
        const int kvh = h - a.NQ - (is_v ? c.NKV : 0);
        const int64_t head = static_cast<int64_t>(keep ? id : 0) * c.NKV + kvh;
        if (!is_v) {
            uint32_t word = 0;
            constexpr int order[8] = {0, 2, 4, 6, 1, 3, 5, 7};
#pragma unroll
            for (int n = 0; n < 8; ++n) word |= q[order[n]] << (4 * n);
            if (keep)
                stg(reinterpret_cast<uint32_t*>(c.k_pages + (head * c.page + slot) * (HD / 2)) + W * (o & 3) + (o >> 2),
                    word);
        } else {
            // lane o = 8 u + 2 n + e holds dimensions 64 u + 16 n + 8 e + j, j < 8; unit (m = 8 e + j, u) wants its
            // nibbles n = 0 .. 3 from the four lanes of one (u, e): a 4 x 4 transpose of nibble pairs (j, j + 4)
            uint32_t v = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) v |= (q[j] | (q[j + 4] << 4)) << (8 * j);  // byte j: dimensions j, j + 4
            {
                const uint32_t p = dpp_u<0x4e>(v);  // lane ^ 2: n ^ 1
                v = (o & 2) ? (v & 0xff00ff00u) | ((p >> 8) & 0x00ff00ffu) : (v & 0x00ff00ffu) | ((p & 0x00ff00ffu) << 8);
                const uint32_t r = xor_u<4>(v);     // lane ^ 4: n ^ 2
                v = (o & 4) ? (v & 0xffff0000u) | (r >> 16) : (v & 0x0000ffffu) | (r << 16);
            }
            // now byte n' of lane (u, n, e) is byte n of lane (u, n', e): dimensions n and n + 4 of nibble n'
            const uint32_t lo = v & 0x0f0f0f0fu, hi = (v >> 4) & 0x0f0f0f0fu;
            auto squeeze = [](uint32_t b4) {  // four nibbles in bytes -> 16 bits
                b4 = (b4 | (b4 >> 4)) & 0x00ff00ffu;
                return static_cast<uint16_t>(b4 | (b4 >> 8));
            };
            const int u = o >> 3, m = 8 * (o & 1) + ((o >> 1) & 3);
            uint16_t* units = reinterpret_cast<uint16_t*>(c.v_pages + head * c.page * (HD / 2));
            if (keep) {
                const int64_t at = (static_cast<int64_t>((slot >> 2) * 16 + m) * (HD / 64) + u) * 4 + (slot & 3);
                stg(units + at, squeeze(lo));
                stg(units + at + 4 * (HD / 64) * 4, squeeze(hi));  // unit m + 4
            }
        }
        if (keep && o % (GS / 8) == 0)
            stg((is_v ? c.v_scale : c.k_scale) + (head * (HD / GS) + o / (GS / 8)) * c.page + slot, s);
    }
}

// The cached rows of packed tokens as binary16, k_out and v_out [T, NKV, hd]: the same lanes as the append. A value is
// one rounding of code x scale. Tokens whose position has no page read as zeros.
template <int HD, int GS>
__global__ __launch_bounds__(256) void kv4_read_kernel(const int32_t* __restrict__ cu, const Kv4Cache c,
                                                       uint16_t* __restrict__ k_out, uint16_t* __restrict__ v_out, int T,
                                                       int heads_per_wave) {
    constexpr int LPT = HD / 8, TPW = kWave / LPT, W = HD / 32;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int o = lane % LPT, i = lane / LPT;
    const int t0 = static_cast<int>(blockIdx.x) * TPW, t = t0 + i;
    const int h0 = (static_cast<int>(blockIdx.y) * 4 + wave) * heads_per_wave;
    if (h0 >= c.NKV) return;  // wave-uniform
    int b, pos;
    const bool found = kv4_locate<TPW>(cu, c.lens, c.B, t0, i, lane, b, pos) && t < T;
    const int id = found ? kv4_page(c, b, pos) : -1;
    const int slot = id >= 0 ? pos & (c.page - 1) : 0;
    for (int h = h0; h < h0 + heads_per_wave && h < c.NKV; ++h) {
        const int64_t head = static_cast<int64_t>(id >= 0 ? id : 0) * c.NKV + h;
        const int64_t srow = (head * (HD / GS) + o / (GS / 8)) * c.page + slot;
        const uint32_t kw = ldg(reinterpret_cast<const uint32_t*>(c.k_pages + (head * c.page + slot) * (HD / 2)) +
                                W * (o & 3) + (o >> 2));
        const uint16_t* units = reinterpret_cast<const uint16_t*>(c.v_pages + head * c.page * (HD / 2));
        const int u = o >> 3, n = (o >> 1) & 3, m0 = 8 * (o & 1);
        uint32_t vw = 0;  // AWQ order, so that one unpacking serves both
        constexpr int place[8] = {0, 4, 1, 5, 2, 6, 3, 7};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t unit =
                ldg(units + (static_cast<int64_t>((slot >> 2) * 16 + m0 + j) * (HD / 64) + u) * 4 + (slot & 3));
            vw |= ((unit >> (4 * n)) & 15u) << (4 * place[j]);
        }
        const uint16_t ks = ldg(c.k_scale + srow), vs = ldg(c.v_scale + srow);
        if (!found) continue;
        auto put = [&](uint16_t* out, uint32_t word, uint16_t s) {
            f16x2 v[4];
            dequant_int4x8_bitfield(word, v);
            const f16 sh = __builtin_bit_cast(f16, s);
            u32x4 r;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f16x2 p = v[j] * f16x2{sh, sh};
                r[j] = id >= 0 ? __builtin_bit_cast(uint32_t, p) : 0u;
            }
            stg(reinterpret_cast<u32x4*>(out + (static_cast<int64_t>(t) * c.NKV + h) * HD) + o, r);
        };
        put(k_out, kw, ks);
        put(v_out, vw, vs);
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
    SOI_REQUIRE(T >= 0 && T <= (int64_t(1) << 30), "%s: the token count must be in [0, 2^30], got %lld", what, (long long)T);
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
    SOI_REQUIRE(T >= 0 && T <= (int64_t(1) << 30), "%s: the token count must be in [0, 2^30], got %lld", what, (long long)T);
    if (T == 0) return SOI_OK;
    SOI_REQUIRE(cu_seqlens && k_out && v_out && k_out != v_out, "%s: null pointer or k_out = v_out", what);
    SOI_REQUIRE(aligned16(k_out) && aligned16(v_out), "%s: k_out and v_out must be 16-byte aligned", what);
    const int64_t tw = ceil_div64(T, kWave / (hd / 8));
    const int hpw = kv4_heads_per_wave(tw, cache->num_kv_heads);
    const dim3 grid(static_cast<unsigned>(tw), static_cast<unsigned>(ceil_div64(cache->num_kv_heads, 4 * hpw)));
    const Kv4Cache c = kv4_device(cache);
#define SOI_X(H, G)                                                                                               \
    hipLaunchKernelGGL((kv4_read_kernel<H, G>), grid, dim3(256), 0, as_stream(stream), cu_seqlens, c, k_out, v_out, \
                       static_cast<int>(T), hpw)
    SOI_KV4_SHAPES(SOI_X);
#undef SOI_X
    return launch_status(what);
}
