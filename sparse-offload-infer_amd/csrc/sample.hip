// The next token of each row of logits by temperature, top-k, top-p and min-p, from given random numbers (gfx950).
//
//   w_i = exp(-z_i), z_i = (max l - l_i) / T; tokens in order of falling logits, the lower index first among equals.
//   top-k keeps the first k; top-p, of these, every token in front of which the weights add up to less than p times their
//   sum; min-p, of these, the tokens of w >= min_p. Each keeps a prefix of the order, so the kept set is one number K, the
//   sum of its weights, and the token is the first whose running sum exceeds u K.
//
// Weights are whole numbers, rint(2^44 w) (w in binary64 to 2^-46): sums of up to 2^19 of them are exact in 64 bits, so no
// result depends on the order of an addition, on how a row is split, or on the rows beside it. Tokens below 2^-45 of the
// largest weight count as 0 and are never drawn.
//
// No sort of the row. Its weights go into kBins bins of equal width in z (a histogram in LDS of each chunk, added up in
// memory); the running sums over the bins say which bins the k-th token, the p border, the min_p border and the drawn token
// can lie in; only the tokens of those few bins are collected, sorted (a few hundred), and looked at one by one. Rows with a
// top-k of up to kMostK need no weights before that: the bins down to the k-th token are counted and collected whole.
// Bins that hold more than kList tokens (many equal logits) are searched by radix passes over the row instead.
//
// Four launches: largest and smallest logit, bins, collect, decide. Bound by latency for few rows and by the three passes
// over the logits, the binary64 exponentials of the second and its LDS atomics for many.
#include "soi_host.h"
#include "soi_device.h"

#include <type_traits>

namespace soi {

constexpr int kBins = 1024, kThreads = 1024, kList = 4096, kMostK = 2048, kPiece = 8, kChunk = kThreads * kPiece;
constexpr int kIdxBits = 20;                      // of a token's index in its place in the order (the vocabulary: 2^19)
constexpr double kZMost = 45 * 0.6931471805599453;  // 2^44 exp(-z) rounds to 0 from here on
constexpr uint32_t kKeyInf = 0xff800000u, kKeyNegInf = 0x007fffffu;

struct SampleRow {  // of the workspace
    uint64_t weight[kBins];
    uint32_t count[kBins];
    uint32_t listed, pad[3];
    uint64_t list[kList];
};
struct SamplePart {  // a chunk's extremes
    uint64_t top;    // key of the largest, ~index
    uint32_t low;    // key of the smallest number that is not -inf
    uint32_t pad;
};

struct SampleArgs {
    const void* logits;
    int64_t stride;
    const float* u;
    const float *temperature, *top_p, *min_p;  // or null: the same number for every row
    const int32_t* top_k;
    float temperature_all, top_p_all, min_p_all;
    int top_k_all;
    int32_t* tokens;
    SampleRow* rows;
    SamplePart* parts;
    int B, V, chunks, chunk;  // chunks of `chunk` logits a row
};

// Ascending with the number; NaN on top, both zeros one.
__device__ __forceinline__ uint32_t key_of(float v) {
    if (v != v) return 0xffffffffu;
    const uint32_t b = __builtin_bit_cast(uint32_t, v == 0.0f ? 0.0f : v);
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __builtin_bit_cast(float, key >> 31 ? key & 0x7fffffffu : ~key);
}
// place in the order: ascending from the first token
__device__ __forceinline__ uint64_t place_of(uint32_t key, int i) {
    return static_cast<uint64_t>(~key) << kIdxBits | static_cast<uint32_t>(i);
}
__device__ __forceinline__ uint32_t place_key(uint64_t c) { return ~static_cast<uint32_t>(c >> kIdxBits); }
__device__ __forceinline__ int place_index(uint64_t c) { return static_cast<int>(c & ((1u << kIdxBits) - 1)); }

// Calls f(key, index) for the logits i of [lo, hi) that thread `tid` of kThreads has.
template <class LT, class F>
__device__ __forceinline__ void each_logit(const SampleArgs& a, int row, int lo, int hi, int tid, F f) {
    const LT* p = static_cast<const LT*>(a.logits) + row * a.stride;
    for (int i = lo + tid * kPiece; i < hi; i += kChunk) {
        float v[kPiece];
        if (i + kPiece <= a.V) {
            if constexpr (sizeof(LT) == 2) {
                const u32x4 r = ldg_any(p + i);
#pragma unroll
                for (int e = 0; e < kPiece; ++e) v[e] = f16_bits_to_f32(static_cast<uint16_t>(r[e >> 1] >> (16 * (e & 1))));
            } else {
                const u32x4 r0 = ldg_any(p + i), r1 = ldg_any(p + i + 4);
                // (lanes copied to scalars first: a bit cast of a vector's lane was compiled as one of lane 0)
                const uint32_t w[kPiece] = {r0.x, r0.y, r0.z, r0.w, r1.x, r1.y, r1.z, r1.w};
#pragma unroll
                for (int e = 0; e < kPiece; ++e) v[e] = __builtin_bit_cast(float, w[e]);
            }
#pragma unroll
            for (int e = 0; e < kPiece; ++e) f(key_of(v[e]), i + e);
        } else {
            for (int e = i; e < a.V; ++e) {
                if constexpr (sizeof(LT) == 2) f(key_of(f16_bits_to_f32(ldg(p + e))), e);
                else f(key_of(ldg(p + e)), e);
            }
        }
    }
}

template <class LT>
__global__ __launch_bounds__(kThreads) void sample_extremes_kernel(const SampleArgs a) {
    __shared__ uint64_t s_top[kThreads / kWave];
    __shared__ uint32_t s_low[kThreads / kWave];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.y, chunk = blockIdx.x;
    if (chunk == 0) {
        SampleRow* w = a.rows + row;
        stg(&w->weight[tid], uint64_t(0));
        stg(&w->count[tid], 0u);
        if (tid == 0) stg(&w->listed, 0u);
    }
    uint64_t top = 0;
    uint32_t low = 0xffffffffu;
    each_logit<LT>(a, row, chunk * a.chunk, min(a.V, (chunk + 1) * a.chunk), tid, [&](uint32_t key, int i) {
        const uint64_t t = static_cast<uint64_t>(key) << 32 | ~static_cast<uint32_t>(i);
        top = t > top ? t : top;
        low = key > kKeyNegInf && key < low ? key : low;
    });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint64_t t = __shfl_xor(top, o);
        const uint32_t l = __shfl_xor(low, o);
        top = t > top ? t : top;
        low = l < low ? l : low;
    }
    if (lane == 0) {
        s_top[wave] = top;
        s_low[wave] = low;
    }
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kThreads / kWave; ++w) {
            top = s_top[w] > top ? s_top[w] : top;
            low = s_low[w] < low ? s_low[w] : low;
        }
        SamplePart* p = a.parts + static_cast<int64_t>(row) * a.chunks + chunk;
        stg(&p->top, top);
        stg(&p->low, low);
    }
}

// What a row's launches have in common.
struct SamplePlan {
    bool greedy;  // the token is the first largest one
    int first;    // that token
    double max, inv_t, z_limit, per_z;  // tokens with z <= z_limit count; bins per unit of z
    double min_z;                       // min-p: tokens with z <= min_z stay (infinity: no min-p)
    double p;                           // 1: no top-p
    int k;                              // 0: no top-k
    bool by_count;                      // the tokens down to the k-th are all collected
    __device__ __forceinline__ double z(uint32_t key) const { return (max - static_cast<double>(value_of(key))) * inv_t; }
    __device__ __forceinline__ bool counts(uint32_t key, double z) const { return key > kKeyNegInf && z <= z_limit; }
    __device__ __forceinline__ int bin(double z) const {
        const double b = z * per_z;
        return b < kBins - 1 ? static_cast<int>(b) : kBins - 1;
    }
};

__device__ __forceinline__ SamplePlan sample_plan(const SampleArgs& a, int row) {
    const int lane = threadIdx.x & 63;
    const SamplePart* p = a.parts + static_cast<int64_t>(row) * a.chunks;
    uint64_t top = 0;
    uint32_t low = 0xffffffffu;
    for (int c = lane; c < a.chunks; c += kWave) {
        const uint64_t t = ldg(&p[c].top);
        const uint32_t l = ldg(&p[c].low);
        top = t > top ? t : top;
        low = l < low ? l : low;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint64_t t = __shfl_xor(top, o);
        const uint32_t l = __shfl_xor(low, o);
        top = t > top ? t : top;
        low = l < low ? l : low;
    }
    const float T = a.temperature ? ldg(a.temperature + row) : a.temperature_all;
    const float tp = a.top_p ? ldg(a.top_p + row) : a.top_p_all, mp = a.min_p ? ldg(a.min_p + row) : a.min_p_all;
    const int k = a.top_k ? ldg(a.top_k + row) : a.top_k_all;
    const uint32_t key = static_cast<uint32_t>(top >> 32);
    SamplePlan s;
    s.first = static_cast<int>(~static_cast<uint32_t>(top));
    s.greedy = !(T > 0.0f) || key >= kKeyInf || key <= kKeyNegInf;
    if (s.greedy) return s;
    s.max = static_cast<double>(value_of(key));
    s.inv_t = 1.0 / static_cast<double>(T);
    s.p = tp < 1.0f ? static_cast<double>(tp) : 1.0;  // (NaN: 1)
    s.k = k > 0 ? k : 0;
    s.min_z = mp > 0.0f ? (mp < 1.0f ? -log(static_cast<double>(mp)) : 0.0) : __builtin_inf();
    // without top-p, what min-p drops does not count for anything
    s.z_limit = s.p == 1.0 && s.min_z < kZMost ? s.min_z : kZMost;
    const double most = s.z(low), span = most < s.z_limit ? most : s.z_limit;
    s.per_z = span > 1e-290 ? kBins / span : 0.0;
    s.by_count = s.k > 0 && s.k <= kMostK;
    return s;
}

// rint(2^44 exp(-z)) for 0 <= z <= kZMost: 2^n e^r, |r| <= ln 2 / 2, by the exponential series to r^12 (error 2^-50), and the
// rounding of a number below 2^52 by adding 2^52.
__device__ __forceinline__ uint64_t weight_of(double z) {
    const double n = __builtin_rint(z * -1.4426950408889634);
    const double r = fma(n, -0.6931471805599453, -z);  // (n times the constant's error: below 2^-49)
    double e = 1.0 / 479001600;
    e = fma(e, r, 1.0 / 39916800);
    e = fma(e, r, 1.0 / 3628800);
    e = fma(e, r, 1.0 / 362880);
    e = fma(e, r, 1.0 / 40320);
    e = fma(e, r, 1.0 / 5040);
    e = fma(e, r, 1.0 / 720);
    e = fma(e, r, 1.0 / 120);
    e = fma(e, r, 1.0 / 24);
    e = fma(e, r, 1.0 / 6);
    e = fma(e, r, 0.5);
    e = fma(e, r, 1.0);
    e = fma(e, r, 1.0);
    const double w = __builtin_amdgcn_ldexp(e, static_cast<int>(n) + 44);
    return __builtin_bit_cast(uint64_t, w + 4503599627370496.0) & ((uint64_t(1) << 52) - 1);
}

template <class LT>
__global__ __launch_bounds__(kThreads) void sample_bins_kernel(const SampleArgs a) {
    __shared__ uint64_t s_weight[kBins];
    __shared__ uint32_t s_count[kBins];
    const int tid = threadIdx.x, row = blockIdx.y, chunk = blockIdx.x;
    const SamplePlan s = sample_plan(a, row);
    if (s.greedy) return;
    s_weight[tid] = 0;
    s_count[tid] = 0;
    __syncthreads();
    const bool weights = !s.by_count, counts = s.k > 0;
    each_logit<LT>(a, row, chunk * a.chunk, min(a.V, (chunk + 1) * a.chunk), tid, [&](uint32_t key, int) {
        const double z = s.z(key);
        if (!s.counts(key, z)) return;
        const int b = s.bin(z);
        if (weights) atomicAdd(reinterpret_cast<unsigned long long*>(&s_weight[b]), weight_of(z));
        if (counts) atomicAdd(&s_count[b], 1u);
    });
    __syncthreads();
    SampleRow* w = a.rows + row;
    if (s_weight[tid]) atomicAdd(reinterpret_cast<unsigned long long*>(&w->weight[tid]), s_weight[tid]);
    if (s_count[tid]) atomicAdd(&w->count[tid], s_count[tid]);
}

// Inclusive sums over the workgroup's threads; s_part: one number a wave. Every thread may call it again at once.
template <class N>
__device__ __forceinline__ N scan_threads(N v, N* s_part) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const N x = __shfl_up(v, o);
        v += lane >= o ? x : 0;
    }
    if (lane == 63) s_part[wave] = v;
    __syncthreads();
    N base = 0;
    for (int w = 0; w < kThreads / kWave; ++w) base += w < wave ? s_part[w] : 0;
    __syncthreads();
    return v + base;
}

// The bins' running sums; thread b has bin b.
struct SampleBins {
    uint64_t weight, to_weight;  // the bin's, and up to and with it
    uint32_t count, to_count;
};

struct SampleShared {
    uint64_t part[kThreads / kWave];
    uint32_t part32[kThreads / kWave];
    uint64_t before, to;  // answers
    int at;
};

__device__ __forceinline__ SampleBins sample_bins(const SampleArgs& a, int row, SampleShared& sh) {
    const SampleRow* w = a.rows + row;
    SampleBins b;
    b.weight = ldg(&w->weight[threadIdx.x]);
    b.count = ldg(&w->count[threadIdx.x]);
    b.to_weight = scan_threads(b.weight, sh.part);
    b.to_count = scan_threads(b.count, sh.part32);
    return b;
}

// A bin, with the weights in front of it and with it.
struct BinAt {
    int bin;
    uint64_t before, to;
};

// The bin in which the running sum reaches x, 1 <= x <= the sum of all (the last bin otherwise).
__device__ __forceinline__ BinAt bin_of_weight(const SampleBins& b, uint64_t x, SampleShared& sh) {
    if ((b.to_weight >= x && b.to_weight - b.weight < x) || (threadIdx.x == kBins - 1 && b.to_weight < x)) {
        sh.at = threadIdx.x;
        sh.before = b.to_weight - b.weight;
        sh.to = b.to_weight;
    }
    __syncthreads();
    const BinAt r{sh.at, sh.before, sh.to};
    __syncthreads();
    return r;
}

__device__ __forceinline__ BinAt bin_at(const SampleBins& b, int bin, SampleShared& sh) {
    if (static_cast<int>(threadIdx.x) == bin) {
        sh.before = b.to_weight - b.weight;
        sh.to = b.to_weight;
    }
    __syncthreads();
    const BinAt r{bin, sh.before, sh.to};
    __syncthreads();
    return r;
}

// The bin of the k-th token, and how many there are in front of it and with it (k > 0, at most all).
__device__ __forceinline__ BinAt bin_of_count(const SampleBins& b, uint32_t k, SampleShared& sh) {
    if (b.to_count >= k && b.to_count - b.count < k) {
        sh.at = threadIdx.x;
        sh.before = b.to_count - b.count;
        sh.to = b.to_count;
    }
    __syncthreads();
    const BinAt r{sh.at, sh.before, sh.to};
    __syncthreads();
    return r;
}

// The running sum that top-p's last token reaches first, of a sum of `all`; and the one that the drawn token does, of the kept
// weights `kept`.
__device__ __forceinline__ uint64_t p_border(double p, uint64_t all) {
    const uint64_t x = static_cast<uint64_t>(ceil(p * static_cast<double>(all)));
    return x < 1 ? 1 : x > all ? all : x;
}
__device__ __forceinline__ uint64_t u_border(float u, uint64_t kept) {
    if (kept == 0) return 1;
    if (u >= 1.0f) return kept;
    const uint64_t x = u > 0.0f ? static_cast<uint64_t>(floor(static_cast<double>(u) * static_cast<double>(kept))) : 0;  // (NaN: 0)
    return (x < kept - 1 ? x : kept - 1) + 1;
}

template <class LT>
__global__ __launch_bounds__(kThreads) void sample_collect_kernel(const SampleArgs a) {
    __shared__ SampleShared sh;
    __shared__ uint8_t s_wanted[kBins];
    __shared__ uint64_t s_list[kList];
    __shared__ uint32_t s_n, s_at;
    const int tid = threadIdx.x, row = blockIdx.y, chunk = blockIdx.x;
    const SamplePlan s = sample_plan(a, row);
    if (s.greedy) return;
    const SampleBins b = sample_bins(a, row, sh);
    if (tid == kBins - 1) {
        s_at = b.to_count;
        sh.to = b.to_weight;
    }
    if (tid == 0) s_n = 0;
    __syncthreads();
    const uint32_t all_count = s_at;
    uint64_t all_lo = sh.to, all_hi = sh.to;
    __syncthreads();
    bool wanted = false;
    if (s.by_count) {
        const uint32_t k = static_cast<uint32_t>(s.k);
        wanted = b.to_count - b.count < k;  // the bins that any of the first k are in
    } else {
        // The sums after each rule, as far as the bins say: between lo and hi.
        if (s.k > 0 && static_cast<uint32_t>(s.k) < all_count) {
            const BinAt c = bin_of_count(b, s.k, sh), w = bin_at(b, c.bin, sh);
            const bool whole = c.to == static_cast<uint64_t>(s.k);
            wanted |= tid == c.bin && !whole;
            all_lo = whole ? w.to : w.before;
            all_hi = w.to;
        }
        uint64_t lo = all_lo, hi = all_hi;
        if (s.p < 1.0) {
            lo = all_lo ? p_border(s.p, all_lo) : 1;
            const BinAt x = bin_of_weight(b, lo, sh), y = bin_of_weight(b, p_border(s.p, all_hi), sh);
            wanted |= tid >= x.bin && tid <= y.bin;
            hi = y.to < all_hi ? y.to : all_hi;
        }
        if (s.min_z < s.z_limit) {
            const BinAt m = bin_at(b, s.bin(s.min_z), sh);
            wanted |= tid == m.bin && m.before < hi;
            lo = m.before < lo ? m.before : lo;
            hi = m.to < hi ? m.to : hi;
        }
        const float u = ldg(a.u + row);
        const BinAt x = bin_of_weight(b, u_border(u, lo), sh), y = bin_of_weight(b, u_border(u, hi), sh);
        wanted |= tid >= x.bin && tid <= y.bin;
    }
    s_wanted[tid] = wanted;
    __syncthreads();
    each_logit<LT>(a, row, chunk * a.chunk, min(a.V, (chunk + 1) * a.chunk), tid, [&](uint32_t key, int i) {
        const double z = s.z(key);
        if (!s.counts(key, z) || !s_wanted[s.bin(z)]) return;
        const uint32_t n = atomicAdd(&s_n, 1u);
        if (n < kList) s_list[n] = place_of(key, i);
    });
    __syncthreads();
    SampleRow* w = a.rows + row;
    if (tid == 0) s_at = s_n ? atomicAdd(&w->listed, s_n) : 0;
    __syncthreads();
    const uint32_t n = s_n < kList ? s_n : kList, at = s_at;
    for (uint32_t i = tid; i < n; i += kThreads)
        if (at + i < kList) stg(&w->list[at + i], s_list[i]);
}

// Tokens of the bins lo .. hi, in front of which the weights add up to `before`.
struct Segment {
    int lo, hi;
    uint64_t before;
};
struct Found {
    uint64_t to;  // the running sum with the token
    int index;
};

// The collected tokens in order, with the running sums of their weights.
struct Sorted {
    const SamplePlan& s;
    SampleShared& sh;
    const uint64_t *place, *sum;  // [n] in LDS
    int n;
    __device__ __forceinline__ int bin(int i) const { return s.bin(s.z(place_key(place[i]))); }
    // position of the segment's first token
    __device__ __forceinline__ int start(const Segment& g) const {
        if (threadIdx.x == 0) sh.at = n;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += kThreads)
            if (bin(i) >= g.lo && (i == 0 || bin(i - 1) < g.lo)) sh.at = i;
        __syncthreads();
        const int r = sh.at;
        __syncthreads();
        return r;
    }
    __device__ __forceinline__ uint64_t until(int i) const { return i > 0 ? sum[i - 1] : 0; }
    // the running sum with the segment's j-th token (from 1)
    __device__ __forceinline__ uint64_t nth(const Segment& g, uint64_t j) const {
        const int first = start(g), i = first + static_cast<int>(j);
        return g.before + until(i < n ? i : n) - until(first);
    }
    // the first token with which the running sum reaches x
    __device__ __forceinline__ Found reach(const Segment& g, uint64_t x) const {
        const uint64_t base = until(start(g));
        if (threadIdx.x == 0) {
            sh.at = 0;
            sh.to = g.before;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const int b = bin(i);
            if (b < g.lo || b > g.hi) continue;
            const uint64_t to = g.before + sum[i] - base, before = g.before + until(i) - base;
            if (to >= x && before < x) {
                sh.at = place_index(place[i]);
                sh.to = to;
            }
        }
        __syncthreads();
        const Found r{sh.to, sh.at};
        __syncthreads();
        return r;
    }
    // the running sum with the segment's last token of z <= z_max
    __device__ __forceinline__ uint64_t within(const Segment& g, double z_max) const {
        const uint64_t base = until(start(g));
        if (threadIdx.x == 0) sh.to = g.before;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const double z = s.z(place_key(place[i]));
            const int b = s.bin(z);
            if (b < g.lo || b > g.hi || z > z_max) continue;
            const int nb = i + 1 < n ? bin(i + 1) : kBins;
            if (nb > g.hi || s.z(place_key(place[i + 1])) > z_max) sh.to = g.before + sum[i] - base;
        }
        __syncthreads();
        const uint64_t r = sh.to;
        __syncthreads();
        return r;
    }
};

// The same answers from passes over the row, where a segment holds more tokens than the list: the place is found ten bits at a
// time by histograms of what the segment's tokens weigh (or count).
template <class LT>
struct Searched {
    const SampleArgs& a;
    const SamplePlan& s;
    SampleShared& sh;
    uint64_t* hist;  // [kBins] in LDS
    int row;
    template <class F>
    __device__ __forceinline__ void each(const Segment& g, F f) const {
        each_logit<LT>(a, row, 0, a.V, threadIdx.x, [&](uint32_t key, int i) {
            const double z = s.z(key);
            if (!s.counts(key, z)) return;
            const int b = s.bin(z);
            if (b >= g.lo && b <= g.hi) f(key, i, z);
        });
    }
    __device__ __forceinline__ uint64_t total(const Segment& g, uint64_t last, double z_max) const {
        uint64_t w = 0;
        each(g, [&](uint32_t key, int i, double z) {
            if (place_of(key, i) <= last && z <= z_max) w += weight_of(z);
        });
        w = scan_threads(w, sh.part);
        if (threadIdx.x == kThreads - 1) sh.to = w;
        __syncthreads();
        const uint64_t r = g.before + sh.to;
        __syncthreads();
        return r;
    }
    // the place of the first token with which the sum from the segment's start reaches x (1 <= x)
    __device__ __forceinline__ uint64_t place(const Segment& g, uint64_t x, bool by_count) const {
        uint64_t lo = 0;
        for (int shift = 32 + kIdxBits - 10;; shift = shift > 10 ? shift - 10 : 0) {
            hist[threadIdx.x] = 0;
            __syncthreads();
            each(g, [&](uint32_t key, int i, double z) {
                const uint64_t d = place_of(key, i) - lo;
                if (place_of(key, i) >= lo && d >> shift < kBins)
                    atomicAdd(reinterpret_cast<unsigned long long*>(&hist[d >> shift]), by_count ? 1ull : weight_of(z));
            });
            __syncthreads();
            const uint64_t own = hist[threadIdx.x], to = scan_threads(own, sh.part);
            if (threadIdx.x == 0) {
                sh.at = kBins - 1;
                sh.before = 0;
            }
            __syncthreads();
            if (to >= x && to - own < x) {
                sh.at = threadIdx.x;
                sh.before = to - own;
            }
            __syncthreads();
            lo += static_cast<uint64_t>(sh.at) << shift;
            x -= sh.before;
            __syncthreads();
            if (shift == 0) return lo;
        }
    }
    __device__ __forceinline__ uint64_t nth(const Segment& g, uint64_t j) const {
        return total(g, place(g, j, true), __builtin_inf());
    }
    __device__ __forceinline__ Found reach(const Segment& g, uint64_t x) const {
        const uint64_t c = place(g, x - g.before, false);
        return {total(g, c, __builtin_inf()), place_index(c)};
    }
    __device__ __forceinline__ uint64_t within(const Segment& g, double z_max) const { return total(g, ~uint64_t(0), z_max); }
};

template <class Q>
__device__ __forceinline__ int sample_decide(const SamplePlan& s, const SampleBins& b, float u, const Q& q, SampleShared& sh) {
    if (threadIdx.x == kBins - 1) {
        sh.to = b.to_weight;
        sh.at = static_cast<int>(b.to_count);
    }
    __syncthreads();
    uint64_t kept = sh.to;
    const int count = sh.at;
    __syncthreads();
    Segment g{0, kBins - 1, 0};  // by_count: everything that was collected
    if (s.by_count) {
        const int k = s.k < count ? s.k : count;
        const BinAt c = bin_of_count(b, k, sh);
        g.hi = c.bin;
        kept = q.nth(g, k);
    } else if (s.k > 0 && s.k < count) {
        const BinAt c = bin_of_count(b, s.k, sh), w = bin_at(b, c.bin, sh);
        if (c.to == static_cast<uint64_t>(s.k)) kept = w.to;
        else kept = q.nth(Segment{c.bin, c.bin, w.before}, s.k - c.before);
    }
    auto segment = [&](uint64_t x) {  // where the running sum reaches x
        if (s.by_count) return g;
        const BinAt w = bin_of_weight(b, x, sh);
        return Segment{w.bin, w.bin, w.before};
    };
    if (s.p < 1.0) {
        const uint64_t x = p_border(s.p, kept);
        kept = q.reach(segment(x), x).to;
    }
    if (s.min_z < s.z_limit) {
        Segment m = g;
        if (!s.by_count) {
            const BinAt w = bin_at(b, s.bin(s.min_z), sh);
            m = Segment{w.bin, w.bin, w.before};
        }
        if (m.before < kept) {
            const uint64_t most = q.within(m, s.min_z);
            kept = most < kept ? most : kept;
        }
    }
    const uint64_t x = u_border(u, kept);
    return q.reach(segment(x), x).index;
}

template <class LT>
__global__ __launch_bounds__(kThreads) void sample_decide_kernel(const SampleArgs a) {
    __shared__ SampleShared sh;
    __shared__ uint64_t s_place[kList], s_sum[kList];
    const int tid = threadIdx.x, row = blockIdx.x;
    const SamplePlan s = sample_plan(a, row);
    if (s.greedy) {
        if (tid == 0) stg(a.tokens + row, s.first);
        return;
    }
    const SampleBins b = sample_bins(a, row, sh);
    const SampleRow* w = a.rows + row;
    const uint32_t listed = ldg(&w->listed);
    const float u = ldg(a.u + row);
    int token;
    if (listed <= kList) {
        const int n = static_cast<int>(listed);
        int size = 2;
        while (size < n) size <<= 1;
        for (int i = tid; i < size; i += kThreads) s_place[i] = i < n ? ldg(&w->list[i]) : ~uint64_t(0);
        __syncthreads();
        for (int k = 2; k <= size; k <<= 1)  // bitonic
            for (int j = k >> 1; j > 0; j >>= 1) {
                for (int t = tid; t < size / 2; t += kThreads) {
                    const int i = 2 * t - (t & (j - 1)), o = i + j;
                    const uint64_t x = s_place[i], y = s_place[o];
                    if ((x > y) == ((i & k) == 0)) {
                        s_place[i] = y;
                        s_place[o] = x;
                    }
                }
                __syncthreads();
            }
        uint64_t base = 0;
        for (int i0 = 0; i0 < n; i0 += kThreads) {  // running sums
            const int i = i0 + tid;
            const uint64_t v = scan_threads(i < n ? weight_of(s.z(place_key(s_place[i]))) : uint64_t(0), sh.part) + base;
            if (i < n) s_sum[i] = v;
            if (tid == kThreads - 1) sh.to = v;
            __syncthreads();
            base = sh.to;
            __syncthreads();
        }
        token = sample_decide(s, b, u, Sorted{s, sh, s_place, s_sum, n}, sh);
    } else {
        token = sample_decide(s, b, u, Searched<LT>{a, s, sh, s_place, row}, sh);
    }
    if (tid == 0) stg(a.tokens + row, token);
}

// Chunks of a row: as many as give about two workgroups to a CU, each of at least one piece a thread.
static int sample_chunks(int64_t B, int64_t V) {
    const int64_t most = ceil_div64(V, kChunk), want = ceil_div64(512, B);
    return static_cast<int>(want < most ? want : most);
}

}  // namespace soi

using namespace soi;

extern "C" size_t soi_sample_tokens_workspace_bytes(int64_t batch, int64_t vocab) {
    if (batch < 1 || batch > 65535 || vocab < 1 || vocab > (1 << 19)) return 0;
    return static_cast<size_t>(batch) * (sizeof(SampleRow) + sample_chunks(batch, vocab) * sizeof(SamplePart));
}

extern "C" int soi_sample_tokens(const void* logits, int logits_f32, int64_t stride, int64_t batch, int64_t vocab, const float* u,
                                 const float* temperature, float temperature_all, const int32_t* top_k, int32_t top_k_all,
                                 const float* top_p, float top_p_all, const float* min_p, float min_p_all, int32_t* tokens,
                                 void* workspace, size_t workspace_bytes, void* stream) {
    const char* what = "soi_sample_tokens";
    SOI_REQUIRE(batch >= 0 && batch <= 65535, "%s: the number of rows must be in [0, 65535], got %lld", what, (long long)batch);
    SOI_REQUIRE(vocab >= 1 && vocab <= (1 << 19), "%s: a row must hold 1 to 524288 logits, got %lld", what, (long long)vocab);
    SOI_REQUIRE(stride >= vocab || batch <= 1, "%s: rows overlap: stride %lld below %lld", what, (long long)stride,
                (long long)vocab);
    if (batch == 0) return SOI_OK;
    SOI_REQUIRE(logits && u && tokens, "%s: null pointer", what);
    const size_t need = soi_sample_tokens_workspace_bytes(batch, vocab);
    if (!workspace || workspace_bytes < need || !aligned16(workspace)) {
        set_last_error("%s: workspace of %zu bytes (16-byte aligned) needed, got %zu", what, need, workspace_bytes);
        return SOI_ERR_WORKSPACE;
    }
    SampleArgs a{logits, stride, u, temperature, top_p, min_p, top_k, temperature_all, top_p_all, min_p_all, top_k_all, tokens,
                 static_cast<SampleRow*>(workspace), nullptr, static_cast<int>(batch), static_cast<int>(vocab), 0, 0};
    a.parts = reinterpret_cast<SamplePart*>(a.rows + batch);
    a.chunks = sample_chunks(batch, vocab);
    a.chunk = static_cast<int>(ceil_div64(ceil_div64(vocab, a.chunks), kPiece) * kPiece);
    a.chunks = static_cast<int>(ceil_div64(vocab, a.chunk));
    const dim3 grid(static_cast<unsigned>(a.chunks), static_cast<unsigned>(batch)), block(kThreads);
    hipStream_t st = as_stream(stream);
    const bool draws = temperature || temperature_all > 0.0f;  // otherwise every row's token is its largest
    auto launch = [&](auto type) {
        using LT = decltype(type);
        hipLaunchKernelGGL(sample_extremes_kernel<LT>, grid, block, 0, st, a);
        if (draws) {
            hipLaunchKernelGGL(sample_bins_kernel<LT>, grid, block, 0, st, a);
            hipLaunchKernelGGL(sample_collect_kernel<LT>, grid, block, 0, st, a);
        }
        hipLaunchKernelGGL(sample_decide_kernel<LT>, dim3(static_cast<unsigned>(batch)), block, 0, st, a);
    };
    if (logits_f32) launch(float{});
    else launch(uint16_t{});
    return launch_status(what);
}
