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
// can lie in; only the tokens of those few bins are collected (a few hundred, in flat rows a thousand or two), and sorted, or
// searched by radix passes in LDS. The bins' width follows from the row's lowest logits, a few far below the others left aside:
// with the smallest logit, one of -1e4 or -infinity in a row of 151936 of deviation 0.35 spread its tokens over a tenth of the
// bins, and it took 200 to 505 us instead of 26 to 28.
// Rows with a top-k of up to kMostK need no weights before that: the bins down to the k-th token are counted and collected whole,
// and of the other tokens only those are looked at that reach the smallest of the first launch's threads' largest logits (one a
// thread does, which are at least k).
// Bins that hold more than kList tokens (many equal logits, or nearly so beside others far below) are searched by the same passes
// over the row, by one workgroup.
//
// Four launches: largest and smallest logit, bins, collect, decide. Bound by latency for one row (151936 binary16 logits: 4.6, 4.3,
// 7.0 and 9.9 us), for many by the three passes over the logits and the binary64 exponentials and LDS atomics of the second (200
// rows, each with its own settings: 18, 37, 32 and 20 us; one pass at a large copy's rate is 12 us). The collected tokens of a row
// are sorted, by one wave where they are up to 256 (one row 29 -> 23 us beside radix passes for all), by the workgroup up to 2048
// (the last launch of the 200 rows 34 -> 17 us).
#include "soi_host.h"
#include "soi_device.h"

#include <type_traits>

namespace soi {

constexpr int kBins = 1024, kThreads = 1024, kList = 4096, kMostK = 2048, kPiece = 8, kChunk = kThreads * kPiece;
constexpr int kBinThreads = 512;                  // of the bins' workgroups: rows differ in work, and half as much each evens out (40 -> 37 us)
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
    uint32_t low;    // key that stands for its smallest numbers: the median of its waves' smallest
    uint32_t bound;  // key of the smallest of the threads' largest: one token a thread reaches it
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
    int bin_chunk;            // logits of a workgroup of the bins
    int threads;              // of a row's that have a logit
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

// Eight logits i .. i + 7 (those past the row: -infinity).
struct Piece {
    float v[kPiece];
};
template <class LT>
__device__ __forceinline__ Piece load_piece(const SampleArgs& a, int row, int i) {
    const LT* p = static_cast<const LT*>(a.logits) + row * a.stride + i;
    Piece x;
    if (i + kPiece <= a.V) {
        // (lanes copied to scalars first: a bit cast of a vector's lane was compiled as one of lane 0)
        if constexpr (sizeof(LT) == 2) {
            const u32x4 r = ldg_any(p);
            const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int e = 0; e < kPiece; ++e) x.v[e] = f16_bits_to_f32(static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1))));
        } else {
            const u32x4 r0 = ldg_any(p), r1 = ldg_any(p + 4);
            const uint32_t w[kPiece] = {r0.x, r0.y, r0.z, r0.w, r1.x, r1.y, r1.z, r1.w};
#pragma unroll
            for (int e = 0; e < kPiece; ++e) x.v[e] = __builtin_bit_cast(float, w[e]);
        }
        return x;
    }
#pragma unroll
    for (int e = 0; e < kPiece; ++e) {
        x.v[e] = -__builtin_inff();
        if (i + e < a.V) {
            if constexpr (sizeof(LT) == 2) x.v[e] = f16_bits_to_f32(ldg(p + e));
            else x.v[e] = ldg(p + e);
        }
    }
    return x;
}

// Calls f(logit, index) for the logits of [lo, hi) that thread `tid` of NT has (and for -infinity past the row's end);
// first: its first piece, requested before.
template <class LT, int NT = kThreads, class F>
__device__ __forceinline__ void each_logit(const SampleArgs& a, int row, int lo, int hi, int tid, Piece first, F f) {
    for (int i = lo + tid * kPiece; i < hi; i += NT * kPiece) {
        const Piece x = first;
        if (i + NT * kPiece < hi) first = load_piece<LT>(a, row, i + NT * kPiece);
#pragma unroll
        for (int e = 0; e < kPiece; ++e) f(x.v[e], i + e);
    }
}

// Inclusive sums over a wave's lanes, and the largest of them in every lane.
template <int CTRL, int ROWS, class N>
__device__ __forceinline__ N lane_move(N v) {  // zeros where nothing comes from
    if constexpr (sizeof(N) == 8) {
        const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, false);
        const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), CTRL, ROWS, 0xf, false);
        return static_cast<uint64_t>(hi) << 32 | lo;
    } else {
        return static_cast<N>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, false));
    }
}
template <class N, class Op>
__device__ __forceinline__ N wave_run(N v, Op op) {
    v = op(v, lane_move<0x111, 0xf>(v));
    v = op(v, lane_move<0x112, 0xf>(v));
    v = op(v, lane_move<0x114, 0xf>(v));
    v = op(v, lane_move<0x118, 0xf>(v));
    v = op(v, lane_move<0x142, 0xa>(v));
    v = op(v, lane_move<0x143, 0xc>(v));
    return v;
}
// The largest of the lanes, valid in lane 63.
template <class N>
__device__ __forceinline__ N wave_top(N v) {
    return wave_run(v, [](N a, N b) { return a > b ? a : b; });
}

// The median (of an even number: the lower one) of the first n lanes' keys, 1 <= n <= 16, but for their last four bits.
__device__ __forceinline__ uint32_t median_key(uint32_t key, int n) {
    constexpr int kMost = 16;
    const int lane = threadIdx.x & 63;
    const uint32_t mine = lane < n ? (key & ~(kMost - 1u)) | static_cast<uint32_t>(lane) : 0xffffffffu;
    int rank = 0;
#pragma unroll
    for (int j = 0; j < kMost; ++j) rank += static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(mine), j)) < mine;
    const int at = __builtin_ctzll(ballot(rank == (n - 1) / 2));
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(mine), at)) & ~(kMost - 1u);
}

template <class LT>
__global__ __launch_bounds__(kThreads) void sample_extremes_kernel(const SampleArgs a) {
    __shared__ uint64_t s_top[kThreads / kWave];
    __shared__ uint32_t s_low[kThreads / kWave], s_bound[kThreads / kWave];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.y, chunk = blockIdx.x;
    if (chunk == 0) {
        SampleRow* w = a.rows + row;
        stg(&w->weight[tid], uint64_t(0));
        stg(&w->count[tid], 0u);
        if (tid == 0) stg(&w->listed, 0u);
    }
    // A thread keeps its largest and smallest number (NaN aside), the piece that the largest came with first, and the largest
    // pattern without its sign, which tells whether there is a NaN. The index is looked up at the end by those that have the wave's.
    const int lo = chunk * a.chunk, hi = min(a.V, lo + a.chunk);
    float best = -__builtin_inff(), least = __builtin_inff();
    uint32_t pattern = 0;
    int from = lo + tid * kPiece, at = from;
    Piece x;  // the piece at `at`
    {
        Piece next = load_piece<LT>(a, row, from);
        for (int i = from; i < hi; i += kChunk) {
            x = next;
            at = i;
            if (i + kChunk < hi) next = load_piece<LT>(a, row, i + kChunk);
            float most = x.v[0];
#pragma unroll
            for (int e = 1; e < kPiece; ++e) most = fmaxf(most, x.v[e]);
#pragma unroll
            for (int e = 0; e < kPiece; ++e) {
                if (i + e < a.V) least = fminf(least, x.v[e]);
                const uint32_t m = __builtin_bit_cast(uint32_t, x.v[e]) & 0x7fffffffu;
                pattern = m > pattern ? m : pattern;
            }
            from = most > best ? i : from;
            best = most > best ? most : best;
        }
    }
    if (pattern > 0x7f800000u) {  // the first NaN is this thread's largest
        best = __builtin_nanf("");
        for (int i = lo + tid * kPiece; i < hi; i += kChunk) {
            x = load_piece<LT>(a, row, i);
            bool here = false;
#pragma unroll
            for (int e = 0; e < kPiece; ++e) here |= x.v[e] != x.v[e];
            from = at = i;
            if (here) break;
        }
    }
    const uint32_t best_key = key_of(best);
    uint32_t low = least == -__builtin_inff() ? kKeyNegInf : key_of(least);
    const bool any = lo + tid * kPiece < hi;
    const uint32_t top_key = __builtin_amdgcn_readlane(static_cast<int>(wave_top(any ? best_key : 0u)), 63);
    uint64_t top = 0;
    if (any && best_key == top_key) {
        if (from != at) x = load_piece<LT>(a, row, from);
        int i = a.V;
#pragma unroll
        for (int e = kPiece - 1; e >= 0; --e) i = from + e < a.V && key_of(x.v[e]) == top_key ? from + e : i;
        top = static_cast<uint64_t>(top_key) << 32 | ~static_cast<uint32_t>(i);
    }
    uint32_t bound = any ? best_key : 0xffffffffu;
    bound = ~wave_top(~bound);
    top = wave_top(top);
    low = ~wave_top(~low);
    if (lane == 63) {
        s_top[wave] = top;
        s_low[wave] = low;
        s_bound[wave] = bound;
    }
    __syncthreads();
    if (wave == 0) {
        top = wave_top(lane < kThreads / kWave ? s_top[lane] : uint64_t(0));
        low = median_key(s_low[lane & (kThreads / kWave - 1)], min(kThreads / kWave, (hi - lo + kWave * kPiece - 1) / (kWave * kPiece)));
        bound = ~wave_top(lane < kThreads / kWave ? ~s_bound[lane] : 0u);
    }
    if (tid == 63) {
        SamplePart* p = a.parts + static_cast<int64_t>(row) * a.chunks + chunk;
        stg(&p->top, top);
        stg(&p->low, low);
        stg(&p->bound, bound);
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
    __device__ __forceinline__ double z(float v) const { return (max - static_cast<double>(v)) * inv_t; }
    __device__ __forceinline__ bool counts(double z) const { return z <= z_limit; }  // (-infinity: z is infinite or NaN)
    __device__ __forceinline__ int bin(double z) const {  // of a z that counts
        return static_cast<int>(fmin(z * per_z, kBins - 1.0));
    }
};

__device__ __forceinline__ SamplePlan sample_plan(const SampleArgs& a, int row) {
    const int lane = threadIdx.x & 63;
    const SamplePart* p = a.parts + static_cast<int64_t>(row) * a.chunks;  // (the lanes' chunks)
    uint64_t top = 0;
    uint32_t low = 0xffffffffu, bound = 0xffffffffu;
    static_assert((1 << 19) <= kChunk * kWave, "a lane for each chunk");
    if (lane < a.chunks) {
        top = ldg(&p[lane].top);
        low = ldg(&p[lane].low);
        bound = ldg(&p[lane].bound);
    }
    const auto last = [](uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 63)); };
    top = wave_top(top);
    top = static_cast<uint64_t>(last(static_cast<uint32_t>(top >> 32))) << 32 | last(static_cast<uint32_t>(top));
    bound = ~last(wave_top(~bound));
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
    s.p = tp < 1.0f ? static_cast<double>(fmaxf(tp, 0.0f)) : 1.0;  // (NaN: 1; a negative sum is no whole number of p_border's)
    s.k = k > 0 ? k : 0;
    s.min_z = mp > 0.0f ? (mp < 1.0f ? -log(static_cast<double>(mp)) : 0.0) : __builtin_inf();
    // without top-p, what min-p drops does not count for anything
    s.z_limit = s.p == 1.0 && s.min_z < kZMost ? s.min_z : kZMost;
    s.by_count = s.k > 0 && s.k <= kMostK;
    if (s.by_count && s.k <= a.threads && bound > kKeyNegInf) {  // as many tokens as threads are at least `bound`
        const double z = s.z(value_of(bound));
        s.z_limit = z < s.z_limit ? z : s.z_limit;
    }
    // The bins reach to the lowest of the chunks' numbers that is at most four times as far from the largest as is usual among
    // them (their mean on the float's pattern, which is one of logarithms): a few logits far below the rest (masks of -1e4 or
    // -infinity) leave the others their bins.
    const double far = lane < a.chunks && low > kKeyNegInf ? s.z(value_of(low)) : 1e300;
    const uint32_t base = __builtin_bit_cast(uint32_t, 0.01f);
    const uint32_t log_far = __builtin_bit_cast(uint32_t, fminf(fmaxf(static_cast<float>(far), 0.01f), 128.0f)) - base;
    const uint32_t logs = last(wave_run(lane < a.chunks ? log_far >> 3 : 0u, [](uint32_t v, uint32_t w) { return v + w; }));
    const float usual = __builtin_bit_cast(float, base + (logs / static_cast<uint32_t>(a.chunks) << 3));
    const uint32_t lowest = ~last(wave_top(static_cast<float>(far) <= 4.0f * usual ? ~low : 0u));
    double span = s.z_limit;
    if (lowest < kKeyInf) {
        const double most = s.z(value_of(lowest));
        span = most < span ? most : span;
    }
    s.per_z = span > 1e-290 ? kBins / span : 0.0;
    for (double* d : {&s.max, &s.inv_t, &s.z_limit, &s.per_z, &s.min_z, &s.p}) {  // to scalar registers
        const uint64_t v = __builtin_bit_cast(uint64_t, *d);
        const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<int>(v)), hi = __builtin_amdgcn_readfirstlane(static_cast<int>(v >> 32));
        *d = __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
    }
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
__global__ __launch_bounds__(kBinThreads) void sample_bins_kernel(const SampleArgs a) {
    __shared__ uint64_t s_weight[kBins];
    __shared__ uint32_t s_count[kBins];
    const int tid = threadIdx.x, row = blockIdx.y, lo = static_cast<int>(blockIdx.x) * a.bin_chunk, hi = min(a.V, lo + a.bin_chunk);
    const Piece first = load_piece<LT>(a, row, lo + tid * kPiece);
#pragma unroll
    for (int i = tid; i < kBins; i += kBinThreads) {
        s_weight[i] = 0;
        s_count[i] = 0;
    }
    const SamplePlan s = sample_plan(a, row);
    if (s.greedy) return;
    __syncthreads();
    auto pass = [&](auto WEIGHTS, auto COUNTS) {
        each_logit<LT, kBinThreads>(a, row, lo, hi, tid, first, [&](float v, int) {
            const double z = s.z(v);
            if (!s.counts(z)) return;
            const int b = s.bin(z);
            if (WEIGHTS) atomicAdd(reinterpret_cast<unsigned long long*>(&s_weight[b]), weight_of(z));
            if (COUNTS) atomicAdd(&s_count[b], 1u);
        });
    };
    if (s.by_count) pass(std::false_type{}, std::true_type{});
    else if (s.k > 0) pass(std::true_type{}, std::true_type{});
    else pass(std::true_type{}, std::false_type{});
    __syncthreads();
    SampleRow* w = a.rows + row;
#pragma unroll
    for (int i = tid; i < kBins; i += kBinThreads) {
        if (s_weight[i]) atomicAdd(reinterpret_cast<unsigned long long*>(&w->weight[i]), s_weight[i]);
        if (s_count[i]) atomicAdd(&w->count[i], s_count[i]);
    }
}

// Inclusive sums over the workgroup's threads; s_part: one number a wave. Every thread may call it again at once.
template <class N>
__device__ __forceinline__ N scan_threads(N v, N* s_part) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    v = wave_run(v, [](N a, N b) { return a + b; });
    if (lane == 63) s_part[wave] = v;
    __syncthreads();
    // the waves' sums in the first lanes: their running sum, of which this wave takes its own
    const N part = wave_run(lane < kThreads / kWave ? s_part[lane] : N(0), [](N a, N b) { return a + b; });
    N base;
    if constexpr (sizeof(N) == 8) {
        const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(part), wave > 0 ? wave - 1 : 0);
        const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(part >> 32), wave > 0 ? wave - 1 : 0);
        base = static_cast<uint64_t>(hi) << 32 | lo;
    } else {
        base = __builtin_amdgcn_readlane(static_cast<int>(part), wave > 0 ? wave - 1 : 0);
    }
    __syncthreads();
    return v + (wave > 0 ? base : N(0));
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
    unsigned long long least, most;
    int at, n;
};

__device__ __forceinline__ void sum_bins(SampleBins& b, SampleShared& sh) {
    b.to_weight = scan_threads(b.weight, sh.part);
    b.to_count = scan_threads(b.count, sh.part32);
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
    __shared__ int s_lo, s_hi;
    const int tid = threadIdx.x, row = blockIdx.y, chunk = blockIdx.x, lo_i = chunk * a.chunk, hi_i = min(a.V, lo_i + a.chunk);
    SampleRow* w = a.rows + row;
    const Piece first = load_piece<LT>(a, row, lo_i + tid * kPiece);
    SampleBins b;
    b.weight = ldg(&w->weight[tid]);
    b.count = ldg(&w->count[tid]);
    const float u = ldg(a.u + row);
    const SamplePlan s = sample_plan(a, row);
    if (s.greedy) return;
    sum_bins(b, sh);
    if (tid == kBins - 1) {
        s_at = b.to_count;
        sh.to = b.to_weight;
    }
    if (tid == 0) {
        s_n = 0;
        s_lo = kBins;
        s_hi = -1;
    }
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
        const BinAt x = bin_of_weight(b, u_border(u, lo), sh), y = bin_of_weight(b, u_border(u, hi), sh);
        wanted |= tid >= x.bin && tid <= y.bin;
    }
    s_wanted[tid] = wanted;
    {  // the first and the last of them: most tokens are past it
        const uint64_t any = ballot(wanted);
        if (any && (tid & 63) == 0) {
            atomicMin(&s_lo, tid + __builtin_ctzll(any));
            atomicMax(&s_hi, tid + 63 - __builtin_clzll(any));
        }
    }
    __syncthreads();
    const int b_lo = s_lo, b_hi = s_hi;
    each_logit<LT>(a, row, lo_i, hi_i, tid, first, [&](float v, int i) {
        const double z = s.z(v);
        if (!s.counts(z)) return;
        const int bin = s.bin(z);
        if (bin < b_lo || bin > b_hi || !s_wanted[bin]) return;
        const uint32_t n = atomicAdd(&s_n, 1u);
        if (n < kList) s_list[n] = place_of(key_of(v), i);
    });
    __syncthreads();
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

// The collected tokens, or, where a segment holds more of them than the list, the row's.
struct Listed {
    const SamplePlan& s;
    const uint64_t *place, *weight;  // [n] in LDS
    int n;
    template <class F>
    __device__ __forceinline__ void each(const Segment& g, F f) const {
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const double z = s.z(value_of(place_key(place[i])));
            const int b = s.bin(z);
            if (b >= g.lo && b <= g.hi) f(place[i], z, [&] { return weight[i]; });
        }
    }
};
template <class LT>
struct InRow {
    const SampleArgs& a;
    const SamplePlan& s;
    int row;
    template <class F>
    __device__ __forceinline__ void each(const Segment& g, F f) const {
        each_logit<LT>(a, row, 0, a.V, threadIdx.x, load_piece<LT>(a, row, threadIdx.x * kPiece), [&](float v, int i) {
            const double z = s.z(v);
            if (s.counts(z)) {
                const int b = s.bin(z);
                if (b >= g.lo && b <= g.hi) f(place_of(key_of(v), i), z, [&] { return weight_of(z); });
            }
            __builtin_amdgcn_sched_barrier(0);  // (eight logits at once would spill)
        });
    }
};

// Finds tokens of a segment: their place, ten bits at a time, by histograms of what the segment's tokens weigh and count, until
// one token is left where the sum crosses.
template <class Source>
struct Search {
    const Source& q;
    SampleShared& sh;
    uint64_t* hist;    // [kBins] in LDS
    uint32_t* counts;  // likewise
    // the first token with which the running sum (or, by_count, the number of tokens) of the segment reaches x >= 1
    __device__ __forceinline__ Found find(const Segment& g, uint64_t x, bool by_count) const {
        const int tid = threadIdx.x;
        // the segment's range of places
        uint64_t least = ~uint64_t(0), most = 0;
        q.each(g, [&](uint64_t c, double, auto) {
            least = c < least ? c : least;
            most = c > most ? c : most;
        });
        least = ~wave_top(~least);
        most = wave_top(most);
        if (tid == 0) {
            sh.least = ~0ull;
            sh.most = 0;
        }
        __syncthreads();
        if ((tid & 63) == 63) {
            atomicMin(&sh.least, least);
            atomicMax(&sh.most, most);
        }
        __syncthreads();
        uint64_t lo = sh.least, before = 0;
        const uint64_t range = sh.most >= lo ? sh.most - lo : 0;
        int shift = 0;
        while (range >> shift >= kBins) shift += 10;
        for (;; shift = shift > 10 ? shift - 10 : 0) {
            hist[tid] = 0;
            counts[tid] = 0;
            __syncthreads();
            q.each(g, [&](uint64_t c, double, auto weight) {
                const uint64_t d = (c - lo) >> shift;
                if (c < lo || d >= kBins) return;
                atomicAdd(reinterpret_cast<unsigned long long*>(&hist[d]), weight());
                atomicAdd(&counts[d], 1u);
            });
            __syncthreads();
            const uint64_t w = hist[tid], to_w = scan_threads(w, sh.part);
            const uint32_t n = counts[tid], to_n = scan_threads(n, sh.part32);
            const uint64_t own = by_count ? n : w, to = by_count ? to_n : to_w;
            if (tid == 0) {
                sh.at = kBins - 1;
                sh.before = sh.to = 0;
                sh.n = 0;
            }
            __syncthreads();
            if (to >= x && to - own < x) {
                sh.at = tid;
                sh.before = to_w - w;
                sh.to = to - own;
                sh.n = static_cast<int>(n);
            }
            __syncthreads();
            const uint64_t bin = static_cast<uint64_t>(sh.at);
            const int left = sh.n;
            before += sh.before;
            x -= sh.to;
            lo += bin << shift;
            __syncthreads();
            if (left <= 1 || shift == 0) break;
        }
        // the token itself: of the places lo .. lo + 2^shift - 1, of which one is taken
        if (tid == 0) {
            sh.at = 0;
            sh.to = 0;
        }
        __syncthreads();
        q.each(g, [&](uint64_t c, double, auto weight) {
            if (c < lo || (c - lo) >> shift) return;
            sh.at = place_index(c);
            sh.to = weight();
        });
        __syncthreads();
        const Found r{g.before + before + sh.to, sh.at};
        __syncthreads();
        return r;
    }
    // the running sum with the segment's last token of z <= z_max
    __device__ __forceinline__ uint64_t within(const Segment& g, double z_max) const {
        uint64_t w = 0;
        q.each(g, [&](uint64_t, double z, auto weight) {
            if (z <= z_max) w += weight();
        });
        w = scan_threads(w, sh.part);
        if (threadIdx.x == kThreads - 1) sh.to = w;
        __syncthreads();
        const uint64_t r = g.before + sh.to;
        __syncthreads();
        return r;
    }
};

// Up to kShort collected tokens: the first wave sorts them in registers, four a lane, and answers from their running sums.
constexpr int kShort = 4 * kWave;

// The value of lane (l ^ MASK).
template <int MASK>
__device__ __forceinline__ uint64_t other_lane(uint64_t v) {
    const uint32_t lo = __builtin_bit_cast(uint32_t, xor_lanes<MASK>(__builtin_bit_cast(float, static_cast<uint32_t>(v))));
    const uint32_t hi = __builtin_bit_cast(uint32_t, xor_lanes<MASK>(__builtin_bit_cast(float, static_cast<uint32_t>(v >> 32))));
    return static_cast<uint64_t>(hi) << 32 | lo;
}

// Bitonic steps from (K, J) on, of numbers 4 lane + e.
template <int K, int J>
__device__ __forceinline__ void sort_short(uint64_t (&x)[4], int lane) {
    if constexpr (J >= 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint64_t o = other_lane<J / 4>(x[e]);
            const bool least = ((lane & (J / 4)) == 0) == (((4 * lane + e) & K) == 0);
            x[e] = (x[e] < o) == least ? x[e] : o;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (e & J) continue;
            const uint64_t a = x[e], b = x[e + J];
            const bool swap = (a > b) == (((4 * lane + e) & K) == 0);
            x[e] = swap ? b : a;
            x[e + J] = swap ? a : b;
        }
    }
    if constexpr (J > 1) sort_short<K, J / 2>(x, lane);
    else if constexpr (K < kShort) sort_short<2 * K, K>(x, lane);
}

struct Short {
    const SamplePlan& s;
    SampleShared& sh;
    uint64_t place[4], sum[4];  // (of the first wave; past the last token: the largest place)
    int bin[4];
    __device__ __forceinline__ Short(const SamplePlan& s, SampleShared& sh, const uint64_t* list, int n) : s(s), sh(sh) {
        const int lane = threadIdx.x & 63;
        if (threadIdx.x >= kWave) return;
#pragma unroll
        for (int e = 0; e < 4; ++e) place[e] = 4 * lane + e < n ? list[4 * lane + e] : ~uint64_t(0);
        sort_short<2, 1>(place, lane);
        uint64_t w[4], mine = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool is = 4 * lane + e < n;
            const double z = s.z(value_of(place_key(place[e])));
            bin[e] = is ? s.bin(z) : kBins;
            w[e] = is ? weight_of(z) : 0;
            mine += w[e];
        }
        uint64_t run = wave_run(mine, [](uint64_t a, uint64_t b) { return a + b; }) - mine;
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] = run += w[e];
    }
    template <class F>
    __device__ __forceinline__ int how_many(F f) const {
        int n = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) n += __popcll(ballot(f(e)));
        return n;
    }
    static __device__ __forceinline__ uint64_t of_lane(uint64_t v, int lane) {
        const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(v), lane), hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane);
        return static_cast<uint64_t>(hi) << 32 | lo;
    }
    static __device__ __forceinline__ uint64_t at(const uint64_t (&x)[4], int i) {  // the i-th number
        const uint64_t a = i & 1 ? x[1] : x[0], b = i & 1 ? x[3] : x[2];
        return of_lane(i & 2 ? b : a, i >> 2);
    }
    __device__ __forceinline__ Found find(const Segment& g, uint64_t x, bool by_count) const {
        if (threadIdx.x < kWave) {
            const int first = how_many([&](int e) { return bin[e] < g.lo; });
            const uint64_t base = first ? at(sum, first - 1) : 0;
            int i = first + static_cast<int>(x) - 1;
            if (!by_count) i = how_many([&](int e) { return bin[e] < g.lo || (bin[e] < kBins && sum[e] - base < x); });
            i = i < kShort ? i : kShort - 1;
            const uint64_t to = g.before + at(sum, i) - base;
            const int index = place_index(at(place, i));
            if (threadIdx.x == 0) {
                sh.to = to;
                sh.at = index;
            }
        }
        __syncthreads();
        const Found r{sh.to, sh.at};
        __syncthreads();
        return r;
    }
    __device__ __forceinline__ uint64_t within(const Segment& g, double z_max) const {
        if (threadIdx.x < kWave) {
            const int first = how_many([&](int e) { return bin[e] < g.lo; });
            const int end = how_many([&](int e) { return bin[e] < g.lo || (bin[e] <= g.hi && s.z(value_of(place_key(place[e]))) <= z_max); });
            const uint64_t to = g.before + (end ? at(sum, end - 1) : 0) - (first ? at(sum, first - 1) : 0);
            if (threadIdx.x == 0) sh.to = to;
        }
        __syncthreads();
        const uint64_t r = sh.to;
        __syncthreads();
        return r;
    }
};

// Up to E tokens a thread: the workgroup sorts them (in registers and lanes, across waves through LDS), and every wave answers
// for itself from their running sums in LDS.
template <int E>
struct Sorted {
    static constexpr int kMost = E * kThreads;
    const SamplePlan& s;
    const uint64_t *place, *sum;  // [kMost] in LDS, in order; sums with the token
    int n;
    // bitonic steps from (K, J) on, of numbers E tid + e; buffer: 2 kMost numbers, of which each exchange takes a half
    template <int K, int J>
    static __device__ __forceinline__ void sort(uint64_t (&x)[E], uint64_t* buffer, int half) {
        const int tid = threadIdx.x;
        if constexpr (J >= E) {
            if constexpr (J / E >= kWave) {
#pragma unroll
                for (int e = 0; e < E; ++e) buffer[half * kMost + E * tid + e] = x[e];
                __syncthreads();
            }
#pragma unroll
            for (int e = 0; e < E; ++e) {
                uint64_t o;
                if constexpr (J / E >= kWave) o = buffer[half * kMost + ((E * tid + e) ^ J)];
                else o = other_lane<J / E>(x[e]);
                const bool least = ((E * tid + e) & J) == 0 ? ((E * tid + e) & K) == 0 : ((E * tid + e) & K) != 0;
                x[e] = (x[e] < o) == least ? x[e] : o;
            }
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (e & J) continue;
                const uint64_t a = x[e], b = x[e + J];
                const bool swap = (a > b) == (((E * tid + e) & K) == 0);
                x[e] = swap ? b : a;
                x[e + J] = swap ? a : b;
            }
        }
        constexpr int kNext = J / E >= kWave ? 1 : 0;  // (the other half: this one may still be read)
        if constexpr (J > 1) sort<K, J / 2>(x, buffer, half ^ kNext);
        else if constexpr (K < kMost) sort<2 * K, K>(x, buffer, half ^ kNext);
    }
    // list: x[e] of each thread in any order, ~0 past the last; buffer: 2 kMost numbers of LDS, sums: kMost
    __device__ __forceinline__ Sorted(const SamplePlan& s, SampleShared& sh, uint64_t (&x)[E], uint64_t* buffer, uint64_t* sums, int n)
        : s(s), place(buffer), sum(sums), n(n) {
        const int tid = threadIdx.x;
        sort<2, 1>(x, buffer, 0);
        uint64_t w[E], mine = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            w[e] = E * tid + e < n ? weight_of(s.z(value_of(place_key(x[e])))) : 0;
            mine += w[e];
        }
        uint64_t run = scan_threads(mine, sh.part) - mine;  // (its barriers are behind the last reads of the buffer)
#pragma unroll
        for (int e = 0; e < E; ++e) {
            buffer[E * tid + e] = x[e];
            sums[E * tid + e] = run += w[e];
        }
        __syncthreads();
    }
    __device__ __forceinline__ double z(int i) const { return s.z(value_of(place_key(place[i]))); }
    // how many tokens f(i) is true of; it is for the first ones and no other
    template <class F>
    __device__ __forceinline__ int how_many(F f) const {
        constexpr int kPart = kMost / kWave;
        const int lane = threadIdx.x & 63;
        const int i = kPart * lane + kPart - 1;
        const int part = __popcll(ballot(i < n && f(i)));
        const int j = kPart * part + lane;
        return kPart * part + __popcll(ballot(lane < kPart && j < n && f(j)));
    }
    __device__ __forceinline__ Found find(const Segment& g, uint64_t x, bool by_count) const {
        const int first = how_many([&](int i) { return s.bin(z(i)) < g.lo; });
        const uint64_t base = first ? sum[first - 1] : 0;
        int i = first + static_cast<int>(x) - 1;
        if (!by_count) i = how_many([&](int i) { return i < first || sum[i] - base < x; });
        i = i < n ? i : n - 1;
        return Found{g.before + sum[i] - base, place_index(place[i])};
    }
    __device__ __forceinline__ uint64_t within(const Segment& g, double z_max) const {
        const int first = how_many([&](int i) { return s.bin(z(i)) < g.lo; });
        const int end = how_many([&](int i) { return i < first || (s.bin(z(i)) <= g.hi && z(i) <= z_max); });
        return g.before + (end ? sum[end - 1] : 0) - (first ? sum[first - 1] : 0);
    }
};

template <class Q>
__device__ __forceinline__ int sample_decide(const SamplePlan& s, const SampleBins& b, float u, const Q& q, SampleShared& sh) {
    if (threadIdx.x == kBins - 1) {
        sh.to = b.to_weight;
        sh.at = static_cast<int>(b.to_count);
    }
    __syncthreads();
    uint64_t kept = sh.to;  // the sum of the weights that are left
    const int count = sh.at;
    __syncthreads();
    Segment all{0, kBins - 1, 0};  // by_count: everything that was collected
    int index = 0;
    for (int rule = 0; rule < 3; ++rule) {  // top-k, top-p, the draw
        Segment g = all;
        uint64_t x;
        if (rule == 0) {
            if (s.k == 0 || (!s.by_count && s.k >= count)) continue;
            x = s.k < count ? s.k : count;
            const BinAt c = bin_of_count(b, static_cast<uint32_t>(x), sh);
            if (s.by_count) {
                all.hi = g.hi = c.bin;
            } else {
                const BinAt w = bin_at(b, c.bin, sh);
                kept = w.to;
                if (c.to == x) continue;
                g = Segment{c.bin, c.bin, w.before};
                x -= c.before;
            }
        } else {
            if (rule == 1 && s.p >= 1.0) continue;
            if (rule == 2 && s.min_z < s.z_limit) {
                if (!s.by_count) {
                    const BinAt w = bin_at(b, s.bin(s.min_z), sh);
                    g = Segment{w.bin, w.bin, w.before};
                }
                if (g.before < kept) {
                    const uint64_t most = q.within(g, s.min_z);
                    kept = most < kept ? most : kept;
                }
            }
            x = rule == 1 ? p_border(s.p, kept) : u_border(u, kept);
            if (!s.by_count) {
                const BinAt w = bin_of_weight(b, x, sh);
                g = Segment{w.bin, w.bin, w.before};
            }
            x -= g.before;
        }
        const Found f = q.find(g, x, rule == 0);
        if (rule < 2) kept = f.to;
        index = f.index;
    }
    return index;
}

template <class LT>
__global__ __launch_bounds__(kThreads) void sample_decide_kernel(const SampleArgs a) {
    __shared__ SampleShared sh;
    __shared__ uint64_t s_place[kList], s_weight[kList], s_hist[kBins];
    __shared__ uint32_t s_count[kBins];
    const int tid = threadIdx.x, row = blockIdx.x;
    const SampleRow* w = a.rows + row;
    // everything is requested before the first of it is needed (what the launches before left out is whatever was there)
    SampleBins b;
    b.weight = ldg(&w->weight[tid]);
    b.count = ldg(&w->count[tid]);
    uint64_t place = ldg(&w->list[tid]);
    const uint32_t listed = ldg(&w->listed);
    const float u = ldg(a.u + row);
    __shared__ SamplePlan s_plan;  // (in scalar registers it spilled some)
    {
        const SamplePlan p = sample_plan(a, row);
        if (p.greedy) {
            if (tid == 0) stg(a.tokens + row, p.first);
            return;
        }
        if (tid == 0) s_plan = p;
    }
    sum_bins(b, sh);  // (its barriers are behind the plan's writes)
    const SamplePlan& s = s_plan;
    int token;
    if (listed <= kList) {
        const int n = static_cast<int>(listed);
        if (n > kShort && n <= kThreads) {
            uint64_t x[1] = {tid < n ? place : ~uint64_t(0)};
            token = sample_decide(s, b, u, Sorted<1>(s, sh, x, s_place, s_weight, n), sh);
        } else if (n > kThreads && n <= 2 * kThreads) {
            uint64_t x[2] = {place, tid + kThreads < n ? ldg(&w->list[tid + kThreads]) : ~uint64_t(0)};
            token = sample_decide(s, b, u, Sorted<2>(s, sh, x, s_place, s_weight, n), sh);
        } else {
            for (int i = tid; i < n; i += kThreads) {
                if (i >= kThreads) place = ldg(&w->list[i]);
                s_place[i] = place;
                s_weight[i] = weight_of(s.z(value_of(place_key(place))));
            }
            __syncthreads();
            if (n <= kShort) {
                token = sample_decide(s, b, u, Short(s, sh, s_place, n), sh);
            } else {
                const Listed q{s, s_place, s_weight, n};
                token = sample_decide(s, b, u, Search<Listed>{q, sh, s_hist, s_count}, sh);
            }
        }
    } else {
        const InRow<LT> q{a, s, row};
        token = sample_decide(s, b, u, Search<InRow<LT>>{q, sh, s_hist, s_count}, sh);
    }
    if (tid == 0) stg(a.tokens + row, token);
}

// Chunks of a row: as many as give four workgroups of 1024 threads to a CU, two at a time, each of at least one piece a thread
// where the row allows it. 200 rows of 151936 fp16 logits, by workgroups to a CU, extremes + bins + collect: 2: 19 + 52 + 35 us
// (rows differ in how many of their weights count, and one round of them waits for the slowest); 4: 20 + 41 + 33; 8:
// 27 + 46 + 44; 16: 40 + 53 + 60 (each workgroup's histogram is cleared and added up).
static int sample_chunks(int64_t B, int64_t V) {
    const int64_t most = ceil_div64(V, kChunk), want = B < 1024 ? 1024 / B : 1;
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
                 static_cast<SampleRow*>(workspace), nullptr, static_cast<int>(batch), static_cast<int>(vocab), 0, 0, 0, 0};
    a.parts = reinterpret_cast<SamplePart*>(a.rows + batch);
    a.chunks = sample_chunks(batch, vocab);
    a.chunk = static_cast<int>(ceil_div64(ceil_div64(vocab, a.chunks), kPiece) * kPiece);
    a.chunks = static_cast<int>(ceil_div64(vocab, a.chunk));
    a.bin_chunk = static_cast<int>(ceil_div64(a.chunk, 2 * kPiece) * kPiece);
    const auto with_logits = [](int64_t n) { return n < kChunk ? ceil_div64(n, kPiece) : int64_t(kThreads); };
    a.threads = static_cast<int>((a.chunks - 1) * with_logits(a.chunk) + with_logits(vocab - int64_t(a.chunks - 1) * a.chunk));
    const dim3 grid(static_cast<unsigned>(a.chunks), static_cast<unsigned>(batch)), block(kThreads);
    hipStream_t st = as_stream(stream);
    const bool draws = temperature || temperature_all > 0.0f;  // otherwise every row's token is its largest
    auto launch = [&](auto type) {
        using LT = decltype(type);
        hipLaunchKernelGGL(sample_extremes_kernel<LT>, grid, block, 0, st, a);
        if (draws) {
            hipLaunchKernelGGL(sample_bins_kernel<LT>, dim3(static_cast<unsigned>(ceil_div64(vocab, a.bin_chunk)), grid.y),
                               dim3(kBinThreads), 0, st, a);
            hipLaunchKernelGGL(sample_collect_kernel<LT>, grid, block, 0, st, a);
        }
        hipLaunchKernelGGL(sample_decide_kernel<LT>, dim3(static_cast<unsigned>(batch)), block, 0, st, a);
    };
    if (logits_f32) launch(float{});
    else launch(uint16_t{});
    return launch_status(what);
}
