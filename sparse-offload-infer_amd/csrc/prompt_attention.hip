// Causal attention of packed prompts over binary16 q, k, v on the matrix cores (gfx950).
//
// Sequence b owns query rows cu_q[b] .. cu_q[b + 1] - 1 and key rows cu_k[b] .. cu_k[b + 1] - 1. Query i of nq sees keys
// j <= i + nk - nq of nk (the last query sees every key; nk > nq continues a context), and
//   out[i, h] = sum_j softmax_j(scale q[i, h] . k[j, h / rep]) v[j, h / rep];
// a query that sees no key gives zeros. The framework's other prompt attention (prompt.hip) takes one sequence over a
// contiguous cache in the decode step's order of sums, on v_dot2; this one takes the tile order the matrix cores want.
//
// A workgroup of NW waves owns 32 NW queries of one head, or fewer of two or four heads of one KV head; a wave owns 32 of one
// head (v_mfma_f32_32x32x16_f16, lane n = lane & 31 is a query, h = lane >> 5):
//   * S^T = K Q^T: lane (n, h) ends with the scores of query n and keys 8 (r >> 2) + 4 h + (r & 3), r < 16, of each
//     32-key tile: a row's maximum is a lane's own but for one swap with lane + 32;
//   * O^T = V^T P^T takes these scores, exponentiated, as its B operand as they lie. The k slots of V are then
//     tokens 16 j + 4 h + 0 .. 3 and + 8 .. 11, four tokens of one dimension a lane, which ds_read_b64_tr_b16 reads
//     straight from the row-major V tile;
//   * the output's rescaling is lane-wise too (a lane's accumulators are all of its own query).
// K and V tiles go from memory into LDS without passing through registers (buffer_load .. lds, whose descriptor ends with
// the sequence's last row, so that rows behind it arrive as zeros), the next tiles' loads in flight during a tile's
// products; 16-byte chunks are XOR-swizzled on the way so that the operand reads spread over the banks (conflicts: 0.1 %
// of the busy cycles). The queries come in and the outputs leave through LDS too, as whole rows.
//
// Bound: 4 hd operations a (query, key, head) on the matrix cores, one exponential each on the vector units (at head_dim
// 64 both take 512 cycles for 32 x 64 scores). The running sum takes the binary16 weights that the products use, the
// base of the exponents lies 7 to 15 binades below the row's maximum. One sequence of 16384 tokens, 16 / 8 heads of
// 128: 1.05 ms, 1050 TFLOP/s (at the 1.8 GHz that the power limit leaves; a matrix product of 8192 reaches 1160, or 1360
// by its kernel alone), matrix units busy 63 % of the cycles, vector units 58 %. Twenty prompts of 1 to 1000 tokens, 32 / 8
// heads: 91 to 93 us.
//
// Tile, buffers and occupancy, 128 dimensions: 32 keys, three buffers (two tiles in flight), three workgroups to a CU
// against 64 keys, two buffers, two workgroups: 1.07 / 1.07 ms and 119 / 135 us for the two above, and against 32 keys,
// four buffers, two workgroups: 1.10 ms and 137 us. Many workgroups hide each other's starts and masked tiles. No
// instance may spill (the build sees to it): a version that did came back with a register of Q lost, why was never found.
// The instance above 128 dimensions, one workgroup to a CU, keeps its accumulators in accumulation registers, where its
// products write them, and moves all of them for every tile: 8192 tokens, 8 / 4 heads of 256, 359 us (765 TFLOP/s). These
// moves are of whole registers: nothing between the first tile and the last changes which lanes run.
//
// Tiles that the wave sees in full run a loop without masks. In the others a value that is not finite has to stay out of
// the rows that do not see its key, though their weight for it is 0: the products take the largest finite number in its
// place, and a rare last pass adds it where it is seen.
#include "soi_host.h"
#include "soi_device.h"
#include "soi_attn.h"

#include <type_traits>

namespace soi {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef __attribute__((address_space(3))) f16x8 lds_f16x8;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// A row's largest weight lies between 2^kPaLow and 2^kPaHigh (below 65504): weights are rounded by 2^-11 of themselves down to
// 2^-21 of the largest, and end in 0 below 2^-32 of it.
constexpr float kPaLow = 7.0f, kPaHigh = 15.0f;

struct PaArgs {
    const uint16_t *q, *k, *v;
    uint16_t* out;
    int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, o_ts, o_hs;  // token and head strides, in elements
    const int32_t *cu_q, *cu_k;
    float* part;  // split rows: acc [nsplit][Tq][NQ][hd], then (m, l) [nsplit][Tq][NQ][2]
    int Tq, Tk, NQ, NKV, hd, nsplit;
    int hshift;  // a workgroup's queries are those of 2^hshift heads of one KV head
    float scale_log2;
};

// The rows and keys of one workgroup: `rows` queries from q0 of sequence b.
struct PaRows {
    int q_lo, nq, k_lo, nk, off, q0, tiles;
    __device__ __forceinline__ PaRows(const PaArgs& a, int b, int qtile, int rows, int keys_per_tile) {
        auto clamp = [](int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; };
        auto uniform = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
        q_lo = clamp(uniform(ldg(a.cu_q + b)), 0, a.Tq);
        nq = clamp(uniform(ldg(a.cu_q + b + 1)), q_lo, a.Tq) - q_lo;
        k_lo = clamp(uniform(ldg(a.cu_k + b)), 0, a.Tk);
        nk = clamp(uniform(ldg(a.cu_k + b + 1)), k_lo, a.Tk) - k_lo;
        off = nk - nq;
        q0 = qtile * rows;
        const int keys = clamp(min(q0 + rows, nq) + off, 0, nk);  // seen by the last query
        tiles = (keys + keys_per_tile - 1) / keys_per_tile;
    }
};

// Key tiles per split, for at most nsplit splits of at least kPaSplitTiles tiles.
constexpr int kPaSplitTiles = 4;
__device__ __forceinline__ int pa_split_tiles(int tiles, int nsplit) {
    const int most = (tiles + kPaSplitTiles - 1) / kPaSplitTiles, ns = most < nsplit ? most : nsplit;
    return ns <= 1 ? (tiles < 1 ? 1 : tiles) : (tiles + ns - 1) / ns;
}

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
// flight (the kernel waits for them itself, at the barrier; no register but m0 is written). m0 holds the LDS address. The
// compiler does not count wait states inside assembly: with the s_nop the load is 5 of them behind whatever came before, as
// many as a vector instruction's write to the descriptor's registers (a readfirstlane or readlane) has to be ahead of it.
template <int LOADS>
__device__ __forceinline__ void pa_load(const uint16_t* base, int bytes, const uint32_t (&off)[LOADS], uint32_t lds) {
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

// 16 bytes to any address
__device__ __forceinline__ void stg_any(void* p, const u32x4& v) {
    typedef __attribute__((address_space(1))) u32x4_any gT;
    *(gT*)(p) = v;
}

template <int HD, int NW, int KT, int NBUF, int OCC>
__global__ __launch_bounds__(NW * kWave, OCC) void prompt_attention_kernel(const PaArgs a) {
    constexpr int kPaKeys = KT;
    constexpr int CPR = HD / 8, ROWB = HD * 2, TILEB = kPaKeys * ROWB;  // chunks and bytes of a row, bytes of a tile
    constexpr int KK = HD / 16, DT = HD / 32, NT = kPaKeys / 32, NJ = kPaKeys / 16;
    // Operand addresses of every chunk in registers and a loop of three tiles, one a buffer, whose offsets the reads then
    // carry: 14 vector instructions fewer a tile. 16384 tokens, 16 / 8 heads: 1176 -> 1150 us on one card. (The other
    // instances have no registers left for it.)
    constexpr bool PRE = HD == 128 && NBUF == 3;
    constexpr int LOADS = TILEB / 1024 / NW;  // 1 KB loads per wave and tile
    static_assert(TILEB % (1024 * NW) == 0, "whole loads per wave");
    __shared__ __attribute__((aligned(1024))) uint8_t s_kv[NBUF][2][TILEB];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, hh = lane >> 5;
    // heads of one KV head lie NKV apart in x: with NKV a multiple of 8 they run on one XCD and share its L2
    const int split = static_cast<int>(blockIdx.x) / a.NQ, hx = static_cast<int>(blockIdx.x) % a.NQ;
    const int kvh = hx % a.NKV, rep = a.NQ / a.NKV, hmask = (1 << a.hshift) - 1;
    const int head = kvh * rep + ((hx / a.NKV) & ~hmask) + (wave & hmask);
    // Neighbours in x have the other parts of the same 32 NW queries, and the longest rows come first. Which neighbour has
    // which part changes with y and z: workgroups go to the CUs in turn, and the same CUs would get all the long ones.
    const int part = (hx / a.NKV + static_cast<int>(blockIdx.y + blockIdx.z)) & hmask;
    const int qtile = static_cast<int>(gridDim.z - 1 - blockIdx.z) << a.hshift | part;
    const PaRows w(a, blockIdx.y, qtile, 32 * NW >> a.hshift, KT);
    const int q_lo = w.q_lo, nq = w.nq, k_lo = w.k_lo, nk = w.nk, off = w.off, q0 = w.q0;
    if (q0 >= nq) return;
    auto clamp = [](int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; };
    const int per = pa_split_tiles(w.tiles, a.nsplit), t0 = split * per, tiles = min(w.tiles, t0 + per);
    if (split > 0 && t0 >= w.tiles) return;
    const int wq0 = q0 + 32 * (wave >> a.hshift);
    const int last = wq0 + n + off - 4 * hh;  // the last key that the lane's query sees, less the lane's 4 hh

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
    // a wave's 32 queries, loaded like a tile into the buffers that no key tile needs yet
    constexpr int QLOADS = 32 * ROWB / 1024;
    static_assert((NBUF - 1) * 2 * KT >= 32 * NW, "room for the queries");
    uint32_t qo[QLOADS];
#pragma unroll
    for (int i = 0; i < QLOADS; ++i) {
        const int id = i * 64 + lane, r = id / CPR, c = (id % CPR) ^ pa_swz_k<HD>(r);
        qo[i] = 8 * c < a.hd ? static_cast<uint32_t>(r * a.q_ts + 8 * c) * 2 : 0xfffffff0u;
    }
    const uint16_t* kb = a.k + k_lo * a.k_ts + kvh * a.k_hs;
    const uint16_t* vb = a.v + k_lo * a.v_ts + kvh * a.v_hs;
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_u8*)&s_kv[0][0][0]));
    const uint32_t lds = lds0 + wave * LOADS * 1024;
    // the next tile to load: its first key's rows, the keys from there on, its buffer (tiles are loaded in order)
    const int kspan = static_cast<int>(a.k_ts) * 2, vspan = static_cast<int>(a.v_ts) * 2, hd2 = a.hd * 2;  // bytes
    const uint16_t *k_next = kb + static_cast<int64_t>(t0) * KT * a.k_ts, *v_next = vb + static_cast<int64_t>(t0) * KT * a.v_ts;
    int left = nk - t0 * KT, into = 0;
    auto load = [&] {
        const int rows = min(left, KT) - 1;
        pa_load<LOADS>(k_next, rows < 0 ? 0 : rows * kspan + hd2, ko, lds + into);
        pa_load<LOADS>(v_next, rows < 0 ? 0 : rows * vspan + hd2, vof, lds + into + TILEB);
        k_next += KT * a.k_ts;
        v_next += KT * a.v_ts;
        left -= KT;
        into = into == (NBUF - 1) * 2 * TILEB ? 0 : into + 2 * TILEB;
    };

    f32x16 acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] = 0.0f;
    float m = kNegBig, l = 0.0f;
    uint32_t odd = 0;  // not 0: a value that is not finite was replaced in a tile that not all the wave's queries see in full

    // Operand addresses: the lane's part below with bits flipped for the chunk, the row and the buffer added.
    // K: key n of 32, chunk 2 kk + hh
    const uint32_t k_at = lds0 + n * ROWB + ((hh ^ pa_swz_k<HD>(n)) << 4);
    // V: token vr + 8 x + 16 j, four dimensions of chunk 4 d + ...; 8 x flips bit 1 of the swizzle
    const int vr = 4 * hh + ((lane & 15) >> 2);
    const uint32_t v_at = lds0 + TILEB + vr * ROWB +
                          (((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ pa_swz_v<HD>(vr)) << 4) + 8 * (lane & 1);

    // the tiles that the wave's queries see any of, and that they all see in full (none for a wave without queries)
    const int wtiles = wq0 < nq ? (clamp(min(wq0 + 32, nq) + off, 0, nk) + kPaKeys - 1) / kPaKeys : 0;
    const int whole = wq0 >= nq || wq0 + off + 1 < 0 ? 0 : (wq0 + off + 1) / kPaKeys;
    auto mask = [&](f32x16 (&z)[NT], int tile) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int key = tile * kPaKeys + 32 * i + 8 * (r >> 2) + (r & 3);
                z[i][r] = key <= last ? z[i][r] : -__builtin_inff();
            }
    };
    auto highest = [&](const f32x16 (&z)[NT]) {
        float top = z[0][0];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, z[i][r]);
        return fmaxf(top, xor_lanes<32>(top)) * a.scale_log2;
    };
    // m is the base of the exponents, raised only where a weight would pass 2^kPaHigh, and then to where it is 2^kPaLow: most
    // tiles of a long row rescale nothing
    auto raise = [&](float top) {
        if (ballot(top > m + kPaHigh)) {
            const float mn = top > m + kPaHigh ? top - kPaLow : m, w = fast_exp2(m - mn);  // a row does not depend on its neighbours
            m = mn;
            l *= w;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[d][r] *= w;
        }
    };
    // this wave's LDS reads are done, and its loads but for the last `flight`; after the barrier everyone's
    auto meet = [](auto flight) {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0070 | (flight & 15) | (flight >> 4) << 14);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    if (t0 < tiles) {  // (workgroup-uniform)
        const int rows = min(nq - wq0, 32) - 1;
        pa_load<QLOADS>(a.q + (q_lo + min(wq0, nq)) * a.q_ts + head * a.q_hs,
                        rows < 0 ? 0 : static_cast<int>(rows * a.q_ts + a.hd) * 2, qo, lds0 + 2 * TILEB + wave * QLOADS * 1024);
        load();
        meet(std::integral_constant<int, 0>{});
        f16x8 qf[KK];
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
            qf[kk] = *(const lds_f16x8*)((lds_u8*)((k_at + 2 * TILEB + 32 * wave * ROWB) ^ (kk << 5)));
        meet(std::integral_constant<int, 0>{});
#pragma unroll
        for (int i = 1; i < NBUF - 1; ++i) load();
        int at = 0, t = t0;  // LDS offset of tile t
        uint32_t kx[PRE ? KK : 1], vx[PRE ? 2 * DT : 1];
        if constexpr (PRE) {
#pragma unroll
            for (int i = 0; i < KK; ++i) {
                kx[i] = k_at ^ (i << 5);
                asm volatile("" : "+v"(kx[i]));  // (kept: the compiler would flip the bits again for every read)
            }
#pragma unroll
            for (int i = 0; i < 2 * DT; ++i) {
                vx[i] = v_at ^ (i << 5);
                asm volatile("" : "+v"(vx[i]));
            }
        }
        auto tile = [&](auto MASKED, auto BUF) {  // BUF: the tile's buffer, -1 where only `at` says it
            if (t > t0) meet(std::integral_constant<int, (NBUF - 2) * 2 * LOADS>{});
            load();
            const int cur = BUF < 0 ? at : BUF * 2 * TILEB;
            if (BUF < 0) at = at == (NBUF - 1) * 2 * TILEB ? 0 : at + 2 * TILEB;
            if (MASKED && t >= wtiles) return;  // wave-uniform: nothing of this tile is seen here
            f32x16 z[NT];
            const uint32_t ka = k_at + cur, va = v_at + cur;
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                f16x8 kf[KK];
#pragma unroll
                for (int kk = 0; kk < KK; ++kk)
                    kf[kk] = *(const lds_f16x8*)((lds_u8*)(PRE ? kx[PRE ? kk : 0] : ka ^ (kk << 5)) + (PRE ? cur : 0) +
                                                 i * 32 * ROWB);
                if (KK <= 8) __builtin_amdgcn_sched_barrier(0);  // all reads first: a product waits for its own only
#pragma unroll
                for (int r = 0; r < 16; ++r) z[i][r] = 0.0f;
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) z[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[kk], qf[kk], z[i], 0, 0, 0);
            }
            auto v_read = [&](int d, int j) {
                s16x4 r[2];
#pragma unroll
                for (int x = 0; x < 2; ++x)
                    r[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (lds_s16x4*)((lds_u8*)(PRE ? vx[PRE ? 2 * d + x : 0] : va ^ (d << 6 | x << 5)) + (PRE ? cur : 0) +
                                     (16 * j + 8 * x) * ROWB));
                return (s16x8)__builtin_shufflevector(r[0], r[1], 0, 1, 2, 3, 4, 5, 6, 7);
            };
            s16x8 vf[2][NJ];  // V of two dimension tiles, one in use and one on its way
            auto v_fetch = [&](int d) {
#pragma unroll
                for (int j = 0; j < NJ; ++j) vf[d & 1][j] = v_read(d, j);
            };
            v_fetch(0);
            __builtin_amdgcn_sched_barrier(0);  // (requested before the softmax, which they do not wait for)
            if (MASKED) mask(z, t);
            raise(highest(z));
            f16x8 pb[NJ];
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    pb[j][e] = static_cast<f16>(fast_exp2(fmaf(z[j >> 1][8 * (j & 1) + e], a.scale_log2, -m)));
            // the sum is that of the weights the products use: rounded p, added in binary32
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int e = 0; e < 8; e += 2)
                    l = dot2(f16x2{pb[j][e], pb[j][e + 1]}, f16x2{(f16)1.0f, (f16)1.0f}, l);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                if (d + 1 < DT) v_fetch(d + 1);
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    s16x8 v = vf[d & 1][j];
                    if (MASKED) {
                        // A weight of 0 does not hide an infinity or NaN (bits from 0x7c00 and from 0xfc00 up): the products
                        // take the largest finite number for it, and the queries that do see it get it added at the end.
                        const u16x8 lo = __builtin_elementwise_min(__builtin_bit_cast(u16x8, v), (u16x8)(uint16_t)0xfbff);
                        const s16x8 f = __builtin_elementwise_min(__builtin_bit_cast(s16x8, lo), (s16x8)(short)0x7bff);
                        const u32x4 was = __builtin_bit_cast(u32x4, v), is = __builtin_bit_cast(u32x4, f), x = was ^ is;
                        odd |= (x.x | x.y) | (x.z | x.w);
                        v = f;
                    }
                    acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, v), pb[j], acc[d], 0, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        const int full = min(whole, tiles);
        using std::integral_constant;
        if constexpr (PRE)
            while (t + NBUF <= full) {
                tile(std::false_type{}, integral_constant<int, 0>{});
                ++t;
                tile(std::false_type{}, integral_constant<int, 1>{});
                ++t;
                tile(std::false_type{}, integral_constant<int, 2>{});
                ++t;
            }
        for (; t < full; ++t) tile(std::false_type{}, integral_constant<int, -1>{});
        for (; t < tiles; ++t) tile(std::true_type{}, integral_constant<int, -1>{});
    }
    const bool patch = ballot(odd != 0) != 0;
    l += xor_lanes<32>(l);
    // the lane once more, from the hardware: nothing of it stays in registers through the tiles
    const int elane = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)), en = elane & 31, ehh = elane >> 5;
    // adds the values left out to the queries that see them: add(r, d, v) for each key, the wave's query r, dimension d
    auto patched = [&](int d0, int d1, auto add) {
        const int first = max(whole, t0) * kPaKeys, end = min(nk, tiles * kPaKeys);
        for (int key = first; key < end; ++key)
            for (int d = d0 + elane; d < min(d1, a.hd); d += kWave) {
                const uint16_t v = ldg(vb + key * a.v_ts + d);
                if ((v & 0x7fff) >= 0x7c00)
                    for (int r = max(0, key - off - wq0); r < 32; ++r) add(r, d, f16_bits_to_f32(v));
            }
    };
    if (w.tiles > per) {  // a split row: its state as it is, 64 dimensions at a time through LDS
        lds_u8* so = (lds_u8*)(lds0 + wave * 32 * 256);
        float* pb = a.part + (static_cast<int64_t>(split) * a.Tq + q_lo + wq0) * a.NQ * a.hd + head * a.hd;
#pragma unroll
        for (int d = 0; d < DT; d += 2) {
            meet(std::integral_constant<int, 0>{});
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                const f32x16& v = acc[d + (x >> 2)];
                const int r = 4 * (x & 3);
                *(__attribute__((address_space(3))) f32x4*)(so + en * 256 + (((2 * x + ehh) ^ (en & 15)) << 4)) =
                    f32x4{v[r], v[r + 1], v[r + 2], v[r + 3]};
            }
            if (patch)
                patched(32 * d, 32 * d + 64, [&](int r, int dim, float v) {
                    const int c = (dim - 32 * d) >> 2;
                    auto* x = (__attribute__((address_space(3))) float*)(so + r * 256 + ((c ^ (r & 15)) << 4) + 4 * (dim & 3));
                    *x += v;
                });
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int r = 4 * i + (elane >> 4), c = elane & 15;
                const f32x4 o = *(const __attribute__((address_space(3))) f32x4*)(so + r * 256 + ((c ^ (r & 15)) << 4));
                if (wq0 + r < nq && 32 * d + 4 * c < a.hd)
                    stg(reinterpret_cast<f32x4*>(pb + static_cast<int64_t>(r) * a.NQ * a.hd + 32 * d + 4 * c), o);
            }
        }
        if (ehh == 0 && wq0 + en < nq) {
            float* ml = a.part + static_cast<int64_t>(a.nsplit) * a.Tq * a.NQ * a.hd +
                        2 * ((static_cast<int64_t>(split) * a.Tq + q_lo + wq0 + en) * a.NQ + head);
            stg(reinterpret_cast<f32x2*>(ml), f32x2{m, l});
        }
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    // out rows leave through LDS, so that a store covers whole rows: 8 bytes of 32 rows at a time otherwise
    meet(std::integral_constant<int, 0>{});
    lds_u8* so = (lds_u8*)(lds0 + wave * 32 * ROWB);
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int x = 0; x < 4; ++x)
            *(__attribute__((address_space(3))) u32x2*)(so + en * ROWB + (((4 * d + x) ^ pa_swz_k<HD>(en)) << 4) + 8 * ehh) =
                u32x2{pack_f16x2(acc[d][4 * x] * inv, acc[d][4 * x + 1] * inv),
                      pack_f16x2(acc[d][4 * x + 2] * inv, acc[d][4 * x + 3] * inv)};
    if (patch)
        patched(0, HD, [&](int r, int dim, float v) {
            auto* x = (__attribute__((address_space(3))) uint16_t*)(so + r * ROWB + (((dim >> 3) ^ pa_swz_k<HD>(r)) << 4) +
                                                                    2 * (dim & 7));
            *x = f32_to_f16_bits(f16_bits_to_f32(*x) + v);
        });
    uint16_t* ob = a.out + head * a.o_hs;
#pragma unroll
    for (int i = 0; i < 32 * ROWB / 1024; ++i) {
        const int id = i * 64 + elane, r = id / CPR, c = id % CPR;  // (a wave's LDS writes and reads are in order)
        const u32x4 o = *(const __attribute__((address_space(3))) u32x4*)(so + r * ROWB + ((c ^ pa_swz_k<HD>(r)) << 4));
        if (wq0 + r < nq && 8 * c < a.hd) stg_any(ob + (q_lo + wq0 + r) * a.o_ts + 8 * c, o);
    }
}

// The split rows' states, in split order: four dimensions of one query and head a thread, kPaCombineRows queries of one
// attention workgroup's `rows` a workgroup (many small workgroups: a thread's loads are two round trips, whatever they move).
constexpr int kPaCombineRows = 8;
constexpr int kPaMaxSplits = 64;
__global__ __launch_bounds__(256) void prompt_combine_kernel(const PaArgs a, int rows, int keys_per_tile) {
    const int head = blockIdx.x, r0 = static_cast<int>(blockIdx.z) * kPaCombineRows;
    const PaRows w(a, blockIdx.y, r0 / rows, rows, keys_per_tile);
    const int per = pa_split_tiles(w.tiles, a.nsplit);
    if (r0 >= w.nq || w.tiles <= per) return;  // written by its one split
    const int ns = (w.tiles + per - 1) / per, quads = a.hd >> 2;
    const int64_t stride = static_cast<int64_t>(a.Tq) * a.NQ;
    const float* ml = a.part + a.nsplit * stride * a.hd;
    const int rows_here = min(kPaCombineRows, w.nq - r0);
    const int64_t row0 = static_cast<int64_t>(w.q_lo + r0) * a.NQ + head;
    // the weights 2^(m_s - M) / l of each row's splits (32 lanes a row, splits j and j + 32 a lane)
    __shared__ float s_w[kPaCombineRows][kPaMaxSplits];
    {
        const int r = threadIdx.x >> 5, j = threadIdx.x & 31;
        const float* p = ml + 2 * (row0 + static_cast<int64_t>(r < rows_here ? r : 0) * a.NQ);
        f32x2 x[2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
            x[e] = j + 32 * e < ns ? ldg(reinterpret_cast<const f32x2*>(p + 2 * (j + 32 * e) * stride)) : f32x2{kNegBig, 0.0f};
        float M = fmaxf(x[0].x, x[1].x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 32));
        const float e0 = fast_exp2(x[0].x - M), e1 = fast_exp2(x[1].x - M);
        float lsum = fmaf(x[0].y, e0, x[1].y * e1);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) lsum += __shfl_xor(lsum, o, 32);
        const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;
        s_w[r][j] = e0 * inv;
        s_w[r][j + 32] = e1 * inv;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows_here * quads; i += 256) {
        const int r = i / quads, d = 4 * (i % quads);
        const float* p = a.part + (row0 + static_cast<int64_t>(r) * a.NQ) * a.hd + d;
        f32x4 v = {0, 0, 0, 0};
        for (int s = 0; s < ns; s += 8) {
            f32x4 x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                x[e] = ldg(reinterpret_cast<const f32x4*>(p + (s + e < ns ? s + e : s) * stride * a.hd));
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float f = s + e < ns ? s_w[r][s + e] : 0.0f;
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = s + e < ns ? fmaf(x[e][k], f, v[k]) : v[k];
            }
        }
        const u32x2 o = {pack_f16x2(v.x, v.y), pack_f16x2(v.z, v.w)};
        stg(reinterpret_cast<u32x2*>(a.out + (w.q_lo + r0 + r) * a.o_ts + head * a.o_hs + d), o);
    }
}

constexpr int kPaWaves = 4;

// Heads that share a workgroup (as a power of two): waves of different heads of one KV head read the same tiles for the same
// queries, so none of them idles while another finishes the tiles of later queries, and few queries fill a workgroup.
// With one / four heads of 32 / 8 (of 128 dimensions) a workgroup: 80 prompts of 16 tokens 22 / 12 us, 80 of 128 48 / 43,
// 20 of 512 81 / 75, 20 of up to 1000 (10577 in all) 122 / 108, 10 of 1024 121 / 118. The parts have to be neighbours (in
// the order of the sequences' rows instead, the 20 ragged prompts take 140 us: K and V leave the L2 between them).
static int pa_hshift(int64_t rep) { return rep % 4 == 0 ? 2 : rep % 2 == 0 ? 1 : 0; }

// Splits of a row's keys: where the heads and the 128-query tiles of all rows together make fewer workgroups than 1024
// (head_dim up to 64), 512 (up to 128) or 256 (above), as many as fit into that. The count is a rough one: it knows neither
// the batch nor the heads that share a workgroup, so that one short sequence with four heads to a workgroup is split into
// fewer workgroups than that, and many sequences of a few queries into more. Four, three and one workgroup fit on a CU;
// every split writes and reads hd + 2 floats a query. Measured with 512 / 768 / 1024 / 1536 workgroups aimed at: five ragged parts of up to 513 queries behind up to
// 4000 keys, 14 heads of 64, 70 / 62 / 57 / 58 us, 1024 queries over 17408 keys, 8 heads of 64, 58 / 57 / 58 / 64 us. With
// 256 / 512 / 768 / 1024: 512 queries over 16896 keys, 16 heads of 128, 123 / 93 / 94 / 105 us, 2048 queries of 8 heads of
// 128, 40 / 31 / 31 / 40 us. 300 queries x 2 over 3300 keys, 14 heads of 256, 67 us with 256 and 98 with 512.
static int64_t pa_nsplit(int64_t Tq, int64_t Tk, int64_t NQ, int64_t hd, int64_t KT) {
    const int64_t groups = NQ * ceil_div64(Tq, 32 * kPaWaves), most = ceil_div64(ceil_div64(Tk, KT), kPaSplitTiles);
    int64_t n = (hd > 128 ? 256 : hd > 64 ? 512 : 1024) / groups;
    n = n < most ? n : most;
    return n < 1 ? 1 : n > kPaMaxSplits ? kPaMaxSplits : n;
}

// Whether two of the rows i ts + j hs + 0 .. hd - 1 (i < T, j < H) share an element: for a distance of dj heads only the two
// distances of tokens nearest to -dj hs / ts can bring them together.
static bool pa_rows_meet(int64_t T, int64_t H, int64_t ts, int64_t hs, int64_t hd) {
    if (hs >= hd && ts >= (H - 1) * hs + hd) return false;  // the usual order
    if (T > 1 && ts < hd && ts > -hd) return true;
    for (int64_t dj = 1; dj < H; ++dj) {
        const int64_t at = dj * hs, near = T > 1 ? -at / ts : 0;
        for (int64_t di = near - 1; di <= near + 1; ++di) {
            const int64_t d = di * ts + at;
            if (di < T && di > -T && d < hd && d > -hd) return true;
        }
    }
    return false;
}

static int64_t pa_keys(int64_t hd) { return hd > 64 && hd <= 128 ? 32 : 64; }

}  // namespace soi

using namespace soi;

extern "C" size_t soi_prompt_attention_workspace_bytes(int64_t Tq, int64_t Tk, int64_t num_q_heads, int64_t head_dim) {
    if (Tq < 1 || Tk < 1 || num_q_heads < 1 || head_dim < 1 || head_dim > 256) return 0;
    const int64_t n = pa_nsplit(Tq, Tk, num_q_heads, head_dim, pa_keys(head_dim));
    return n == 1 ? 0 : static_cast<size_t>(n) * Tq * num_q_heads * (head_dim + 2) * sizeof(float);
}

extern "C" int soi_prompt_attention(const uint16_t* q, int64_t q_token_stride, int64_t q_head_stride, const uint16_t* k,
                                    int64_t k_token_stride, int64_t k_head_stride, const uint16_t* v,
                                    int64_t v_token_stride, int64_t v_head_stride, const int32_t* cu_q,
                                    const int32_t* cu_k, int64_t batch, int64_t Tq, int64_t Tk, int64_t max_q,
                                    int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim, uint16_t* out,
                                    int64_t out_token_stride, int64_t out_head_stride, float scale, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    const char* what = "soi_prompt_attention";
    SOI_REQUIRE(head_dim >= 8 && head_dim % 8 == 0 && head_dim <= 256, "%s: head_dim must be a multiple of 8 up to 256, got %lld",
                what, (long long)head_dim);
    SOI_REQUIRE(num_kv_heads >= 1 && num_q_heads >= 1 && num_q_heads <= 65535 && num_q_heads % num_kv_heads == 0,
                "%s: num_q_heads must be a multiple of num_kv_heads", what);
    SOI_REQUIRE(batch >= 1 && batch <= 65535, "%s: the number of sequences must be in [1, 65535]", what);
    SOI_REQUIRE(Tq >= 0 && Tk >= 0 && Tq < (int64_t(1) << 30) && Tk < (int64_t(1) << 30), "%s: token counts out of range", what);
    SOI_REQUIRE(max_q >= 0 && max_q <= 65535 * kPaCombineRows, "%s: max_q must be in [0, 524280]", what);
    SOI_REQUIRE(scale > 0.0f && scale < __builtin_inff(), "%s: scale must be positive and finite", what);
    if (Tq == 0 || max_q == 0) return SOI_OK;
    SOI_REQUIRE(q && out && cu_q && cu_k && (Tk == 0 || (k && v)), "%s: null pointer", what);
    SOI_REQUIRE(k_token_stride >= 0 && k_token_stride < (int64_t(1) << 22) && v_token_stride >= 0 &&
                    v_token_stride < (int64_t(1) << 22),
                "%s: key and value rows must be less than 2^22 elements apart", what);
    SOI_REQUIRE(q_token_stride >= 0 && q_token_stride < (int64_t(1) << 22), "%s: query rows must be less than 2^22 elements apart",
                what);
    SOI_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && q_token_stride % 8 == 0 &&
                    q_head_stride % 8 == 0 && k_token_stride % 8 == 0 && k_head_stride % 8 == 0 &&
                    v_token_stride % 8 == 0 && v_head_stride % 8 == 0,
                "%s: q, k and v must be 16-byte aligned with strides of whole 16 bytes", what);
    SOI_REQUIRE((reinterpret_cast<uintptr_t>(out) & 7u) == 0 && out_token_stride % 4 == 0 && out_head_stride % 4 == 0,
                "%s: out must be 8-byte aligned with strides of whole 8 bytes", what);
    SOI_REQUIRE(!pa_rows_meet(Tq, num_q_heads, out_token_stride, out_head_stride, head_dim), "%s: rows of out overlap", what);
    const size_t need = soi_prompt_attention_workspace_bytes(Tq, Tk, num_q_heads, head_dim);
    if (need && (!workspace || workspace_bytes < need || !aligned16(workspace))) {
        set_last_error("%s: workspace of %zu bytes (16-byte aligned) needed, got %zu", what, need, workspace_bytes);
        return SOI_ERR_WORKSPACE;
    }
    const int hshift = pa_hshift(num_q_heads / num_kv_heads), rows = 32 * kPaWaves >> hshift;
    const int64_t kt = pa_keys(head_dim), nsplit = pa_nsplit(Tq, Tk, num_q_heads, head_dim, kt);
    const PaArgs a{q, k, v, out, q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride,
                   v_head_stride, out_token_stride, out_head_stride, cu_q, cu_k, static_cast<float*>(workspace),
                   static_cast<int>(Tq), static_cast<int>(Tk), static_cast<int>(num_q_heads),
                   static_cast<int>(num_kv_heads), static_cast<int>(head_dim), static_cast<int>(nsplit), hshift,
                   scale * kLog2e};
    constexpr int NW = kPaWaves;
    const unsigned qtiles = static_cast<unsigned>(ceil_div64(max_q, 32 * NW));
    const dim3 grid(static_cast<unsigned>(num_q_heads * nsplit), static_cast<unsigned>(batch), qtiles);
    hipStream_t st = as_stream(stream);
#define SOI_P(H, KT, NB, OCC) \
    hipLaunchKernelGGL((prompt_attention_kernel<H, NW, KT, NB, OCC>), grid, dim3(NW * kWave), 0, st, a)
    if (head_dim <= 64) SOI_P(64, 64, 2, 4);
    else if (head_dim <= 128) SOI_P(128, 32, 3, 3);
    else SOI_P(256, 64, 2, 1);
#undef SOI_P
    const int status = launch_status(what);
    if (status || nsplit == 1) return status;
    hipLaunchKernelGGL(prompt_combine_kernel, dim3(static_cast<unsigned>(num_q_heads), static_cast<unsigned>(batch),
                            static_cast<unsigned>(ceil_div64(max_q, kPaCombineRows))),
                       dim3(256), 0, st, a, rows, static_cast<int>(kt));
    return launch_status(what);
}
