// The weights of an attention call, accumulated per cached position: score_out[kv head][p] = score_in[kv head][p] + the sum
// over the call's rows and the heads of the group of w = 2^(s - m) / l, where s is the row's score of key p in log2 units, m
// the reference its attention used and l = sum 2^(s - m).  The attention kernels (VAR_TRACK) leave m and l, with l summed in
// fp32 from unrounded weights.
//
// track_step, one row per sequence: the decode kernel kept the scores (16 bytes per position and kv head at four heads,
// beside the 272 bytes of K and V it streams), so the cache is not read again; it runs beside the merge of the split records,
// in the same launch.
// k_track_chunk, a prompt chunk: the scores are formed a second time; only K is read.
#pragma once
#include <cuda.h>

#include "common.cuh"
#include "exact.cuh"
#include "prefill.cuh"
#include "work_cut.h"

namespace battn {
namespace tr {

constexpr int TILE = 64;                    // tiles of the decode kernel's scores

struct StepParams {
    const int* hdr;          // the decode kernel's header, records and scores
    const float* part;
    const float* scores;
    float* out;              // score_out, [partition or table row][kv head][stride]
    const float* in;         // score_in, or null: nothing accumulated yet
    const int* pos;
    const int* kslot;
    const int* act;
    int n_seq, Hkv, G, HD, cph;
    size_t stride;
    int* status;
};
struct StepMerge {           // one launch: blocks below `merge_blocks` merge the outputs, the others accumulate the weights
    MergeParams merge;
    StepParams step;
    int merge_blocks;
};

// (m, 1 / l) of head `h` of an item over the records of the CTAs that hold a piece of it, by one warp
__device__ __forceinline__ float2 item_norm(const StepParams& P, int item, int clo, int chi, int h, int lane) {
    const float* rec = P.part + ((size_t)(clo + item) * P.G + h) * (P.HD + 4) + P.HD;
    const size_t step = (size_t)P.G * (P.HD + 4);
    float M = NEG_BIG, L = 0.f;
    for (int s = lane; s <= chi - clo; s += 32) {
        const float4 r = *reinterpret_cast<const float4*>(rec + s * step);     // m, rounded l, l
        const float Mn = fmaxf(M, r.x);
        L = L * fast_exp2(M - Mn) + r.z * fast_exp2(r.x - Mn);
        M = Mn;
    }
    float Mx = M;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) Mx = fmaxf(Mx, __shfl_xor_sync(0xffffffffu, Mx, o));
    L *= fast_exp2(M - Mx);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    return make_float2(Mx, 1.f / L);
}

// Block `cta` of `n_cta` accumulates its contiguous share of the scores' tiles, a thread per position, several in flight.
template <int THREADS>
__device__ __forceinline__ void track_step(const StepParams& P, int cta, int n_cta) {
    extern __shared__ int s_cum[];                               // [n_seq + 1]
    __shared__ float2 s_norm[8];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int i = tid; i <= P.n_seq; i += THREADS) s_cum[i] = P.hdr[2 + i];
    const int per_cta = P.hdr[0];
    __syncthreads();
    const int total = P.Hkv * s_cum[P.n_seq];
    const int share = (total + n_cta - 1) / n_cta;
    const int g1 = min(total, (cta + 1) * share);
    for (int g = cta * share; g < g1;) {
        const fd::Piece pc = fd::locate(g, g1, s_cum, P.n_seq, P.Hkv);
        const int c0 = s_cum[pc.i], nt = s_cum[pc.i + 1] - c0;
        const int p = P.pos[pc.i], slot = P.kslot ? P.kslot[pc.i] : 0;
        int clo, chi;
        fd::item_ctas(P.cph, per_cta, P.Hkv, c0, nt, pc.kvh, clo, chi);
        // a slot that two active sequences name would get both sums or either one, by chance: neither is written
        bool twice = false;
        if (P.kslot)
            for (int j = tid; j < P.n_seq; j += THREADS) twice |= j != pc.i && P.kslot[j] == slot && !(P.act && P.act[j] == 0);
        if (__syncthreads_or(twice)) {                           // (and the previous piece has used s_norm)
            if (tid == 0) atomicOr(P.status, BATTN_DEV_BAD_POSITION);
            g += pc.n;
            continue;
        }
        if (warp < P.G) {
            const float2 nm = item_norm(P, pc.i * P.Hkv + pc.kvh, clo, chi, warp, lane);
            if (lane == 0) s_norm[warp] = nm;
        }
        __syncthreads();
        const int first = pc.tl * TILE, keys = min(pc.n * TILE, p + 1 - first);
        const float* in = P.in ? P.in + ((size_t)slot * P.Hkv + pc.kvh) * P.stride + first : nullptr;
        float* out = P.out + ((size_t)slot * P.Hkv + pc.kvh) * P.stride + first;
        const float* sc = P.scores + (size_t)g * TILE * P.G;
        constexpr int UN = THREADS == 1024 ? 2 : 4;              // (the big block has 64 registers, and covers 2048 positions)
        if (P.G == 4) {                                          // the usual group: a position's scores are one 16-byte load
            const float2 n0 = s_norm[0], n1 = s_norm[1], n2 = s_norm[2], n3 = s_norm[3];
            for (int k0 = tid; k0 < keys; k0 += UN * THREADS) {
                float4 v[UN];
                float w[UN];
#pragma unroll
                for (int u = 0; u < UN; ++u) {
                    const int k = k0 + u * THREADS;
                    v[u] = k < keys ? *reinterpret_cast<const float4*>(sc + 4 * (size_t)k) : make_float4(0.f, 0.f, 0.f, 0.f);
                    w[u] = in && k < keys && first + k < p ? in[k] : 0.f;   // the call's own position starts from nothing
                }
#pragma unroll
                for (int u = 0; u < UN; ++u) {
                    const int k = k0 + u * THREADS;
                    if (k < keys)
                        out[k] = (fmaf(fast_exp2(v[u].x - n0.x), n0.y, fast_exp2(v[u].y - n1.x) * n1.y) +
                                  fmaf(fast_exp2(v[u].z - n2.x), n2.y, fast_exp2(v[u].w - n3.x) * n3.y)) + w[u];
                }
            }
        } else {
            for (int k = tid; k < keys; k += THREADS) {
                float w = 0.f;
                for (int h = 0; h < P.G; ++h) w = fmaf(fast_exp2(sc[(size_t)k * P.G + h] - s_norm[h].x), s_norm[h].y, w);
                out[k] = w + (in && first + k < p ? in[k] : 0.f);
            }
        }
        g += pc.n;
    }
}

// few items (one or two sequences): the merge is one latency chain, see k_merge_balanced
template <int HD>
__global__ void __launch_bounds__(MERGE_B_THREADS) k_merge_track_few(const StepMerge P) {
    if ((int)blockIdx.x < P.merge_blocks) {
        merge_balanced<HD>(P.merge);
    } else {
        pdl_trigger();
        pdl_wait();
        track_step<MERGE_B_THREADS>(P.step, (int)blockIdx.x - P.merge_blocks, (int)gridDim.x - P.merge_blocks);
    }
}
template <int HD>
__global__ void __launch_bounds__(MERGE_M_THREADS) k_merge_track_many(const StepMerge P) {
    pdl_trigger();
    pdl_wait();
    if ((int)blockIdx.x < P.merge_blocks) {
        const int item = blockIdx.x * (MERGE_M_THREADS / 32) + (threadIdx.x >> 5);
        if (item < P.merge.n_rows * P.merge.Hq) merge_many<HD>(P.merge, item);
    } else {
        track_step<MERGE_M_THREADS>(P.step, (int)blockIdx.x - P.merge_blocks, (int)gridDim.x - P.merge_blocks);
    }
}

struct ChunkParams {
    CUtensorMap q_map;       // fp16 queries [row][head][dim], boxes of 128 / G rows x G heads x 64 dims, 128-byte swizzle
    const void* q;
    const uint8_t* kvk;
    const float2* norm;      // [row][head]: (m, 1 / l)
    float* out;
    const float* in;
    const int* pos;
    const int* kslot;
    const int* act;
    int rows, Hq, Hkv, G, q_f16;
    int pstride, n_slots;
    float scale_log2;
    int* status;
    Paging pg;
};

// ---- the weights of a prompt chunk -------------------------------------------------------------------------------------
// Persistent CTAs, one per SM; a unit is (kv head, 256 keys at head_dim 128, 128 keys at 256).  S^T = K Q^T on tcgen05 with
// 128 keys on the M side, so that a TMEM lane is a key and the sum over the rows is a sum over columns, inside one thread.
//   * K is the tensor-memory A operand and stays there for the unit, in two exact fp16 parts like in the prompt kernels
//     (hi = fp16(d x), lo = d x - hi): the scores carry no rounding of K.  (From shared memory the products run as
//     fast -- 64 cycles for 128 x 128 x 16 either way -- but its 128 KB are the Q ring's.)
//     The low part comes first, here and in the attention kernel's VAR_TRACK instances: every accumulation step drops what
//     lies below the running sum's 24 bits, always towards zero, so that large scores lose, and the low part's steps are
//     free of it only while the sum is small.  (Distance of the weights from 64 bits, 2-norm, 2 rows at 16000 positions: head_dim
//     128 2.7e-6 -> 1.3e-6, 256 6.1e-6 -> 1.0e-6.  At 256 the attention kernel takes the dims in two halves; the same order here,
//     low, high, low, high, gave 3.0e-6.)
//   * Q tiles of 128 (row, head) pairs stream from L2 through a ring as the B operand, by tiled copies that place them swizzled;
//     every one serves all keys of the unit (two M tiles at head_dim 128: half the L2 traffic, which at one would be near 7 TB/s).
//     Loader warps did this before and were the bound: with divisions 390 us, with shifts 245, copies 236.  (fp32 queries are
//     still brought by warps, which round them.)
//   * Two accumulators of 128 columns; each of two groups of four warps takes its own into registers whole, frees it, and adds up
//     w += 2^(s c - m) / l, one exponential per score.  The exponentials (16 per cycle and SM) take as long as the two products:
//     that balance is the bound.
//   * Between units the eight warps convert the next K, whose raw records were fetched ahead.
// 512 rows at 32K, 32/8 heads of 128: 236 us (warp MMAs with scales on fp32 sums took 705) at 1.61 GHz, which is what the power cap
// leaves; exponentials 64 % of their rate, tensor pipe 62 %.  A quarter or half of the exponentials on the FMA pipes: no gain.
constexpr int QN = 128;                     // pairs per Q tile

// one box of a 3-d tensor map into shared memory (no multicast); x is a multiple of 64 halves
__device__ __forceinline__ void tensor_g2s(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar)) : "memory");
}
constexpr int W_Q = 8, W_MMA = 10, W_K = 11;
constexpr int CTHREADS = 12 * 32;           // warps 0-7 convert K and sum weights, 8-9 load Q, 10 issues the MMAs, 11 loads K
constexpr int MAX_PAIRS = MAX_PREFILL * 8;

template <int HD>
struct ChunkCfg {
    static constexpr int NBLK = HD / 32, REC = HD + 2 * NBLK;
    static constexpr int KT = HD == 128 ? 2 : 1;                 // key tiles (M = 128) per unit
    static constexpr int KEYS = 128 * KT;
    static constexpr int Q_SUB = QN * 128;                       // one 64-dim sub-tile [128 pairs][128 B], 128-byte swizzle
    static constexpr int Q_BYTES = (HD / 64) * Q_SUB;
    static constexpr int QST = HD == 128 ? 4 : 2;                // Q ring
    static constexpr int RAW = 128 * REC;                        // raw records of one key tile
    static constexpr int OFF_RAW = QST * Q_BYTES;
    static constexpr int OFF_NORM = OFF_RAW + KT * RAW;          // -m, then 1 / l, of every pair of the unit's kv head
    static constexpr int OFF_XCH = OFF_NORM + MAX_PAIRS * 8;
    static constexpr int OFF_BAR = OFF_XCH + 128 * 4;
    static constexpr int SMEM = OFF_BAR + 16 * 8 + 16 + 1024;    // + slack to align the base to 1024
    static constexpr int T_LO = HD / 2;                          // columns from the high to the low part of a K tile
    static constexpr int T_D = 256;                              // two accumulators of 128 columns
    static_assert(KT * HD == 256 && SMEM <= 226 * 1024, "tensor and shared memory budget");
};
enum { B_RAWF = 0, B_RAWE = 1, B_KRDY = 2, B_QF = 3, B_QE = 7, B_DF = 11, B_DE = 13, N_CBARS = 15 };

template <int HD>
__global__ void __launch_bounds__(CTHREADS, 1) k_track_chunk(const __grid_constant__ ChunkParams P) {
    using namespace pf;
    using C = ChunkCfg<HD>;
    constexpr int NBLK = C::NBLK, REC = C::REC, KT = C::KT, QST = C::QST;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    float* s_nm = reinterpret_cast<float*>(smem + C::OFF_NORM);
    float* s_il = s_nm + MAX_PAIRS;
    float* s_xch = reinterpret_cast<float*>(smem + C::OFF_XCH);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
    volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(smem + C::OFF_BAR + 16 * 8);    // [0] tmem base, [1] abort
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();
    pdl_trigger();
    const SeqRange sr = seq_range(P.pos, P.kslot, P.act, 0, P.rows, 0, 0, P.pstride, P.n_slots, P.status);
    const int n = sr.hi, p0 = sr.p0, G = P.G, lg = __ffs(G) - 1;         // the group divides 128: a power of two
    const int pairs = P.rows * G, n_qt = (pairs + QN - 1) / QN;
    const int units = sr.active ? (n + C::KEYS - 1) / C::KEYS * P.Hkv : 0;
    if ((int)blockIdx.x >= units) return;
    if (tid == 0) {
        mbar_init(&bars[B_RAWF], 1); mbar_init(&bars[B_RAWE], 8); mbar_init(&bars[B_KRDY], 8);
        for (int i = 0; i < QST; ++i) { mbar_init(&bars[B_QF + i], P.q_f16 ? 1 : W_MMA - W_Q); mbar_init(&bars[B_QE + i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&bars[B_DF + i], 1); mbar_init(&bars[B_DE + i], 4); }
        misc[1] = 0;
        mbar_fence_init();
    }
    if (warp == W_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(const_cast<uint32_t*>(&misc[0]))), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = misc[0];
    // bounded wait that degrades to "do not wait" once any wait has run out
    auto wait = [&](int b, uint32_t parity) {
        if (mbar_try_wait(&bars[b], parity)) return;
        if (misc[1]) return;
        if (!mbar_wait_backoff(&bars[b], parity, 20)) {
            atomicOr(P.status, BATTN_DEV_WAIT_TIMEOUT);
            misc[1] = 1;
        }
    };
    // unit u: keys t0 .. of kv head kvh; rows before Q tile qt0 see none of them
    auto unit_t0 = [&](int u) { return u / P.Hkv * C::KEYS; };
    auto unit_qt0 = [&](int t0) { return max(0, t0 - p0) * G / QN; };
    auto unit_tiles = [&](int t0) { return KT == 1 || t0 + 128 >= n ? 1 : KT; };

    if (warp < 8) {
        // ======================= K operand, then the weights: one thread per key and accumulator ====================
        const int grp = warp >> 2, row = tid & 127;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        uint32_t used = 0, steps = 0, unit = 0;                  // accumulators emptied by this group, products so far, units
        for (int u = blockIdx.x; u < units; u += gridDim.x, ++unit) {
            const int kvh = u % P.Hkv, t0 = unit_t0(u), qt0 = unit_qt0(t0);
            // every product of the previous unit has completed (each group has seen its last one), s_nm, s_il and s_xch are read
            named_bar_sync(1, 256);
            wait(B_RAWF, unit & 1);
            if (KT == 1 || grp < unit_tiles(t0)) {
                // head_dim 128: the group's key tile; 256: its half of the dims of the one tile
                const uint8_t* rec = smem + C::OFF_RAW + (KT == 2 ? grp * C::RAW : 0) + row * REC;
                const int d0 = KT == 2 ? 0 : 128 * grp;
                const uint32_t tk = tmem + lane_base + (KT == 2 ? grp * HD : 0) + d0 / 2;
#pragma unroll 1
                for (int half = 0; half < 2; ++half) {
                    uint32_t hi[32], lo[32];
#pragma unroll
                    for (int c = 0; c < 8; ++c) {                // 8 dims each
                        const int d = d0 + 64 * half + 8 * c;
                        const __half2 s2 = __half2half2(reinterpret_cast<const __half*>(rec)[d >> 5]);
                        const uint32_t su = *reinterpret_cast<const uint32_t*>(&s2);
                        const uint2 w = *reinterpret_cast<const uint2*>(rec + 2 * NBLK + d);
                        const uint32_t x = w.x ^ 0x80808080u, y = w.y ^ 0x80808080u;
                        const uint32_t v[4] = {sub1152(widen_lo(x)), sub1152(widen_hi(x)), sub1152(widen_lo(y)), sub1152(widen_hi(y))};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            hi[4 * c + e] = hmul2_u32(v[e], su);
                            lo[4 * c + e] = hfma2_residual(v[e], su, hi[4 * c + e]);
                        }
                    }
                    tmem_st32(tk + 32 * half, hi);
                    tmem_st32(tk + C::T_LO + 32 * half, lo);
                }
                tmem_st_wait();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) { mbar_arrive(&bars[B_RAWE]); mbar_arrive(&bars[B_KRDY]); }
            // the pairs' normalisers, while the first products run (no pair: weight 0)
            for (int i = tid + qt0 * QN; i < n_qt * QN; i += 256) {
                const float2 nm = i < pairs ? P.norm[(size_t)(i >> lg) * P.Hq + kvh * G + (i & (G - 1))] : make_float2(0.f, 0.f);
                s_nm[i] = -nm.x; s_il[i] = nm.y;
            }
            named_bar_sync(1, 256);
            const int key = t0 + (KT == 2 ? 128 * grp : 0) + row;
            const bool mine = KT == 1 || grp < unit_tiles(t0);
            const uint32_t tD = tmem + lane_base + C::T_D + grp * 128;
            const uint64_t c2p = pack_f2(P.scale_log2, P.scale_log2);
            float w = 0.f;
            for (int qt = qt0; qt < n_qt; ++qt, ++steps) {
                if (KT == 2 ? !mine : (int)(steps & 1) != grp) continue;
                wait(B_DF + grp, used & 1);
                ++used;
                tc_fence_after();
                // pairs of this tile that see the key: index at least (key - p0) G
                const int first = (key - p0) * G - qt * QN;
                const bool masked = t0 + C::KEYS - 1 > p0 + qt * QN / G;
// the whole accumulator into registers, so that the next product can have it back before the exponentials
                uint32_t v[128];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32_nowait(tD + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&v[32 * c]));
                tmem_ld_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars[B_DE + grp]);
                const ulonglong2* nm = reinterpret_cast<const ulonglong2*>(s_nm + qt * QN);
                const float4* il = reinterpret_cast<const float4*>(s_il + qt * QN);
                float a[4] = {0.f, 0.f, 0.f, 0.f};               // sums of 32 terms each: what a long sum would round away
                if (masked) {
#pragma unroll
                    for (int i = 0; i < 128; ++i)
                        if (i < first) v[i] = __float_as_uint(-INFINITY);
                }
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const ulonglong2 l = nm[i];
                    const float4 r = il[i];
                    float e0, e1, e2, e3;
                    ffma2(e0, e1, __uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]), c2p, l.x);
                    ffma2(e2, e3, __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]), c2p, l.y);
                    a[0] = fmaf(fast_exp2(e0), r.x, a[0]); a[1] = fmaf(fast_exp2(e1), r.y, a[1]);
                    a[2] = fmaf(fast_exp2(e2), r.z, a[2]); a[3] = fmaf(fast_exp2(e3), r.w, a[3]);
                }
                w += (a[0] + a[1]) + (a[2] + a[3]);
            }
            if (KT == 1) {                                       // the two groups share the keys
                if (grp == 1) s_xch[row] = w;
                named_bar_sync(1, 256);
                if (grp == 0) w += s_xch[row];
            }
            if ((KT == 2 ? mine : grp == 0) && key < n) {
                const size_t at = ((size_t)sr.slot * P.Hkv + kvh) * P.pstride + key;
                if (P.in && key < p0) w += P.in[at];             // the call's own positions start from nothing
                P.out[at] = w;
            }
        }
    } else if (warp < W_MMA) {
        // ======================= Q tiles: [pair][dim], 64-dim sub-tiles, 128-byte swizzle ================================
        uint32_t cnt = 0;
        if (P.q_f16) {
            // one box of the queries' tensor map per sub-tile: 128 / G rows of G heads of 64 dims, zeros past the last row
            if (warp == W_Q && lane == 0) {
                for (int u = blockIdx.x; u < units; u += gridDim.x) {
                    const int kvh = u % P.Hkv;
                    for (int qt = unit_qt0(unit_t0(u)); qt < n_qt; ++qt, ++cnt) {
                        const int st = cnt % QST;
                        if (cnt >= QST) wait(B_QE + st, (cnt / QST - 1) & 1);
                        mbar_expect_tx(&bars[B_QF + st], C::Q_BYTES);
#pragma unroll
                        for (int sub = 0; sub < HD / 64; ++sub)
                            tensor_g2s(smem + st * C::Q_BYTES + sub * C::Q_SUB, &P.q_map, 64 * sub, kvh * G, qt * (QN >> lg), &bars[B_QF + st]);
                    }
                }
            }
        } else {
            // fp32 queries are rounded on the way: thread t has 16-byte chunk `ch` of every PSTEP-th pair
            constexpr int PSTEP = (W_MMA - W_Q) * 32 / (HD / 8);
            const int t = tid - W_Q * 32, ch = t & (HD / 8 - 1), pr0 = t / (HD / 8);
            for (int u = blockIdx.x; u < units; u += gridDim.x) {
                const int kvh = u % P.Hkv;
                for (int qt = unit_qt0(unit_t0(u)); qt < n_qt; ++qt, ++cnt) {
                    const int st = cnt % QST;
                    if (cnt >= QST) wait(B_QE + st, (cnt / QST - 1) & 1);
                    uint8_t* dst = smem + st * C::Q_BYTES + (ch >> 3) * C::Q_SUB;
#pragma unroll 4
                    for (int pr = pr0; pr < QN; pr += PSTEP) {
                        const int pair = qt * QN + pr;
                        uint4 w = make_uint4(0u, 0u, 0u, 0u);
                        if (pair < pairs) {
                            const float* src = reinterpret_cast<const float*>(P.q) +
                                               ((size_t)(pair >> lg) * P.Hq + kvh * G + (pair & (G - 1))) * HD + ch * 8;
                            const float4 x = *reinterpret_cast<const float4*>(src), y = *reinterpret_cast<const float4*>(src + 4);
                            w = make_uint4(pack_h2(x.x, x.y), pack_h2(x.z, x.w), pack_h2(y.x, y.y), pack_h2(y.z, y.w));
                        }
                        *reinterpret_cast<uint4*>(dst + sw128(pr, ch & 7)) = w;
                    }
                    proxy_fence();                               // hand it to the tensor core's proxy
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bars[B_QF + st]);
                }
            }
        }
    } else if (warp == W_MMA) {
        // ======================= the products ============================================================================
        if (lane == 0) {
            const uint32_t id = umma_idesc(128, QN);
            const uint64_t qd0 = umma_desc(smem_u32(smem));
            uint32_t cnt = 0, unit = 0, filled[2] = {0, 0};
            for (int u = blockIdx.x; u < units; u += gridDim.x, ++unit) {
                const int t0 = unit_t0(u), tiles = unit_tiles(t0);
                wait(B_KRDY, unit & 1);
                for (int qt = unit_qt0(t0); qt < n_qt; ++qt, ++cnt) {
                    wait(B_QF + cnt % QST, (cnt / QST) & 1);
                    const uint64_t qd = qd0 + (uint64_t)((cnt % QST) * (C::Q_BYTES >> 4));
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt) {
                        if (kt >= tiles) break;
                        const int b = KT == 2 ? kt : (int)(cnt & 1);
                        const uint32_t f = b ? filled[1] : filled[0];
                        if (f > 0) wait(B_DE + b, (f - 1) & 1);
                        tc_fence_after();
                        const uint32_t d = tmem + C::T_D + b * 128, ka = tmem + kt * HD;
#pragma unroll
                        for (int part = 1; part >= 0; --part)    // the low part first, see above
#pragma unroll
                            for (int ks = 0; ks < HD / 16; ++ks)
                                umma_f16_ts(d, ka + part * C::T_LO + 8 * ks, qd + (uint64_t)((ks >> 2) * (C::Q_SUB >> 4) + 2 * (ks & 3)),
                                            id, part == 0 || ks > 0);
                        umma_commit(&bars[B_DF + b]);
                        if (b) ++filled[1]; else ++filled[0];
                    }
                    umma_commit(&bars[B_QE + cnt % QST]);
                }
            }
        }
    } else if (lane == 0) {
        // ======================= raw K records, one unit ahead ================================================================
        uint32_t unit = 0;
        for (int u = blockIdx.x; u < units; u += gridDim.x, ++unit) {
            const int kvh = u % P.Hkv, t0 = unit_t0(u), tiles = unit_tiles(t0);
            if (unit > 0) wait(B_RAWE, (unit - 1) & 1);
            uint32_t bytes = 0;
            for (int kt = 0; kt < tiles; ++kt) bytes += (uint32_t)min(128, P.pstride - t0 - 128 * kt) * REC;
            mbar_expect_tx(&bars[B_RAWF], bytes);
            for (int kt = 0; kt < tiles; ++kt) {
                const int key = t0 + 128 * kt;
                bulk_g2s(smem + C::OFF_RAW + kt * C::RAW, P.kvk + kv_rec_index(P.pg, sr.slot, kvh, P.Hkv, P.pstride, key, P.status) * (size_t)REC,
                         (uint32_t)min(128, P.pstride - key) * REC, &bars[B_RAWF]);
            }
        }
    }
    __syncthreads();
    if (warp == W_MMA) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

}  // namespace tr
}  // namespace battn
