// Eviction from a full-causal cache by accumulated attention weight: per (sequence, kv head) the records of the first n_sink
// and the last n_recent positions and of the best-scored ones between them stay, in their order, moved to the front.
//
// Two launches.  k_evict_select finds which positions stay: an exact selection of the m best of n scores by a radix descent
// over the scores as ordered 32-bit integers (11 + 11 + 10 bits), then one ordered pass that writes the list.  One cluster
// per (sequence, kv head); the scores are read from HBM once and stay in shared memory as keys.  k_evict_move carries the
// records: one cluster per (sequence, kv head, K|V).  Because the order is kept, the j-th record that stays comes from a
// position >= j, so the move works in place with nothing but an order between rounds: a round covers the next `round`
// target positions of the whole cluster, loads all of its sources into shared memory, and stores after a cluster barrier.
// What it overwrites lies below the targets of the next round, and the sources of every later round lie at or above them.
#pragma once
#include <cooperative_groups.h>

#include "common.cuh"

namespace battn {
namespace ev {

constexpr int MAX_CLUSTER = 8;              // the portable limit
constexpr int SEL_THREADS = 1024, MOVE_THREADS = 256;
constexpr int KEYS_SMEM = 40 * 1024;        // keys a CTA keeps in shared memory (160 KB); a longer share re-reads the rest
constexpr int BINS = 2048;

struct Params {
    uint8_t* kvk;
    uint8_t* kvv;
    float* score;        // [partition or table row][kv head][pstride]
    int* kept;           // [n_seq][kv head][budget]
    int* pos_out;
    int* plan;           // workspace: records that stay of sequence i, -1: nothing to do
    const int* pos;
    const int* kslot;
    const int* kslot_dst;
    const int* act;
    int n_seq, budget, n_sink, n_recent;
    int Hkv, pstride, n_slots;
    int* status;
    Paging pg;
};

// Scores as integers of the same order: NaN below everything, the two zeros alike.
__device__ __forceinline__ uint32_t ordered(float f) {
    if (f != f) return 0u;
    const uint32_t u = __float_as_uint(f + 0.f);
    return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}

// Block-wide exclusive scan of one value per thread; `total` is the block's sum.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* s_warp, uint32_t& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += t;
    }
    __syncthreads();                                 // the previous scan's sums have been read
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    uint32_t w = s_warp[lane];                       // 32 warps
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += t;
    }
    total = __shfl_sync(0xffffffffu, w, 31);
    const uint32_t before = __shfl_sync(0xffffffffu, w, warp == 0 ? 0 : warp - 1);
    return x - v + (warp ? before : 0u);
}

__global__ void __launch_bounds__(SEL_THREADS, 1) k_evict_select(const Params P) {
    namespace cg = cooperative_groups;
    extern __shared__ uint32_t s_key[];              // KEYS_SMEM keys of this CTA's share
    __shared__ uint32_t s_hist[BINS], s_warp[32];
    __shared__ uint32_t s_bin, s_above, s_gt, s_eq;
    __shared__ int s_clash;
    const cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int i = blockIdx.x / C, kvh = blockIdx.y, tid = threadIdx.x;
    if (tid == 0) s_clash = 0;
    pdl_wait();
    pdl_trigger();
    __syncthreads();
    // ---- what the call asks of this sequence; every thread of the cluster finds the same ------------------------
    const bool idle = P.act && P.act[i] == 0;
    const int n = P.pos[i], src = P.kslot ? P.kslot[i] : 0, dst = P.kslot_dst ? P.kslot_dst[i] : src;
    bool bad = n < 0 || n > P.pstride || src < 0 || dst < 0 || (P.kslot && (src >= P.n_slots || dst >= P.n_slots));
    // a target that another sequence of the call reads or writes would be overwritten while it is read
    for (int j = tid; j < P.n_seq; j += SEL_THREADS) {
        if (j == i || (P.act && P.act[j] == 0)) continue;
        const int sj = P.kslot ? P.kslot[j] : 0, dj = P.kslot_dst ? P.kslot_dst[j] : sj;
        if (dj == dst || sj == dst) s_clash = 1;
    }
    __syncthreads();
    bad = bad || s_clash;
    const int stay = min(n, P.budget);
    if (kvh == 0 && rank == 0 && tid == 0) {
        P.plan[i] = idle || bad ? -1 : stay;
        if (bad && !idle) atomicOr(P.status, BATTN_DEV_BAD_POSITION);
    }
    if (idle || bad) return;                         // the whole cluster

    int* kept = P.kept + ((size_t)i * P.Hkv + kvh) * P.budget;
    const int gtid = rank * SEL_THREADS + tid, gthreads = C * SEL_THREADS;
    if (n <= P.budget) {
        for (int j = gtid; j < P.budget; j += gthreads) kept[j] = j < n ? j : -1;
        return;
    }
    for (int j = gtid; j < P.n_sink; j += gthreads) kept[j] = j;
    for (int j = gtid; j < P.n_recent; j += gthreads) kept[P.budget - P.n_recent + j] = n - P.n_recent + j;
    const int cand = n - P.n_sink - P.n_recent, m = P.budget - P.n_sink - P.n_recent;
    if (m == 0) return;
    // ---- this CTA's share of the candidates, as keys ---------------------------------------------------------------
    const float* score = P.score + ((size_t)src * P.Hkv + kvh) * P.pstride + P.n_sink;
    const int per = ((cand + C - 1) / C + 3) & ~3;
    const int a = min(rank * per, cand), len = min(per, cand - a);
    score += a;
    for (int j = tid; j < min(len, KEYS_SMEM); j += SEL_THREADS) s_key[j] = ordered(score[j]);
    auto key = [&](int j) { return j < KEYS_SMEM ? s_key[j] : ordered(score[j]); };

    // ---- the m-th best key, 11 + 11 + 10 bits --------------------------------------------------------------------------
    uint32_t prefix = 0, need = (uint32_t)m;
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11, bins = 1 << bits;
        for (int b = tid; b < bins; b += SEL_THREADS) s_hist[b] = 0;
        __syncthreads();
        for (int j = tid; j < len; j += SEL_THREADS) {
            const uint32_t k = key(j);
            if (pass == 0 || (k >> (shift + bits)) == prefix) atomicAdd(&s_hist[(k >> shift) & (bins - 1)], 1u);
        }
        cl.sync();
        // from the highest bin down: thread t adds up bins - 1 - per_t * t ...
        const int per_t = bins / SEL_THREADS;
        uint32_t c[2] = {0, 0};
        for (int r = 0; r < C; ++r) {
            const uint32_t* h = cl.map_shared_rank(s_hist, r);
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (e < per_t) c[e] += h[bins - 1 - per_t * tid - e];
        }
        uint32_t tot, before = block_scan(c[0] + c[1], s_warp, tot);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if (e < per_t && before < need && before + c[e] >= need) { s_bin = bins - 1 - per_t * tid - e; s_above = before; }
            before += c[e];
        }
        cl.sync();                                   // every CTA has read this one's counts
        prefix = (prefix << bits) | s_bin;
        need -= s_above;
    }
    // ---- better than the m-th, or equal and among the first `need` equal ones: the list, in order -----------------------
    const uint32_t T = prefix;
    if (tid == 0) { s_gt = 0; s_eq = 0; }
    __syncthreads();
    uint32_t gt = 0, eq = 0;
    for (int j = tid; j < len; j += SEL_THREADS) {
        const uint32_t k = key(j);
        gt += k > T; eq += k == T;
    }
    gt = __reduce_add_sync(0xffffffffu, gt);
    eq = __reduce_add_sync(0xffffffffu, eq);
    if ((tid & 31) == 0) { atomicAdd(&s_gt, gt); atomicAdd(&s_eq, eq); }
    cl.sync();
    uint32_t gt0 = 0, eq0 = 0;
    for (int r = 0; r < rank; ++r) { gt0 += *cl.map_shared_rank(&s_gt, r); eq0 += *cl.map_shared_rank(&s_eq, r); }
    kept += P.n_sink;
    for (int base = 0; base < len; base += 4 * SEL_THREADS) {
        uint32_t k[4], mine = 0;                     // two counts of 16 bits: better, equal
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int j = base + 4 * tid + e;
            k[e] = j < len ? key(j) : 0u;
            if (j < len) mine += (k[e] > T ? 0x10000u : 0u) + (k[e] == T ? 1u : 0u);
        }
        uint32_t tot;
        const uint32_t at = block_scan(mine, s_warp, tot);
        uint32_t g = gt0 + (at >> 16), q = eq0 + (at & 0xFFFFu);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int j = base + 4 * tid + e;
            if (j >= len) break;
            if (k[e] > T) { kept[g + min(q, need)] = P.n_sink + a + j; ++g; }
            else if (k[e] == T) { if (q < need) kept[g + q] = P.n_sink + a + j; ++q; }
        }
        gt0 += tot >> 16; eq0 += tot & 0xFFFFu;
    }
    cl.sync();                                       // this CTA's counts are read by the others
}

template <int HD>
struct MoveCfg {
    static constexpr int REC = HD + HD / 16, WORDS = REC / 8;
    static constexpr int ROUND = HD == 128 ? 512 : 256;          // records of a CTA in a round
    static constexpr int SMEM = ROUND * (REC + 8 + 4);           // records, source offsets, scores
};

__device__ __forceinline__ void copy8_async(void* dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

template <int HD>
__global__ void __launch_bounds__(MOVE_THREADS) k_evict_move(const Params P) {
    using C = MoveCfg<HD>;
    namespace cg = cooperative_groups;
    extern __shared__ __align__(16) uint8_t smem[];
    uint2* s_rec = reinterpret_cast<uint2*>(smem);
    long long* s_off = reinterpret_cast<long long*>(smem + C::ROUND * C::REC);      // byte offset of the source, -1: stays
    float* s_score = reinterpret_cast<float*>(s_off + C::ROUND);
    const cg::cluster_group cl = cg::this_cluster();
    const int nb = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int i = blockIdx.x / nb, kvh = blockIdx.y, tid = threadIdx.x;
    const bool isv = blockIdx.z != 0;
    pdl_wait();
    pdl_trigger();
    const int stay = P.plan[i];
    if (stay < 0) return;
    if (kvh == 0 && !isv && rank == 0 && tid == 0) P.pos_out[i] = stay;
    const int src = P.kslot ? P.kslot[i] : 0, dst = P.kslot_dst ? P.kslot_dst[i] : src;
    const int* kept = P.kept + ((size_t)i * P.Hkv + kvh) * P.budget;
    uint8_t* cache = isv ? P.kvv : P.kvk;
    float* sc_src = P.score + ((size_t)src * P.Hkv + kvh) * P.pstride;
    float* sc_dst = P.score + ((size_t)dst * P.Hkv + kvh) * P.pstride;
    for (int j0 = 0; j0 < stay; j0 += nb * C::ROUND) {
        const int first = j0 + rank * C::ROUND, cnt = max(0, min(C::ROUND, stay - first));
        for (int r = tid; r < cnt; r += MOVE_THREADS) {
            const int from = kept[first + r];
            const bool same = from == first + r && src == dst;
            s_off[r] = same ? -1 : (long long)(kv_rec_index(P.pg, src, kvh, P.Hkv, P.pstride, from, P.status) * (size_t)C::REC);
            if (!isv && !same) s_score[r] = sc_src[from];
        }
        __syncthreads();
        for (int w = tid; w < cnt * C::WORDS; w += MOVE_THREADS) {
            const int r = w / C::WORDS, c = w - r * C::WORDS;
            if (s_off[r] >= 0) copy8_async(&s_rec[w], cache + s_off[r] + 8 * c);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        cl.sync();                                   // every source of this round has been read
        for (int w = tid; w < cnt * C::WORDS; w += MOVE_THREADS) {
            const int r = w / C::WORDS, c = w - r * C::WORDS;
            if (s_off[r] < 0) continue;
            const size_t to = kv_rec_index(P.pg, dst, kvh, P.Hkv, P.pstride, first + r, P.status) * (size_t)C::REC;
            *reinterpret_cast<uint2*>(cache + to + 8 * c) = s_rec[w];
        }
        if (!isv)
            for (int r = tid; r < cnt; r += MOVE_THREADS)
                if (s_off[r] >= 0) sc_dst[first + r] = s_score[r];
        __syncthreads();                             // the buffers are free again
    }
}

}  // namespace ev
}  // namespace battn
