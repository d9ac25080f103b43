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
#include "common.cuh"

namespace battn {
namespace ev {

constexpr int MAX_CLUSTER = 8;              // the portable limit
constexpr int MOVE_THREADS = 512;           // 256 where several CTAs share an SM
constexpr int KEYS_SMEM = 40 * 1024;        // keys a CTA keeps in shared memory at most (160 KB); a longer share re-reads the rest
// Candidates that are worth another CTA of the cluster: up to here a pass over them is shorter than the cluster barriers
// (4160 positions, one CTA of eight: 23 -> 10 us)
constexpr int KEYS_PER_CTA = 8192;
constexpr int MATCHES = 2048;               // keys of the first pass's bin that are listed

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
    int cluster;         // CTAs per cluster of this launch
    int keys;            // k_evict_select: keys its shared memory holds
    int round, bufs;     // k_evict_move: records of a CTA in a round, buffers of that many
    int* status;
    Paging pg;
};

// Cluster barriers (CTAs that have left count as arrived) and reads of another CTA's shared memory.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() { cluster_arrive(); cluster_wait(); }
template <int N>
__device__ __forceinline__ void load_rank(const uint32_t* p, int r, uint32_t (&v)[N]) {
    uint32_t ra;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(smem_u32(p)), "r"(r));
    if constexpr (N == 4) asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(ra) : "memory");
    else if constexpr (N == 2) asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(ra) : "memory");
    else                  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v[0]) : "r"(ra) : "memory");
}

// Scores as integers of the same order: NaN below everything, the two zeros alike.
__device__ __forceinline__ uint32_t ordered(float f) {
    if (f != f) return 0u;
    const uint32_t u = __float_as_uint(f + 0.f);
    return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}

// Block-wide exclusive scan of one value per thread; `total` is the block's sum.
template <int THREADS>
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
    uint32_t w = lane < THREADS / 32 ? s_warp[lane] : 0u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += t;
    }
    total = __shfl_sync(0xffffffffu, w, 31);
    const uint32_t before = __shfl_sync(0xffffffffu, w, warp == 0 ? 0 : warp - 1);
    return x - v + (warp ? before : 0u);
}

// One pass of the descent over BITS bits at SHIFT.  `hist` holds this CTA's counts of the keys that match the prefix so
// far; every CTA adds up the cluster's counts itself and finds the same bin.  Counts of the CTAs before this one are kept
// too: above the bin they end up in `gt_low`, in the last pass the bin's own are `eq_low`.
template <int THREADS, int SHIFT, int BITS>
__device__ __forceinline__ void descend(uint32_t* hist, int C, int rank, uint32_t* s_warp, volatile uint32_t* s_found,
                                        uint32_t& prefix, uint32_t& need, uint32_t& gt_low, uint32_t& eq_low) {
    constexpr int PER = (1 << BITS) / THREADS;                   // bins per thread, from the highest down
    const int top = (1 << BITS) - PER * ((int)threadIdx.x + 1);  // lowest of this thread's bins
    uint32_t c[PER], low[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) c[e] = low[e] = 0;
    if (C > 1) {
        cluster_sync();
#pragma unroll
        for (int r = 0; r < MAX_CLUSTER; ++r) {
            if (r >= C) break;
            uint32_t v[PER];
            load_rank<PER>(hist + top, r, v);
#pragma unroll
            for (int e = 0; e < PER; ++e) { c[e] += v[e]; low[e] += r < rank ? v[e] : 0u; }
        }
    } else {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < PER; ++e) c[e] = hist[top + e];
    }
    uint32_t sum = 0, tot;
#pragma unroll
    for (int e = 0; e < PER; ++e) sum += c[e];
    uint32_t before = block_scan<THREADS>(sum, s_warp, tot);
#pragma unroll
    for (int e = PER - 1; e >= 0; --e) {
        if (before < need && before + c[e] >= need) { s_found[0] = top + e; s_found[1] = before; }
        before += c[e];
    }
    __syncthreads();
    const uint32_t bin = s_found[0];
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        if (top + e > (int)bin) gt_low += low[e];
        if (SHIFT == 0 && top + e == (int)bin) eq_low += low[e];
    }
    prefix = (prefix << BITS) | bin;
    need -= s_found[1];
}

// SEL_THREADS: 1024 for few clusters, where a pass over the keys is the time; 512 once they outnumber the SMs, so that three
// CTAs share one (32 sequences of up to 8192: 20 -> 14 us).  That holds where a partition has room for 11,000 positions or fewer: the
// host sizes the keys by the partition, up to 160 KB, and from about 21,000 positions on one CTA of 512 has the SM to itself
// (the whole call on 32 sequences of up to 8192 moved elsewhere: 81 us in partitions of 8192, 87 of 32768, 89 of 131072; in
// place 72, 78, 79).
template <int SEL_THREADS>
__global__ void __launch_bounds__(SEL_THREADS, 1024 / SEL_THREADS) k_evict_select(const Params P) {
    extern __shared__ __align__(16) uint32_t s_key[];            // P.keys keys of this CTA's share
    __shared__ __align__(16) uint32_t s_hist[2048 + 2048 + 1024];
    __shared__ uint32_t s_warp[32], s_found[3][2], s_low[2], s_match, s_list[MATCHES];
    __shared__ int s_clash;
    const int CL = P.cluster, rank = (int)blockIdx.x % CL;
    const int i = blockIdx.x / CL, kvh = blockIdx.y, tid = threadIdx.x;
    for (int b = tid; b < 2048 + 2048 + 1024; b += SEL_THREADS) s_hist[b] = 0;
    if (tid == 0) { s_clash = 0; s_match = 0; s_low[0] = s_low[1] = 0; }
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
    // ... and so would page 0 be in the place of a page that is not mapped
    if (P.pg.table && !bad) {
        const int from = (n + (1 << P.pg.shift) - 1) >> P.pg.shift, to = (min(n, P.budget) + (1 << P.pg.shift) - 1) >> P.pg.shift;
        for (int j = tid; j < from + to; j += SEL_THREADS) {
            const int e = P.pg.table[(size_t)(j < from ? src : dst) * P.pg.max_pages + (j < from ? j : j - from)];
            if ((unsigned)e >= (unsigned)P.pg.n_pages) s_clash = 1;
        }
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
    const int gtid = rank * SEL_THREADS + tid, gthreads = CL * SEL_THREADS;
    if (n <= P.budget) {
        for (int j = gtid; j < P.budget; j += gthreads) kept[j] = j < n ? j : -1;
        return;
    }
    for (int j = gtid; j < P.n_sink; j += gthreads) kept[j] = j;
    for (int j = gtid; j < P.n_recent; j += gthreads) kept[P.budget - P.n_recent + j] = n - P.n_recent + j;
    const int cand = n - P.n_sink - P.n_recent, m = P.budget - P.n_sink - P.n_recent;
    if (m == 0) return;
    // ---- this CTA's share of the candidates, as keys; CTAs that are not needed leave (barriers count who is left) -----
    const int C = min(CL, (cand + KEYS_PER_CTA - 1) / KEYS_PER_CTA);
    if (rank >= C) return;
    const int per = ((cand + C - 1) / C + 3) & ~3;
    const int a = min(rank * per, cand), len = min(per, cand - a);
    const float* score = P.score + ((size_t)src * P.Hkv + kvh) * P.pstride + P.n_sink + a;
    const int held = min(len, P.keys);
    auto key = [&](int j) { return j < held ? s_key[j] : ordered(__ldg(score + j)); };
    constexpr int UN = 8;
    for (int j0 = tid; j0 < len; j0 += UN * SEL_THREADS) {       // the scores' one trip, and the first pass's counts
        float v[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) v[u] = j0 + u * SEL_THREADS < len ? __ldg(score + j0 + u * SEL_THREADS) : 0.f;
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int j = j0 + u * SEL_THREADS;
            if (j < len) {
                const uint32_t k = ordered(v[u]);
                if (j < held) s_key[j] = k;
                atomicAdd(&s_hist[k >> 21], 1u);
            }
        }
    }
    // ---- the m-th best key ------------------------------------------------------------------------------------------------
    uint32_t T = 0, need = (uint32_t)m, gt_low = 0, eq_low = 0;
    descend<SEL_THREADS, 21, 11>(s_hist, C, rank, s_warp, s_found[0], T, need, gt_low, eq_low);
    // one more look at every key; the third pass only needs those that matched, as long as their list has room
    for (int j0 = 4 * tid; j0 < len; j0 += 4 * SEL_THREADS) {
        uint4 k4;
        if (j0 + 4 <= held) k4 = *reinterpret_cast<const uint4*>(s_key + j0);
        else k4 = make_uint4(key(j0), j0 + 1 < len ? key(j0 + 1) : 0u, j0 + 2 < len ? key(j0 + 2) : 0u, j0 + 3 < len ? key(j0 + 3) : 0u);
        const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if ((k[e] >> 21) == T && j0 + e < len) {
                atomicAdd(&s_hist[2048 + ((k[e] >> 10) & 2047)], 1u);
                const uint32_t at = atomicAdd(&s_match, 1u);
                if (at < MATCHES) s_list[at] = k[e];
            }
    }
    descend<SEL_THREADS, 10, 11>(s_hist + 2048, C, rank, s_warp, s_found[1], T, need, gt_low, eq_low);
    const bool listed = s_match <= MATCHES;
    for (int j = tid; j < (listed ? (int)s_match : len); j += SEL_THREADS) {
        const uint32_t k = listed ? s_list[j] : key(j);
        if ((k >> 10) == T) atomicAdd(&s_hist[4096 + (k & 1023)], 1u);
    }
    descend<SEL_THREADS, 0, 10>(s_hist + 4096, C, rank, s_warp, s_found[2], T, need, gt_low, eq_low);
    if (C > 1) cluster_arrive();                                 // this CTA reads no other's counts any more
    // ---- better than the m-th, or equal and among the first `need` equal ones: the list, in order -----------------------
    uint32_t gt0 = 0, eq0 = 0;
    if (C > 1) {
        gt_low = __reduce_add_sync(0xffffffffu, gt_low);
        eq_low = __reduce_add_sync(0xffffffffu, eq_low);
        if ((tid & 31) == 0) { atomicAdd(&s_low[0], gt_low); atomicAdd(&s_low[1], eq_low); }
        __syncthreads();
        gt0 = s_low[0]; eq0 = s_low[1];
    }
    kept += P.n_sink;
    for (int base = 0; base < len; base += 4 * SEL_THREADS) {
        const int j0 = base + 4 * tid;
        uint32_t k[4], mine = 0;                     // two counts of 16 bits: better, equal
        if (j0 + 4 <= held) {
            const uint4 k4 = *reinterpret_cast<const uint4*>(s_key + j0);
            k[0] = k4.x; k[1] = k4.y; k[2] = k4.z; k[3] = k4.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) k[e] = j0 + e < len ? key(j0 + e) : 0u;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (j0 + e < len) mine += (k[e] > T ? 0x10000u : 0u) + (k[e] == T ? 1u : 0u);
        }
        uint32_t tot;
        const uint32_t at = block_scan<SEL_THREADS>(mine, s_warp, tot);
        uint32_t g = gt0 + (at >> 16), q = eq0 + (at & 0xFFFFu);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (j0 + e >= len) break;
            if (k[e] > T) { kept[g + min(q, need)] = P.n_sink + a + j0 + e; ++g; }
            else if (k[e] == T) { if (q < need) kept[g + q] = P.n_sink + a + j0 + e; ++q; }
        }
        gt0 += tot >> 16; eq0 += tot & 0xFFFFu;
    }
    if (C > 1) cluster_wait();                       // the others have read this CTA's counts
}

// A round of a CTA: P.round records, chosen by the host: all of the CTA's part in one round when there are few clusters (the
// SM has the room, and a round costs two trips to memory one after the other: 4096 records of 272 bytes, 15 -> 11 us),
// half of it where the clusters would not all be resident at one CTA per SM (about nine of eight CTAs are: 16 clusters of 151 KB
// ran in two waves, 22 us instead of 19), otherwise 34 KB, so that several CTAs share an SM and two buffers overlap the rounds.
template <int HD>
struct MoveCfg {
    static constexpr int REC = HD + HD / 16, WORDS = REC / 8;
    static constexpr int PER = REC + 8 + 4;                      // bytes of a record's slot: record, source offset, score
    static constexpr int ROUND = HD == 128 ? 256 : 128;
    static constexpr int ROUND_MAX = 200 * 1024 / PER & ~7;      // one buffer that fills the SM, or half of it
    static constexpr int ROUND_HALF = 108 * 1024 / PER & ~7;
};

__device__ __forceinline__ void copy8_async(void* dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4_async(void* dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

// Sources are fetched in pieces of 8 bytes: a record of 136 bytes starts on 8, one of 272 (head_dim 256) would allow 16.
// Targets are one run of 16-byte pieces per round and page.
template <int HD>
__global__ void __launch_bounds__(MOVE_THREADS) k_evict_move(const Params P) {
    using C = MoveCfg<HD>;
    extern __shared__ __align__(16) uint8_t smem[];              // per buffer: records, source offsets, scores
    const int round = P.round, buf_bytes = P.bufs == 2 ? round * C::PER : 0;    // (a multiple of 8 records: 16-byte aligned parts)
    const int nb = P.cluster, rank = (int)blockIdx.x % nb;
    const int i = blockIdx.x / nb, kvh = blockIdx.y, tid = threadIdx.x, nt = blockDim.x;
    const bool isv = blockIdx.z != 0;
    pdl_wait();
    pdl_trigger();
    const int stay = P.plan[i];
    if (stay < 0) return;
    if (kvh == 0 && !isv && rank == 0 && tid == 0) P.pos_out[i] = stay;
    const int src = P.kslot ? P.kslot[i] : 0, dst = P.kslot_dst ? P.kslot_dst[i] : src;
    const int* kept = P.kept + ((size_t)i * P.Hkv + kvh) * P.budget;
    uint8_t* cache = isv ? P.kvv : P.kvk;
    const float* sc_src = P.score + ((size_t)src * P.Hkv + kvh) * P.pstride;
    float* sc_dst = P.score + ((size_t)dst * P.Hkv + kvh) * P.pstride;
    const int rounds = (stay + nb * round - 1) / (nb * round);
    // loads of a round into its buffer; false where every record of this CTA's part is where it belongs already
    auto load = [&](int rd) {
        const int first = (rd * nb + rank) * round, cnt = max(0, min(round, stay - first));
        uint8_t* buf = smem + (rd & 1) * buf_bytes;
        long long* off = reinterpret_cast<long long*>(buf + round * C::REC);
        bool moves = false;
        constexpr int UN = 4;
        for (int r0 = tid; r0 < cnt; r0 += UN * nt) {            // the list and then the table are trips to memory: UN at once
            int from[UN], page[UN];
#pragma unroll
            for (int u = 0; u < UN; ++u) from[u] = r0 + u * nt < cnt ? __ldg(kept + first + r0 + u * nt) : 0;
#pragma unroll
            for (int u = 0; u < UN; ++u)
                page[u] = P.pg.table ? __ldg(P.pg.table + (size_t)src * P.pg.max_pages + (from[u] >> P.pg.shift)) : 0;
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const int r = r0 + u * nt;
                if (r >= cnt) break;
                moves |= from[u] != first + r || src != dst;
                off[r] = (long long)((P.pg.table ? kv_rec_index_page(P.pg, page[u], kvh, P.Hkv, from[u], P.status)
                                                 : ((size_t)src * P.Hkv + kvh) * P.pstride + from[u]) * (size_t)C::REC);
                if (!isv) copy4_async(buf + round * (C::REC + 8) + 4 * r, sc_src + from[u]);
            }
        }
        moves = __syncthreads_or(moves);
        if (moves)
#pragma unroll 4
            for (int w = tid; w < cnt * C::WORDS; w += nt) {
                const int r = w / C::WORDS, c = w - r * C::WORDS;
                copy8_async(buf + 8 * w, cache + off[r] + 8 * c);
            }
        asm volatile("cp.async.commit_group;" ::: "memory");
        return moves;
    };
    bool moves = load(0);
    for (int rd = 0; rd < rounds; ++rd) {
        bool next = false;
        if (P.bufs == 2) {
            if (rd + 1 < rounds) next = load(rd + 1);            // what is stored below lies under every source of this round
            else asm volatile("cp.async.commit_group;" ::: "memory");
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        if (nb > 1) cluster_sync(); else __syncthreads();        // every source of round rd has been read
        if (moves) {
            const int first = (rd * nb + rank) * round, cnt = min(round, stay - first);
            const uint8_t* buf = smem + (rd & 1) * buf_bytes;
#pragma unroll 4
            for (int w = tid; w < cnt * C::REC / 16; w += nt) {
                // (an odd last record leaves a half piece, stored below; a piece never spans two pages)
                const int r = 16 * w / C::REC;
                uint8_t* to = cache + kv_rec_index(P.pg, dst, kvh, P.Hkv, P.pstride, first + r, P.status) * (size_t)C::REC +
                              (16 * w - r * C::REC);
                *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(buf + 16 * w);
            }
            if (tid == 0 && (cnt * C::REC & 8)) {
                const int at = cnt * C::REC - 8;
                uint8_t* to = cache + kv_rec_index(P.pg, dst, kvh, P.Hkv, P.pstride, first + cnt - 1, P.status) * (size_t)C::REC +
                              (C::REC - 8);
                *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(buf + at);
            }
            if (!isv)
                for (int r = tid; r < cnt; r += nt)
                    sc_dst[first + r] = reinterpret_cast<const float*>(buf + round * (C::REC + 8))[r];
        }
        __syncthreads();                             // the buffer is free again
        if (P.bufs == 1 && rd + 1 < rounds) next = load(rd + 1);
        moves = next;
    }
}

}  // namespace ev
}  // namespace battn
