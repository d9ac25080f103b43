// The weights of an attention call, accumulated per cached position: score_out[kv head][p] = score_in[kv head][p] + the sum
// over the call's rows and the heads of the group of w = 2^(s - lse), where s is the row's score of key p in log2 units and
// lse its log-sum-exp.  The attention kernels (VAR_TRACK) leave what is needed for lse, with denominators summed in fp32
// from unrounded weights.
//
// k_track_step, one row per sequence: the decode kernel kept the scores (16 bytes per position and kv head at four heads,
// beside the 272 bytes of K and V it streams), so the cache is not read again; a thread owns a position.
// k_track_chunk, a prompt chunk: the scores are formed a second time, S^T = K Q^T with the keys on the MMA rows, so that a
// thread holds all rows of its keys in turn and the sum over rows stays in its registers; only K is read.
#pragma once
#include "common.cuh"
#include "work_cut.h"

namespace battn {
namespace tr {

constexpr int TILE = 64;                    // tiles of the decode kernel's scores
constexpr int STEP_THREADS = 256;

struct StepParams {
    const int* hdr;          // the decode kernel's header, records and scores
    const float* part;
    const float* scores;
    float* out;              // score_out, [partition or table row][kv head][stride]
    const float* in;         // score_in, or null: nothing accumulated yet
    const int* pos;
    const int* kslot;
    int n_seq, Hkv, G, HD, cph;
    size_t stride;
};

__global__ void __launch_bounds__(STEP_THREADS) k_track_step(const StepParams P) {
    extern __shared__ int s_cum[];                               // [n_seq + 1]
    __shared__ float s_lse[8];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_wait();
    pdl_trigger();
    for (int i = tid; i <= P.n_seq; i += STEP_THREADS) s_cum[i] = P.hdr[2 + i];
    const int per_cta = P.hdr[0];
    __syncthreads();
    const int total = P.Hkv * s_cum[P.n_seq];
    const int share = (total + (int)gridDim.x - 1) / (int)gridDim.x;
    const int g1 = min(total, ((int)blockIdx.x + 1) * share);
    for (int g = blockIdx.x * share; g < g1;) {
        const fd::Piece pc = fd::locate(g, g1, s_cum, P.n_seq, P.Hkv);
        const int c0 = s_cum[pc.i], nt = s_cum[pc.i + 1] - c0;
        const int p = P.pos[pc.i], slot = P.kslot ? P.kslot[pc.i] : 0;
        // lse of every head of the group over the records of the CTAs that hold a piece of this item
        int clo, chi;
        fd::item_ctas(P.cph, per_cta, P.Hkv, c0, nt, pc.kvh, clo, chi);
        __syncthreads();
        if (warp < P.G) {
            const float* rec = P.part + ((size_t)(clo + pc.i * P.Hkv + pc.kvh) * P.G + warp) * (P.HD + 4) + P.HD;
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
            if (lane == 0) s_lse[warp] = Mx + log2f(L);
        }
        __syncthreads();
        const size_t base = ((size_t)slot * P.Hkv + pc.kvh) * P.stride;
        for (int k = tid; k < pc.n * TILE; k += STEP_THREADS) {
            const int key = pc.tl * TILE + k;
            if (key > p) break;
            const float* sc = P.scores + ((size_t)g * TILE + k) * P.G;
            float w = 0.f;
            for (int h = 0; h < P.G; ++h) w += fast_exp2(sc[h] - s_lse[h]);
            if (P.in && key < p) w += P.in[base + key];           // the call's own position starts from nothing
            P.out[base + key] = w;
        }
        g += pc.n;
    }
}

struct ChunkParams {
    const void* q;
    const uint8_t* kvk;
    const float* lse;        // [row][head]
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

constexpr int CW = 8;                       // warps; each owns 16 keys of a 128-key tile
constexpr int CTHREADS = CW * 32, CKEYS = 16 * CW;
constexpr int CPAIRS = 64;                  // (row, head) pairs of a Q tile

template <int HD>
struct ChunkCfg {
    static constexpr int NBLK = HD / 32, REC = HD + 2 * NBLK;
    static constexpr int QSTR = HD + 32;                        // halves per staged Q row (as in flash_decode.cuh)
    static constexpr int Q_BYTES = CPAIRS * QSTR * 2;
    static constexpr int SMEM = 2 * Q_BYTES + 2 * CPAIRS * 8;   // two Q tiles, their (lse, position) pairs
};

// One unit = (kv head, 128 keys).  The warp's 16 keys are the A operand of every product of the unit: the exact integers of
// the records, kept in registers, with the block scales applied to the fp32 sums of each 32-dim block afterwards, so the
// scores carry no rounding of K.  Q tiles of 64 pairs are double-buffered in shared memory.
template <int HD>
__global__ void __launch_bounds__(CTHREADS) k_track_chunk(const ChunkParams P) {
    using C = ChunkCfg<HD>;
    constexpr int NBLK = C::NBLK, REC = C::REC, QSTR = C::QSTR;
    extern __shared__ __align__(16) uint8_t smem[];
    __half* s_q = reinterpret_cast<__half*>(smem);
    float2* s_st = reinterpret_cast<float2*>(smem + 2 * C::Q_BYTES);       // (lse, last visible position as int bits)
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, t4 = lane & 3;
    pdl_wait();
    pdl_trigger();
    const SeqRange sr = seq_range(P.pos, P.kslot, P.act, 0, P.rows, 0, 0, P.pstride, P.n_slots, P.status);
    if (!sr.active) return;
    const int n = sr.hi, pairs = P.rows * P.G, n_qt = (pairs + CPAIRS - 1) / CPAIRS;
    const int tiles = (n + CKEYS - 1) / CKEYS, units = tiles * P.Hkv;
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
        const int kvh = u % P.Hkv, t0 = (u / P.Hkv) * CKEYS;
        // ---- this thread's parts of the records of keys k0, k1 (MMA rows gid, gid + 8) --------------------------------
        const int k0 = t0 + warp * 16 + gid, k1 = k0 + 8;
        uint32_t a[NBLK][2][4];
        float d0[NBLK], d1[NBLK];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int key = e ? k1 : k0;
            const bool in = key < n;
            const uint8_t* rec = P.kvk;
            if (in) rec += kv_rec_index(P.pg, sr.slot, kvh, P.Hkv, P.pstride, key, P.status) * (size_t)REC;
#pragma unroll
            for (int b = 0; b < NBLK; ++b) {
                const float d = in ? __half2float(reinterpret_cast<const __half*>(rec)[b]) : 0.f;
                if (e) d1[b] = d; else d0[b] = d;
                const uint2 w = in ? *reinterpret_cast<const uint2*>(rec + 2 * NBLK + b * 32 + t4 * 8) : make_uint2(0u, 0u);
                const uint32_t x = w.x ^ 0x80808080u, y = w.y ^ 0x80808080u;
                a[b][0][e] = sub1152(widen_lo(x)); a[b][0][2 + e] = sub1152(widen_hi(x));
                a[b][1][e] = sub1152(widen_lo(y)); a[b][1][2 + e] = sub1152(widen_hi(y));
            }
        }
        float w0 = 0.f, w1 = 0.f;
        // rows before qt0 see none of these keys
        const int qt0 = max(0, t0 - sr.p0) * P.G / CPAIRS;
        auto load = [&](int qt, int buf) {
            for (int idx = tid; idx < CPAIRS * (HD / 8); idx += CTHREADS) {
                const int pr = idx / (HD / 8), ch = idx - pr * (HD / 8), pair = qt * CPAIRS + pr;
                __half* dst = s_q + buf * (C::Q_BYTES / 2) + pr * QSTR + ch * 8;
                if (pair < pairs) {
                    const int r = pair / P.G, h = pair - r * P.G;
                    const size_t qi = ((size_t)r * P.Hq + kvh * P.G + h) * HD + ch * 8;
                    if (P.q_f16) {
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)),
                                     "l"(reinterpret_cast<const __half*>(P.q) + qi) : "memory");
                    } else {
                        const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(P.q) + qi);
                        const float4 y = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(P.q) + qi + 4);
                        *reinterpret_cast<uint4*>(dst) = make_uint4(pack_h2(x.x, x.y), pack_h2(x.z, x.w), pack_h2(y.x, y.y), pack_h2(y.z, y.w));
                    }
                } else {
                    *reinterpret_cast<uint4*>(dst) = make_uint4(0u, 0u, 0u, 0u);
                }
            }
            if (tid < CPAIRS) {
                const int pair = qt * CPAIRS + tid, r = pair / P.G, h = pair - r * P.G;
                s_st[buf * CPAIRS + tid] = pair < pairs ? make_float2(P.lse[(size_t)r * P.Hq + kvh * P.G + h], __int_as_float(sr.p0 + r))
                                                        : make_float2(0.f, __int_as_float(-1));
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        __syncthreads();                                        // the previous unit's tiles have been used
        load(qt0, qt0 & 1);
        for (int qt = qt0; qt < n_qt; ++qt) {
            const int buf = qt & 1;
            if (qt + 1 < n_qt) load(qt + 1, buf ^ 1);
            else asm volatile("cp.async.commit_group;" ::: "memory");
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            __syncthreads();
            const __half* qs = s_q + buf * (C::Q_BYTES / 2);
            const bool masked = t0 + CKEYS - 1 > sr.p0 + qt * CPAIRS / P.G || (qt + 1) * CPAIRS > pairs;
#pragma unroll 2
            for (int nt = 0; nt < CPAIRS / 8; ++nt) {
                float sv[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int b = 0; b < NBLK; ++b) {
                    const uint4 qv = *reinterpret_cast<const uint4*>(qs + (nt * 8 + gid) * QSTR + b * 32 + t4 * 8);
                    float acc[4] = {0.f, 0.f, 0.f, 0.f};
                    mma16816(acc, a[b][0], qv.x, qv.y);
                    mma16816(acc, a[b][1], qv.z, qv.w);
                    sv[0] = fmaf(d0[b], acc[0], sv[0]);
                    sv[1] = fmaf(d0[b], acc[1], sv[1]);
                    sv[2] = fmaf(d1[b], acc[2], sv[2]);
                    sv[3] = fmaf(d1[b], acc[3], sv[3]);
                }
                // columns 2 t4, 2 t4 + 1: their (lse, position) are neighbours
                const float4 st = *reinterpret_cast<const float4*>(&s_st[buf * CPAIRS + nt * 8 + 2 * t4]);
                float e0 = fast_exp2(fmaf(sv[0], P.scale_log2, -st.x)), e1 = fast_exp2(fmaf(sv[1], P.scale_log2, -st.z));
                float e2 = fast_exp2(fmaf(sv[2], P.scale_log2, -st.x)), e3 = fast_exp2(fmaf(sv[3], P.scale_log2, -st.z));
                if (masked) {
                    const int l0 = __float_as_int(st.y), l1 = __float_as_int(st.w);
                    if (k0 > l0) e0 = 0.f;
                    if (k0 > l1) e1 = 0.f;
                    if (k1 > l0) e2 = 0.f;
                    if (k1 > l1) e3 = 0.f;
                }
                w0 += e0 + e1;
                w1 += e2 + e3;
            }
            __syncthreads();                                    // the buffer is refilled next
        }
        w0 += __shfl_xor_sync(0xffffffffu, w0, 1); w0 += __shfl_xor_sync(0xffffffffu, w0, 2);
        w1 += __shfl_xor_sync(0xffffffffu, w1, 1); w1 += __shfl_xor_sync(0xffffffffu, w1, 2);
        if (t4 < 2) {
            const int key = t4 ? k1 : k0;
            if (key < n) {
                const size_t at = ((size_t)sr.slot * P.Hkv + kvh) * P.pstride + key;
                float w = t4 ? w1 : w0;
                if (P.in && key < sr.p0) w += P.in[at];
                P.out[at] = w;
            }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

}  // namespace tr
}  // namespace battn
