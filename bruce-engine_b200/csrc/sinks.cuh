// The sink buffers of a sliding-window layer: copies of the first positions of every sequence, taken from the ring while
// it still holds them (the attention side of sinks is VAR_SINK of the attention kernels, see SinkView in common.cuh).
#pragma once
#include "common.cuh"

namespace battn {

struct SinkStoreParams {
    const uint8_t* kvk;
    const uint8_t* kvv;
    uint8_t* sk;
    uint8_t* sv;
    const int* pos;
    const int* kslot;
    const int* act;
    int rows, Hkv, rec, ring, cap, n_slots;
    int* status;
};

// One block per (sequence, kv head, K|V): the records of positions [pos, pos + rows) that lie below cap, 8 bytes per thread
// and step (a record is a multiple of 8 bytes and starts on one).  A step that is past cap, every step but a sequence's
// first few, reads one position and returns.
__global__ void __launch_bounds__(256) k_sinks_store(const SinkStoreParams P) {
    pdl_wait();
    pdl_trigger();
    const int i = blockIdx.x, kvh = blockIdx.y;
    if (P.act && P.act[i] == 0) return;
    const int slot = P.kslot ? P.kslot[i] : 0, p0 = P.pos[i];
    if (p0 < 0 || slot < 0 || (P.kslot && slot >= P.n_slots)) {
        if (threadIdx.x == 0) atomicOr(P.status, BATTN_DEV_BAD_POSITION);
        return;
    }
    if (p0 >= P.cap) return;
    const int n = min(P.rows, P.cap - p0), wpr = P.rec / 8;
    const size_t head = (size_t)slot * P.Hkv + kvh;
    const uint2* src = reinterpret_cast<const uint2*>((blockIdx.z ? P.kvv : P.kvk) + head * P.ring * P.rec);
    uint2* dst = reinterpret_cast<uint2*>((blockIdx.z ? P.sv : P.sk) + head * P.cap * P.rec);
    for (int w = threadIdx.x; w < n * wpr; w += blockDim.x) {
        const int r = w / wpr, c = w - r * wpr, p = p0 + r;      // (below cap; its words may pass 32 bits)
        dst[(size_t)p * wpr + c] = src[(size_t)(p & (P.ring - 1)) * wpr + c];
    }
}

}  // namespace battn
