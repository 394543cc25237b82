// What the kernels of the paged key/value cache share: the device view of a
// batch's sequences, the rounding to the cache's type, and the host's checks.
#pragma once

#include "zest_b200.h"
#include "zest_device.cuh"
#include "zest_internal.h"

#include <cmath>
#include <cuda_fp16.h>

namespace zest {

// One sequence of a batch as the kernels see it: its first row, its new
// tokens and all its tokens. ok is false where the batch's arrays contradict
// its bounds: the sequence is then skipped (and ZEST_ERR_BAD_SEQ raised).
struct kv_seq {
    int q0, n, kv;
    bool ok;
};

__device__ __forceinline__ kv_seq kv_seq_from(const zest_kv_batch &b, int page_size, int a, int e, int kv) {
    kv_seq r;
    r.q0 = a;
    r.kv = kv;
    r.ok = a >= 0 && e >= a && e <= b.T && (int64_t) e - a <= b.max_q && r.kv >= 0 && r.kv <= b.max_kv &&
           r.kv <= b.table_stride * page_size;
    r.n = r.ok ? e - a : 0;
    return r;
}

__device__ __forceinline__ kv_seq kv_seq_of(const zest_kv_batch &b, int page_size, int s) {
    return kv_seq_from(b, page_size, b.q_start[s], b.q_start[s + 1], b.kv_len[s]);
}

// The bits of lo and hi, each rounded once (nearest even) to the cache's type.
// fp16 values past 65504 become infinite, as the format's rounding has it.
template <bool F16>
__device__ __forceinline__ uint32_t kv_bits2(float lo, float hi) {
    uint32_t p;
    if (F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(p) : "f"(hi), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(p) : "f"(hi), "f"(lo));
    return p;
}

template <bool F16>
__device__ __forceinline__ float kv_value(uint16_t bits) {
    return F16 ? __half2float(__ushort_as_half(bits)) : __uint_as_float((uint32_t) bits << 16);
}

// The host's checks of a cache and a batch. Null, or why they are refused.
inline const char *kv_cache_fault(const zest_kv_cache *c, int64_t layer) {
    if (!c) return "no cache";
    if (c->type != ZEST_TYPE_BF16 && c->type != ZEST_TYPE_F16) return "the cache's type is not BF16 or F16";
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128 && c->page_size != 256)
        return "page_size is not 16, 32, 64, 128 or 256";
    if (c->kv_heads < 1 || c->kv_heads > 65535 || c->d < 8 || c->d > 256 || c->d % 8)
        return "heads of 8 to 256 values, a multiple of 8, and at least one of them";
    if (c->layers < 1 || c->pages < 1 || c->pages > 0x7fffffff - 1) return "no layers or pages";
    if (layer < 0 || layer >= c->layers) return "no such layer";
    // a dimension of one entry has no stride to speak of
    const int64_t big = int64_t(1) << 38;  // bytes below the 2^40 of a tensor map's stride
    const struct { int64_t n, s; } dim[4] = { { c->layers, c->layer_stride }, { c->pages, c->page_stride },
                                              { c->page_size, c->token_stride }, { c->kv_heads, c->head_stride } };
    for (const auto &x : dim)
        if (x.n > 1 && (x.s < c->d || x.s % 8 || x.s > big)) return "strides are multiples of 8 values, at least d";
    if (!c->k || !c->v || ((uintptr_t) c->k & 15) || ((uintptr_t) c->v & 15)) return "pools are not 16-byte aligned";
    return nullptr;
}

inline const char *kv_batch_fault(const zest_kv_batch *b) {
    if (!b) return "no batch";
    if (b->n_seqs < 0 || b->n_seqs > 65535) return "0 to 65535 sequences";
    // the kernels count rows and keys in 32 bits, up to a tile past the last
    const int64_t most = 0x7fffffff - 4096;
    if (b->T < 0 || b->T > most || b->max_q < 0 || b->max_q > 0x7fffffff || b->max_kv < 0 || b->max_kv > most)
        return "row and token counts below 2^31 - 4096";
    if (b->n_seqs > 0 && (!b->q_start || !b->kv_len)) return "no q_start or kv_len";
    if (b->table_stride < 0 || b->table_stride > 0x7fffffff || (b->n_seqs > 0 && b->table_stride > 0 && !b->table))
        return "no page table";
    return nullptr;
}

int kv_refuse(const char *call, const char *why);

}  // namespace zest
