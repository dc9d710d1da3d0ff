// attn_shared.cuh -- arguments and work items of the shared-prefix attention's
// kernels (attn_shared.cu, attn_prefix.cu).
#pragma once
#include <cuda.h>  // CUtensorMap (the encoder is reached through the runtime's driver entry point)

#include "mma.cuh"
#include "umma.cuh"

namespace loom {

struct AttnArgs {
    const void *q, *pk, *pv, *ok, *ov;
    void *out;
    const uint32_t *seq_rows, *seq_len;
    // parts: [slot][row][head] (m, l) pairs and [slot][row][head][hd] sums; the
    // prefix's n_pre slots come first, then the n_own slots of the row's own cache
    float2 *ml;
    float *acc;
    int64_t q_stride, out_stride, ppos, phead, opos, ohead, oseq;
    int n_seqs, n_rows, nh, nkv, group, hd;
    int prefix, cap;
    int pre_chunk, own_chunk, n_pre, n_own, pre_tiles, pre_rows;
    int first;    // first item of a launch that leaves the prefix's to another
    int split;    // f32 products were made of tf32 terms
    int fail;     // the waits give up (loom_cuda_attn_fail_waits)
    float scale;  // of the scores in base 2: scale * log2(e)
};

// A sequence's rows and the own positions that all of them see; every value is
// held to the call's sizes, so wrong device arrays give wrong numbers, not
// addresses outside the tensors.
struct SeqView {
    int row0, rows, len, common;
};
__device__ __forceinline__ SeqView seq_view(const AttnArgs &a, int b) {
    SeqView s;
    s.row0 = (int)min(a.seq_rows[b], (uint32_t)a.n_rows);
    s.rows = max((int)min(a.seq_rows[b + 1], (uint32_t)a.n_rows) - s.row0, 0);
    s.len = (int)min(a.seq_len[b], (uint32_t)a.cap);
    s.common = max(s.len - max(s.rows - 1, 0), 0);
    return s;
}

// A CTA's work: query rows r0 .. r1-1 (row * group + head of the group) of one KV
// head against positions p0 .. p1-1 of a cache, and the slot for the parts.
template <class T> struct Item {
    int slot, r0, r1, p0, p1, seq;
    bool own;  // of the own cache of sequence `seq`, else of the prefix
    const T *k, *v;
    int64_t pos_stride;
};
template <class T> __device__ __forceinline__ Item<T> item_of(const AttnArgs &a, int item, int kvh) {
    Item<T> o;
    if (item < a.n_pre * a.pre_tiles) {
        o.slot = item / a.pre_tiles;
        o.own = false;
        o.seq = 0;
        o.r0 = (item % a.pre_tiles) * a.pre_rows;
        o.r1 = min(o.r0 + a.pre_rows, a.n_rows * a.group);
        o.p0 = o.slot * a.pre_chunk;
        o.p1 = min(o.p0 + a.pre_chunk, a.prefix);
        o.pos_stride = a.ppos;
        o.k = static_cast<const T *>(a.pk) + kvh * a.phead;
        o.v = static_cast<const T *>(a.pv) + kvh * a.phead;
    } else {
        item -= a.n_pre * a.pre_tiles;
        const int b = item / a.n_own, c = item % a.n_own;
        const SeqView s = seq_view(a, b);
        o.own = true;
        o.seq = b;
        o.slot = a.n_pre + c;
        o.r0 = s.row0 * a.group;
        o.r1 = o.r0 + s.rows * a.group;
        o.p0 = c * a.own_chunk;
        o.p1 = min(o.p0 + a.own_chunk, s.common);
        o.pos_stride = a.opos;
        o.k = static_cast<const T *>(a.ok) + b * a.oseq + kvh * a.ohead;
        o.v = static_cast<const T *>(a.ov) + b * a.oseq + kvh * a.ohead;
    }
    return o;
}
__device__ __forceinline__ size_t part_at(const AttnArgs &a, int slot, int hr, int kvh) {
    return ((size_t)slot * a.n_rows + hr / a.group) * a.nh + kvh * a.group + hr % a.group;
}

// The caches as the copy engine sees them; those without a position are not used.
struct AttnMaps {
    CUtensorMap pk, pv, ok, ov;
};
// one box of a cache (dimension x, position y, KV head z, sequence w) to shared memory
__device__ __forceinline__ void attn_tma(uint32_t dst, const CUtensorMap *map, int x, int y, int z, int w, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void attn_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// A wait gives up after about a second (a poll that finds nothing sleeps 4 us). The
// limits are constants: read from the arguments they cost the kernels 1 to 7 %.
constexpr uint32_t ATTN_POLLS = 64;  // polls of a wait between looks at the CTA's error flag,
constexpr int ATTN_LOOKS = 1 << 12;  // and looks before it gives up
// After a wait gave up: the copies to this CTA's memory that are under way, before that is given back.
__device__ __forceinline__ void attn_drain(uint64_t *bar, uint32_t parity) { mbar_wait_hint(bar, parity, 1u << 12, 2000); }

// The prefix items of a 16-bit call (head_dim <= 128, scale > 0, pre_rows <= 256,
// pre_chunk a multiple of the box of ATTN_PREFIX_N positions) on the 5th-generation
// tensor cores.
constexpr int ATTN_PREFIX_N = 64;
cudaError_t attn_prefix_run(int type, const AttnArgs &a, const AttnMaps &maps, cudaStream_t st);
cudaError_t attn_prefix_gave_up(unsigned *v, cudaStream_t st);  // to v: CTAs of which a wait gave up, ever
cudaError_t attn_shared_gave_up(unsigned (&v)[2], cudaStream_t st);  // the same of all the operator's kernels
int attn_shared_error();  // 128 after a wait of the operator's kernels gave up; -1 when the device is in error

}  // namespace loom
