// attn_shared.cu -- attention of a batch whose sequences share a prefix
// (include/loom_cuda.h, loom_cuda_attn_shared).
//
// Row r of sequence b (rows seq_rows[b] .. seq_rows[b+1]-1, its last token and
// its drafts) attends to the prefix_len rows of the shared cache and to its
// sequence's own cache rows 0 .. len_b - (n_b - 1 - j) - 1, j = r - seq_rows[b]:
//
//   o = sum_i p_i v_i,  p = softmax_i(scale q . k_i)
//
// The positions are cut in chunks. A chunk's part of a row is (m, l, o~) with
// m = max s_i, l = sum e^(s_i - m), o~ = sum e^(s_i - m) v_i, and parts join
// exactly: M = max m, o = sum e^(m - M) o~ / sum e^(m - M) l. So the prefix is
// read once for the rows of all sequences, and each own cache once for its
// sequence's rows.
//
// The own rows that only some rows of a sequence see (its last n_b - 1: the
// drafts see one another causally) are left to the join, which adds them row by
// row. The chunk kernels then have one length for a whole sequence and no mask
// but that length, and a cache row that a query may not see never meets it, not
// even as 0 times infinity.
#include <cfloat>

#include "../../include/loom_cuda.h"
#include "serve.cuh"

namespace loom {
namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int MAX_HD = 256;

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
    int pre_chunk, own_chunk, n_pre, n_own, pre_tiles;
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

// ---- any shape ---------------------------------------------------------------
// One CTA per chunk of positions and KV head. 32 positions at a time go to
// shared memory as f32; 16 query rows (row, head of the group) share them, a
// lane taking one position for the scores and hd / 32 dimensions for the sums.
constexpr int G_TP = 32, G_TR = 16, G_WARPS = 4;

template <class T>
__global__ void __launch_bounds__(G_WARPS * 32) k_attn_shared_any(AttnArgs a) {
    extern __shared__ float sm[];
    const int hd = a.hd, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, kvh = blockIdx.y;
    float *sq = sm, *sk = sq + G_TR * hd, *sv = sk + G_TP * (hd + 1), *ss = sv + G_TP * hd;
    int item = blockIdx.x, slot, r0, r1, p0, p1;
    const T *kb, *vb;
    int64_t ps;
    if (item < a.n_pre * a.pre_tiles) {
        slot = item / a.pre_tiles;
        const int rows = a.n_rows * a.group, per = (rows + a.pre_tiles - 1) / a.pre_tiles;
        r0 = (item % a.pre_tiles) * per;
        r1 = min(r0 + per, rows);
        p0 = slot * a.pre_chunk;
        p1 = min(p0 + a.pre_chunk, a.prefix);
        ps = a.ppos;
        kb = static_cast<const T *>(a.pk) + kvh * a.phead;
        vb = static_cast<const T *>(a.pv) + kvh * a.phead;
    } else {
        item -= a.n_pre * a.pre_tiles;
        const int b = item / a.n_own, c = item % a.n_own;
        const SeqView s = seq_view(a, b);
        slot = a.n_pre + c;
        r0 = s.row0 * a.group;
        r1 = r0 + s.rows * a.group;
        p0 = c * a.own_chunk;
        p1 = min(p0 + a.own_chunk, s.common);
        ps = a.opos;
        kb = static_cast<const T *>(a.ok) + b * a.oseq + kvh * a.ohead;
        vb = static_cast<const T *>(a.ov) + b * a.oseq + kvh * a.ohead;
    }
    if (p0 >= p1) return;  // the join does not read this slot
    for (int t0 = r0; t0 < r1; t0 += G_TR) {
        __syncthreads();
        for (int i = tid; i < G_TR * hd; i += G_WARPS * 32) {
            const int hr = t0 + i / hd;
            sq[i] = hr < r1 ? to_f32(static_cast<const T *>(a.q)[(hr / a.group) * a.q_stride +
                                                                  (int64_t)(kvh * a.group + hr % a.group) * hd + i % hd]) * a.scale
                            : 0.0f;
        }
        float m[4], l[4], acc[4][MAX_HD / 32];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            m[j] = -INFINITY;
            l[j] = 0.0f;
#pragma unroll
            for (int d = 0; d < MAX_HD / 32; d++) acc[j][d] = 0.0f;
        }
        for (int p = p0; p < p1; p += G_TP) {
            __syncthreads();
            for (int i = tid; i < G_TP * hd; i += G_WARPS * 32) {
                const int j = i / hd, d = i % hd;
                const bool in = p + j < p1;
                sk[j * (hd + 1) + d] = in ? to_f32(kb[(p + j) * ps + d]) : 0.0f;
                sv[i] = in ? to_f32(vb[(p + j) * ps + d]) : 0.0f;
            }
            __syncthreads();
            float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int d = 0; d < hd; d++) {
                const float k = sk[lane * (hd + 1) + d];
#pragma unroll
                for (int j = 0; j < 4; j++) s[j] = fmaf(k, sq[(warp * 4 + j) * hd + d], s[j]);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (p + lane >= p1) s[j] = -INFINITY;
                const float mn = fmaxf(m[j], warp_max(s[j]));
                const float base = mn == -INFINITY ? 0.0f : mn;
                const float e = exp2f(s[j] - base), fix = exp2f(m[j] - base);
                l[j] = l[j] * fix + warp_sum(e);
                m[j] = mn;
                ss[(warp * 4 + j) * G_TP + lane] = e;
#pragma unroll
                for (int d = 0; d < MAX_HD / 32; d++) acc[j][d] *= fix;
            }
            __syncwarp();
            const int n = min(G_TP, p1 - p);
            for (int i = 0; i < n; i++) {
#pragma unroll
                for (int d = 0; d < MAX_HD / 32; d++) {
                    const int dd = d * 32 + lane;
                    if (dd < hd) {
                        const float v = sv[i * hd + dd];
#pragma unroll
                        for (int j = 0; j < 4; j++) acc[j][d] = fmaf(ss[(warp * 4 + j) * G_TP + i], v, acc[j][d]);
                    }
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int hr = t0 + warp * 4 + j;
            if (hr >= r1) break;
            const size_t at = ((size_t)slot * a.n_rows + hr / a.group) * a.nh + kvh * a.group + hr % a.group;
            if (lane == 0) a.ml[at] = make_float2(m[j], l[j]);
#pragma unroll
            for (int d = 0; d < MAX_HD / 32; d++)
                if (d * 32 + lane < hd) a.acc[at * hd + d * 32 + lane] = acc[j][d];
        }
    }
}

// ---- join ----------------------------------------------------------------------
// One warp per (row, head): the parts of the chunks, then the own rows that not
// every row of the sequence sees, then the division. A row that sees nothing
// gives zeros.
template <class T> __global__ void __launch_bounds__(128) k_attn_shared_join(AttnArgs a) {
    const int lane = threadIdx.x & 31;
    const int64_t rh = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (rh >= (int64_t)a.n_rows * a.nh) return;
    const int r = (int)(rh / a.nh), h = (int)(rh % a.nh), kvh = h / a.group;
    // the sequence of row r: the last b with seq_rows[b] <= r
    int lo = 0, hi = a.n_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if ((int)min(a.seq_rows[mid], 0x7FFFFFFFu) <= r) lo = mid; else hi = mid;
    }
    const int b = lo;
    SeqView s = {0, 0, 0, 0};
    if (a.n_seqs) s = seq_view(a, b);
    const bool mine = r >= s.row0 && r < s.row0 + s.rows;
    const int own = mine ? (s.common + a.own_chunk - 1) / a.own_chunk : 0;
    const int tail = mine ? max(s.len - (s.row0 + s.rows - 1 - r), 0) : 0;  // own positions this row sees
    float m = -INFINITY, l = 0.0f, acc[MAX_HD / 32];
#pragma unroll
    for (int d = 0; d < MAX_HD / 32; d++) acc[d] = 0.0f;
    const int n = a.n_pre + own;
    for (int i = 0; i < n; i++) {
        const size_t at = ((size_t)i * a.n_rows + r) * a.nh + h;
        const float2 p = a.ml[at];
        if (p.y == 0.0f) continue;  // nothing but weights of zero (a NaN goes on)
        const float mn = fmaxf(m, p.x), fa = exp2f(m - mn), fb = exp2f(p.x - mn);
        l = l * fa + p.y * fb;
        m = mn;
#pragma unroll
        for (int d = 0; d < MAX_HD / 32; d++)
            if (d * 32 + lane < a.hd) acc[d] = acc[d] * fa + a.acc[at * a.hd + d * 32 + lane] * fb;
    }
    const T *q = static_cast<const T *>(a.q) + r * a.q_stride + (int64_t)h * a.hd;
    for (int p = s.common; p < tail; p++) {
        const T *k = static_cast<const T *>(a.ok) + b * a.oseq + p * a.opos + kvh * a.ohead;
        const T *v = static_cast<const T *>(a.ov) + b * a.oseq + p * a.opos + kvh * a.ohead;
        float x = 0.0f;
#pragma unroll
        for (int d = 0; d < MAX_HD / 32; d++)
            if (d * 32 + lane < a.hd) x = fmaf(to_f32(q[d * 32 + lane]) * a.scale, to_f32(k[d * 32 + lane]), x);
        x = warp_sum(x);
        if (x == -INFINITY) continue;
        const float mn = fmaxf(m, x), fa = exp2f(m - mn), fb = exp2f(x - mn);
        l = l * fa + fb;
        m = mn;
#pragma unroll
        for (int d = 0; d < MAX_HD / 32; d++)
            if (d * 32 + lane < a.hd) acc[d] = acc[d] * fa + to_f32(v[d * 32 + lane]) * fb;
    }
    T *out = static_cast<T *>(a.out) + r * a.out_stride + (int64_t)h * a.hd;
#pragma unroll
    for (int d = 0; d < MAX_HD / 32; d++)
        if (d * 32 + lane < a.hd) out[d * 32 + lane] = from_f32<T>(l != 0.0f ? acc[d] / l : 0.0f);
}

const char *check(const loom_attn_shared_desc *d) {
    if (!d) return "attn_shared: no descriptor";
    if (!elem_bytes(d->type)) return "attn_shared: type must be LOOM_F32, LOOM_F16 or LOOM_BF16";
    if (!d->n_heads || !d->n_kv_heads || d->n_heads % d->n_kv_heads)
        return "attn_shared: n_heads must be a multiple of n_kv_heads";
    if (!d->head_dim || d->head_dim > MAX_HD) return "attn_shared: head_dim must be 1..256";
    if (d->n_heads > 65535) return "attn_shared: at most 65535 heads";
    if (d->n_rows > (1u << 20) || d->n_rows * d->n_heads > (1u << 28)) return "attn_shared: too many rows";
    if (d->n_seqs > (1u << 20)) return "attn_shared: too many sequences";
    if (d->prefix_len > (1u << 30) || d->own_cap > (1u << 30)) return "attn_shared: at most 2^30 positions";
    if (!(d->scale == d->scale)) return "attn_shared: scale is NaN";
    return nullptr;
}

// The cut of the positions. Chunks are sized so that prefix and own items
// together give the GPU a few CTAs per SM, no smaller than 64 positions.
void plan(const loom_attn_shared_desc *d, AttnArgs &a) {
    a.n_seqs = (int)d->n_seqs;
    a.n_rows = (int)d->n_rows;
    a.nh = (int)d->n_heads;
    a.nkv = (int)d->n_kv_heads;
    a.group = a.nh / a.nkv;
    a.hd = (int)d->head_dim;
    a.prefix = (int)d->prefix_len;
    a.cap = (int)d->own_cap;
    a.scale = d->scale * LOG2E;
    a.q_stride = (int64_t)d->q_stride;
    a.out_stride = (int64_t)d->out_stride;
    a.ppos = (int64_t)d->prefix_pos_stride;
    a.phead = (int64_t)d->prefix_head_stride;
    a.opos = (int64_t)d->own_pos_stride;
    a.ohead = (int64_t)d->own_head_stride;
    a.oseq = (int64_t)d->own_seq_stride;
    auto up = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
    const int want = 4 * 148;
    a.pre_tiles = (int)up((int64_t)a.n_rows * a.group, 64);
    const int64_t pre_per = std::max<int64_t>(1, up(want, (int64_t)std::max(a.pre_tiles, 1) * a.nkv));
    a.pre_chunk = (int)std::max<int64_t>(64, up(up(std::max(a.prefix, 1), pre_per), G_TP) * G_TP);
    a.n_pre = (int)up(a.prefix, a.pre_chunk);
    const int64_t own_per = std::max<int64_t>(1, up(want, (int64_t)std::max(a.n_seqs, 1) * a.nkv));
    a.own_chunk = (int)std::max<int64_t>(64, up(up(std::max(a.cap, 1), own_per), G_TP) * G_TP);
    a.n_own = a.n_seqs ? (int)up(a.cap, a.own_chunk) : 0;
}

size_t ml_bytes(const AttnArgs &a) {
    return (((size_t)(a.n_pre + a.n_own) * a.n_rows * a.nh * sizeof(float2)) + 255) / 256 * 256;
}
size_t ws_bytes_of(const AttnArgs &a) {
    return ml_bytes(a) + (size_t)(a.n_pre + a.n_own) * a.n_rows * a.nh * a.hd * sizeof(float);
}

template <class T> cudaError_t launch(const AttnArgs &a, cudaStream_t st) {
    const size_t smem = (size_t)(G_TR * a.hd + G_TP * (a.hd + 1) + G_TP * a.hd + G_TR * G_TP) * sizeof(float);
    const int items = a.n_pre * a.pre_tiles + a.n_seqs * a.n_own;
    if (items) {
        cudaError_t e = cudaFuncSetAttribute(k_attn_shared_any<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        k_attn_shared_any<T><<<dim3(items, a.nkv), G_WARPS * 32, smem, st>>>(a);
        count_launch();
    }
    k_attn_shared_join<T><<<(unsigned)(((int64_t)a.n_rows * a.nh + 3) / 4), 128, 0, st>>>(a);
    count_launch();
    return cudaGetLastError();
}

}  // namespace
}  // namespace loom

using namespace loom;

extern "C" {

size_t loom_cuda_attn_shared_workspace(const loom_attn_shared_desc *d) {
    if (check(d)) return 0;
    AttnArgs a{};
    plan(d, a);
    return ws_bytes_of(a);
}

int loom_cuda_attn_shared(const loom_attn_shared_desc *d, const void *d_q, const void *d_prefix_k,
                          const void *d_prefix_v, const void *d_own_k, const void *d_own_v, const uint32_t *d_seq_rows,
                          const uint32_t *d_seq_len, void *d_out, void *d_ws, size_t ws_bytes, void *stream) {
    if (int rc = rt_need_init()) return rc;
    if (const char *why = check(d)) return rt_decline(why);
    if (d->n_rows == 0) return LOOM_CUDA_OK;
    if (!d_q || !d_out) return rt_decline("attn_shared: q and out are required");
    if (d->prefix_len && (!d_prefix_k || !d_prefix_v)) return rt_decline("attn_shared: a prefix needs its caches");
    if (d->n_seqs && (!d_seq_rows || !d_seq_len)) return rt_decline("attn_shared: sequences need seq_rows and seq_len");
    if (d->n_seqs && d->own_cap && (!d_own_k || !d_own_v)) return rt_decline("attn_shared: own positions need their caches");
    AttnArgs a{};
    plan(d, a);
    if (ws_bytes < ws_bytes_of(a) || (!d_ws && ws_bytes_of(a))) return rt_decline("attn_shared: workspace too small");
    if (reinterpret_cast<uintptr_t>(d_ws) % 16) return rt_decline("attn_shared: workspace not aligned to 16 bytes");
    a.q = d_q;
    a.pk = d_prefix_k;
    a.pv = d_prefix_v;
    a.ok = d_own_k;
    a.ov = d_own_v;
    a.out = d_out;
    a.seq_rows = d_seq_rows;
    a.seq_len = d_seq_len;
    a.ml = static_cast<float2 *>(d_ws);
    a.acc = reinterpret_cast<float *>(static_cast<uint8_t *>(d_ws) + ml_bytes(a));
    const cudaError_t e = by_type(d->type, [&](auto t) { return launch<decltype(t)>(a, rt_stream(stream)); });
    return e == cudaSuccess ? LOOM_CUDA_OK : rt_fail("attn_shared", e);
}

}  // extern "C"
