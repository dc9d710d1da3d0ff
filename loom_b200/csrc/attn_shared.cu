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
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "../../include/loom_cuda.h"
#include "attn_shared.cuh"

namespace loom {
namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int MAX_HD = 256;

__device__ unsigned g_gave_up;  // CTAs of which a wait gave up
std::atomic<int> g_fail{0};

// The end of a CTA. The chunk kernel may run beside the prefix's (attn_prefix.cu),
// and the join waits for the chunk kernel alone: so one CTA of it, and with it the
// kernel, ends after the prefix's. (Were it all of them, they would keep their
// places on the SMs: the two kernels took 206 us, one after the other 223.)
__device__ __forceinline__ void after_prefix() {
    if (blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1) pdl_wait_();
}

// ---- any shape ---------------------------------------------------------------
// One CTA per chunk of positions and KV head. 32 positions at a time go to
// shared memory as f32; 16 query rows (row, head of the group) share them, a
// lane taking one position for the scores and hd / 32 dimensions for the sums. Takes
// what the copy engine cannot: odd head widths, strides off 16 bytes.
constexpr int G_TP = 32, G_TR = 16, G_WARPS = 4;

template <class T>
__global__ void __launch_bounds__(G_WARPS * 32) k_attn_shared_any(AttnArgs a) {
    extern __shared__ float sm[];
    pdl_trigger_();
    const int hd = a.hd, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, kvh = blockIdx.y;
    float *sq = sm, *sk = sq + G_TR * hd, *sv = sk + G_TP * (hd + 1), *ss = sv + G_TP * hd;
    const Item<T> it = item_of<T>(a, a.first + blockIdx.x, kvh);
    const int slot = it.slot, r0 = it.r0, r1 = it.r1, p0 = it.p0, p1 = it.p1;
    const T *kb = it.k, *vb = it.v;
    const int64_t ps = it.pos_stride;
    if (p0 >= p1) {  // the join does not read this slot
        after_prefix();
        return;
    }
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
            const size_t at = part_at(a, slot, hr, kvh);
            if (lane == 0) a.ml[at] = make_float2(m[j], l[j]);
#pragma unroll
            for (int d = 0; d < MAX_HD / 32; d++)
                if (d * 32 + lane < hd) a.acc[at * hd + d * 32 + lane] = acc[j][d];
        }
    }
    after_prefix();
}

// ---- tensor cores, a few query rows per tile ------------------------------------
// Four warps over up to 64 query rows: a warp has 16 of them, and warps that are
// left over when the rows are fewer share the rows and split the positions (a
// decode step's 8 heads of a group: all four do), joining at the end. Positions
// come in tiles of 64 (f32: 32) through two shared-memory stages, copied by TMA in
// blocks of 128 bytes of dimensions, swizzled; one thread asks for them (the
// addresses of 16-byte copies by all threads were half of their instructions).
// Scores, maxima and sums are f32. The weights are rounded to the element type for
// their product with the values (2^-9 or 2^-12 of each, the size of the output's
// own rounding) and summed as rounded, so that they still add up to one; f32
// operands go as three tf32 products (mma.cuh), and each step's leading products
// are added to the running sums by f32 additions: the tensor core truncates its
// own, which along a row of 128 dimensions cost 2.1e-6 of the result, where this costs
// 3e-7. Bound by latency and issue at the 8 (16-bit: 12) warps that registers leave an
// SM, and in long 16-bit caches by reading them: 32 f32 rows of 32 heads over 1,536
// shared and up to 512 own positions 52 us (0.7 TB/s of caches, issue slots 39 % used,
// tensor pipe 29 %), the bf16 own caches of 128 sequences, 349 MB, 69 us (5.1 TB/s).
template <class T> constexpr int mma_tp() { return sizeof(T) == 4 ? 32 : 64; }
template <class T> constexpr size_t mma_block() { return mma_tp<T>() * 128; }  // 128 bytes of a tile's rows
template <class T, int HDP> constexpr size_t mma_tile() { return HDP * sizeof(T) / 128 * mma_block<T>(); }
constexpr size_t maxz(size_t a, size_t b) { return a > b ? a : b; }
template <class T, int HDP> constexpr size_t mma_smem() {  // stages (or the warps' sums), then f32 queries
    return maxz(4 * mma_tile<T, HDP>(), (size_t)64 * (HDP + 8) * 4) + (sizeof(T) == 4 ? (size_t)64 * (HDP + 4) * 4 : 0);
}

template <class T, int HDP>
__global__ void __launch_bounds__(128, sizeof(T) == 2 && HDP <= 128 ? 3 : 1) k_attn_shared_mma(AttnArgs a, const __grid_constant__ AttnMaps maps) {
    constexpr int TP = mma_tp<T>(), E = 128 / (int)sizeof(T);  // positions of a tile, dimensions of a block
    constexpr uint32_t BLK = mma_block<T>(), TILE = mma_tile<T, HDP>();
    constexpr bool F = sizeof(T) == 4;
    constexpr int KS = F ? 1 : HDP / 16;  // query fragments held in registers (16-bit types)
    extern __shared__ __align__(1024) uint8_t smb[];
    __shared__ float s_m[4][16], s_l[4][16];
    __shared__ uint64_t s_full[2], s_empty[2];
    __shared__ int s_err;
    pdl_trigger_();
    const int hd = a.hd, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int kvh = blockIdx.y;
    const Item<T> it = item_of<T>(a, a.first + blockIdx.x, kvh);
    if (it.p0 >= it.p1) {  // the join does not read this slot
        after_prefix();
        return;
    }
    const uint32_t sm0 = smem_u32(smb);
    float *sq = reinterpret_cast<float *>(smb + maxz(4 * TILE, (size_t)64 * (HDP + 8) * 4));
    constexpr int QST = HDP + 4;
    const int blocks = (hd + E - 1) / E, wide = F ? blocks * E : (hd + 15) / 16 * 16;
    const int tiles = (it.p1 - it.p0 + TP - 1) / TP, left = it.p1 - it.p0 - (tiles - 1) * TP;
    auto wait = [&](uint64_t *bar, uint32_t parity) {  // false once any wait of the CTA has given up
        for (int i = 0; i < ATTN_LOOKS; i++) {
            if (mbar_wait(bar, parity, ATTN_POLLS)) return true;
            if (*reinterpret_cast<volatile int *>(&s_err)) return false;
        }
        *reinterpret_cast<volatile int *>(&s_err) = 1;
        return false;
    };
    uint32_t issued = 0;              // tiles asked for (thread 0), over all blocks of rows
    auto fetch = [&](int s, int i) {  // tile i into stage s; what lies outside the cache reads as zero
        issued++;
        const uint32_t dst = sm0 + s * 2 * TILE;
        mbar_expect_tx(&s_full[s], 2 * blocks * BLK);
        for (int b = 0; b < blocks; b++) {
            attn_tma(dst + b * BLK, it.own ? &maps.ok : &maps.pk, b * E, it.p0 + i * TP, kvh, it.seq, &s_full[s]);
            attn_tma(dst + TILE + b * BLK, it.own ? &maps.ov : &maps.pv, b * E, it.p0 + i * TP, kvh, it.seq, &s_full[s]);
        }
    };
    if (tid == 0) {
        for (int s = 0; s < 2; s++) {
            mbar_init_nf(&s_full[s], 1);
            mbar_init_nf(&s_empty[s], 4);
        }
        s_err = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    uint32_t seen = 0;  // tiles of the blocks of rows before
    bool ok = true;
    for (int rb = it.r0; rb < it.r1; rb += 64) {
        const int rows = min(64, it.r1 - rb);
        const int nps = rows <= 16 ? 4 : rows <= 32 ? 2 : 1;  // warps that share 16 rows
        const int rt = warp / nps, ps = warp % nps;
        const int row_a = rb + rt * 16 + g, row_b = row_a + 8;
        const bool in_a = row_a < it.r1, in_b = row_b < it.r1, busy = rt * 16 < rows;
        auto q_row = [&](int hr) {
            return static_cast<const T *>(a.q) + (int64_t)(hr / a.group) * a.q_stride +
                   (int64_t)(kvh * a.group + hr % a.group) * hd;
        };
        fence_async_smem();  // zeros written below, before the copies that follow
        if (__syncthreads_or(!ok)) break;
        if (tid == 0) {  // both stages are free: every tile before has been read
            fetch(seen & 1, 0);
            if (tiles > 1) fetch((seen + 1) & 1, 1);
        }
        if (a.fail) ok = false;
        uint32_t qf[KS][4];
        if constexpr (F) {
            // All of a thread's pieces in flight at once. Up to 32 rows are split here, once
            // for every tile: the first terms in their rows, the second 32 rows further.
            const int lanes = wide / 4, there = (rows + 15) / 16 * 16;
            for (int j = tid; j < there * lanes; j += 128) {
                const int r = j / lanes, d = j % lanes * 4;
                const float *src = reinterpret_cast<const float *>(q_row(min(rb + r, it.r1 - 1))) + d;
                float *dst = sq + r * QST + d;
                if (r >= rows || d >= hd) {
                    *reinterpret_cast<float4 *>(dst) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                } else if (d + 4 <= hd && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
                    cp_async16(smem_u32(dst), src, true);
                } else {
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        if (d + k < hd)
                            cp_async4(smem_u32(dst + k), src + k);
                        else
                            dst[k] = 0.0f;
                    }
                }
            }
            cp_async_wait_all();
            if (nps > 1)
                for (int j = tid; j < there * lanes; j += 128) {  // the thread's own pieces
                    float4 *p = reinterpret_cast<float4 *>(sq + j / lanes * QST + j % lanes * 4);
                    const float4 x = *p;
                    uint4 hi, lo;
                    split_tf32(x.x, hi.x, lo.x);
                    split_tf32(x.y, hi.y, lo.y);
                    split_tf32(x.z, hi.z, lo.z);
                    split_tf32(x.w, hi.w, lo.w);
                    *reinterpret_cast<uint4 *>(p) = hi;
                    *reinterpret_cast<uint4 *>(reinterpret_cast<float *>(p) + 32 * QST) = lo;
                }
            __syncthreads();
        } else {
            // pairs of dimensions; whole words where rows lie on 4 bytes (hd is even)
            const uint16_t *qa = reinterpret_cast<const uint16_t *>(q_row(in_a ? row_a : rb)) + 2 * t;
            const uint16_t *qb = reinterpret_cast<const uint16_t *>(q_row(in_b ? row_b : rb)) + 2 * t;
            const bool words = ((reinterpret_cast<uintptr_t>(qa) | reinterpret_cast<uintptr_t>(qb)) & 3) == 0;
            auto two = [&](bool in, const uint16_t *p, int d) -> uint32_t {
                if (!in || d + 2 * t >= hd) return 0u;
                return words ? *reinterpret_cast<const uint32_t *>(p + d) : (uint32_t)p[d] | ((uint32_t)p[d + 1] << 16);
            };
#pragma unroll
            for (int k = 0; k < KS; k++) {
                qf[k][0] = two(in_a, qa, k * 16);
                qf[k][1] = two(in_b, qb, k * 16);
                qf[k][2] = two(in_a, qa, k * 16 + 8);
                qf[k][3] = two(in_b, qb, k * 16 + 8);
            }
        }
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
        float o[HDP / 8][4];
#pragma unroll
        for (int i = 0; i < HDP / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
        for (int i = 0; i < tiles; i++, seen++) {
            const int s = seen & 1, here = i == tiles - 1 ? left : TP;
            ok = ok && wait(&s_full[s], (seen >> 1) & 1);
            const uint32_t tk = sm0 + s * 2 * TILE, tv = tk + TILE;
            if (here < TP) {  // what lies past the length may be anything, and 0 times it is not 0
                __syncthreads();
                for (int j = tid; j < (TP - here) * blocks * 8; j += 128)
                    *reinterpret_cast<uint4 *>(smb + (tv - sm0) + (j >> 3) % blocks * BLK + (here + (j >> 3) / blocks) * 128 +
                                               (j & 7) * 16) = make_uint4(0, 0, 0, 0);
                __syncthreads();
            }
            // 8 NT positions from `sub` on
            auto step = [&](auto nt, const int sub) {
                constexpr int NT = decltype(nt)::value;
                float c[NT][4];
#pragma unroll
                for (int n = 0; n < NT; n++) c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.0f;
                if constexpr (F) {
                    // lane t has dimensions 8t .. 8t + 7 of 32, in pieces 2t and 2t + 1, two
                    // for each of four products: any order sums to the same scores
                    // (products that add to one result wait for one another: the tiles and the
                    // two small terms take turns)
                    constexpr int NS = NT == 4 ? 1 : 2;  // four tiles are turns enough
                    float small[NS][NT][4];
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int j = 0; j < 4; j++) small[0][n][j] = small[NS - 1][n][j] = 0.0f;
                    const float *qa = sq + (rt * 16 + g) * QST + 8 * t, *qb = qa + 8 * QST;
                    const uint8_t *kr = smb + (tk - sm0) + (sub + g) * 128;
#pragma unroll 1  // two at once miss the instruction cache (32 sequences: 65 us, not 61)
                    for (int d = 0; d < blocks; d++) {
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            uint32_t ah[2][4], al[2][4], bh[NT][4], bl[NT][4];
                            const float4 ua = *reinterpret_cast<const float4 *>(qa + d * 32 + h * 4);
                            const float4 ub = *reinterpret_cast<const float4 *>(qb + d * 32 + h * 4);
                            if constexpr (NT == 4) {
                                split_tf32(ua.x, ah[0][0], al[0][0]);
                                split_tf32(ub.x, ah[0][1], al[0][1]);
                                split_tf32(ua.y, ah[0][2], al[0][2]);
                                split_tf32(ub.y, ah[0][3], al[0][3]);
                                split_tf32(ua.z, ah[1][0], al[1][0]);
                                split_tf32(ub.z, ah[1][1], al[1][1]);
                                split_tf32(ua.w, ah[1][2], al[1][2]);
                                split_tf32(ub.w, ah[1][3], al[1][3]);
                            } else {  // split already
                                const float4 va = *reinterpret_cast<const float4 *>(qa + 32 * QST + d * 32 + h * 4);
                                const float4 vb = *reinterpret_cast<const float4 *>(qb + 32 * QST + d * 32 + h * 4);
                                auto four_of = [](uint32_t (&r)[2][4], const float4 &a4, const float4 &b4) {
                                    r[0][0] = __float_as_uint(a4.x), r[0][1] = __float_as_uint(b4.x);
                                    r[0][2] = __float_as_uint(a4.y), r[0][3] = __float_as_uint(b4.y);
                                    r[1][0] = __float_as_uint(a4.z), r[1][1] = __float_as_uint(b4.z);
                                    r[1][2] = __float_as_uint(a4.w), r[1][3] = __float_as_uint(b4.w);
                                };
                                four_of(ah, ua, ub);
                                four_of(al, va, vb);
                            }
                            float e[NT][4];
#pragma unroll
                            for (int n = 0; n < NT; n++) {
                                const float4 kk = *reinterpret_cast<const float4 *>(kr + d * BLK + n * 1024 + (((2 * t + h) ^ g) << 4));
                                split_tf32(kk.x, bh[n][0], bl[n][0]);
                                split_tf32(kk.y, bh[n][1], bl[n][1]);
                                split_tf32(kk.z, bh[n][2], bl[n][2]);
                                split_tf32(kk.w, bh[n][3], bl[n][3]);
                                e[n][0] = e[n][1] = e[n][2] = e[n][3] = 0.0f;
                            }
#pragma unroll
                            for (int u = 0; u < 2; u++) {
#pragma unroll
                                for (int n = 0; n < NT; n++) mma_tf32(e[n], ah[u], bh[n][2 * u], bh[n][2 * u + 1]);
#pragma unroll
                                for (int n = 0; n < NT; n++) mma_tf32(small[0][n], al[u], bh[n][2 * u], bh[n][2 * u + 1]);
#pragma unroll
                                for (int n = 0; n < NT; n++) mma_tf32(small[NS - 1][n], ah[u], bl[n][2 * u], bl[n][2 * u + 1]);
                            }
#pragma unroll
                            for (int n = 0; n < NT; n++)
#pragma unroll
                                for (int j = 0; j < 4; j++) c[n][j] += e[n][j];
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int j = 0; j < 4; j++) c[n][j] += NS == 1 ? small[0][n][j] : small[0][n][j] + small[NS - 1][n][j];
                } else {
                    // 16-byte piece c of a row is at c ^ (row % 8) of its block
                    const uint32_t row = tk + (sub + (lane >> 4) * 8 + (lane & 7)) * 128, x = ((lane >> 3) & 1) ^ (lane & 7);
#pragma unroll
                    for (int k = 0; k < KS; k++) {
                        if (k * 16 < wide) {
#pragma unroll
                            for (int n = 0; n < NT; n += 2) {
                                uint32_t b[4];
                                ldmatrix_x4(b, row + n * 1024 + (k >> 2) * BLK + ((((2 * k) & 7) ^ x) << 4));
                                mma_k16<T>(c[n], qf[k], b[0], b[1]);
                                mma_k16<T>(c[n + 1], qf[k], b[2], b[3]);
                            }
                        }
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int j = 0; j < 4; j++) c[n][j] *= a.scale;
                if (sub + 8 * NT > here) {
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            if (sub + n * 8 + 2 * t + (j & 1) >= here) c[n][j] = -INFINITY;
                }
                float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    x0 = fmaxf(x0, fmaxf(c[n][0], c[n][1]));
                    x1 = fmaxf(x1, fmaxf(c[n][2], c[n][3]));
                }
                x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1));
                x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
                x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2));
                x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2));
                const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
                const float b0 = n0 == -INFINITY ? 0.0f : n0, b1 = n1 == -INFINITY ? 0.0f : n1;
                if (__any_sync(0xffffffffu, n0 > m0 || n1 > m1)) {  // the maxima settle after a few tiles
                    const float f0 = ex2(m0 - b0), f1 = ex2(m1 - b1);
                    l0 *= f0;
                    l1 *= f1;
#pragma unroll
                    for (int i2 = 0; i2 < HDP / 8; i2++) {
                        o[i2][0] *= f0;
                        o[i2][1] *= f0;
                        o[i2][2] *= f1;
                        o[i2][3] *= f1;
                    }
                    m0 = n0;
                    m1 = n1;
                }
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    c[n][0] = ex2(c[n][0] - b0);
                    c[n][1] = ex2(c[n][1] - b0);
                    c[n][2] = ex2(c[n][2] - b1);
                    c[n][3] = ex2(c[n][3] - b1);
                }
                if constexpr (F) {
                    uint32_t ah[NT][4], al[NT][4];
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        split_tf32(c[n][0], ah[n][0], al[n][0]);  // depth t is position 2t, depth t + 4 is 2t + 1
                        split_tf32(c[n][2], ah[n][1], al[n][1]);
                        split_tf32(c[n][1], ah[n][2], al[n][2]);
                        split_tf32(c[n][3], ah[n][3], al[n][3]);
                        l0 += c[n][0] + c[n][1];
                        l1 += c[n][2] + c[n][3];
                    }
                    const uint8_t *v0 = smb + (tv - sm0) + (sub + 2 * t) * 128 + (g & 3) * 4;
                    constexpr int NP = NT > 2 ? 2 : NT;  // positions of a turn, in eights
#pragma unroll 1
                    for (int n0 = 0; n0 < NT; n0 += NP, v0 += NP * 1024) {
#pragma unroll
                        for (int i4 = 0; i4 < HDP / 8; i4 += 4) {  // a block of 32 dimensions, zeros past hd
                            if (i4 * 8 < hd) {
                                const uint8_t *v = v0 + (i4 >> 2) * BLK;
                                float e[4][4];
#pragma unroll
                                for (int i = 0; i < 4; i++) e[i][0] = e[i][1] = e[i][2] = e[i][3] = 0.0f;
#pragma unroll
                                for (int n = 0; n < NP; n++) {
                                    uint32_t bh[4][2], bl[4][2];
#pragma unroll
                                    for (int i = 0; i < 4; i++) {
                                        const int piece = 2 * i + (g >> 2);
                                        split_tf32(*reinterpret_cast<const float *>(v + n * 1024 + ((piece ^ (2 * t)) << 4)), bh[i][0],
                                                   bl[i][0]);
                                        split_tf32(*reinterpret_cast<const float *>(v + n * 1024 + 128 + ((piece ^ (2 * t + 1)) << 4)),
                                                   bh[i][1], bl[i][1]);
                                    }
#pragma unroll
                                    for (int i = 0; i < 4; i++) mma_tf32(e[i], al[n], bh[i][0], bh[i][1]);
#pragma unroll
                                    for (int i = 0; i < 4; i++) mma_tf32(e[i], ah[n], bl[i][0], bl[i][1]);
#pragma unroll
                                    for (int i = 0; i < 4; i++) mma_tf32(e[i], ah[n], bh[i][0], bh[i][1]);
                                }
#pragma unroll
                                for (int i = 0; i < 4; i++)
#pragma unroll
                                    for (int j = 0; j < 4; j++) o[i4 + i][j] += e[i][j];
                            }
                        }
#pragma unroll
                        for (int n = 0; n + NP < NT; n++)  // the next turn's weights
#pragma unroll
                            for (int j = 0; j < 4; j++) ah[n][j] = ah[n + NP][j], al[n][j] = al[n + NP][j];
                    }
                } else {
                    uint32_t pf[NT / 2][4];
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        const uint32_t pa = pack2<T>(c[n][0], c[n][1]), pb = pack2<T>(c[n][2], c[n][3]);
                        pf[n / 2][n % 2 * 2] = pa;
                        pf[n / 2][n % 2 * 2 + 1] = pb;
                        const float2 ra = unpack2<T>(pa), rb = unpack2<T>(pb);
                        l0 += ra.x + ra.y;
                        l1 += rb.x + rb.y;
                    }
                    const uint32_t row = tv + (sub + ((lane >> 3) & 1) * 8 + (lane & 7)) * 128, x = (lane >> 4) ^ (lane & 7);
#pragma unroll
                    for (int n = 0; n < NT / 2; n++)
#pragma unroll
                        for (int i2 = 0; i2 < HDP / 16; i2++) {
                            if (i2 * 16 < wide) {
                                uint32_t b[4];
                                ldmatrix_x4_trans(b, row + n * 2048 + (i2 >> 2) * BLK + ((((2 * i2) & 7) ^ x) << 4));
                                mma_k16<T>(o[2 * i2], pf[n], b[0], b[1]);
                                mma_k16<T>(o[2 * i2 + 1], pf[n], b[2], b[3]);
                            }
                        }
                }
            };
            // 32 positions at a time where the warp has as many: fewer maxima, and f32 queries
            // are split once for all of them
            if (busy) {
                if constexpr (!F) {
                    if (nps == 4) {
                        if (ps * 16 < here) step(std::integral_constant<int, 2>{}, ps * 16);
                    } else {
                        for (int sub = ps * 32; sub < here; sub += nps * 32) step(std::integral_constant<int, 4>{}, sub);
                    }
                } else if (nps == 1) {
                    step(std::integral_constant<int, 4>{}, 0);
                } else if (nps == 2) {
                    if (ps * 16 < here) step(std::integral_constant<int, 2>{}, ps * 16);
                } else if (ps * 8 < here) {
                    step(std::integral_constant<int, 1>{}, ps * 8);
                }
            }
            __syncwarp();
            if (lane == 0) attn_arrive(&s_empty[s]);
            if (tid == 0 && i + 2 < tiles) {
                ok = ok && wait(&s_empty[s], (seen >> 1) & 1);
                if (ok) fetch(s, i + 2);
            }
            __syncwarp();
        }
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
        l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
        if (nps == 1) {
#pragma unroll
            for (int half = 0; half < 2; half++) {
                if (half ? !in_b : !in_a) continue;
                const size_t at = part_at(a, it.slot, half ? row_b : row_a, kvh);
                if (t == 0) a.ml[at] = half ? make_float2(m1, l1) : make_float2(m0, l0);
                float *dst = a.acc + at * hd;
#pragma unroll
                for (int i = 0; i < HDP / 8; i++)
                    if (i * 8 + 2 * t < hd)  // hd is even
                        *reinterpret_cast<float2 *>(dst + i * 8 + 2 * t) = make_float2(o[i][2 * half], o[i][2 * half + 1]);
            }
            continue;
        }
        if (t == 0) {
            s_m[warp][g] = m0;
            s_m[warp][g + 8] = m1;
            s_l[warp][g] = l0;
            s_l[warp][g + 8] = l1;
        }
        __syncthreads();  // the tiles are read: the sums of the warps take their place
        constexpr int SST = HDP + 8;  // rows g and pairs t of a store touch every bank once
        float *sums = reinterpret_cast<float *>(smb);
        {
            float t0 = -INFINITY, t1 = -INFINITY;
            for (int w = rt * nps; w < (rt + 1) * nps; w++) {
                t0 = fmaxf(t0, s_m[w][g]);
                t1 = fmaxf(t1, s_m[w][g + 8]);
            }
            const float f0 = m0 == -INFINITY ? 0.0f : ex2(m0 - t0), f1 = m1 == -INFINITY ? 0.0f : ex2(m1 - t1);
            float *so = sums + (warp * 16 + g) * SST + 2 * t;
#pragma unroll
            for (int i = 0; i < HDP / 8; i++) {
                *reinterpret_cast<float2 *>(so + i * 8) = make_float2(o[i][0] * f0, o[i][1] * f0);
                *reinterpret_cast<float2 *>(so + 8 * SST + i * 8) = make_float2(o[i][2] * f1, o[i][3] * f1);
            }
        }
        __syncthreads();
        if (tid < rows) {
            const int w0 = (tid / 16) * nps, jr = tid % 16;
            float top = -INFINITY, l = 0.0f;
            for (int w = w0; w < w0 + nps; w++) top = fmaxf(top, s_m[w][jr]);
            for (int w = w0; w < w0 + nps; w++) l += s_l[w][jr] * (s_m[w][jr] == -INFINITY ? 0.0f : ex2(s_m[w][jr] - top));
            a.ml[part_at(a, it.slot, rb + tid, kvh)] = make_float2(top, l);
        }
        // a warp's rows four at a time (one after the other 32 rows took 3 us more)
        constexpr int RU = 4, NP = (HDP + 63) / 64;
        for (int j0 = warp; j0 < rows; j0 += 4 * RU) {
            float2 v[RU][NP];
#pragma unroll
            for (int u = 0; u < RU; u++) {
                const int j = min(j0 + 4 * u, rows - 1);
                const float *from = sums + ((j / 16) * nps * 16 + j % 16) * SST + 2 * lane;
#pragma unroll
                for (int d = 0; d < NP; d++) {
                    v[u][d] = make_float2(0.0f, 0.0f);
                    if (d * 64 + 2 * lane < HDP)
                        for (int w = 0; w < nps; w++) {
                            const float2 x = *reinterpret_cast<const float2 *>(from + w * 16 * SST + d * 64);
                            v[u][d].x += x.x;
                            v[u][d].y += x.y;
                        }
                }
            }
#pragma unroll
            for (int u = 0; u < RU; u++) {
                const int j = j0 + 4 * u;
                if (j >= rows) break;
                float *dst = a.acc + part_at(a, it.slot, rb + j, kvh) * hd + 2 * lane;
#pragma unroll
                for (int d = 0; d < NP; d++)
                    if (d * 64 + 2 * lane < hd) *reinterpret_cast<float2 *>(dst + d * 64) = v[u][d];  // hd is even
            }
        }
    }
    if (__syncthreads_or(!ok)) {  // a copy that does not come: no result
        if (tid == 0) {
            for (uint32_t i = max(issued, 2u) - 2; i < issued; i++) attn_drain(&s_full[i & 1], (i >> 1) & 1);
            atomicAdd(&g_gave_up, 1u);
        }
        for (int hr = it.r0 + tid; hr < it.r1; hr += 128) a.ml[part_at(a, it.slot, hr, kvh)] = make_float2(NAN, NAN);
    }
    after_prefix();
}

// ---- join ----------------------------------------------------------------------
// WPH warps per (row, head), one warp where the parts are few: their maxima and
// sums a lane each, then the parts weighted by e^(m - M), eight in flight; before
// them, while the chunk kernels may still run, the own rows that not every row of the
// sequence sees, four at a time; at the end the division. A lane has four dimensions of each 128. A row that sees nothing gives
// zeros. Bound by reading the parts: 128 sequences of up to two rows of 32 heads, 26 MB
// of parts, in 18 us.
// elements d .. d + 3 of a row of n, zeros past it; one access where it is aligned
template <class T> __device__ __forceinline__ float4 four(const T *p, int d, int n, bool whole) {
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (whole && d < n) {  // n is a multiple of 4
        if constexpr (sizeof(T) == 4) {
            v = *reinterpret_cast<const float4 *>(p + d);
        } else {
            const uint2 u = *reinterpret_cast<const uint2 *>(p + d);
            const float2 a = unpack2<T>(u.x), b = unpack2<T>(u.y);
            v = make_float4(a.x, a.y, b.x, b.y);
        }
    } else if (d < n) {
        v.x = to_f32(p[d]);
        if (d + 1 < n) v.y = to_f32(p[d + 1]);
        if (d + 2 < n) v.z = to_f32(p[d + 2]);
        if (d + 3 < n) v.w = to_f32(p[d + 3]);
    }
    return v;
}
__device__ __forceinline__ void mul_add(float4 &a, float f, const float4 &v) {
    a.x = fmaf(v.x, f, a.x);
    a.y = fmaf(v.y, f, a.y);
    a.z = fmaf(v.z, f, a.z);
    a.w = fmaf(v.w, f, a.w);
}
__device__ __forceinline__ void scale_by(float4 &a, float f) {
    a.x *= f;
    a.y *= f;
    a.z *= f;
    a.w *= f;
}

// Row r of head h by one warp in plain f32 over everything it sees (`see` own positions
// of sequence b): the two tf32 terms of an infinite operand are an infinity and a NaN,
// and a row that came out NaN is taken again so that it has what f32 arithmetic gives
// (32 rows of 32 heads over 2,048 positions, all NaN: 0.9 ms).
template <class T, int ND> __device__ __noinline__ void row_plain(const AttnArgs &a, int r, int h, int b, int see) {
    const int lane = threadIdx.x & 31, hd = a.hd, kvh = h / a.group;
    float m = -INFINITY, l = 0.0f;
    float acc[ND * 4], q[ND * 4];
    auto at = [&](int i) { return lane + 32 * i; };  // a lane's i-th dimension
#pragma unroll
    for (int i = 0; i < ND * 4; i++) {
        acc[i] = 0.0f;
        q[i] = at(i) < hd ? to_f32(static_cast<const T *>(a.q)[r * a.q_stride + (int64_t)h * hd + at(i)]) : 0.0f;
    }
    auto cache = [&](const T *k0, const T *v0, int n, int64_t pos) {
        for (int p = 0; p < n; p++) {
            const T *k = k0 + p * pos, *v = v0 + p * pos;
            float x = 0.0f, e[ND * 4];
#pragma unroll
            for (int i = 0; i < ND * 4; i++) {
                x = fmaf(q[i], at(i) < hd ? to_f32(k[at(i)]) : 0.0f, x);
                e[i] = at(i) < hd ? to_f32(v[at(i)]) : 0.0f;
            }
            x = warp_sum(x) * a.scale;
            if (x == -INFINITY) continue;
            const float mn = fmaxf(m, x), fa = ex2(m - mn), fb = ex2(x - mn);
            l = l * fa + fb;
            m = mn;
#pragma unroll
            for (int i = 0; i < ND * 4; i++) acc[i] = fmaf(e[i], fb, acc[i] * fa);
        }
    };
    cache(static_cast<const T *>(a.pk) + kvh * a.phead, static_cast<const T *>(a.pv) + kvh * a.phead, a.prefix, a.ppos);
    cache(static_cast<const T *>(a.ok) + b * a.oseq + kvh * a.ohead, static_cast<const T *>(a.ov) + b * a.oseq + kvh * a.ohead, see, a.opos);
    T *out = static_cast<T *>(a.out) + r * a.out_stride + (int64_t)h * hd;
#pragma unroll
    for (int i = 0; i < ND * 4; i++)
        if (at(i) < hd) out[at(i)] = from_f32<T>(l != 0.0f ? acc[i] / l : 0.0f);
}

// ND: groups of 128 dimensions; whole, whole_out: rows of queries and own caches, of out
// lie on four elements. Six CTAs to an SM where registers allow: 64 sequences of up to 5
// rows, 78.4 us a call, with four 82.2 (f32: 55 with six, 53 as it is).
template <class T, int WPH, int ND> __global__ void __launch_bounds__(128, sizeof(T) == 2 && WPH == 1 && ND == 1 ? 6 : 1)
    k_attn_shared_join(const __grid_constant__ AttnArgs a, bool whole, bool whole_out) {
    __shared__ float4 s_acc[WPH > 1 ? 4 : 1][ND * 32];
    __shared__ float2 s_ml[4];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % WPH, hd = a.hd;
    const int64_t rh = (int64_t)blockIdx.x * (4 / WPH) + warp / WPH;
    if (rh >= (int64_t)a.n_rows * a.nh) {
        pdl_wait_();
        return;
    }
    const int r = (int)(rh / a.nh), h = (int)(rh % a.nh), kvh = h / a.group;
    // the sequence of row r: the last b with seq_rows[b] <= r
    int lo = 0, hi = a.n_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.seq_rows[mid] <= (uint32_t)r) lo = mid; else hi = mid;
    }
    const int b = lo;
    SeqView s = {0, 0, 0, 0};
    if (a.n_seqs) s = seq_view(a, b);
    const bool mine = r >= s.row0 && r < s.row0 + s.rows;
    const int n = a.n_pre + (mine ? (s.common + a.own_chunk - 1) / a.own_chunk : 0);
    const int see = mine ? max(s.len - (s.row0 + s.rows - 1 - r), 0) : 0;  // own positions this row sees
    float m = -INFINITY, l = 0.0f;
    float4 acc[ND], q[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) {
        acc[d] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        q[d] = four(static_cast<const T *>(a.q) + r * a.q_stride + (int64_t)h * hd, d * 128 + lane * 4, hd, whole);
    }
    // no kernel of the call writes these
    const T *k0 = static_cast<const T *>(a.ok) + b * a.oseq + kvh * a.ohead, *v0 = static_cast<const T *>(a.ov) + b * a.oseq + kvh * a.ohead;
    for (int p0 = part ? see : s.common; p0 < see; p0 += 4) {
        float x[4];
        float4 v[4][ND];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            x[j] = 0.0f;
            const int64_t at = (int64_t)min(p0 + j, see - 1) * a.opos;
#pragma unroll
            for (int d = 0; d < ND; d++) {
                const float4 k = four(k0 + at, d * 128 + lane * 4, hd, whole);
                v[j][d] = four(v0 + at, d * 128 + lane * 4, hd, whole);
                x[j] = fmaf(q[d].x, k.x, fmaf(q[d].y, k.y, fmaf(q[d].z, k.z, fmaf(q[d].w, k.w, x[j]))));
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            x[j] = warp_sum(x[j]) * a.scale;
            if (p0 + j >= see || x[j] == -INFINITY) continue;
            const float mn = fmaxf(m, x[j]), fa = ex2(m - mn), fb = ex2(x[j] - mn);
            l = l * fa + fb;
            m = mn;
#pragma unroll
            for (int d = 0; d < ND; d++) {
                scale_by(acc[d], fa);
                mul_add(acc[d], fb, v[j][d]);
            }
        }
    }
    const int64_t step = (int64_t)a.n_rows * a.nh;  // (row, head) pairs from part to part
    pdl_wait_();
    for (int i0 = 0; i0 < n; i0 += 32 * WPH) {
        const int i = i0 + lane * WPH + part;
        const float2 p = i < n ? a.ml[i * step + rh] : make_float2(-INFINITY, 0.0f);
        const float top = fmaxf(m, warp_max(p.y == 0.0f ? -INFINITY : p.x));
        const float base = top == -INFINITY ? 0.0f : top;
        // a part of zero weight counts for nothing; a NaN goes on
        const float f = p.y == 0.0f ? 0.0f : ex2(p.x - base), fix = ex2(m - base);
        l = l * fix + warp_sum(p.y * f);
        m = top;
#pragma unroll
        for (int d = 0; d < ND; d++) scale_by(acc[d], fix);
        const int here = min(32, (n - i0 - part + WPH - 1) / WPH);
        const float *src = a.acc + ((i0 + part) * step + rh) * hd;
        for (int j0 = 0; j0 < here; j0 += 8) {
#pragma unroll
            for (int d = 0; d < ND; d++) {
                float4 v[8];
#pragma unroll
                for (int j = 0; j < 8; j++)
                    v[j] = j0 + j < here ? four(src + (int64_t)(j0 + j) * WPH * step * hd, d * 128 + lane * 4, hd, hd % 4 == 0)
                                         : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float w = __shfl_sync(0xffffffffu, f, (j0 + j) & 31);
                    if (j0 + j < here && w != 0.0f) mul_add(acc[d], w, v[j]);
                }
            }
        }
    }
    if constexpr (WPH > 1) {
        if (lane == 0) s_ml[warp] = make_float2(m, l);
#pragma unroll
        for (int d = 0; d < ND; d++) s_acc[warp][d * 32 + lane] = acc[d];
        __syncthreads();
        if (part) return;
        float top = -INFINITY;
        for (int w = 0; w < WPH; w++) top = fmaxf(top, s_ml[w].x);
        const float base = top == -INFINITY ? 0.0f : top;
        m = top;
        l = 0.0f;
#pragma unroll
        for (int d = 0; d < ND; d++) acc[d] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int w = 0; w < WPH; w++) {
            const float f = s_ml[w].y == 0.0f ? 0.0f : ex2(s_ml[w].x - base);
            l += s_ml[w].y * f;
#pragma unroll
            for (int d = 0; d < ND; d++) mul_add(acc[d], f, s_acc[w][d * 32 + lane]);
        }
    }
    if constexpr (sizeof(T) == 4) {
        bool nan = l != l;
#pragma unroll
        for (int d = 0; d < ND; d++) nan = nan || acc[d].x != acc[d].x || acc[d].y != acc[d].y || acc[d].z != acc[d].z || acc[d].w != acc[d].w;
        if (a.split && __any_sync(0xffffffffu, nan)) {
            row_plain<T, ND>(a, r, h, b, see);
            return;
        }
    }
    T *out = static_cast<T *>(a.out) + r * a.out_stride + (int64_t)h * hd;
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int d = 0; d < ND; d++) {
        const int at = d * 128 + lane * 4;
        if (at >= hd) continue;
        T e[4] = {from_f32<T>(0.0f), from_f32<T>(0.0f), from_f32<T>(0.0f), from_f32<T>(0.0f)};
        if (l != 0.0f) e[0] = from_f32<T>(acc[d].x * inv), e[1] = from_f32<T>(acc[d].y * inv), e[2] = from_f32<T>(acc[d].z * inv), e[3] = from_f32<T>(acc[d].w * inv);
        if (whole_out) {
            struct alignas(4 * sizeof(T)) Four { T e[4]; };
            *reinterpret_cast<Four *>(out + at) = Four{{e[0], e[1], e[2], e[3]}};
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (at + k < hd) out[at + k] = e[k];
        }
    }
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

// Whether the prefix goes to attn_prefix.cu, as far as the call's sizes say: 16-bit
// types, a scale above zero (its masked scores are -inf before they are scaled, and its
// maxima are taken there), dimensions that fit its tiles, a quarter of a tile's rows and products enough
// to make up for its longer start. Both kernels, bf16, 8 query heads to each of 4 KV
// heads of 128, us of a call: 2^27 products (256 rows, prefix 1,024 / 64 rows, 4,096)
// 15.9 / 13.5 here and 15.5 / 13.0 there, half of them (256 rows, 512) 12.0 and 14.6,
// four times (128 rows, 8,192) 20.9 and 17.7, 2^32 (256 rows, 32,768) 84 and 42; 8 and
// 16 rows over 32,768 positions 18.2 and 19.9 here, 21.1 and 21.3 there, 32 rows 24.6
// and 22.1. Heads of 64 meet at twice the positions.
bool prefix_tc(const loom_attn_shared_desc *d) {
    const double rows = (double)d->n_rows * (d->n_heads / d->n_kv_heads);
    return d->type != T_F32 && d->head_dim <= 128 && d->head_dim % 8 == 0 && d->scale > 0.0f && rows >= 32 &&
           rows * d->n_kv_heads * d->prefix_len * d->head_dim >= (double)(1 << 28);
}

// The cut of the positions, chunks of 64 or more: the prefix in 3 CTAs per SM, the own
// caches in 4. More parts cost the join more than the SMs gain (1 row of 8 heads, f32,
// prefix 8,192: 22 us, at 6 CTAs 28; 70 rows, bf16, own caches of 1,024: 38.8 us, at 6
// 42.5), fewer leave them idle (128 sequences' own caches of 2,048: 167 us of a call, at
// 3 174). attn_prefix.cu takes one CTA per SM in one round, of one tile of 128 rows
// where that leaves it few steps (256 rows over 4,096 positions of 4 heads: 20 us, with
// two tiles 25.5; 1,024 over 8,192 43.6 and 42.6; 512 over 32,768 62.0 and 59.6).
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
    const int64_t rows = std::max<int64_t>((int64_t)a.n_rows * a.group, 1);
    if (prefix_tc(d)) {
        a.pre_tiles = (int)up(rows, rows * a.nkv * a.prefix <= ((int64_t)1 << 24) ? 128 : 256);
        a.pre_rows = (int)up(rows, a.pre_tiles);
        const int64_t per = std::max<int64_t>(1, 148 / ((int64_t)a.pre_tiles * a.nkv));
        a.pre_chunk = (int)(up(up(std::max(a.prefix, 1), per), 128) * 128);
    } else {
        a.pre_rows = 64;
        a.pre_tiles = (int)up(rows, a.pre_rows);
        const int64_t per = up(3 * 148, (int64_t)a.pre_tiles * a.nkv);
        a.pre_chunk = (int)(up(up(std::max(a.prefix, 1), per), 64) * 64);
    }
    a.n_pre = (int)up(a.prefix, a.pre_chunk);
    const int64_t own_per = std::max<int64_t>(1, up(4 * 148, (int64_t)std::max(a.n_seqs, 1) * a.nkv));
    a.own_chunk = (int)std::max<int64_t>(64, up(up(std::max(a.cap, 1), own_per), 64) * 64);
    a.n_own = a.n_seqs ? (int)up(a.cap, a.own_chunk) : 0;
}

size_t ml_bytes(const AttnArgs &a) {
    return (((size_t)(a.n_pre + a.n_own) * a.n_rows * a.nh * sizeof(float2)) + 255) / 256 * 256;
}
size_t ws_bytes_of(const AttnArgs &a) {
    return ml_bytes(a) + (size_t)(a.n_pre + a.n_own) * a.n_rows * a.nh * a.hd * sizeof(float);
}

// Whether the copy engine can take the caches: whole 16-byte pieces in every row,
// and rows of whole pieces apart.
bool pieces(const AttnArgs &a, size_t size) {
    auto whole = [&](int64_t elems) { return elems * (int64_t)size % 16 == 0; };
    auto ptr = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    return whole(a.hd) && whole(a.ppos) && whole(a.phead) && whole(a.opos) && whole(a.ohead) && whole(a.oseq) &&
           ptr(a.pk) && ptr(a.pv) && ptr(a.ok) && ptr(a.ov);
}

typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                             const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encoder() {
    static EncodeFn f = nullptr;
    if (!f) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            f = reinterpret_cast<EncodeFn>(p);
    }
    return f;
}

// [seqs][KV heads][positions][head_dim] of a cache in boxes of `box` positions x 128
// bytes of dimensions; what lies outside reads as zero
bool attn_map(CUtensorMap &m, int type, const void *base, const AttnArgs &a, int len, int64_t pos, int64_t head, int seqs,
              int64_t seq, uint32_t box) {
    EncodeFn enc = encoder();
    if (!enc || !base) return false;
    const cuuint64_t size = elem_bytes(type);
    const cuuint64_t dims[4] = {(cuuint64_t)a.hd, (cuuint64_t)len, (cuuint64_t)a.nkv, (cuuint64_t)seqs};
    auto stride = [&](int64_t s, int n) { return (cuuint64_t)(n > 1 ? s : pos) * size; };  // of one element: unused
    const cuuint64_t strides[3] = {stride(pos, 2), stride(head, a.nkv), stride(seq, seqs)};
    const cuuint32_t boxes[4] = {(cuuint32_t)(128 / size), box, 1, 1}, es[4] = {1, 1, 1, 1};
    const CUtensorMapDataType ty = type == T_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                 : type == T_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    return enc(&m, ty, 4, const_cast<void *>(base), dims, strides, boxes, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <auto K, class... M>
cudaError_t launch_items(size_t smem, int items, int threads, const AttnArgs &a, cudaStream_t st, const M &...maps) {
    cudaError_t e = allow_smem<K>(smem);
    if (e != cudaSuccess) return e;
    // beside the prefix's kernel where that came before (neither reads what the other writes)
    if (a.first) return launch_pdl_(K, dim3(items, a.nkv), dim3(threads), smem, st, a, maps...);
    K<<<dim3(items, a.nkv), threads, smem, st>>>(a, maps...);
    count_launch();
    return cudaGetLastError();
}

template <class T, int ND> cudaError_t launch_join(const AttnArgs &a, int items, cudaStream_t st) {
    // Four warps share a (row, head) where one would read many parts in turn and the
    // rows alone leave SMs idle (bf16 calls of 32 heads, us with one and with four: 1 row
    // of prefix 32,768 25.8 and 18.1, 16 rows of 4,096 26.3 and 24.0, 32 rows of 8,192
    // 29.0 and 30.3, 64 rows of 4,096 32.4 and 37.7).
    const int64_t pairs = (int64_t)a.n_rows * a.nh;
    const bool few = a.n_pre + a.n_own > 16 && pairs <= 4 * 148;
    const auto on = [&](int64_t elems) { return elems % 4 == 0; };
    const auto at = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T)) == 0; };
    const bool whole = on(a.hd) && on(a.q_stride) && on(a.opos) && on(a.ohead) && on(a.oseq) && at(a.q) && at(a.ok) && at(a.ov);
    const bool whole_out = on(a.hd) && on(a.out_stride) && at(a.out);
    const dim3 grid((unsigned)(few ? pairs : (pairs + 3) / 4));
    if (items)
        return few ? launch_pdl_(k_attn_shared_join<T, 4, ND>, grid, dim3(128), 0, st, a, whole, whole_out)
                   : launch_pdl_(k_attn_shared_join<T, 1, ND>, grid, dim3(128), 0, st, a, whole, whole_out);
    k_attn_shared_join<T, 1, ND><<<grid, 128, 0, st>>>(a, whole, whole_out);  // reads seq_rows before its wait: only behind its own kernel
    count_launch();
    return cudaGetLastError();
}

template <class T> cudaError_t launch(AttnArgs a, bool tc, cudaStream_t st) {
    const int all = a.n_pre * a.pre_tiles + a.n_seqs * a.n_own;
    constexpr int type = sizeof(T) == 4 ? (int)T_F32 : std::is_same<T, __half>::value ? (int)T_F16 : T_BF16;
    cudaError_t e = cudaSuccess;
    AttnMaps maps;
    bool mapped = pieces(a, sizeof(T));
    tc = tc && mapped;
    const uint32_t pre_box = tc ? (uint32_t)ATTN_PREFIX_N : mma_tp<T>();
    if (mapped && a.n_pre)
        mapped = attn_map(maps.pk, type, a.pk, a, a.prefix, a.ppos, a.phead, 1, 0, pre_box) &&
                 attn_map(maps.pv, type, a.pv, a, a.prefix, a.ppos, a.phead, 1, 0, pre_box);
    if (mapped && a.n_own)
        mapped = attn_map(maps.ok, type, a.ok, a, a.cap, a.opos, a.ohead, a.n_seqs, a.oseq, mma_tp<T>()) &&
                 attn_map(maps.ov, type, a.ov, a, a.cap, a.opos, a.ohead, a.n_seqs, a.oseq, mma_tp<T>());
    if (mapped && tc) {
        e = attn_prefix_run(type, a, maps, st);
        if (e != cudaSuccess) return e;
        a.first = a.n_pre * a.pre_tiles;
    }
    a.split = mapped && sizeof(T) == 4;
    if (const int items = all - a.first) {
        if (!mapped)
            e = launch_items<k_attn_shared_any<T>>((size_t)(G_TR * a.hd + G_TP * (a.hd + 1) + G_TP * a.hd + G_TR * G_TP) * 4,
                                                   items, G_WARPS * 32, a, st);
        else if (a.hd <= 64)
            e = launch_items<k_attn_shared_mma<T, 64>>(mma_smem<T, 64>(), items, 128, a, st, maps);
        else if (a.hd <= 128)
            e = launch_items<k_attn_shared_mma<T, 128>>(mma_smem<T, 128>(), items, 128, a, st, maps);
        else
            e = launch_items<k_attn_shared_mma<T, 256>>(mma_smem<T, 256>(), items, 128, a, st, maps);
        if (e != cudaSuccess) return e;
    }
    return a.hd <= 128 ? launch_join<T, 1>(a, all, st) : launch_join<T, 2>(a, all, st);
}

}  // namespace

cudaError_t attn_shared_gave_up(unsigned (&v)[2], cudaStream_t st) {
    const cudaError_t e = cudaMemcpyFromSymbolAsync(&v[0], g_gave_up, sizeof v[0], 0, cudaMemcpyDeviceToHost, st);
    return e == cudaSuccess ? attn_prefix_gave_up(&v[1], st) : e;
}

int attn_shared_error() {
    unsigned v[2] = {0, 0};
    if (attn_shared_gave_up(v, nullptr) != cudaSuccess || cudaStreamSynchronize(nullptr) != cudaSuccess) return -1;
    return v[0] || v[1] ? 128 : 0;
}

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
    a.fail = g_fail;
    const cudaError_t e = by_type(d->type, [&](auto t) { return launch<decltype(t)>(a, prefix_tc(d), rt_stream(stream)); });
    return e == cudaSuccess ? LOOM_CUDA_OK : rt_fail("attn_shared", e);
}

int loom_cuda_attn_fail_waits(int on) { return g_fail.exchange(on != 0); }

}  // extern "C"
