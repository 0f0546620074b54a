/*
 * serve_step.cu — the small kernels of a serving step over a paged latent
 * cache (include/waste_cuda.h): the step's maps from the requests' lengths,
 * the new latents written to their cache rows, and the logits made ready
 * for sampling. The attention between them is mla_tree.cu.
 */
#include "vq3r_common.cuh"
#include "waste_cuda.h"
#include "wc_launch.h"

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

using namespace wc;
namespace cg = cooperative_groups;

namespace {

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f(float v) { return v; }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }

/* ---- the step's maps -------------------------------------------------------
 * need_r = max(0, ceil((ctx + q) / page) - held), its prefix sum gives each
 * request's place in the free list, the prefix sum of q its token rows.
 *
 * A few KB in and out: launch and dependent loads are all there is, so one
 * launch, a token a thread. Every CTA makes both prefix sums for itself (B <=
 * 4096 lengths, 8 a thread at most), which costs less than handing them round,
 * keeps them in shared memory, and takes its share of the tokens and table
 * entries. Where the counts are updated in place the CTAs are one cluster (at
 * most 8): its barrier stands between the last read of an input and the first
 * write. 64 requests of one token take 4.2 us in a captured graph, 256 trees of
 * up to 31 nodes 6.4 (7.5 and 8.2 called one by one, which is the host's rate).
 * Which slot a token gets follows from the old table (blocks held) or the free
 * list (blocks taken now), so no table entry written here is read here. */
constexpr int kPlanThreads = 512;
constexpr int kPlanMaxB = 4096;
constexpr int kPlanPer = kPlanMaxB / kPlanThreads;

struct PlanSmem {
    int qstart[kPlanMaxB + 1];       /* prefix of q                              */
    int fstart[kPlanMaxB];           /* first free-list entry, -1: not served     */
    int held[kPlanMaxB];             /* blocks held before the step               */
    int red[2][kPlanThreads / 32];
};

__global__ void __launch_bounds__(kPlanThreads) kv_plan_kernel(
    const waste_cuda_kv_plan_desc d, unsigned int *err)
{
    extern __shared__ __align__(16) unsigned char smp[];
    PlanSmem &s = *reinterpret_cast<PlanSmem *>(smp);
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = (int)blockIdx.x, ncta = (int)gridDim.x;
    const int per = (d.B + kPlanThreads - 1) / kPlanThreads, r0 = tid * per;
    int q[kPlanPer], need[kPlanPer], held[kPlanPer];
    int sq = 0, sn = 0;
    unsigned int bad = 0, okm = 0;
    const int head0 = *d.free_head, head = max(0, head0), avail = max(0, d.n_free - head);
    if (head0 < 0 || head0 > d.n_free) bad |= WASTE_CUDA_DERR_BAD_BLOCK;
#pragma unroll
    for (int k = 0; k < kPlanPer; k++) {
        q[k] = need[k] = held[k] = 0;
        const int r = r0 + k;
        if (k >= per || r >= d.B) continue;
        const int ctx = d.ctx_len[r];
        held[k] = d.n_blocks[r];
        q[k] = d.q_len[r];
        bool ok = ctx >= 0 && q[k] >= 0 && held[k] >= 0;
        if (q[k] < 0) q[k] = 0;
        const long long blocks = ((long long)ctx + q[k] + d.page - 1) / d.page;
        ok = ok && blocks <= d.max_blocks && held[k] <= d.max_blocks;
        if (!ok) bad |= WASTE_CUDA_DERR_BAD_BLOCK;
        if (d.mask && q[k] > 32 * d.mask_words) { ok = false; bad |= WASTE_CUDA_DERR_BAD_TREE; }
        if (ok) okm |= 1u << k;
        need[k] = ok ? max(0, (int)blocks - held[k]) : 0;
        /* the token rows stop at T: sums of larger counts cannot overflow */
        sq = (int)min((long long)sq + q[k], (long long)0x3fffffff);
        sn = (int)min((long long)sn + need[k], (long long)0x3fffffff);
    }
    int iq = sq, in = sn;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, iq, o), b = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) { iq = min(iq + a, 0x3fffffff); in = min(in + b, 0x3fffffff); }
    }
    if (lane == 31) { s.red[0][warp] = iq; s.red[1][warp] = in; }
    __syncthreads();
    int pq = iq - sq, pn = in - sn;
    for (int w = 0; w < warp; w++) {
        pq = min(pq + s.red[0][w], 0x3fffffff);
        pn = min(pn + s.red[1][w], 0x3fffffff);
    }
    int total = 0;
    for (int w = 0; w < kPlanThreads / 32; w++) total = min(total + s.red[1][w], 0x3fffffff);
    if (tid == 0) s.qstart[0] = 0;
    int given = 0;
#pragma unroll
    for (int k = 0; k < kPlanPer; k++) {
        const int r = r0 + k;
        if (k >= per || r >= d.B) continue;
        const bool served = ((okm >> k) & 1) && (need[k] == 0 || pn + need[k] <= avail);
        s.fstart[r] = !served ? -1 : need[k] ? head + pn : 0;        /* 0: takes none, any place */
        if (served && need[k]) given = max(given, pn + need[k]);
        s.held[r] = held[k];
        pn = min(pn + need[k], 0x3fffffff);
        pq = min(pq + q[k], 0x3fffffff);
        s.qstart[r + 1] = pq;
    }
    /* blocks taken: the largest served end (served needs are a prefix) */
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) given = max(given, __shfl_xor_sync(0xffffffffu, given, o));
    __syncthreads();
    if (lane == 0) s.red[0][warp] = given;
    __syncthreads();
    for (int w = 0; w < kPlanThreads / 32; w++) given = max(given, s.red[0][w]);
    const int T = min(s.qstart[d.B], d.T);
    if (s.qstart[d.B] > d.T) bad |= WASTE_CUDA_DERR_BAD_TREE;
    /* every input that an output may stand in for has been read */
    if (cl.num_blocks() > 1) cl.sync(); else __syncthreads();
    if (rank == 0) {
#pragma unroll
        for (int k = 0; k < kPlanPer; k++) {
            const int r = r0 + k;
            if (k >= per || r >= d.B) continue;
            const bool served = s.fstart[r] >= 0;
            d.n_blocks_out[r] = held[k] + (served ? need[k] : 0);
            /* the rows with the new ones that have one of T's: a longer length would
             * make cached rows of those that are there */
            const int end = min(s.qstart[r + 1], d.T);
            d.kv_len[r] = served ? d.ctx_len[r] + (end - min(s.qstart[r], d.T)) : 0;
            d.q_indptr[r + 1] = end;
        }
        if (tid == 0) {
            d.q_indptr[0] = 0;
            *d.free_head_out = head + given;
            *d.short_blocks = max(0, total - avail);
        }
    }
    /* the taken blocks into the table: a thread per request, its few entries */
    const int stride = ncta * kPlanThreads, t0 = rank * kPlanThreads + tid;
    for (int r = t0; r < d.B; r += stride) {
        const int f = s.fstart[r];
        if (f < 0) continue;
        const int h = s.held[r];
        const long long want = ((long long)d.ctx_len[r] + (s.qstart[r + 1] - s.qstart[r]) + d.page - 1) / d.page;
        for (int j = h; j < want; j++) d.block_table[(size_t)r * d.max_blocks + j] = d.free_blocks[f + j - h];
    }
    /* the tokens */
    for (int t = t0; t < T; t += stride) {
        int lo = 0, hi = d.B;                    /* the last r with qstart[r] <= t */
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s.qstart[mid] <= t) lo = mid; else hi = mid;
        }
        const int r = lo, i = t - s.qstart[r], ctx = d.ctx_len[r];
        const int f = s.fstart[r];
        /* ancestors: parents are smaller, so one walk upwards meets the
         * mask's words in descending order */
        int depth = 0;
        if (d.parent) {
            uint32_t *row = d.mask ? d.mask + (size_t)t * d.mask_words : nullptr;
            const bool fits = row && i < 32 * d.mask_words;
            int w = fits ? i >> 5 : 0, j = i;
            uint32_t bits = 0;
            if (row)
                for (int z = fits ? w + 1 : 0; z < d.mask_words; z++) row[z] = 0;
            for (;;) {
                if (fits) {
                    while (w > (j >> 5)) { row[w--] = bits; bits = 0; }
                    bits |= 1u << (j & 31);
                }
                /* a tree too large for its mask is not served: no walk from its far nodes,
                 * whose length only T would bound */
                if (!fits) break;
                const int p = d.parent[s.qstart[r] + j];
                if (p < 0 || p >= j) {
                    if (p != -1) bad |= WASTE_CUDA_DERR_BAD_TREE;
                    break;
                }
                j = p;
                depth++;
            }
            if (fits)
                while (w >= 0) { row[w--] = bits; bits = 0; }
        } else {
            depth = i;
            if (d.mask)
                for (int w = 0; w < d.mask_words; w++)
                    d.mask[(size_t)t * d.mask_words + w] =
                        i >= 32 * w + 31 ? 0xffffffffu : (i < 32 * w ? 0u : (2u << (i - 32 * w)) - 1u);
        }
        d.pos[t] = ctx + depth;
        int64_t slot = -1;
        if (f >= 0) {
            const int at = ctx + i, b = at / d.page, h = s.held[r];
            const int id = b < h ? d.block_table[(size_t)r * d.max_blocks + b] : d.free_blocks[f + b - h];
            if (id < 0) bad |= WASTE_CUDA_DERR_BAD_BLOCK;
            else slot = (int64_t)id * d.page + at % d.page;
        }
        d.slot[t] = slot;
    }
    if (bad) atomicOr(err, bad);
}

/* ---- the new latents to their cache rows ------------------------------------
 * y = x / sqrt(sum x^2 / kl + eps) * w, rotary pairs, one rounding.
 * One warp a row, the row in registers (512 values; longer rows are read
 * again), so x crosses memory once: the bytes bound it at prompt lengths, a
 * launch and one row's latency at decode. Everything a row needs is loaded
 * before anything waits; where rows allow it four values a load (VEC 4), which
 * took 8191 rows of 512 + 64 floats to fp16 from 12.5 us a call to 7.4, the
 * host's rate; in a captured graph they take 4.5, 64 rows 1.8. */
constexpr int kRowsWarps = 4;
constexpr int kRowRegs = 16;         /* 512 latents */

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Pack { T v[VEC]; };

template <typename TX, typename TC, int VEC>
__global__ void __launch_bounds__(kRowsWarps * 32) mla_rows_kernel(
    const waste_cuda_mla_rows_desc d, unsigned int *err)
{
    constexpr int K = kRowRegs / VEC, kStep = 32 * VEC;
    const int lane = threadIdx.x & 31, t = blockIdx.x * kRowsWarps + (threadIdx.x >> 5);
    if (t >= d.T) return;
    const TX *x = static_cast<const TX *>(d.x) + (size_t)t * d.x_stride;
    const int64_t slot = d.slot[t];
    const int there = d.n_tokens ? *d.n_tokens : d.T;
    const int pos = d.inv_freq ? d.pos[t] : 0;
    Pack<TX, VEC> v[K];
    Pack<float, VEC> w[K];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int i = lane * VEC + kStep * k;
        if (i < d.kl) v[k] = *reinterpret_cast<const Pack<TX, VEC> *>(x + i);
        else
#pragma unroll
            for (int z = 0; z < VEC; z++) v[k].v[z] = from_f<TX>(0.0f);
    }
    const int half = d.rope / 2;
    TX ra = from_f<TX>(0.0f), rb = ra;                        /* the lane's first pair       */
    float fr = 0.0f;
    if (lane < half) {
        ra = x[d.kl + 2 * lane];
        rb = x[d.kl + 2 * lane + 1];
        if (d.inv_freq) fr = d.inv_freq[lane];
    }
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int i = lane * VEC + kStep * k;
        if (i < d.kl) w[k] = *reinterpret_cast<const Pack<float, VEC> *>(d.norm_w + i);
    }
    const bool short_of = there < 0 || there > d.T;
    if (short_of || t >= there || slot < 0 || slot >= d.n_rows) {
        if ((short_of || (t < there && slot >= 0)) && lane == 0) atomicOr(err, WASTE_CUDA_DERR_BAD_BLOCK);
        return;
    }
    TC *y = static_cast<TC *>(d.cache) + (size_t)slot * d.row_stride;
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
        for (int z = 0; z < VEC; z++) s = fmaf(to_f(v[k].v[z]), to_f(v[k].v[z]), s);
    for (int i = lane + 32 * kRowRegs; i < d.kl; i += 32) {
        const float u = to_f(x[i]);
        s = fmaf(u, u, s);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float r = 1.0f / sqrtf(s / (float)d.kl + d.eps);
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int i = lane * VEC + kStep * k;
        if (i >= d.kl) break;
        Pack<TC, VEC> o;
#pragma unroll
        for (int z = 0; z < VEC; z++) o.v[z] = from_f<TC>(to_f(v[k].v[z]) * r * w[k].v[z]);
        *reinterpret_cast<Pack<TC, VEC> *>(y + i) = o;
    }
    for (int i = lane + 32 * kRowRegs; i < d.kl; i += 32)
        y[i] = from_f<TC>(to_f(x[i]) * r * d.norm_w[i]);
    for (int j = lane; j < half; j += 32) {
        if (j >= 32) {
            ra = x[d.kl + 2 * j];
            rb = x[d.kl + 2 * j + 1];
            if (d.inv_freq) fr = d.inv_freq[j];
        }
        float a = to_f(ra), b = to_f(rb);
        if (d.inv_freq) {
            /* the angle in 64 bits, taken to [-pi, pi] there: at far positions
             * 32 bits lose its fraction of a turn */
            const double ang = (double)pos * (double)fr;
            const double turn = 6.283185307179586476925;
            float sn, cs;
            sincosf((float)fma(-turn, rint(ang * (1.0 / turn)), ang), &sn, &cs);
            const float e = a, o = b;
            a = e * cs - o * sn;
            b = e * sn + o * cs;
        }
        y[d.kl + 2 * j] = from_f<TC>(a);
        y[d.kl + 2 * j + 1] = from_f<TC>(b);
    }
}

/* ---- logits -----------------------------------------------------------------
 * A CTA takes a slice of the ids for up to kLogRows rows of one request. Half
 * of its warps copy the slice of each row, disallowed ids set to -infinity, 16
 * bytes a thread and load, eight in flight: the bytes bound it. The other half
 * finds meanwhile what the history, the drafts and the biases name: marked in
 * a bitmap, numbered by its prefix counts and counted by number (integer
 * atomics: any order gives the same counts). Then all set the named ids'
 * values again; a row's branch of drafted tokens is counted where a drafted id
 * is met. A count per named id and not per id lets the CTAs of a whole batch
 * be resident at once; where a slice's named ids are more than kLogCap they
 * are taken in the widest pieces that hold no more, each of which reads the
 * history again. 4096 of them leave most of an SM's L1 to the history and the
 * named values: with 8192, which two CTAs an SM still have room for, the cases
 * below took 21 us, and 103 on either side of 4096 named ids.
 * 64 rows of 163840 16-bit logits take 18 us (43 MB: 6.6 us of copying), 187
 * fp32 rows of 16 trees 75 to 78 us (247 MB: 38 us) where no slice names more
 * than kLogCap ids, and 100 to 105 where one does (165 with pieces of always
 * kLogCap ids). Measured and slower: counts for every id, in several waves (33 us), the rows staged in shared memory (67),
 * the sparse half following the copy row by row (20 and 85), the sparse work
 * as a kernel of its own under the copy (24 and 94).
 *
 * A count word holds the times produced, bit 31 for "in the prompt" and bit
 * 30 for "drafted". */
constexpr int kLogThreads = 512;
constexpr int kLogHalf = kLogThreads / 2;
constexpr int kLogSlice = 65536;     /* the widest slice                          */
constexpr int kLogCap = 4096;
constexpr int kLogDrafts = 256;      /* drafted tokens of a slice that are listed */
constexpr int kLogBranch = 4096;     /* rows of a request that drafts are followed for:
                                        without the list their cost grows with its square */
constexpr int kLogRows = 4;          /* rows a CTA takes at most                  */
constexpr int kLogKeep = 16;         /* tokens a thread keeps between its two uses */
constexpr uint32_t kPrompt = 0x80000000u, kDrafted = 0x40000000u;

struct alignas(16) LogitSmem {
    uint32_t id[kLogCap], cnt[kLogCap], bias[kLogCap];
    uint32_t named[kLogSlice / 32];
    uint16_t before[kLogSlice / 32]; /* named ids before a word, from the piece's start */
    int warp[kLogHalf / 32];
    int n, nlist, list_j[kLogDrafts], list_u[kLogDrafts];
    int mask[kLogRows];              /* a row's mask, -1: none                     */
};

template <typename T> __device__ __forceinline__ void mask_vec(uint4 &v, uint32_t ok)
{
    T *e = reinterpret_cast<T *>(&v);
#pragma unroll
    for (int z = 0; z < 16 / (int)sizeof(T); z++)
        if (!(ok >> z & 1)) e[z] = from_f<T>(-INFINITY);
}

template <typename T>
__global__ void __launch_bounds__(kLogThreads, 2) logits_kernel(const waste_cuda_logits_desc d, int vs,
                                                                unsigned int *err)
{
    constexpr int E = 16 / sizeof(T), U = 8;
    extern __shared__ __align__(16) unsigned char sml[];
    LogitSmem &s = *reinterpret_cast<LogitSmem *>(sml);
    const int tid = threadIdx.x, lane = tid & 31, v0 = blockIdx.x * vs, nv = min(vs, d.V - v0);
    const int words = (nv + 31) >> 5;
    /* the request and its rows: chunk blockIdx.y of all requests' chunks */
    int r = blockIdx.y, q0 = r, q1 = r + 1, t0 = r, rows = 1;
    if (d.q_indptr) {                                         /* each warp for itself        */
        const int per = (d.B + 31) / 32, first = lane * per, last = min(first + per, d.B);
        auto begin = [&](int i) { return min(max(d.q_indptr[i], 0), d.R); };
        auto chunks = [&](int i) { return (max(begin(i + 1) - begin(i), 0) + kLogRows - 1) / kLogRows; };
        int sum = 0;
        bool wrong = false;
        for (int i = first; i < last; i++) {
            wrong |= d.q_indptr[i] < 0 || d.q_indptr[i + 1] < d.q_indptr[i] || d.q_indptr[i + 1] > d.R;
            sum += chunks(i);
        }
        /* ranges that go backwards overlap, or have more chunks than the grid: every
         * CTA sees them, none writes */
        if (__any_sync(0xffffffffu, wrong)) {
            if (tid == 0 && (blockIdx.x | blockIdx.y) == 0) atomicOr(err, WASTE_CUDA_DERR_BAD_BLOCK);
            return;
        }
        int at = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, at, o);
            if (lane >= o) at += v;
        }
        at -= sum;
        const int want = blockIdx.y;
        const bool here = at <= want && want < at + sum;
        const unsigned who = __ballot_sync(0xffffffffu, here);
        if (!who) return;                                     /* the grid is a bound         */
        if (here)
            for (r = first; want >= at + chunks(r); r++) at += chunks(r);
        r = __shfl_sync(0xffffffffu, r, __ffs(who) - 1);
        at = __shfl_sync(0xffffffffu, at, __ffs(who) - 1);
        q0 = begin(r);
        q1 = begin(r + 1);
        t0 = q0 + (want - at) * kLogRows;
        rows = min(kLogRows, q1 - t0);
    }
    const T *x = static_cast<const T *>(d.logits) + (size_t)t0 * d.ld + v0;
    T *y = static_cast<T *>(d.out) + (size_t)t0 * d.ld_out + v0;
    auto mask_of = [&](int t) -> const uint32_t * {           /* of the chunk's row t        */
        return s.mask[t] >= 0 ? d.allow + (size_t)s.mask[t] * d.allow_words + (v0 >> 5) : nullptr;
    };
    const int hn = d.hist ? min(max(d.hist_len[r], 0), (int)min(d.hist_stride, (size_t)0x7fffffff)) : 0;
    const int hm = d.prompt_len ? d.prompt_len[r] : 0;
    const int *hist = d.hist + (size_t)r * d.hist_stride;
    const int b0 = d.bias_indptr ? max(d.bias_indptr[r], 0) : 0, bn = d.bias_indptr ? d.bias_indptr[r + 1] - b0 : 0;
    const int nd = !d.draft || q1 - q0 > kLogBranch ? 0 : q1 - q0;
    if (tid == 0 && blockIdx.x == 0) {
        if ((d.draft && q1 - q0 > kLogBranch) || (d.tree && q1 - q0 > 32 * d.tree_words))
            atomicOr(err, WASTE_CUDA_DERR_BAD_TREE);
        if (d.hist && hn != d.hist_len[r]) atomicOr(err, WASTE_CUDA_DERR_BAD_BLOCK);
    }
    const int ht = tid - kLogHalf;                            /* of the half that counts     */
    /* what a thread needs twice is loaded once: under the copy a load takes long */
    int keep[kLogKeep], id_b = -1, id_d = -1;
    const float rep = d.rep ? d.rep[r] : 1.0f, freq = d.freq ? d.freq[r] : 0.0f, pres = d.pres ? d.pres[r] : 0.0f;
    if (tid < rows) {
        const int a = !d.allow ? -1 : d.allow_row ? d.allow_row[t0 + tid] : t0 + tid;
        s.mask[tid] = a < d.n_allow ? a : -1;
        if (d.allow && a >= d.n_allow) atomicOr(err, WASTE_CUDA_DERR_BAD_MASK);
    }
    if (ht >= 0) {
#pragma unroll
        for (int k = 0; k < kLogKeep; k++) keep[k] = ht + k * kLogHalf < hn ? hist[ht + k * kLogHalf] : -1;
        if (ht < bn) id_b = d.bias_id[b0 + ht];
        if (ht < nd) id_d = d.draft[q0 + ht];
        for (int i = ht; i < words; i += kLogHalf) s.named[i] = 0;
        if (ht == 0) s.nlist = 0;
    }
    __syncthreads();
    /* ids [32 w0, 32 (w0 + wn)) of the slice numbered; how many are named */
    auto sync_half = [] { asm volatile("bar.sync 1, %0;" ::"n"(kLogHalf) : "memory"); };
    auto numbered = [&](int w0, int wn) {
        const int per = (wn + kLogHalf - 1) / kLogHalf, ws = w0 + ht * per, we = min(ws + per, w0 + wn);
        int sum = 0;
        for (int k = ws; k < we; k++) sum += __popc(s.named[k]);
        int at = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, at, o);
            if (lane >= o) at += v;
        }
        if (lane == 31) s.warp[ht >> 5] = at;
        sync_half();
        const int v = lane < kLogHalf / 32 ? s.warp[lane] : 0;
        const int n = __reduce_add_sync(0xffffffffu, v);
        at += __reduce_add_sync(0xffffffffu, lane < (ht >> 5) ? v : 0) - sum;
        if (ht == 0) s.n = n;
        if (n <= kLogCap) {
            for (int k = ws; k < we; k++) {
                s.before[k] = (uint16_t)at;
                at += __popc(s.named[k]);
            }
            for (int i = ht; i < n; i += kLogHalf) s.cnt[i] = s.bias[i] = 0;
            sync_half();
            /* words that are full lie side by side: a thread takes every 256th */
            for (int k = w0 + ht; k < w0 + wn; k += kLogHalf) {
                int to = s.before[k];
                for (uint32_t m = s.named[k]; m; m &= m - 1) s.id[to++] = 32 * k + __ffs(m) - 1;
            }
        }
        sync_half();
        return n;
    };
    /* their counts */
    auto counted = [&](int w0, int wn) {
        auto number = [&](int id) {
            const unsigned u = (unsigned)id - (unsigned)v0, w = (u >> 5) - (unsigned)w0;
            return u < (unsigned)nv && w < (unsigned)wn
                       ? (int)s.before[u >> 5] + __popc(s.named[u >> 5] & ((1u << (u & 31)) - 1u)) : -1;
        };
        auto count = [&](int i, int id) {
            const int k = number(id);
            if (k < 0) return;
            if (i < hm) atomicOr(&s.cnt[k], kPrompt);
            else atomicAdd(&s.cnt[k], 1u);
        };
#pragma unroll
        for (int k = 0; k < kLogKeep; k++) count(ht + k * kLogHalf, keep[k]);
#pragma unroll 8
        for (int i = ht + kLogKeep * kLogHalf; i < hn; i += kLogHalf) count(i, hist[i]);
        for (int i = ht; i < bn; i += kLogHalf) {
            const int k = number(i == ht ? id_b : d.bias_id[b0 + i]);
            if (k >= 0) atomicMax(&s.bias[k], (uint32_t)(i + 1));
        }
        for (int j = ht; j < nd; j += kLogHalf) {
            const int k = number(j == ht ? id_d : d.draft[q0 + j]);
            if (k >= 0) atomicOr(&s.cnt[k], kDrafted);
        }
    };
    if (ht < 0) {
        /* ---- the copy, row by row. Loaded words are not looked at before all loads
         * are out ---- */
        const bool wide = (((uintptr_t)x | (uintptr_t)y) & 15) == 0 &&
                          (rows == 1 || (d.ld % E == 0 && d.ld_out % E == 0));
        for (int t = 0; t < rows; t++) {
            const uint32_t *allow = mask_of(t);
            const T *xr = x + (size_t)t * d.ld;
            T *yr = y + (size_t)t * d.ld_out;
            const uint4 *xv = reinterpret_cast<const uint4 *>(xr);
            uint4 *yv = reinterpret_cast<uint4 *>(yr);
            const int nvec = wide ? nv / E : 0;
            for (int c = tid; c < nvec; c += U * kLogHalf) {
                uint4 v[U];
                uint32_t w[U];
                if (allow) {
#pragma unroll
                    for (int k = 0; k < U; k++) w[k] = __ldg(allow + (min(c + k * kLogHalf, nvec - 1) * E >> 5));
                }
#pragma unroll
                for (int k = 0; k < U; k++) v[k] = __ldcs(xv + min(c + k * kLogHalf, nvec - 1));
                if (allow) {
#pragma unroll
                    for (int k = 0; k < U; k++) mask_vec<T>(v[k], w[k] >> ((c + k * kLogHalf) * E & 31));
                }
#pragma unroll
                for (int k = 0; k < U; k++)
                    if (c + k * kLogHalf < nvec) yv[c + k * kLogHalf] = v[k];
            }
#pragma unroll 8
            for (int i = nvec * E + tid; i < nv; i += kLogHalf)
                yr[i] = !allow || (allow[i >> 5] >> (i & 31) & 1) ? xr[i] : from_f<T>(-INFINITY);
        }
    }
    if (ht >= 0) {
        /* ---- what is named ---- */
        auto mark = [&](int id) {
            const unsigned u = (unsigned)id - (unsigned)v0;
            if (u >= (unsigned)nv) return false;
            atomicOr(&s.named[u >> 5], 1u << (u & 31));
            return true;
        };
#pragma unroll
        for (int k = 0; k < kLogKeep; k++) mark(keep[k]);
#pragma unroll 8
        for (int i = ht + kLogKeep * kLogHalf; i < hn; i += kLogHalf) mark(hist[i]);
        mark(id_b);
        for (int i = ht + kLogHalf; i < bn; i += kLogHalf) mark(d.bias_id[b0 + i]);
        for (int j = ht; j < nd; j += kLogHalf) {
            const int id = j == ht ? id_d : d.draft[q0 + j];
            if (!mark(id)) continue;
            const int k = atomicAdd(&s.nlist, 1);
            if (k < kLogDrafts) { s.list_j[k] = j; s.list_u[k] = id - v0; }
        }
        sync_half();
        if (numbered(0, words) <= kLogCap) counted(0, words);
    }
    __syncthreads();
    /* ---- the named ids again ---- */
    auto on = [&](int t, int j) {
        return d.tree ? j < 32 * d.tree_words &&
                            ((d.tree[(size_t)(t0 + t) * d.tree_words + (j >> 5)] >> (j & 31)) & 1)
                      : j <= t0 + t - q0;
    };
    /* times the branch of row t drafts id u of the slice */
    auto drafted = [&](int t, int u) {
        uint32_t n = 0;
        if (s.nlist <= kLogDrafts) {
            for (int k = 0; k < s.nlist; k++)
                if (s.list_u[k] == u) n += on(t, s.list_j[k]);
        } else {
            for (int j = 0; j < nd; j++)
                if (d.draft[q0 + j] == v0 + u) n += on(t, j);
        }
        return n;
    };
    auto again = [&](int t, int n) {
        constexpr int Z = 4;
        const uint32_t *allow = mask_of(t);
        const T *xr = x + (size_t)t * d.ld;
        T *yr = y + (size_t)t * d.ld_out;
        for (int k0 = tid; k0 < n; k0 += Z * kLogThreads) {
            T raw[Z];
            uint32_t w[Z];
#pragma unroll
            for (int z = 0; z < Z; z++) {
                const int i = (int)s.id[min(k0 + z * kLogThreads, n - 1)];
                raw[z] = yr[i];
                w[z] = allow ? __ldg(allow + (i >> 5)) : 0xffffffffu;
            }
#pragma unroll
            for (int z = 0; z < Z; z++) {
                const int k = k0 + z * kLogThreads;
                if (k >= n) break;
                const int i = (int)s.id[k];
                if (!(w[z] >> (i & 31) & 1)) continue;
                const uint32_t b = s.bias[k];
                uint32_t c = s.cnt[k];
                if (c & kDrafted) c = (c & ~kDrafted) + drafted(t, i);
                float f = to_f(raw[z]);
                if (c) {
                    f = f > 0.0f ? f / rep : f * rep;
                    const uint32_t m = c & ~kPrompt;
                    f -= freq * (float)m + (m ? pres : 0.0f);
                }
                if (b) f += d.bias_val[b0 + b - 1];
                if (c | b) yr[i] = from_f<T>(f);
            }
        }
    };
    const int total = s.n;
    if (total <= kLogCap) {
        for (int t = 0; t < rows; t++) again(t, total);
        return;
    }
    /* pieces as wide as fit: each reads the history again, so few of them. A piece
     * of kLogCap ids always fits */
    for (int w0 = 0, wn = (words + 1) / 2; w0 < words;) {
        wn = min(wn, words - w0);
        __syncthreads();
        if (ht >= 0 && numbered(w0, wn) <= kLogCap) counted(w0, wn);
        __syncthreads();
        const int n = s.n;
        if (n > kLogCap) {
            wn = (wn + 1) / 2;
            continue;
        }
        for (int t = 0; t < rows; t++) again(t, n);
        w0 += wn;
        wn *= 2;
    }
}

__global__ void clear_bits_kernel(unsigned int *word, unsigned int bits) { atomicAnd(word, ~bits); }

template <typename TX, typename TC>
cudaError_t rows_launch(const waste_cuda_mla_rows_desc *d, unsigned int *err, cudaStream_t s)
{
    const dim3 grid((d->T + kRowsWarps - 1) / kRowsWarps), block(kRowsWarps * 32);
    const bool vec = (d->kl | d->x_stride | d->row_stride) % 4 == 0 && (uintptr_t)d->x % (4 * sizeof(TX)) == 0 &&
                     (uintptr_t)d->cache % (4 * sizeof(TC)) == 0 && (uintptr_t)d->norm_w % 16 == 0;
    if (vec) mla_rows_kernel<TX, TC, 4><<<grid, block, 0, s>>>(*d, err);
    else mla_rows_kernel<TX, TC, 1><<<grid, block, 0, s>>>(*d, err);
    return cudaGetLastError();
}

template <typename TX>
cudaError_t rows_launch(const waste_cuda_mla_rows_desc *d, unsigned int *err, cudaStream_t s)
{
    if (d->dtype == WASTE_CUDA_F32) return rows_launch<TX, float>(d, err, s);
    if (d->dtype == WASTE_CUDA_F16) return rows_launch<TX, __half>(d, err, s);
    return rows_launch<TX, __nv_bfloat16>(d, err, s);
}

template <typename T>
cudaError_t logits_launch(const waste_cuda_logits_desc *d, unsigned int *err, int sms, cudaStream_t s)
{
    /* as many slices as are resident at once, two CTAs an SM: a few more wait for
     * a whole turn, fewer read the history less often */
    int chunks = d->B;
    if (d->q_indptr) {
        const long long bound = (long long)d->R / kLogRows + d->B;
        chunks = (int)(bound < d->R ? bound : d->R);
    }
    const int most = 2 * sms / chunks > 1 ? 2 * sms / chunks : 1;
    int vs = ((d->V + most - 1) / most + 1023) & ~1023;
    if (vs > kLogSlice) vs = kLogSlice;
    cudaError_t e = cudaFuncSetAttribute(logits_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)sizeof(LogitSmem));
    if (e != cudaSuccess) return e;
    logits_kernel<T><<<dim3((d->V + vs - 1) / vs, chunks), kLogThreads, sizeof(LogitSmem), s>>>(*d, vs, err);
    return cudaGetLastError();
}

} /* namespace */

extern "C" {

int wc_kv_plan_launch(const waste_cuda_kv_plan_desc *d, unsigned int *err, int sms, void *stream)
{
    const size_t smem = sizeof(PlanSmem);
    cudaError_t e = cudaFuncSetAttribute(kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)smem);
    if (e != cudaSuccess) return (int)e;
    /* a token a thread. Counts updated in place need the cluster's barrier, so
     * a portable cluster's size; else any number of CTAs, one an SM at most */
    const bool inplace = d->n_blocks == d->n_blocks_out || d->free_head == d->free_head_out;
    int n = (d->T + kPlanThreads - 1) / kPlanThreads;
    n = n < 1 ? 1 : n;
    if (inplace) {
        int c = 1;
        while (c < 8 && c < n) c <<= 1;
        n = c;
    } else if (n > sms) {
        n = sms;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(n);
    cfg.blockDim = dim3(kPlanThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = inplace ? n : 1;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kv_plan_kernel, *d, err);
    wc_count_launches(1);
    return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

int wc_mla_rows_launch(const waste_cuda_mla_rows_desc *d, unsigned int *err, void *stream)
{
    const cudaStream_t s = (cudaStream_t)stream;
    wc_count_launches(1);
    if (d->x_dtype == WASTE_CUDA_F32) return (int)rows_launch<float>(d, err, s);
    if (d->x_dtype == WASTE_CUDA_F16) return (int)rows_launch<__half>(d, err, s);
    return (int)rows_launch<__nv_bfloat16>(d, err, s);
}

int wc_logits_launch(const waste_cuda_logits_desc *d, unsigned int *err, int sms, void *stream)
{
    const cudaStream_t s = (cudaStream_t)stream;
    wc_count_launches(1);
    if (d->dtype == WASTE_CUDA_F32) return (int)logits_launch<float>(d, err, sms, s);
    if (d->dtype == WASTE_CUDA_F16) return (int)logits_launch<__half>(d, err, sms, s);
    return (int)logits_launch<__nv_bfloat16>(d, err, sms, s);
}

int wc_clear_bits_launch(unsigned int *word, unsigned int bits, void *stream)
{
    clear_bits_kernel<<<1, 1, 0, (cudaStream_t)stream>>>(word, bits);
    wc_count_launches(1);
    return (int)cudaGetLastError();
}

} /* extern "C" */
