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
 * launch of one cluster (at most 8 CTAs of 512 threads, by the token count).
 * Every CTA makes both prefix sums for itself (B <= 4096 lengths, 8 a thread
 * at most), which costs less than handing them round, keeps them in shared
 * memory, and takes its share of the tokens and table entries. The outputs
 * may be the inputs' arrays: the cluster's barrier stands between the last
 * read of an input and the first write. Which slot a token gets follows from
 * the old table (blocks held) or the free list (blocks taken now), so no
 * table entry written here is read here. */
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
    const int rank = (int)cl.block_rank(), ncta = (int)cl.num_blocks();
    const int per = (d.B + kPlanThreads - 1) / kPlanThreads, r0 = tid * per;
    int q[kPlanPer], need[kPlanPer], held[kPlanPer];
    int sq = 0, sn = 0;
    unsigned int bad = 0, okm = 0;
    const int head = max(0, *d.free_head), avail = max(0, d.n_free - head);
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
        s.fstart[r] = served ? head + pn : -1;
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
    if (ncta > 1) cl.sync(); else __syncthreads();
    if (rank == 0) {
#pragma unroll
        for (int k = 0; k < kPlanPer; k++) {
            const int r = r0 + k;
            if (k >= per || r >= d.B) continue;
            const bool served = s.fstart[r] >= 0;
            d.n_blocks_out[r] = held[k] + (served ? need[k] : 0);
            d.kv_len[r] = served ? d.ctx_len[r] + q[k] : 0;
            d.q_indptr[r + 1] = min(s.qstart[r + 1], d.T);
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
 * One warp a row, the row in registers (kRowRegs floats a lane; longer rows
 * are read again), so x crosses memory once: the bytes bound it at prompt
 * lengths, a launch and one row's latency at decode. */
constexpr int kRowsWarps = 4;
constexpr int kRowRegs = 16;         /* 512 latents */

template <typename TX, typename TC>
__global__ void __launch_bounds__(kRowsWarps * 32) mla_rows_kernel(
    const waste_cuda_mla_rows_desc d, unsigned int *err)
{
    const int lane = threadIdx.x & 31, t = blockIdx.x * kRowsWarps + (threadIdx.x >> 5);
    if (t >= d.T) return;
    const int64_t slot = d.slot[t];
    if (slot < 0 || slot >= d.n_rows) {
        if (slot >= 0 && lane == 0) atomicOr(err, WASTE_CUDA_DERR_BAD_BLOCK);
        return;
    }
    const TX *x = static_cast<const TX *>(d.x) + (size_t)t * d.x_stride;
    TC *y = static_cast<TC *>(d.cache) + (size_t)slot * d.row_stride;
    float v[kRowRegs], s = 0.0f;
#pragma unroll
    for (int k = 0; k < kRowRegs; k++) {
        const int i = lane + 32 * k;
        v[k] = i < d.kl ? to_f(x[i]) : 0.0f;
    }
#pragma unroll
    for (int k = 0; k < kRowRegs; k++) s = fmaf(v[k], v[k], s);
    for (int i = lane + 32 * kRowRegs; i < d.kl; i += 32) {
        const float u = to_f(x[i]);
        s = fmaf(u, u, s);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float r = 1.0f / sqrtf(s / (float)d.kl + d.eps);
#pragma unroll
    for (int k = 0; k < kRowRegs; k++) {
        const int i = lane + 32 * k;
        if (i < d.kl) y[i] = from_f<TC>(v[k] * r * d.norm_w[i]);
    }
    for (int i = lane + 32 * kRowRegs; i < d.kl; i += 32)
        y[i] = from_f<TC>(to_f(x[i]) * r * d.norm_w[i]);
    for (int j = lane; j < d.rope / 2; j += 32) {
        float a = to_f(x[d.kl + 2 * j]), b = to_f(x[d.kl + 2 * j + 1]);
        if (d.inv_freq) {
            /* the angle in 64 bits, taken to [-pi, pi] there: at far positions
             * 32 bits lose its fraction of a turn */
            const double ang = (double)d.pos[t] * (double)d.inv_freq[j];
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
 * A CTA takes a slice of the ids of one request: the request's tokens that
 * fall into the slice are counted in shared memory (integer atomics: any
 * order gives the same counts), then the slice of each of the request's rows
 * is read, adjusted and written once. Each row's branch of drafted tokens is
 * counted before its slice and taken out again behind it. The bytes of the
 * logits bound it; the history is read again by each slice, from L2, so
 * slices are as wide as leaves enough CTAs to fill the GPU (wc_logits_launch).
 *
 * A count word holds the times produced, and bit 31 for "in the prompt". */
constexpr int kLogThreads = 256;
constexpr uint32_t kPrompt = 0x80000000u;

struct LogitRow {
    float rep, freq, pres;
    const float *bias;
};

__device__ __forceinline__ float adjust(float x, uint32_t c, uint32_t b, bool ok, const LogitRow &p)
{
    if (c) {
        x = x > 0.0f ? x / p.rep : x * p.rep;
        const uint32_t n = c & ~kPrompt;
        x -= p.freq * (float)n + (n ? p.pres : 0.0f);
    }
    if (b) x += p.bias[b - 1];
    return ok ? x : -INFINITY;
}

template <typename T>
__global__ void __launch_bounds__(kLogThreads) logits_kernel(const waste_cuda_logits_desc d, int vs)
{
    extern __shared__ __align__(16) uint32_t sml[];
    uint32_t *cnt = sml, *bia = sml + vs;
    const int tid = threadIdx.x, r = blockIdx.y, v0 = blockIdx.x * vs, nv = min(vs, d.V - v0);
    int q0 = r, q1 = r + 1;
    if (d.q_indptr) {
        q0 = min(max(d.q_indptr[r], 0), d.R);
        q1 = min(max(d.q_indptr[r + 1], q0), d.R);
    }
    if (q0 >= q1) return;
    for (int i = tid; i < vs; i += kLogThreads) {
        cnt[i] = 0;
        if (d.bias_indptr) bia[i] = 0;
    }
    __syncthreads();
    if (d.hist) {
        const int n = min(max(d.hist_len[r], 0), (int)min(d.hist_stride, (size_t)0x7fffffff));
        const int m = d.prompt_len ? d.prompt_len[r] : 0;
        const int *h = d.hist + (size_t)r * d.hist_stride;
#pragma unroll 4
        for (int i = tid; i < n; i += kLogThreads) {
            const unsigned u = (unsigned)h[i] - (unsigned)v0;
            if (u < (unsigned)nv) {
                if (i < m) atomicOr(&cnt[u], kPrompt);
                else atomicAdd(&cnt[u], 1u);
            }
        }
    }
    LogitRow p = { d.rep ? d.rep[r] : 1.0f, d.freq ? d.freq[r] : 0.0f, d.pres ? d.pres[r] : 0.0f, nullptr };
    if (d.bias_indptr) {
        const int b0 = max(d.bias_indptr[r], 0), b1 = d.bias_indptr[r + 1];
        p.bias = d.bias_val + b0;
        for (int i = b0 + tid; i < b1; i += kLogThreads) {
            const unsigned u = (unsigned)d.bias_id[i] - (unsigned)v0;
            if (u < (unsigned)nv) atomicMax(&bia[u], (uint32_t)(i - b0 + 1));
        }
    }
    __syncthreads();
    for (int t = q0; t < q1; t++) {
        if (d.draft) {
            for (int j = tid; j < q1 - q0; j += kLogThreads) {
                const bool on = d.tree ? j < 32 * d.tree_words &&
                                             ((d.tree[(size_t)t * d.tree_words + (j >> 5)] >> (j & 31)) & 1)
                                       : j <= t - q0;
                const unsigned u = (unsigned)d.draft[q0 + j] - (unsigned)v0;
                if (on && u < (unsigned)nv) atomicAdd(&cnt[u], 1u);
            }
            __syncthreads();
        }
        const uint32_t *allow = nullptr;
        if (d.allow) {
            const int a = d.allow_row ? d.allow_row[t] : t;
            if (a >= 0 && a < d.n_allow) allow = d.allow + (size_t)a * d.allow_words;
        }
        const T *x = static_cast<const T *>(d.logits) + (size_t)t * d.ld + v0;
        T *y = static_cast<T *>(d.out) + (size_t)t * d.ld_out + v0;
        for (int i = tid; i < nv; i += kLogThreads) {
            const bool ok = !allow || ((allow[(v0 + i) >> 5] >> ((v0 + i) & 31)) & 1);
            y[i] = from_f<T>(adjust(to_f(x[i]), cnt[i], d.bias_indptr ? bia[i] : 0u, ok, p));
        }
        if (d.draft) {
            __syncthreads();
            for (int j = tid; j < q1 - q0; j += kLogThreads) {
                const bool on = d.tree ? j < 32 * d.tree_words &&
                                             ((d.tree[(size_t)t * d.tree_words + (j >> 5)] >> (j & 31)) & 1)
                                       : j <= t - q0;
                const unsigned u = (unsigned)d.draft[q0 + j] - (unsigned)v0;
                if (on && u < (unsigned)nv) atomicSub(&cnt[u], 1u);
            }
            __syncthreads();
        }
    }
}

template <typename TX>
cudaError_t rows_launch(const waste_cuda_mla_rows_desc *d, unsigned int *err, cudaStream_t s)
{
    const dim3 grid((d->T + kRowsWarps - 1) / kRowsWarps), block(kRowsWarps * 32);
    if (d->dtype == WASTE_CUDA_F32) mla_rows_kernel<TX, float><<<grid, block, 0, s>>>(*d, err);
    else if (d->dtype == WASTE_CUDA_F16) mla_rows_kernel<TX, __half><<<grid, block, 0, s>>>(*d, err);
    else mla_rows_kernel<TX, __nv_bfloat16><<<grid, block, 0, s>>>(*d, err);
    return cudaGetLastError();
}

template <typename T>
cudaError_t logits_launch(const waste_cuda_logits_desc *d, int vs, cudaStream_t s)
{
    const size_t smem = (size_t)vs * 2 * sizeof(uint32_t);
    cudaError_t e = cudaFuncSetAttribute(logits_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)smem);
    if (e != cudaSuccess) return e;
    logits_kernel<T><<<dim3((d->V + vs - 1) / vs, d->B), kLogThreads, smem, s>>>(*d, vs);
    return cudaGetLastError();
}

} /* namespace */

extern "C" {

int wc_kv_plan_launch(const waste_cuda_kv_plan_desc *d, unsigned int *err, void *stream)
{
    const size_t smem = sizeof(PlanSmem);
    cudaError_t e = cudaFuncSetAttribute(kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)smem);
    if (e != cudaSuccess) return (int)e;
    /* one token a thread, up to a portable cluster */
    int n = 1;
    while (n < 8 && n * kPlanThreads < d->T) n <<= 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(n);
    cfg.blockDim = dim3(kPlanThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = n;
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

int wc_logits_launch(const waste_cuda_logits_desc *d, void *stream)
{
    /* the widest slice that still leaves four CTAs an SM */
    int vs = 8192;
    while (vs > 1024 && (long long)d->B * ((d->V + vs - 1) / vs) < 4 * 148) vs >>= 1;
    const cudaStream_t s = (cudaStream_t)stream;
    wc_count_launches(1);
    if (d->dtype == WASTE_CUDA_F32) return (int)logits_launch<float>(d, vs, s);
    if (d->dtype == WASTE_CUDA_F16) return (int)logits_launch<__half>(d, vs, s);
    return (int)logits_launch<__nv_bfloat16>(d, vs, s);
}

} /* extern "C" */
