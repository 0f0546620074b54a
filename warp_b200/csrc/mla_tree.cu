/*
 * mla_tree.cu — absorbed MLA attention of one or several new tokens a
 * request over a paged latent cache (waste_cuda_mla_tree_attn_dev in
 * include/waste_cuda.h). All heads share a request's cache rows, so a
 * request's new tokens times its heads are the rows of one product against
 * them:
 *   s[i][p] = scale * q_i . c_p,  o_i = sum_p softmax(s_i)_p c_p[:kl]
 * with the running maximum and sum of the softmax, so a cache row crosses
 * memory once per tile of query rows.
 *
 * The work is units of (query tile, key tile), flattened over all requests
 * and cut into equal contiguous ranges, one per CTA, from the lengths on the
 * device: the host knows none of them, and neither ragged lengths nor a
 * single long request leave SMs idle. A query tile whose units fall to one
 * CTA is finished there; otherwise each CTA leaves its partial sums
 * (unnormalised o, maximum, sum) in the workspace, at most two a CTA, and
 * mla_combine_kernel joins them in key order.
 */
#include "pdl.cuh"
#include "vq3r_common.cuh"
#include "waste_cuda.h"
#include "wc_launch.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

using namespace wc;

namespace {

constexpr int kMaxKl = 512;
constexpr int kMaxRope = 128;

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f(float v) { return v; }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }

/* ---- the schedule -----------------------------------------------------------
 * Request r of n tokens has rows token * heads + head, in tiles of NT; a
 * tile's keys come in tiles of KT. unit_prefix(i) is the number of units
 * before its tile i. In a chain of several tiles an early tile sees fewer
 * keys; its units are counted by a bound with a closed prefix sum,
 *   floor(sum_{j<i} (ctx + 1 + (j+1) NT/heads) / KT) + i,
 * which is at least the key tiles it sees and at most about one more (a unit
 * past them is empty). */
struct Req {
    int r, q0, n, ctx, kv, nt;       /* kv: rows seen at most, 0: nothing        */
    int bad;
};

struct Shape {
    waste_cuda_mla_tree_desc d;
    int NT, KT;
    unsigned int *err;
    float *part;                     /* [2 * grid][NT][kl] partial sums          */
    float *stat;                     /* [2 * grid][NT][2] their maxima and sums  */
    int4 *meta;                      /* [grid] the tile that starts to be split there */
};

__device__ __forceinline__ Req req_at(const Shape &p, int r)
{
    const waste_cuda_mla_tree_desc &d = p.d;
    Req q;
    q.r = r;
    q.q0 = min(max(d.q_indptr[r], 0), d.T);
    q.n = min(max(d.q_indptr[r + 1], q.q0), d.T) - q.q0;
    const long long cap = (long long)d.max_blocks * d.page;
    int kv = d.kv_len[r];
    q.bad = kv > cap;
    if (q.bad) kv = (int)cap;
    q.kv = kv < q.n ? 0 : kv;
    q.ctx = q.kv - (q.kv ? q.n : 0);
    q.nt = (int)(((long long)q.n * d.heads + p.NT - 1) / p.NT);
    return q;
}

__device__ __forceinline__ long long unit_prefix(const Shape &p, const Req &q, int i)
{
    if (!p.d.mask && q.nt > 1 && q.kv) {
        const long long H2 = 2ll * p.d.heads;
        return (H2 * i * (q.ctx + 1ll) + (long long)p.NT * i * (i + 1ll)) / (H2 * p.KT) + i;
    }
    return (long long)i * max(1, (q.kv + p.KT - 1) / p.KT);
}

/* One CTA's share of one query tile: key tiles [k0, k1). */
struct Seg {
    Req q;
    int tile, k0, k1;
    int vis;                         /* keys the tile's last row sees             */
    bool first, last;                /* the tile's units all before / behind are here */
    long long units;                 /* nominal units of this segment             */
    int row0, rows;                  /* rows of the request                       */
    long long tile_u0, tile_u1;      /* the tile's units, global                  */
};

struct Walk {
    long long u, u1, base;           /* next unit, end, the request's first unit  */
    int r;
    Req q;
};

/* All threads: the CTA's range of units and where it starts. `red` holds 66
 * long longs of shared memory. Returns false when the range is empty. */
__device__ bool walk_begin(const Shape &p, Walk &w, long long *red, long long &total)
{
    const int nt = blockDim.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = nt >> 5;
    const int per = (p.d.B + nt - 1) / nt, r0 = tid * per;
    long long sum = 0;
    for (int k = 0; k < per && r0 + k < p.d.B; k++) {
        const Req q = req_at(p, r0 + k);
        if (q.bad && blockIdx.x == 0) atomicOr(p.err, WASTE_CUDA_DERR_BAD_BLOCK);
        sum += unit_prefix(p, q, q.nt);
    }
    long long inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long a = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += a;
    }
    if (lane == 31) red[warp] = inc;
    __syncthreads();
    long long at = inc - sum, all = 0;
    for (int k = 0; k < nw; k++) {
        if (k < warp) at += red[k];
        all += red[k];
    }
    total = all;
    /* with fewer units than CTAs, the first CTAs take one each */
    const long long G = max(1ll, min((long long)gridDim.x, all)), c = blockIdx.x;
    w.u = c < G ? c * all / G : all;
    w.u1 = c < G ? (c + 1) * all / G : all;
    if (sum > 0 && at <= w.u && w.u < at + sum) {
        for (int k = 0; k < per && r0 + k < p.d.B; k++) {
            const Req q = req_at(p, r0 + k);
            const long long n = unit_prefix(p, q, q.nt);
            if (w.u < at + n) { red[64] = r0 + k; red[65] = at; break; }
            at += n;
        }
    }
    __syncthreads();
    if (w.u >= w.u1) return false;
    w.r = (int)red[64];
    w.base = red[65];
    w.q = req_at(p, w.r);
    return true;
}

__device__ __forceinline__ bool walk_next(const Shape &p, Walk &w, Seg &s)
{
    if (w.u >= w.u1) return false;
    long long n = unit_prefix(p, w.q, w.q.nt);
    while (w.u >= w.base + n) {
        w.base += n;
        w.q = req_at(p, ++w.r);
        n = unit_prefix(p, w.q, w.q.nt);
    }
    int lo = 0, hi = w.q.nt;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (w.base + unit_prefix(p, w.q, mid) <= w.u) lo = mid; else hi = mid;
    }
    const int H = p.d.heads;
    s.q = w.q;
    s.tile = lo;
    s.tile_u0 = w.base + unit_prefix(p, w.q, lo);
    s.tile_u1 = w.base + unit_prefix(p, w.q, lo + 1);
    const long long end = min(s.tile_u1, w.u1);
    s.first = w.u == s.tile_u0;
    s.last = end == s.tile_u1;
    s.row0 = lo * p.NT;
    s.rows = min(p.NT, w.q.n * H - s.row0);
    s.vis = p.d.mask || !w.q.kv ? w.q.kv : min(w.q.kv, w.q.ctx + (s.row0 + s.rows - 1) / H + 1);
    const int kt = (s.vis + p.KT - 1) / p.KT;
    s.k0 = (int)min((long long)kt, w.u - s.tile_u0);
    s.k1 = (int)min((long long)kt, end - s.tile_u0);
    w.u = end;
    return true;
}

/* Whether new token i of the request sees its new row j. */
__device__ __forceinline__ bool sees(const Shape &p, const Req &q, int i, int j)
{
    if (!p.d.mask) return j <= i;
    return j < 32 * p.d.mask_words &&
           ((__ldg(p.d.mask + (size_t)(q.q0 + i) * p.d.mask_words + (j >> 5)) >> (j & 31)) & 1);
}

/* The workspace slot of a split tile's segment: a CTA's range can begin
 * inside one tile and end inside another. */
__device__ __forceinline__ int part_slot(const Seg &s) { return 2 * blockIdx.x + (s.first ? 1 : 0); }

/* The CTA that holds a tile's first units names the tile for the combine:
 * {first row in tokens * heads, rows, last CTA, 1}. */
__device__ __forceinline__ void note_split(const Shape &p, const Seg &s, long long total)
{
    if (s.first && !s.last) {
        const long long G = min((long long)gridDim.x, total), c1 = (s.tile_u1 * G - 1) / total;
        p.meta[blockIdx.x] = make_int4(s.q.q0 * p.d.heads + s.row0, s.rows, (int)c1, 1);
    }
}

/* ---- any type, size, stride and page ---------------------------------------
 * fp32 arithmetic throughout. A CTA of 256 threads takes 32 query rows by
 * tiles of 64 keys. Scores: a warp takes 8 keys, 4 at a time, their values
 * strided over the lanes in registers, against 8 query rows at a time from
 * shared memory; the 32 sums of a batch are reduced across the lanes
 * together (31 shuffles), one (row, key) to a lane. Products: a thread owns
 * two of the kl columns for all 32 rows (64 sums in registers), the weights
 * broadcast from shared memory, the cache rows read again through L2. The
 * FMA rate bounds it from a few rows on. */
constexpr int kGenThreads = 256;
constexpr int kGenRows = 32;
constexpr int kGenKeys = 64;
constexpr int kGenJ = (kMaxKl + kMaxRope) / 32;

struct GenSmem {
    float p[kGenKeys][kGenRows];     /* scores, then weights                      */
    float m[kGenRows], l[kGenRows], a[kGenRows];
    long long off[kGenKeys];         /* element offset of a key's row, -1: none   */
    long long red[66];
};

template <typename T>
__global__ void __launch_bounds__(kGenThreads, 1) mla_gen_kernel(const __grid_constant__ Shape p)
{
    extern __shared__ __align__(16) unsigned char smg[];
    GenSmem &s = *reinterpret_cast<GenSmem *>(smg);
    float *qs = reinterpret_cast<float *>(smg + sizeof(GenSmem));    /* [32][D] */
    const waste_cuda_mla_tree_desc &d = p.d;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int H = d.heads, kl = d.kl, D = d.kl + d.rope, nj = (D + 31) / 32;
    const T *cache = static_cast<const T *>(d.cache);
    wc_pdl::trigger();
    if (tid == 0) p.meta[blockIdx.x] = make_int4(0, 0, 0, 0);
    Walk w;
    long long total;
    if (!walk_begin(p, w, s.red, total)) return;
    Seg g;
    while (walk_next(p, w, g)) {
        const int rows = g.rows;
        __syncthreads();
        for (int i = tid; i < kGenRows * D; i += kGenThreads) {
            const int row = i / D, j = i - row * D, at = g.row0 + row;
            qs[i] = row < rows ? to_f(static_cast<const T *>(d.q)[(size_t)(g.q.q0 + at / H) * d.q_token_stride +
                                                                 (size_t)(at % H) * d.q_head_stride + j])
                               : 0.0f;
        }
        if (tid < kGenRows) { s.m[tid] = -INFINITY; s.l[tid] = 0.0f; }
        float acc[2][kGenRows];
#pragma unroll
        for (int i = 0; i < kGenRows; i++) acc[0][i] = acc[1][i] = 0.0f;
        for (int kt = g.k0; kt < g.k1; kt++) {
            const int k0 = kt * kGenKeys, nk = min(kGenKeys, g.vis - k0);
            const bool tail = k0 + nk > g.q.ctx;
            __syncthreads();
            if (tid < nk) {
                const int key = k0 + tid, b = key / d.page;
                const int id = d.block_table[(size_t)g.q.r * d.max_blocks + b];
                const bool ok = id >= 0 && id < d.n_blocks;
                if (!ok) atomicOr(p.err, WASTE_CUDA_DERR_BAD_BLOCK);
                s.off[tid] = ok ? ((long long)id * d.page + (key - b * d.page)) * (long long)d.row_stride : -1;
            }
            __syncthreads();
#pragma unroll 1
            for (int kb = warp * 8; kb < warp * 8 + 8; kb += 4) {
                float c[4][kGenJ];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const long long off = kb + k < nk ? s.off[kb + k] : -1;
#pragma unroll
                    for (int j = 0; j < kGenJ; j++)
                        c[k][j] = j < nj && off >= 0 && lane + 32 * j < D ? to_f(cache[off + lane + 32 * j]) : 0.0f;
                }
#pragma unroll 1
                for (int rb = 0; rb < rows; rb += 8) {
                    float sum[32];                       /* [8 rows][4 keys] */
#pragma unroll
                    for (int i = 0; i < 32; i++) sum[i] = 0.0f;
#pragma unroll
                    for (int j = 0; j < kGenJ; j++) {
                        if (j >= nj) break;
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const float q = lane + 32 * j < D ? qs[(rb + i) * D + lane + 32 * j] : 0.0f;
#pragma unroll
                            for (int k = 0; k < 4; k++) sum[i * 4 + k] = fmaf(q, c[k][j], sum[i * 4 + k]);
                        }
                    }
                    /* halve the sums a lane holds at each step: lane l ends
                     * with sum l */
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) {
                        const bool up = lane & o;
#pragma unroll
                        for (int i = 0; i < o; i++) {
                            const float give = up ? sum[i] : sum[i + o];
                            const float got = __shfl_xor_sync(0xffffffffu, give, o);
                            sum[i] = (up ? sum[i + o] : sum[i]) + got;
                        }
                    }
                    const int row = rb + (lane >> 2), k = kb + (lane & 3), key = k0 + k;
                    const int tok = (g.row0 + row) / H;
                    bool see = row < rows && k < nk && s.off[k] >= 0;
                    if (see && key >= g.q.ctx) see = sees(p, g.q, tok, key - g.q.ctx);
                    s.p[k][row] = see ? sum[0] * d.scale : -INFINITY;
                }
            }
            __syncthreads();
            /* softmax of 4 rows a warp; two keys a lane */
#pragma unroll
            for (int i = 0; i < kGenRows / 8; i++) {
                const int row = warp * (kGenRows / 8) + i;
                if (row >= rows) break;
                const float x0 = lane < nk ? s.p[lane][row] : -INFINITY;
                const float x1 = lane + 32 < nk ? s.p[lane + 32][row] : -INFINITY;
                float mx = fmaxf(x0, x1);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                const float m0 = s.m[row], m1 = fmaxf(m0, mx), ref = m1 == -INFINITY ? 0.0f : m1;
                /* a masked key weighs exactly nothing; a NaN score stays one */
                const float e0 = x0 == -INFINITY ? 0.0f : expf(x0 - ref);
                const float e1 = x1 == -INFINITY ? 0.0f : expf(x1 - ref);
                float sum = e0 + e1;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                s.p[lane][row] = e0;
                s.p[lane + 32][row] = e1;
                __syncwarp();
                if (lane == 0) {
                    const float a = m0 == -INFINITY ? 0.0f : expf(m0 - ref);
                    s.a[row] = a;
                    s.l[row] = s.l[row] * a + sum;
                    s.m[row] = m1;
                }
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kGenRows; i++) {
                const float a = i < rows ? s.a[i] : 0.0f;
                acc[0][i] *= a;
                acc[1][i] *= a;
            }
            const bool c0 = tid < kl, c1 = tid + kGenThreads < kl;
#pragma unroll 4
            for (int k = 0; k < nk; k++) {
                const long long off = s.off[k];
                const float v0 = c0 && off >= 0 ? to_f(cache[off + tid]) : 0.0f;
                const float v1 = c1 && off >= 0 ? to_f(cache[off + tid + kGenThreads]) : 0.0f;
                const float4 *pk = reinterpret_cast<const float4 *>(s.p[k]);
                /* a row that does not see a new key is not to meet its
                 * values: they may be no numbers */
                const bool finite = isfinite(v0) && isfinite(v1);
#pragma unroll
                for (int i = 0; i < kGenRows / 4; i++) {
                    const float4 e = pk[i];
                    const float ee[4] = { e.x, e.y, e.z, e.w };
#pragma unroll
                    for (int z = 0; z < 4; z++) {
                        if (finite || !tail) {
                            acc[0][4 * i + z] = fmaf(ee[z], v0, acc[0][4 * i + z]);
                            acc[1][4 * i + z] = fmaf(ee[z], v1, acc[1][4 * i + z]);
                        } else if (ee[z] != 0.0f) {
                            acc[0][4 * i + z] += ee[z] * v0;
                            acc[1][4 * i + z] += ee[z] * v1;
                        }
                    }
                }
            }
        }
        __syncthreads();
        const bool whole = g.first && g.last;
        const int slot = part_slot(g);
#pragma unroll
        for (int i = 0; i < kGenRows; i++) {
            if (i >= rows) break;
            const int at = g.row0 + i;
            const float l = s.l[i], inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
            for (int z = 0; z < 2; z++) {
                const int j = tid + z * kGenThreads;
                if (j >= kl) continue;
                if (whole)
                    static_cast<T *>(d.o)[(size_t)(g.q.q0 + at / H) * d.o_token_stride +
                                          (size_t)(at % H) * d.o_head_stride + j] =
                        from_f<T>(l == 0.0f ? 0.0f : acc[z][i] * inv);
                else
                    p.part[((size_t)slot * kGenRows + i) * kl + j] = acc[z][i];
            }
        }
        if (tid < rows) {
            const float m = s.m[tid], l = s.l[tid];
            if (whole) {
                if (d.lse)
                    d.lse[(size_t)g.q.q0 * H + g.row0 + tid] = l == 0.0f ? -INFINITY : m + logf(l);
            } else {
                p.stat[((size_t)slot * kGenRows + tid) * 2] = m;
                p.stat[((size_t)slot * kGenRows + tid) * 2 + 1] = l;
            }
        }
        if (tid == 0) note_split(p, g, total);
    }
}

/* ---- split tiles joined ------------------------------------------------------
 * grid (CTAs of the attention, rows of a tile): the tile whose first units
 * CTA c held, one row. o = sum_s e^(m_s - M) o_s / sum_s e^(m_s - M) l_s over
 * its segments in key order. Bound by reading the partial sums, from L2.
 * LOG2: the maxima are in units of log2. */
constexpr int kCombThreads = 128;

template <typename T, int LOG2>
__global__ void __launch_bounds__(kCombThreads) mla_combine_kernel(const __grid_constant__ Shape p)
{
    wc_pdl::wait();
    const int c = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
    const int4 t = p.meta[c];
    if (!t.w || row >= t.y) return;
    const waste_cuda_mla_tree_desc &d = p.d;
    const int kl = d.kl;
    const float ln2 = 0.693147180559945f;
    float M = -INFINITY;
    for (int k = c; k <= t.z; k++) {
        const int slot = k == c ? 2 * c + 1 : 2 * k;
        M = fmaxf(M, p.stat[((size_t)slot * p.NT + row) * 2]);
    }
    const float ref = M == -INFINITY ? 0.0f : M;
    float acc[kMaxKl / kCombThreads] = {}, L = 0.0f;
    for (int k = c; k <= t.z; k++) {
        const int slot = k == c ? 2 * c + 1 : 2 * k;
        const float m = p.stat[((size_t)slot * p.NT + row) * 2], l = p.stat[((size_t)slot * p.NT + row) * 2 + 1];
        if (l == 0.0f) continue;                     /* saw nothing: its sums are not set */
        const float e = LOG2 ? exp2f(m - ref) : expf(m - ref);
        L = fmaf(e, l, L);
        const float *o = p.part + ((size_t)slot * p.NT + row) * kl;
#pragma unroll
        for (int j = 0; j < kMaxKl / kCombThreads; j++)
            if (tid + j * kCombThreads < kl) acc[j] = fmaf(e, o[tid + j * kCombThreads], acc[j]);
    }
    const int at = t.x + row, tok = at / d.heads, h = at - tok * d.heads;
    T *o = static_cast<T *>(d.o) + (size_t)tok * d.o_token_stride + (size_t)h * d.o_head_stride;
#pragma unroll
    for (int j = 0; j < kMaxKl / kCombThreads; j++)
        if (tid + j * kCombThreads < kl)
            o[tid + j * kCombThreads] = from_f<T>(L == 0.0f ? 0.0f : acc[j] / L);
    if (tid == 0 && d.lse)
        d.lse[at] = L == 0.0f ? -INFINITY : (LOG2 ? (M + log2f(L)) * ln2 : M + logf(L));
}

/* the workspace: partial sums | their statistics | the split tiles */
void carve(Shape *p, int grid)
{
    char *w = static_cast<char *>(p->d.ws);
    p->part = reinterpret_cast<float *>(w);
    w += (size_t)2 * grid * p->NT * p->d.kl * sizeof(float);
    p->stat = reinterpret_cast<float *>(w);
    w += (size_t)2 * grid * p->NT * 2 * sizeof(float);
    p->meta = reinterpret_cast<int4 *>(w);
}

constexpr int kTileMax = 64;         /* the largest NT */

template <typename T>
cudaError_t gen_launch(Shape &p, int sms, cudaStream_t s)
{
    p.NT = kGenRows;
    p.KT = kGenKeys;
    carve(&p, sms);
    const size_t smem = sizeof(GenSmem) + (size_t)kGenRows * (p.d.kl + p.d.rope) * sizeof(float);
    cudaError_t e = cudaFuncSetAttribute(mla_gen_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)smem);
    if (e != cudaSuccess) return e;
    mla_gen_kernel<T><<<sms, kGenThreads, smem, s>>>(p);
    wc_count_launches(1);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    e = wc_pdl::launch(mla_combine_kernel<T, 0>, dim3(sms, p.NT), dim3(kCombThreads), 0, s, true, p);
    wc_count_launches(1);
    return e;
}

} /* namespace */

extern "C" {

size_t wc_mla_tree_ws_bytes(int kl, int sms)
{
    return (size_t)2 * sms * kTileMax * (kl + 2) * sizeof(float) + (size_t)sms * sizeof(int4);
}

int wc_mla_tree_launch(const waste_cuda_mla_tree_desc *d, unsigned int *err, int sms, void *stream)
{
    Shape p = {};
    p.d = *d;
    p.err = err;
    const cudaStream_t s = (cudaStream_t)stream;
    if (d->dtype == WASTE_CUDA_F32) return (int)gen_launch<float>(p, sms, s);
    if (d->dtype == WASTE_CUDA_F16) return (int)gen_launch<__half>(p, sms, s);
    return (int)gen_launch<__nv_bfloat16>(p, sms, s);
}

} /* extern "C" */
