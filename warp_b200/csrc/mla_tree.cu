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
#include <type_traits>

using namespace wc;

namespace {

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
 *   floor(sum_{j<i} (ctx + 1 + (j+1) NT/heads) / KT) + i
 * (NT/heads in 2^-16, rounded up), which is at least the key tiles it sees
 * and at most about one more (a unit past them is empty). Units are 32 bits
 * wide: the host refuses calls whose sizes could pass that. At a kernel's
 * start every instruction is a cold fetch, so this is kept short: the one
 * thread that finds the CTA's first tile hands it to the others. */
struct Req {
    int r, q0, n, ctx, kv, nt;       /* kv: rows seen at most, 0: nothing        */
};

struct Shape {
    waste_cuda_mla_tree_desc d;
    int NT, KT, kt_log;              /* KT = 1 << kt_log                         */
    unsigned int step;               /* NT / (2 heads) in 2^-16, rounded up       */
    unsigned int *err;
    float *part;                     /* [2 * grid][NT][part_ld] partial sums      */
    float *stat;                     /* [2 * grid][NT][2] their maxima and sums  */
    int4 *meta;                      /* [grid] the tile that starts to be split there */
    int part_ld;                     /* kl in whole float4s                       */
};

__device__ __forceinline__ Req req_at(const Shape &p, int r)
{
    const waste_cuda_mla_tree_desc &d = p.d;
    Req q;
    const int a = d.q_indptr[r], b = d.q_indptr[r + 1], kv = d.kv_len[r];
    q.r = r;
    q.q0 = min(max(a, 0), d.T);
    q.n = min(max(b, q.q0), d.T) - q.q0;
    q.kv = min(kv, d.max_blocks * d.page);           /* longer: reported at the start */
    q.kv = q.kv < q.n ? 0 : q.kv;
    q.ctx = q.kv - (q.kv ? q.n : 0);
    q.nt = (int)(((unsigned)q.n * (unsigned)d.heads + p.NT - 1u) / (unsigned)p.NT);
    return q;
}

__device__ __forceinline__ int unit_prefix(const Shape &p, const Req &q, int i)
{
    if (!p.d.mask && q.nt > 1 && q.kv) {
        const unsigned long long k = (unsigned long long)i * (q.ctx + 1u);
        return (int)((k + ((unsigned long long)i * (i + 1u) * p.step >> 16)) >> p.kt_log) + i;
    }
    return i * max(1, (q.kv + p.KT - 1) >> p.kt_log);
}

/* A CTA's place in the units: CTA c of G has [c * all / G, (c+1) * all / G)
 * up to rounding; with fewer units than CTAs, the first CTAs have one each. */
__device__ __forceinline__ int cta_of_unit(int u, int all)
{
    const int G = min((int)gridDim.x, all), per = all / G, rem = all - per * G, lim = rem * (per + 1);
    return u < lim ? u / (per + 1) : rem + (u - lim) / per;
}

/* One CTA's share of one query tile: key tiles [k0, k1). */
struct Seg {
    Req q;
    int k0, k1;
    int vis;                         /* keys the tile's last row sees             */
    bool first, last;                /* the tile's first / last units are here    */
    int row0, rows;                  /* rows of the request                       */
    int tile_u1;                     /* behind the tile's last unit               */
};

struct Walk {
    int u, u1;                       /* next unit, end                            */
    int tile, tile_u0;               /* the next tile, its first unit             */
    Req q;
    int all;                         /* units of all CTAs                         */
};

struct WalkSmem {
    int sum[32];                     /* units of a warp's requests                */
    Walk w;
};

/* All threads (kWarps warps): the CTA's range of units and where it starts,
 * in s.w; u == u1 where it has none. */
template <int kWarps> __device__ __forceinline__ void walk_begin(const Shape &p, WalkSmem &s)
{
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (p.d.B + kWarps * 32 - 1) / (kWarps * 32), r0 = tid * per;
    int sum = 0;
    bool wrong = false;
    for (int k = 0; k < per && r0 + k < p.d.B; k++) {
        const Req q = req_at(p, r0 + k);
        const int a = p.d.q_indptr[r0 + k], b = p.d.q_indptr[r0 + k + 1];
        wrong |= a < 0 || b < a || b > p.d.T;
        const int kv = p.d.kv_len[r0 + k];
        if (blockIdx.x == 0 && (kv < 0 || kv > p.d.max_blocks * p.d.page))
            atomicOr(p.err, WASTE_CUDA_DERR_BAD_BLOCK);
        if (blockIdx.x == 0 && p.d.mask && q.n > 32 * p.d.mask_words) atomicOr(p.err, WASTE_CUDA_DERR_BAD_TREE);
        sum += unit_prefix(p, q, q.nt);
    }
    int at = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, at, o);
        if (lane >= o) at += a;
    }
    if (lane == 31) s.sum[warp] = at;
    /* requests whose tokens go backwards overlap, and their units could pass 32
     * bits; tokens cut off at T would take others for cached ones: every CTA sees
     * them, none has work */
    wrong = __syncthreads_or(wrong);
    if (wrong && blockIdx.x == 0 && tid == 0) atomicOr(p.err, WASTE_CUDA_DERR_BAD_BLOCK);
    int v = lane < kWarps ? s.sum[lane] : 0;
    int all = __reduce_add_sync(0xffffffffu, v);
    if (wrong) all = 0;
    v = __reduce_add_sync(0xffffffffu, lane < warp ? v : 0);
    at += v - sum;
    const int G = min((int)gridDim.x, all), c = blockIdx.x;
    int u = 0, u1 = 0;
    if (c < G) {
        const int each = all / G, rem = all - each * G;
        u = c * each + min(c, rem);
        u1 = u + each + (c < rem);
    }
    if (tid == 0 && u == u1) s.w.u = s.w.u1 = 0;
    if (u < u1 && at <= u && u < at + sum) {
        for (int k = 0; k < per; k++) {
            const Req q = req_at(p, r0 + k);
            const int n = unit_prefix(p, q, q.nt);
            if (u < at + n) {
                int lo = 0, hi = q.nt;
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (at + unit_prefix(p, q, mid) <= u) lo = mid; else hi = mid;
                }
                s.w = { u, u1, lo, at + unit_prefix(p, q, lo), q, all };
                break;
            }
            at += n;
        }
    }
    __syncthreads();
}

__device__ __forceinline__ bool walk_next(const Shape &p, Walk &w, Seg &s)
{
    if (w.u >= w.u1) return false;
    int base = w.tile_u0 - unit_prefix(p, w.q, w.tile);
    while (w.tile == w.q.nt) {
        base = w.tile_u0;
        w.q = req_at(p, w.q.r + 1);
        w.tile = 0;
    }
    const int H = p.d.heads, u0 = w.tile_u0;
    s.q = w.q;
    s.tile_u1 = w.tile_u0 = base + unit_prefix(p, w.q, w.tile + 1);
    const int end = min(s.tile_u1, w.u1);
    s.first = w.u == u0;
    s.last = end == s.tile_u1;
    s.row0 = w.tile * p.NT;
    s.rows = min(p.NT, w.q.n * H - s.row0);
    s.vis = p.d.mask || !w.q.kv ? w.q.kv : min(w.q.kv, w.q.ctx + (s.row0 + s.rows - 1) / H + 1);
    const int kt = (s.vis + p.KT - 1) >> p.kt_log;
    s.k0 = min(kt, w.u - u0);
    s.k1 = min(kt, end - u0);
    w.u = end;
    w.tile++;
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
__device__ __forceinline__ void note_split(const Shape &p, const Seg &s, int all)
{
    if (s.first && !s.last)
        p.meta[blockIdx.x] = make_int4(s.q.q0 * p.d.heads + s.row0, s.rows, cta_of_unit(s.tile_u1 - 1, all), 1);
}

/* ---- any type, size, stride and page ---------------------------------------
 * fp32 arithmetic throughout. A CTA of 256 threads takes 32 query rows by
 * tiles of 32 keys, both as fp32 rows in shared memory, rows 16 bytes past a
 * multiple of 128 apart so that float4 loads of successive rows meet no bank
 * twice. Scores and softmax: a lane has a key, a warp 4 rows, which its lanes
 * read together; the scores never leave the registers. Products: a thread owns
 * two of the kl columns for all rows, the weights read together (10 loads'
 * worth of shared memory for 64 FMAs a key). Shared memory bounds the scores
 * (32 x 32 rows of 512 + 64: 15 k cycles), the FMA rate the products (7 k). A
 * lone token of 32 heads over 4096 rows, one tile a CTA, takes 29 us with the
 * joining, a third of it cold starts: code that runs once is kept small.
 * Where rows are fp32 and 16-byte aligned the next tile's are copied asynchronously
 * meanwhile, if two tiles fit. */
constexpr int kGenThreads = 256;
constexpr int kGenRows = 32;
constexpr int kGenKeys = 32;

struct alignas(16) GenSmem {
    float p[kGenKeys][kGenRows + 4]; /* weights (key, row)                        */
    float m[kGenRows], l[kGenRows], a[kGenRows];
    long long off[kGenRows];         /* a row's elements in o                     */
    int tok[kGenRows];               /* a row's token in the request              */
    int bad[kGenKeys];               /* a new row that holds no finite number     */
    WalkSmem walk;
};

static_assert(sizeof(GenSmem) % 16 == 0, "rows behind it are read as float4");

__host__ __device__ constexpr int gen_ld(int D) { return ((D + 31) & ~31) + 4; }

template <typename T>
__global__ void __launch_bounds__(kGenThreads, 1) mla_gen_kernel(const __grid_constant__ Shape p, int bufs,
                                                                 int async)
{
    extern __shared__ __align__(16) unsigned char smg[];
    GenSmem &s = *reinterpret_cast<GenSmem *>(smg);
    const waste_cuda_mla_tree_desc &d = p.d;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int H = d.heads, kl = d.kl, D = d.kl + d.rope, ld = gen_ld(D), nv = (D + 3) / 4;
    float *qs = reinterpret_cast<float *>(smg + sizeof(GenSmem));    /* [32][ld]       */
    float *ks = qs + kGenRows * ld;                                  /* [bufs][32][ld] */
    const T *cache = static_cast<const T *>(d.cache);
    wc_pdl::trigger();
    if (tid == 0) p.meta[blockIdx.x] = make_int4(0, 0, 0, 0);
    /* the columns between D and the next float4 stay zero */
    for (int i = tid; i < (1 + bufs) * kGenRows * 4; i += kGenThreads)
        if (D + (i & 3) < nv * 4) qs[(i >> 2) * ld + D + (i & 3)] = 0.0f;
    walk_begin<kGenThreads / 32>(p, s.walk);
    Walk w = s.walk.w;
    Seg g;
    /* tile kt of the segment into buffer `buf`: 8 threads a key, rows past the
     * last seen one zero */
    auto fetch = [&](const Seg &g, int kt, int buf) {
        const int k = tid >> 3, sub = tid & 7, key = kt * kGenKeys + k;
        float *dst = ks + (buf * kGenKeys + k) * ld;
        bool in = key < g.vis;
        const T *src = cache;
        if (in) {
            const int b = key / d.page, id = d.block_table[(size_t)g.q.r * d.max_blocks + b];
            in = id >= 0 && id < d.n_blocks;
            if (!in && sub == 0) atomicOr(p.err, WASTE_CUDA_DERR_BAD_BLOCK);
            if (in) src += ((long long)id * d.page + (key - b * d.page)) * (long long)d.row_stride;
        }
        if (async & 1) {
            for (int i = sub; i < nv; i += 8)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                             ::"r"(smem_u32(dst + i * 4)), "l"(src + i * 4), "r"(in ? 16 : 0) : "memory");
        } else {
#pragma unroll 8
            for (int i = sub; i < D; i += 8) dst[i] = in ? to_f(src[i]) : 0.0f;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    while (walk_next(p, w, g)) {
        const int rows = g.rows;
        __syncthreads();
        if (g.k0 < g.k1) fetch(g, g.k0, 0);
        if (tid < kGenRows) {
            s.m[tid] = -INFINITY;
            s.l[tid] = 0.0f;
            s.tok[tid] = (g.row0 + tid) / H;
        }
        __syncthreads();
        /* a segment without keys waits for no copies, so it issues none: they would be
         * under way when the next segment's go to the same place */
        if (g.k0 < g.k1) {
            const int i = tid >> 3, tok = s.tok[i], h = g.row0 + i - tok * H;
            const T *src = static_cast<const T *>(d.q);
            if (i < rows) src += (size_t)(g.q.q0 + tok) * d.q_token_stride + (size_t)h * d.q_head_stride;
            if (async & 2) {
                for (int j = tid & 7; j < nv; j += 8)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                                 ::"r"(smem_u32(qs + i * ld + j * 4)), "l"(src + j * 4), "r"(i < rows ? 16 : 0) : "memory");
                asm volatile("cp.async.commit_group;" ::: "memory");
            } else {
#pragma unroll 8
                for (int j = tid & 7; j < D; j += 8) qs[i * ld + j] = i < rows ? to_f(src[j]) : 0.0f;
            }
        }
        /* the products' threads: two columns each, and where kl leaves threads over,
         * a part of the rows (in quads from quad0) */
        const int ct = kl > 256 ? 256 : kl > 128 ? 128 : kl > 64 ? 64 : 32, nq = kGenRows / 4 * ct / kGenThreads;
        const int c0 = 2 * (tid % ct), quad0 = tid / ct * nq;
        float acc[2][kGenRows];
#pragma unroll
        for (int i = 0; i < kGenRows; i++) acc[0][i] = acc[1][i] = 0.0f;
        for (int kt = g.k0; kt < g.k1; kt++) {
            const int k0 = kt * kGenKeys, buf = bufs == 2 ? (kt - g.k0) & 1 : 0;
            const bool tail = k0 + kGenKeys > g.q.ctx || k0 + kGenKeys > g.vis;
            float *kb = ks + buf * kGenKeys * ld;
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncthreads();
            if (bufs == 2 && kt + 1 < g.k1) fetch(g, kt + 1, buf ^ 1);
            if (tail) {
                /* a new row that holds a NaN or an infinity is zeros to the products;
                 * who sees it gets NaN weights, who does not is not touched */
                const int k = tid >> 3, key = k0 + k;
                float *row = kb + k * ld;
                bool bad = false;
                if (key >= g.q.ctx && key < g.vis)
                    for (int i = tid & 7; i < kl; i += 8) bad |= !isfinite(row[i]);
                bad = (__ballot_sync(0xffffffffu, bad) >> (lane & 24)) & 0xff;
                if ((tid & 7) == 0) s.bad[k] = bad;
                if (bad)
                    for (int i = tid & 7; i < kl; i += 8) row[i] = 0.0f;
                __syncthreads();
            }
            const int r0 = 4 * warp;
            if (r0 < rows) {
                float4 sum[4] = {};                           /* four chains a row           */
                const float4 *kp = reinterpret_cast<const float4 *>(kb + lane * ld);
                const float4 *qp = reinterpret_cast<const float4 *>(qs + r0 * ld);
#pragma unroll 4
                for (int v = 0; v < nv; v++) {
                    const float4 k = kp[v];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float4 q = qp[i * (ld / 4) + v];
                        sum[i].x = fmaf(q.x, k.x, sum[i].x);
                        sum[i].y = fmaf(q.y, k.y, sum[i].y);
                        sum[i].z = fmaf(q.z, k.z, sum[i].z);
                        sum[i].w = fmaf(q.w, k.w, sum[i].w);
                    }
                }
                const int key = k0 + lane;
                float e[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float x = ((sum[i].x + sum[i].y) + (sum[i].z + sum[i].w)) * d.scale;
                    if (tail) {
                        const bool see = key < g.vis && (key < g.q.ctx || (r0 + i < rows && sees(p, g.q, s.tok[r0 + i], key - g.q.ctx)));
                        if (!see) x = -INFINITY;
                        else if (s.bad[lane]) x = __int_as_float(0x7fc00000);
                    }
                    float mx = x;
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                    const float m0 = s.m[r0 + i], m1 = fmaxf(m0, mx), ref = m1 == -INFINITY ? 0.0f : m1;
                    /* a masked key weighs exactly nothing; a NaN score stays one */
                    e[i] = x == -INFINITY ? 0.0f : expf(x - ref);
                    float sum = e[i];
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    __syncwarp();
                    if (lane == 0) {
                        const float a = m0 == -INFINITY ? 0.0f : expf(m0 - ref);
                        s.a[r0 + i] = a;
                        s.l[r0 + i] = s.l[r0 + i] * a + sum;
                        s.m[r0 + i] = m1;
                    }
                }
                *reinterpret_cast<float4 *>(&s.p[lane][r0]) = make_float4(e[0], e[1], e[2], e[3]);
            }
            __syncthreads();
            /* rows by 8: rows past the tile's own are not looked at */
            auto products = [&](auto quads) {
                constexpr int kQuads = decltype(quads)::value;
#pragma unroll
                for (int i = 0; i < kQuads; i++) {
                    const float4 a = *reinterpret_cast<const float4 *>(s.a + 4 * (quad0 + i));
                    acc[0][4 * i] *= a.x; acc[0][4 * i + 1] *= a.y; acc[0][4 * i + 2] *= a.z; acc[0][4 * i + 3] *= a.w;
                    acc[1][4 * i] *= a.x; acc[1][4 * i + 1] *= a.y; acc[1][4 * i + 2] *= a.z; acc[1][4 * i + 3] *= a.w;
                }
#pragma unroll 2
                for (int k = 0; k < kGenKeys; k++) {
                    const float2 v = *reinterpret_cast<const float2 *>(kb + k * ld + c0);
                    const float4 *pk = reinterpret_cast<const float4 *>(s.p[k]) + quad0;
#pragma unroll
                    for (int i = 0; i < kQuads; i++) {
                        const float4 e = pk[i];
                        const float ee[4] = { e.x, e.y, e.z, e.w };
#pragma unroll
                        for (int z = 0; z < 4; z++) {
                            acc[0][4 * i + z] = fmaf(ee[z], v.x, acc[0][4 * i + z]);
                            acc[1][4 * i + z] = fmaf(ee[z], v.y, acc[1][4 * i + z]);
                        }
                    }
                }
            };
            if (c0 < kl && 4 * quad0 < rows) {
                if (nq == 8 && rows > 8) products(std::integral_constant<int, 8>());
                else if (nq == 4) products(std::integral_constant<int, 4>());
                else if (nq == 1) products(std::integral_constant<int, 1>());
                else products(std::integral_constant<int, 2>());
            }
            if (bufs == 1 && kt + 1 < g.k1) {
                __syncthreads();
                fetch(g, kt + 1, 0);
            }
        }
        __syncthreads();
        const bool whole = g.first && g.last;
        const int slot = part_slot(g), mine = min(rows - 4 * quad0, 4 * nq);      /* rows of this thread */
        if (whole) {
            if (tid < kGenRows) {
                const int tok = s.tok[tid], h = g.row0 + tid - tok * H;
                s.a[tid] = tid < rows && s.l[tid] != 0.0f ? 1.0f / s.l[tid] : 0.0f;
                s.off[tid] = (long long)(g.q.q0 + tok) * (long long)d.o_token_stride + (long long)h * d.o_head_stride;
            }
            __syncthreads();
        }
        /* little code a row: it is fetched cold, once (32 divisions and both ways of
         * storing, unrolled, took 24 k cycles) */
        if (whole) {
            T *o = static_cast<T *>(d.o) + c0;
#pragma unroll
            for (int i = 0; i < kGenRows; i++)
                if (i < mine && c0 < kl) {
                    const float inv = s.a[4 * quad0 + i];
                    T *to = o + s.off[4 * quad0 + i];
                    to[0] = from_f<T>(inv == 0.0f ? 0.0f : acc[0][i] * inv);
                    if (c0 + 1 < kl) to[1] = from_f<T>(inv == 0.0f ? 0.0f : acc[1][i] * inv);
                }
        } else if (c0 < p.part_ld) {
            float *o = p.part + ((size_t)slot * kGenRows + 4 * quad0) * p.part_ld + c0;
#pragma unroll
            for (int i = 0; i < kGenRows; i++)
                if (i < mine) *reinterpret_cast<float2 *>(o + i * p.part_ld) = make_float2(acc[0][i], acc[1][i]);
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
        if (tid == 0) note_split(p, g, w.all);
    }
}

/* ---- 16-bit caches on the tensor cores ---------------------------------------
 * Transposed: the cache rows are the M side of both products, so 32 rows of
 * queries (one token of 32 heads) fill an N of 32 and nothing is padded to
 * 128:
 *   S^T [128 keys x N]   = C [128 x (kl+rope)] . Q^T     A K-major
 *   O^T [kl x N]        += C^T [kl x 128] . P^T          A M-major, same bytes
 * One copy of the tile in shared memory serves both. N is 32 where a
 * request's rows fit that, else 64: the cache is read once per 32 or 64 rows
 * (the second by 64: one token of 64 heads, or two of 32). The rule is the mean
 * of the call's rows a request, which the host knows: 64 tokens of 32 heads in
 * 64 requests take 61 us at N = 32 and 74 at 64; trees of up to 16 nodes 133
 * and 109; 2 trees of up to 5 over 131003 rows 224 and 183; 512 tokens over
 * 8192 rows 657 and 433. In one call (L2 flushed before each) 512 tokens behind
 * 4096 rows beside 63 single ones take 488 and 361, 64 beside them 125 and 125.
 * Rows of T behind the last request's count towards the mean.
 *
 * Shared memory (1 CTA an SM): a ring of 32 KB pairs (128 keys x 2 swizzled
 * 64-column chunks) that TMA fills page by page, 5 pairs at N = 32 and 4 at
 * N = 64; the rope chunk; the query tile; P. A tile's pairs are held from
 * its first product to its last, which frees them one by one, so the next
 * tile's loads run under the second product. At N = 64 P lies where the rope
 * chunk was, which is read by then.
 *
 * Roles: warp 0 loads, one lane a box; a lane of warp 1 issues the products;
 * warps 2..17 do the softmax, a thread a key (TMEM lane) and a quarter of the
 * columns. The weights are taken against a reference per column, an earlier
 * tile's maximum, as long as none passes it by more than 2^kLazy (the 32-bit
 * sums and the types' ranges allow that; the results are the same up to
 * rounding): one vote a tile. Only where one does, at a row's start and a few
 * times after, are the tile's maxima found (redux over the lanes, shared
 * memory over the 4 warps), the reference moved and O in TMEM rescaled.
 *
 * What bounds it. N = 32: 64 tokens over 183 k bf16 rows (216 MB) take 61 us
 * with the joining, 3.5 TB/s. Traced tiles took 6.7 to 7.5 k cycles, where
 * 147 KB at an SM's share of HBM would take 6.4 k. At some ten tiles a CTA that
 * accounts for 36 us or so; the start (lengths, table, first tile: loads that
 * wait for one another), the end and the joining are left with the rest. N =
 * 64, the chain of a tile in one SM's shared memory: a tile is loaded (from L2:
 * 2.5 k cycles at 64 rows a box, 3.4 k at 32), its scores (36 products of 48
 * cycles, under the loads), the softmax 1.5 k, the second product 1.6 k. 512
 * tokens of 32 heads over 8192 rows take 434 us, 695 TFLOP/s, at 115 tiles a CTA
 * 7.4 k cycles each, so there the chain is all. Trees of up to 16 nodes for 16
 * requests take 109 us at 16.6 tiles a CTA, 12.9 k each: half of it is the start
 * and end of query tiles and the joining. Two trees over 131003 rows take 183 us,
 * 12.2 k a tile: a request's query tiles sweep its rows out of step, which reads
 * 481 MB from HBM for 246 MB of rows. Measured and slower: V loaded again instead of held,
 * for an N of 96 (554 us where N = 64 took 445), rows sent for towards L2 two
 * tiles ahead (64 tokens: 62 -> 70 us).
 *
 * Every wait is bounded: one that runs out raises WC_ERR_TMA_WAIT and
 * `dead`, upon which the roles run out their loops without waiting, issue
 * nothing more, and drain what is in flight. */
constexpr int kTcSoft = 512;          /* softmax threads */
constexpr int kTcThreads = 64 + kTcSoft;
constexpr int kTcKeys = 128;
constexpr int kPairBytes = 2 * kTcKeys * 128;
constexpr float kLazy = 6.0f;
constexpr int kMaxPairs = 5;

template <int N> struct TcCfg {
    static constexpr int pairs = N == 64 ? 4 : 5;
    static constexpr int NC = N / 4;                          /* columns a thread   */
    static constexpr int p_row = N * 2;                       /* bytes of a P row    */
    static constexpr int off_rope = pairs * kPairBytes;
    static constexpr int off_p = N == 64 ? off_rope : off_rope + kTcKeys * 128;
    static constexpr int off_q = N == 64 ? off_rope + kTcKeys * 128 : off_p + kTcKeys * p_row;
    static constexpr int off_ctl = off_q + 9 * N * 128;
};

template <int N> struct TcCtl {
    uint64_t pair_full[kMaxPairs], pair_empty[kMaxPairs];
    uint64_t rope_full, rope_empty, q_full, s_full, p_ready, o_done, drain;
    uint32_t tmem;
    volatile int dead;
    WalkSmem walk;
    float mx[4][4][N / 4];            /* [quarter][quadrant][column]                  */
    alignas(16) float col[4][2][N / 4]; /* [quarter] a factor and the reference of each column */
    long long qoff[N], ooff[2][N];   /* a tile row's elements in q (-1: no row) and o */
    int tok[N];                      /* its token in the request                     */
    uint32_t krow[kTcKeys];          /* a key's row of the cache, without TMA         */
    unsigned char nan_row[kTcKeys];  /* a new row that holds no finite number        */
    /* the softmax warps' segments: the next is found while some are at the last */
    Seg seg[3];
    int more[3];
    Walk walk_soft;                  /* theirs: the other roles may still read walk's */
};

template <int N>
__device__ __forceinline__ bool tc_wait(TcCtl<N> &c, uint64_t *bar, uint32_t parity, unsigned int *err)
{
    for (int i = 0; i < kMbarLimit; i++) {
        uint32_t done;
        asm volatile("{\n\t.reg .pred p;\n\t"
                     "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                     "selp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
        if (done) return true;
        if (c.dead) return false;
    }
    c.dead = 1;
    atomicOr(err, WC_ERR_TMA_WAIT);
    return false;
}

__device__ __forceinline__ void mbar_arrive(uint64_t *bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool elect()
{
    uint32_t r;
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ void tc_commit(uint64_t *bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];"
                 ::"r"(smem_u32(bar)) : "memory");
}
/* Shared-memory operand descriptors: the low word has the start address and
 * the leading offset, the high word the stride offset, version 1 and the
 * swizzle (128 B: 2, 64 B: 4); offsets in bytes. */
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) { return (addr >> 4) | (lbo >> 4) << 16; }
__host__ __device__ constexpr uint32_t desc_hi(uint32_t sbo, uint32_t swizzle)
{
    return (sbo >> 4) | 1u << 14 | swizzle << 29;
}
template <uint32_t AHI, uint32_t BHI>
__device__ __forceinline__ void tc_mma(uint32_t d, uint32_t alo, uint32_t blo, uint32_t idesc, uint32_t acc)
{
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
                 "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %6};\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}\n"
                 ::"r"(d), "r"(alo), "r"(blo), "r"(idesc), "r"(acc), "n"(AHI), "n"(BHI) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
/* a named barrier of 128 threads that also votes */
__device__ __forceinline__ bool bar_any(int id, bool v)
{
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %2, 0;\n\tbar.red.or.pred p, %1, 128, q;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}" : "=r"(r) : "r"(id), "r"((uint32_t)v) : "memory");
    return r != 0;
}
__device__ __forceinline__ void bar_named(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }

template <int NC> __device__ __forceinline__ void tm_ld(float *v, uint32_t addr)
{
    uint32_t *u = reinterpret_cast<uint32_t *>(v);
#pragma unroll
    for (int k = 0; k + 16 <= NC; k += 16)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                     "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                     : "=r"(u[k]), "=r"(u[k + 1]), "=r"(u[k + 2]), "=r"(u[k + 3]), "=r"(u[k + 4]),
                       "=r"(u[k + 5]), "=r"(u[k + 6]), "=r"(u[k + 7]), "=r"(u[k + 8]), "=r"(u[k + 9]),
                       "=r"(u[k + 10]), "=r"(u[k + 11]), "=r"(u[k + 12]), "=r"(u[k + 13]),
                       "=r"(u[k + 14]), "=r"(u[k + 15])
                     : "r"(addr + k));
    if (NC == 8)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]),
                       "=r"(u[5]), "=r"(u[6]), "=r"(u[7]) : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
template <int NC> __device__ __forceinline__ void tm_st(const float *v, uint32_t addr)
{
    const uint32_t *u = reinterpret_cast<const uint32_t *>(v);
#pragma unroll
    for (int k = 0; k + 16 <= NC; k += 16)
        asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
                     "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                     ::"r"(addr + k), "r"(u[k]), "r"(u[k + 1]), "r"(u[k + 2]), "r"(u[k + 3]), "r"(u[k + 4]),
                       "r"(u[k + 5]), "r"(u[k + 6]), "r"(u[k + 7]), "r"(u[k + 8]), "r"(u[k + 9]),
                       "r"(u[k + 10]), "r"(u[k + 11]), "r"(u[k + 12]), "r"(u[k + 13]),
                       "r"(u[k + 14]), "r"(u[k + 15]) : "memory");
    if (NC == 8)
        asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                     ::"r"(addr), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]),
                       "r"(u[5]), "r"(u[6]), "r"(u[7]) : "memory");
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

/* The largest of the 32 lanes' values, NaN left out, in every lane. */
__device__ __forceinline__ float warp_max(float v)
{
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

/* Sums of NC values over the 32 lanes: lane l ends with that of column
 * l % NC. */
template <int NC> __device__ __forceinline__ float lane_sums(float *v, int lane)
{
#pragma unroll
    for (int o = 16; o >= NC; o >>= 1) {
#pragma unroll
        for (int i = 0; i < NC; i++) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    }
#pragma unroll
    for (int o = NC / 2; o > 0; o >>= 1) {
        const bool up = lane & o;
#pragma unroll
        for (int i = 0; i < o; i++) {
            const float give = up ? v[i] : v[i + o];
            const float got = __shfl_xor_sync(0xffffffffu, give, o);
            v[i] = (up ? v[i + o] : v[i]) + got;
        }
    }
    return v[0];
}

template <typename T, int N, bool TMA>
__global__ void __launch_bounds__(kTcThreads, 1) mla_tc_kernel(const __grid_constant__ Shape p,
                                                               const __grid_constant__ CUtensorMap map,
                                                               int box_rows)
{
    using Cfg = TcCfg<N>;
    constexpr int NC = Cfg::NC;
    constexpr bool kF16 = sizeof(T) == 2 && std::is_same<T, __half>::value;
    /* weights of fp16 are scaled up, so that small ones keep their bits */
    constexpr float kBias = kF16 ? 8.0f : 0.0f;
    extern __shared__ unsigned char smt[];
    unsigned char *sm = smt + ((1024 - (smem_u32(smt) & 1023)) & 1023);
    TcCtl<N> &c = *reinterpret_cast<TcCtl<N> *>(sm + Cfg::off_ctl);
    const waste_cuda_mla_tree_desc &d = p.d;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int npair = (d.kl + 127) / 128, nchunk = d.kl / 64 + (d.rope > 0), H = d.heads;
    const bool odd = d.kl & 64;                               /* the last pair is one chunk  */

    wc_pdl::trigger();
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;"
                     ::"r"(smem_u32(&c.tmem)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (tid == 0) {
        p.meta[blockIdx.x] = make_int4(0, 0, 0, 0);
        for (int i = 0; i < Cfg::pairs; i++) { mbar_init(&c.pair_full[i], TMA ? 1 : 32); mbar_init(&c.pair_empty[i], 1); }
        mbar_init(&c.rope_full, TMA ? 1 : 32);
        mbar_init(&c.rope_empty, 1);
        mbar_init(&c.q_full, kTcSoft / 32);
        mbar_init(&c.s_full, 1);
        mbar_init(&c.p_ready, kTcSoft / 32);
        mbar_init(&c.o_done, 1);
        mbar_init(&c.drain, 1);
        c.dead = 0;
        mbar_fence_init();
    }
    tc_fence_before();
    walk_begin<kTcThreads / 32>(p, c.walk);
    tc_fence_after();
    Walk w = c.walk.w;
    const bool any = w.u < w.u1;
    const uint32_t tmem = c.tmem, tm_s = tmem + 4 * N;            /* O | S^T */
    if (any && warp == 0) {
        Seg g;
        int it = 0, ur = 0;                                   /* pairs and rope chunks issued */
        if (TMA) {
            /* ---- loads: a lane a box of box_rows keys ---- */
            while (walk_next(p, w, g)) {
                for (int kt = g.k0; kt < g.k1; kt++) {
                    const int k0 = kt * kTcKeys, nk = min(kTcKeys, g.vis - k0);
                    const int nbox = (nk + box_rows - 1) / box_rows;
                    int blk = 0, row = 0;
                    if (lane < nbox) {
                        const int key = k0 + lane * box_rows, b = key / d.page;
                        row = key - b * d.page;
                        blk = d.block_table[(size_t)g.q.r * d.max_blocks + b];
                        if (blk < 0 || blk >= d.n_blocks) {
                            atomicOr(p.err, WASTE_CUDA_DERR_BAD_BLOCK);
                            blk = (int)d.n_blocks;                /* reads zeros                 */
                        }
                    }
                    const uint32_t chunk_tx = (uint32_t)(nbox * box_rows) * 128u;
                    for (int j = 0; j <= npair; j++) {
                        const bool rope = j == npair, both = !rope && !(odd && j == npair - 1);
                        if (rope && d.rope == 0) continue;
                        uint64_t *full = rope ? &c.rope_full : &c.pair_full[it % Cfg::pairs];
                        uint64_t *empty = rope ? &c.rope_empty : &c.pair_empty[it % Cfg::pairs];
                        const int use = rope ? ur : it / Cfg::pairs;
                        bool ok = true;
                        if (use > 0) ok = tc_wait(c, empty, (use - 1) & 1, p.err);
                        ok = __all_sync(0xffffffffu, ok && !c.dead);
                        if (!ok) continue;
                        if (lane == 0) mbar_expect_tx(full, both ? 2 * chunk_tx : chunk_tx);
                        __syncwarp();
                        if (lane < nbox) {
                            unsigned char *dst = sm + (rope ? Cfg::off_rope : (it % Cfg::pairs) * kPairBytes) +
                                                 lane * box_rows * 128;
                            tma_load_3d(dst, &map, rope ? d.kl : j * 128, row, blk, full);
                            if (both) tma_load_3d(dst + kTcKeys * 128, &map, j * 128 + 64, row, blk, full);
                        }
                        if (rope) ur++; else it++;
                    }
                }
            }
            if (c.dead) {                                     /* what is in flight lands     */
                for (int i = 0; i < Cfg::pairs; i++)
                    if (it > i) mbar_wait(&c.pair_full[i], ((it - 1 - i) / Cfg::pairs) & 1);
                if (ur > 0) mbar_wait(&c.rope_full, (ur - 1) & 1);
            }
        } else {
            /* ---- loads of other pages: 16 bytes a lane, 8 lanes a row's chunk. What was
             * issued is handed over before any wait for room, and at the end ---- */
            uint64_t *pend[kMaxPairs + 1];
            int npend = 0;
            auto flush = [&]() {
                asm volatile("cp.async.wait_all;" ::: "memory");
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
#pragma unroll
                for (int i = 0; i <= kMaxPairs; i++)
                    if (i < npend) mbar_arrive(pend[i]);
                npend = 0;
            };
            constexpr uint32_t kNoRow = 0xffffffffu;
            const T *cache = static_cast<const T *>(d.cache);
            const int u = lane & 7;
            while (walk_next(p, w, g)) {
                for (int kt = g.k0; kt < g.k1; kt++) {
                    const int k0 = kt * kTcKeys;
                    __syncwarp();
                    for (int i = lane; i < kTcKeys; i += 32) {
                        const int key = k0 + i, b = key / d.page;
                        uint32_t row = kNoRow;
                        if (key < g.vis) {
                            const int id = d.block_table[(size_t)g.q.r * d.max_blocks + b];
                            if (id < 0 || id >= d.n_blocks) atomicOr(p.err, WASTE_CUDA_DERR_BAD_BLOCK);
                            else row = (uint32_t)id * (uint32_t)d.page + (uint32_t)(key - b * d.page);
                        }
                        c.krow[i] = row;
                    }
                    __syncwarp();
                    for (int j = 0; j <= npair; j++) {
                        const bool rope = j == npair, both = !rope && !(odd && j == npair - 1);
                        if (rope && d.rope == 0) continue;
                        uint64_t *full = rope ? &c.rope_full : &c.pair_full[it % Cfg::pairs];
                        uint64_t *empty = rope ? &c.rope_empty : &c.pair_empty[it % Cfg::pairs];
                        const int use = rope ? ur : it / Cfg::pairs;
                        bool ok = true;
                        if (use > 0) {
                            flush();
                            ok = tc_wait(c, empty, (use - 1) & 1, p.err);
                        }
                        ok = __all_sync(0xffffffffu, ok && !c.dead);
                        if (!ok) continue;
                        const uint32_t dst = smem_u32(sm + (rope ? Cfg::off_rope : (it % Cfg::pairs) * kPairBytes));
                        const int col = (rope ? d.kl : j * 128) + u * 8, end = rope ? d.kl + d.rope : d.kl;
                        for (int r = lane >> 3; r < kTcKeys; r += 4) {
                            const uint32_t row = c.krow[r];
                            const bool in = row != kNoRow;
                            const T *src = cache + (in ? (size_t)row * d.row_stride : 0) + (col < end ? col : 0);
                            const uint32_t to = dst + r * 128 + ((u ^ (r & 7)) << 4);
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                                         ::"r"(to), "l"(src), "r"(in && col < end ? 16 : 0) : "memory");
                            if (both)
                                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                                             ::"r"(to + kTcKeys * 128), "l"(src + 64), "r"(in ? 16 : 0) : "memory");
                        }
                        pend[npend++] = full;
                        if (rope) ur++; else it++;
                    }
                }
            }
            flush();
        }
    } else if (any && warp == 1) {
        /* ---- products: one lane ---- */
        if (elect()) {
            Seg g;
            constexpr uint32_t fmt = kF16 ? 0u : 1u;
            constexpr uint32_t id_s = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(N >> 3) << 17) | (8u << 24);
            constexpr uint32_t id_o = id_s | (1u << 15) | (1u << 16);
            constexpr uint32_t kHi = desc_hi(1024, 2), kHiP = desc_hi(8 * Cfg::p_row, N == 64 ? 2 : 4);
            const uint32_t sm0 = smem_u32(sm);
            const uint32_t k_lo = desc_lo(sm0, 16), v_lo = desc_lo(sm0, kTcKeys * 128);
            const uint32_t q_lo = desc_lo(sm0 + Cfg::off_q, 16), p_lo = desc_lo(sm0 + Cfg::off_p, 16);
            const uint32_t r_lo = desc_lo(sm0 + Cfg::off_rope, 16);
            const int rope_steps = (d.rope + 15) / 16;
            int slot = 0, par = 0;                            /* the next pair in the ring   */
            int unit = 0, segs = 0;
            bool ok = true;
            auto step = [&]() {
                if (++slot == Cfg::pairs) { slot = 0; par ^= 1; }
            };
            /* S^T of unit u, whose pairs come next in the ring */
            auto scores = [&](int u) {
                tc_fence_after();
                for (int j = 0; j < npair && ok; j++) {
                    ok = tc_wait(c, &c.pair_full[slot], par, p.err);
                    if (!ok) return;
                    const uint32_t a = k_lo + slot * (kPairBytes / 16), b = q_lo + j * (2 * N * 128 / 16);
                    const int steps = odd && j == npair - 1 ? 4 : 8;
#pragma unroll
                    for (int k = 0; k < 8; k++)
                        if (k < steps)
                            tc_mma<kHi, kHi>(tm_s, a + (k >> 2) * (kTcKeys * 128 / 16) + (k & 3) * 2,
                                             b + (k >> 2) * (N * 128 / 16) + (k & 3) * 2, id_s, (j | k) != 0);
                    step();
                }
                if (d.rope > 0 && ok) {
                    ok = tc_wait(c, &c.rope_full, u & 1, p.err);
                    if (!ok) return;
                    const uint32_t b = q_lo + (d.kl / 64) * (N * 128 / 16);
                    for (int k = 0; k < rope_steps; k++)
                        tc_mma<kHi, kHi>(tm_s, r_lo + k * 2, b + k * 2, id_s, 1u);
                }
                if (!ok) return;
                tc_commit(&c.s_full);
                if (N != 64) tc_commit(&c.rope_empty);
            };
            while (ok && walk_next(p, w, g)) {
                if (g.k0 == g.k1) continue;
                ok = tc_wait(c, &c.q_full, segs & 1, p.err);
                for (int kt = g.k0; kt < g.k1 && ok; kt++, unit++) {
                    const int slot0 = slot, par0 = par;       /* of the tile's pairs, held   */
                    scores(unit);
                    if (ok) ok = tc_wait(c, &c.p_ready, unit & 1, p.err);
                    if (!ok) break;
                    tc_fence_after();
                    slot = slot0;
                    par = par0;
                    for (int j = 0; j < npair; j++) {
                        const uint32_t a = v_lo + slot * (kPairBytes / 16);
#pragma unroll
                        for (int k = 0; k < 8; k++)
                            tc_mma<kHi, kHiP>(tmem + j * N, a + k * (2048 / 16), p_lo + k * (16 * Cfg::p_row / 16),
                                              id_o, kt > g.k0 || k > 0);
                        tc_commit(&c.pair_empty[slot]);
                        step();
                    }
                    if (N == 64) tc_commit(&c.rope_empty);
                }
                if (ok) tc_commit(&c.o_done);
                segs++;
            }
            if (!ok) {                                        /* the products in flight end */
                tc_commit(&c.drain);
                mbar_wait(&c.drain, 0);
            }
        }
        __syncwarp();
    } else if (any && warp >= 2) {
        /* ---- softmax ---- */
        constexpr float kNone = -3e38f;                       /* no reference yet            */
        const int st = tid - 64, quarter = st >> 7, quad = warp & 3, key_row = quad * 32 + lane, c0 = quarter * NC;
        const uint32_t tm_lane = (uint32_t)(quad * 32) << 16;
        const float scale2 = d.scale * 1.4426950408889634f;
        float(*mine)[NC] = c.col[quarter];                    /* the 4 warps write the same  */
        float(*sx)[NC] = c.mx[quarter];
        int unit = 0, segs = 0, pos = 0;                      /* pos: the segment's first pair */
        /* tables of segment i's rows, and its query tile: swizzled 128-byte rows,
         * zeros past its rows and columns, a row's eight 16-byte units of a chunk
         * to eight threads */
        auto tables = [&](int i, int o) {                     /* o: which of the offsets     */
            const Seg &g = c.seg[i];
            if (st < N) {
                const int at = g.row0 + st, tok = at / H, h = at - tok * H;
                const bool in = st < g.rows;
                c.tok[st] = in ? tok : 0x3fffffff;
                c.qoff[st] = in ? (long long)(g.q.q0 + tok) * (long long)d.q_token_stride + (long long)h * (long long)d.q_head_stride : -1ll;
                c.ooff[o][st] = (long long)(g.q.q0 + tok) * (long long)d.o_token_stride + (long long)h * d.o_head_stride;
            }
        };
        auto queries = [&](int i) {
            if (c.seg[i].k0 == c.seg[i].k1) return;
            const int D = d.kl + d.rope, u = st & 7, row = st >> 3;
            if (row < N) {
                const long long off = c.qoff[row];
                const T *src = static_cast<const T *>(d.q) + off + u * 8;
                unsigned char *dst = sm + Cfg::off_q + row * 128 + ((u ^ (row & 7)) << 4);
                uint4 v[9];
#pragma unroll
                for (int k = 0; k < 9; k++)
                    v[k] = off >= 0 && k < nchunk && k * 64 + u * 8 < D
                               ? __ldg(reinterpret_cast<const uint4 *>(src + k * 64)) : make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int k = 0; k < 9; k++)
                    if (k < nchunk) *reinterpret_cast<uint4 *>(dst + k * N * 128) = v[k];
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&c.q_full);
        };
        auto next = [&](int i) {                              /* one thread                  */
            Walk v = c.walk_soft;
            Seg n;
            c.more[i] = walk_next(p, v, n);
            c.walk_soft = v;
            c.seg[i] = n;
        };
        if (st == 0) {
            c.walk_soft = w;
            next(0);
        }
        bar_named(5, kTcSoft);
        tables(0, 0);
        bar_named(5, kTcSoft);
        queries(0);
        for (int cur = 0, which = 0;; which ^= 1) {
            const int then = cur == 2 ? 0 : cur + 1;
            const Seg &g = c.seg[cur];
            if (st == 0) next(then);                          /* while the first tile loads  */
            const bool whole = g.first && g.last;
            const int slot = part_slot(g);
            /* the references (less the fp16 bias) lie in mine[1] */
            if (lane < NC) mine[1][lane] = kNone;
            __syncwarp();
            float l[NC];
#pragma unroll
            for (int i = 0; i < NC; i++) l[i] = 0.0f;
            for (int kt = g.k0; kt < g.k1; kt++, unit++) {
                const bool tail = kt * kTcKeys + kTcKeys > g.q.ctx || kt * kTcKeys + kTcKeys > g.vis;
                float x[NC];
                tc_wait(c, &c.s_full, unit & 1, p.err);
                tc_fence_after();
                tm_ld<NC>(x, tm_s + tm_lane + c0);
                uint32_t seen = 0xffffffffu;                  /* columns that see this key   */
                bool bad = false;
                const int key = kt * kTcKeys + key_row;
                if (tail) {
                    /* rows past the request's are zeros to the second product, and so is
                     * a new row that holds a NaN or an infinity: who sees it gets NaN
                     * weights, who does not is not touched. A quarter takes a pair. */
                    const int at = pos + (kt - g.k0) * npair + quarter, sl = at % Cfg::pairs;
                    unsigned char *mem = sm + sl * kPairBytes + key_row * 128;
                    const int units = odd && quarter == npair - 1 ? 8 : 16;
                    if (quarter < npair) tc_wait(c, &c.pair_full[sl], (at / Cfg::pairs) & 1, p.err);
                    if (quarter == 0) c.nan_row[key_row] = 0;
                    bar_named(5, kTcSoft);
                    if (quarter < npair && key >= g.q.ctx && key < g.vis) {
                        /* an exponent of ones carries into its half's top bit */
                        constexpr uint32_t e = kF16 ? 0x7c007c00u : 0x7f807f80u, one = kF16 ? 0x04000400u : 0x00800080u;
                        uint32_t found = 0;
#pragma unroll 4
                        for (int u = 0; u < units; u++) {
                            const uint4 v = *reinterpret_cast<const uint4 *>(
                                mem + (u >> 3) * kTcKeys * 128 + (((u + key_row) & 7) << 4));
                            found |= ((v.x & e) + one) | ((v.y & e) + one) | ((v.z & e) + one) | ((v.w & e) + one);
                        }
                        if (found & 0x80008000u) c.nan_row[key_row] = 1;
                    }
                    bar_named(5, kTcSoft);
                    bad = c.nan_row[key_row];
                    if (quarter < npair && (bad || key >= g.vis)) {
                        for (int u = 0; u < units; u++)
                            *reinterpret_cast<uint4 *>(mem + (u >> 3) * kTcKeys * 128 + (((u + key_row) & 7) << 4)) =
                                make_uint4(0, 0, 0, 0);
                    }
                    const int nj = key - g.q.ctx;             /* its place among the new rows */
                    const bool in = key < g.vis;
                    int last = -1;
                    bool see = false;
                    seen = 0;
#pragma unroll
                    for (int i = 0; i < NC; i++) {
                        const int tok = c.tok[c0 + i];
                        if (tok != last) {
                            last = tok;
                            see = in && (nj < 0 || (tok < g.q.n && sees(p, g.q, tok, nj)));
                        }
                        if (see) seen |= 1u << i;
                    }
                }
                /* the exponents: x becomes x * scale2 - reference, masked ones -infinity.
                 * The product is rounded as the reference's was, so that the largest key's
                 * difference is 0 at any size of the scores; fused, the product's own
                 * rounding would be left, which at scores of 2^31 is a weight of 0 or
                 * infinity. */
                auto exponents = [&]() {
#pragma unroll
                    for (int i = 0; i < NC; i += 4) {
                        const float4 r = *reinterpret_cast<const float4 *>(&mine[1][i]);
                        x[i] = __fadd_rn(__fmul_rn(x[i], scale2), -r.x);
                        x[i + 1] = __fadd_rn(__fmul_rn(x[i + 1], scale2), -r.y);
                        x[i + 2] = __fadd_rn(__fmul_rn(x[i + 2], scale2), -r.z);
                        x[i + 3] = __fadd_rn(__fmul_rn(x[i + 3], scale2), -r.w);
                    }
                    if (tail) {
#pragma unroll
                        for (int i = 0; i < NC; i++)
                            x[i] = !(seen >> i & 1) ? -INFINITY : bad ? __int_as_float(0x7fc00000) : x[i];
                    }
                };
                exponents();
                float top = x[0];
#pragma unroll
                for (int i = 1; i < NC; i++) top = fmaxf(top, x[i]);
                if (bar_any(1 + quarter, top > kBias + kLazy)) {
                    tm_ld<NC>(x, tm_s + tm_lane + c0);
                    float mx = -INFINITY;                     /* of column c0 + lane         */
#pragma unroll
                    for (int i = 0; i < NC; i++) {
                        const float m = warp_max(seen >> i & 1 ? __fmul_rn(x[i], scale2) : -INFINITY);
                        if (lane == i) mx = m;
                    }
                    const int lc = min(lane, NC - 1);
                    if (lane < NC) sx[quad][lane] = mx;
                    float r = mine[1][lc];
                    bar_named(1 + quarter, 128);
                    mx = fmaxf(fmaxf(sx[0][lc], sx[1][lc]), fmaxf(sx[2][lc], sx[3][lc]));
                    float a = 1.0f;
                    /* the same difference that the vote saw, and a reference not below
                     * mx - kBias: from 2^25 on sums with these constants round, and a
                     * weight of 2^16 is no fp16 */
                    if (__fsub_rn(mx, r) > kBias + kLazy) {
                        const float to = __fsub_ru(mx, kBias);
                        a = ex2(r - to);
                        r = to;
                    }
                    if (lane < NC) { mine[0][lane] = a; mine[1][lane] = r; }
                    bar_named(1 + quarter, 128);              /* and sx is read              */
#pragma unroll
                    for (int i = 0; i < NC; i++) l[i] *= mine[0][i];
                    exponents();
                    if (kt > g.k0) {
                        /* the products before are done: S's commit followed them */
#pragma unroll 1
                        for (int j = 0; j < npair; j++) {
#pragma unroll 1
                            for (int h = 0; h < NC; h += 8) {
                                float o[8];
                                tm_ld<8>(o, tmem + tm_lane + j * N + c0 + h);
#pragma unroll
                                for (int i = 0; i < 8; i++) o[i] *= mine[0][h + i];
                                tm_st<8>(o, tmem + tm_lane + j * N + c0 + h);
                            }
                        }
                    }
                    __syncwarp();
                }
                /* the weights in the type of the rows, as the products take both operands
                 * in one type: each is off by half a step at most (2^-8 in bf16, 2^-11 in
                 * fp16), independent errors that leave o of 64 tokens in bf16 2.0e-3
                 * from 64 bits where weights of 32 bits leave 1.7e-3, its own rounding.
                 * Weights in two parts would double the product. The sums are of the
                 * unrounded ones. */
                uint32_t pk[NC / 2];
#pragma unroll
                for (int i = 0; i < NC; i += 2) {
                    const float e0 = ex2(x[i]), e1 = ex2(x[i + 1]);
                    l[i] += e0;
                    l[i + 1] += e1;
                    pk[i / 2] = pack2<T>(e0, e1);
                }
                unsigned char *pr = sm + Cfg::off_p + key_row * Cfg::p_row;
                const int sw = N == 64 ? key_row & 7 : (key_row >> 1) & 3;
#pragma unroll
                for (int u = 0; u < NC / 8; u++)
                    *reinterpret_cast<uint4 *>(pr + (((c0 / 8 + u) ^ sw) << 4)) =
                        make_uint4(pk[4 * u], pk[4 * u + 1], pk[4 * u + 2], pk[4 * u + 3]);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                tc_fence_before();
                __syncwarp();                                 /* an arrival a warp: they are serial */
                if (lane == 0) mbar_arrive(&c.p_ready);
            }
            pos += (g.k1 - g.k0) * npair;
            /* the next segment's queries first: its products run under what follows */
            bar_named(5, kTcSoft);
            const bool more = c.more[then];
            if (more) {
                tables(then, which ^ 1);
                bar_named(5, kTcSoft);
                queries(then);
            }
            /* ---- the segment's result ---- */
            const int lc = min(lane, NC - 1);
            const float m = mine[1][lc];                      /* of column c0 + lc           */
            float sum = lane_sums<NC>(l, lane);
            if (lane < NC) sx[quad][lane] = sum;
            bar_named(1 + quarter, 128);
            sum = (sx[0][lc] + sx[1][lc]) + (sx[2][lc] + sx[3][lc]);
            if (lane < NC) mine[0][lane] = sum == 0.0f ? 0.0f : 1.0f / sum;
            bar_named(1 + quarter, 128);                      /* sx is read                  */
            const int row = c0 + lane;
            if (quad == 0 && lane < NC && row < g.rows) {
                if (whole) {
                    if (d.lse)
                        d.lse[(size_t)g.q.q0 * H + g.row0 + row] =
                            sum == 0.0f ? -INFINITY : (m + log2f(sum)) * 0.693147180559945f;
                } else {
                    p.stat[((size_t)slot * N + row) * 2] = sum == 0.0f ? -INFINITY : m;
                    p.stat[((size_t)slot * N + row) * 2 + 1] = sum;
                }
            }
            const bool some = g.k0 < g.k1;
            if (some) {
                tc_wait(c, &c.o_done, segs & 1, p.err);
                tc_fence_after();
                segs++;
            }
            if (some || whole) {
                const int nc = min(NC, g.rows - c0);
#pragma unroll 1
                for (int j = 0; j < npair; j++) {
                    float o[NC];
                    if (some) tm_ld<NC>(o, tmem + tm_lane + j * N + c0);
                    const int cd = j * 128 + key_row;
                    if (cd >= d.kl) continue;                 /* the last chunk has no pair   */
                    if (whole) {
                        T *dst = static_cast<T *>(d.o) + cd;
#pragma unroll
                        for (int i = 0; i < NC; i++)
                            if (i < nc)
                                dst[c.ooff[which][c0 + i]] = from_f<T>(some && mine[0][i] != 0.0f ? o[i] * mine[0][i] : 0.0f);
                    } else {
                        float *dst = p.part + (slot * N + c0) * p.part_ld + cd;
#pragma unroll
                        for (int i = 0; i < NC; i++)
                            if (i < nc) dst[i * p.part_ld] = o[i];
                    }
                }
            }
            tc_fence_before();
            if (st == 0) note_split(p, g, w.all);
            if (!more) break;
            cur = then;
        }
    }
    __syncthreads();
    tc_fence_after();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

/* ---- split tiles joined ------------------------------------------------------
 * o = sum_s w_s o_s / sum_s w_s l_s, w_s = e^(m_s - M), over a split tile's
 * segments in key order. Bound by reading the partial sums from L2, so each
 * thread has kCombDeep segments' loads in flight. The blocks (four an SM, all
 * resident) share out the list of split tiles that the attention left: with
 * few segments two rows at a time, 128 threads of float4s each; with many (a
 * long row alone on the GPU) a quarter of a row's columns, a warp an eighth of
 * the segments in turns, the warps' sums added in order. LOG2: the maxima are
 * in units of log2. */
constexpr int kCombThreads = 256;
constexpr int kCombDeep = 8;
constexpr int kCombMax = 256;        /* CTAs of the attention at most             */

template <typename T, int LOG2>
__global__ void __launch_bounds__(kCombThreads, 4) mla_combine_kernel(const __grid_constant__ Shape p, int ctas)
{
    __shared__ int4 meta[kCombMax];
    __shared__ int start[kCombMax + 1];
    __shared__ float sw[kCombMax], red[8], redl[8];
    __shared__ __align__(16) float4 part_s[8][32];
    wc_pdl::wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const waste_cuda_mla_tree_desc &d = p.d;
    const int kl = d.kl, ld = p.part_ld / 4;
    const float4 *part = reinterpret_cast<const float4 *>(p.part);
    const float2 *stat = reinterpret_cast<const float2 *>(p.stat);
    {
        const int4 t = tid < ctas ? p.meta[tid] : make_int4(0, 0, 0, 0);
        const int items = !t.w ? 0 : t.z - tid < kCombDeep ? (t.y + 1) / 2 : 4 * t.y;
        int at = items;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, at, o);
            if (lane >= o) at += v;
        }
        meta[tid] = t;
        if (lane == 31) start[warp] = at;
        __syncthreads();
        int v = lane < 8 ? start[lane] : 0;
        v = __reduce_add_sync(0xffffffffu, lane < warp ? v : 0);
        __syncthreads();
        start[tid] = at + v - items;
        if (tid == kCombMax - 1) start[kCombMax] = at + v;
        __syncthreads();
    }
    const int items = start[kCombMax];
    auto store = [&](int row, int col, float4 acc, float L, float M) {
        const int tok = row / d.heads, h = row - tok * d.heads;
        T *o = static_cast<T *>(d.o) + (size_t)tok * d.o_token_stride + (size_t)h * d.o_head_stride + col * 4;
        const float vals[4] = { acc.x, acc.y, acc.z, acc.w };
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (col * 4 + j < kl) o[j] = from_f<T>(L == 0.0f ? 0.0f : vals[j] * inv);
        if (col == 0 && d.lse)
            d.lse[row] = L == 0.0f ? -INFINITY : (LOG2 ? (M + log2f(L)) * 0.693147180559945f : M + logf(L));
    };
    auto add = [](float4 &a, float e, float4 v) {
        a.x = fmaf(e, v.x, a.x);
        a.y = fmaf(e, v.y, a.y);
        a.z = fmaf(e, v.z, a.z);
        a.w = fmaf(e, v.w, a.w);
    };
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
        int c = 0;                                            /* the last with start <= item */
#pragma unroll
        for (int o = kCombMax / 2; o > 0; o >>= 1)
            if (start[c + o] <= item) c += o;
        const int4 t = meta[c];
        const int n = t.z - c + 1, at = item - start[c];
        auto slot = [&](int k, int row) { return (size_t)((k == 0 ? 2 * c + 1 : 2 * (c + k)) * p.NT + row); };
        if (n <= kCombDeep) {
            const int row = at * 2 + (tid >> 7), col = tid & 127;
            if (row >= t.y) continue;
            float2 ml[kCombDeep];
            float4 v[kCombDeep];
#pragma unroll
            for (int u = 0; u < kCombDeep; u++) {
                ml[u] = u < n ? stat[slot(u, row)] : make_float2(-INFINITY, 0.0f);
                v[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (u < n && col < ld) v[u] = part[slot(u, row) * ld + col];
            }
            float M = -INFINITY, L = 0.0f;
#pragma unroll
            for (int u = 0; u < kCombDeep; u++) M = fmaxf(M, ml[u].x);
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int u = 0; u < kCombDeep; u++) {
                /* a segment that saw nothing weighs nothing: its sums are not set */
                if (ml[u].y == 0.0f) continue;
                const float x = ml[u].x - (M == -INFINITY ? 0.0f : M), e = LOG2 ? exp2f(x) : expf(x);
                L = fmaf(e, ml[u].y, L);
                add(acc, e, v[u]);
            }
            store(t.x + row, col, acc, L, M);
            continue;
        }
        const int row = at >> 2, col = (at & 3) * 32 + lane;
        float2 ml = make_float2(-INFINITY, 0.0f);             /* segment tid's               */
        if (tid < n) ml = stat[slot(tid, row)];
        float M = ml.x;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
        if (lane == 0) red[warp] = M;
        __syncthreads();
        M = red[0];
#pragma unroll
        for (int k = 1; k < 8; k++) M = fmaxf(M, red[k]);
        const float x = ml.x - (M == -INFINITY ? 0.0f : M);
        const float e = ml.y == 0.0f ? 0.0f : (LOG2 ? exp2f(x) : expf(x));
        sw[tid] = e;
        float L = e * ml.y;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
        if (lane == 0) redl[warp] = L;
        __syncthreads();
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int k0 = warp * kCombDeep; k0 < n; k0 += 8 * kCombDeep) {
            float4 v[kCombDeep];
#pragma unroll
            for (int u = 0; u < kCombDeep; u++)
                v[u] = col < ld && k0 + u < n && sw[k0 + u] != 0.0f ? part[slot(k0 + u, row) * ld + col]
                                                                     : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int u = 0; u < kCombDeep; u++)
                if (k0 + u < n) add(acc, sw[k0 + u], v[u]);
        }
        part_s[warp][lane] = acc;
        __syncthreads();
        if (warp == 0 && col < ld) {
            L = redl[0];
#pragma unroll
            for (int k = 1; k < 8; k++) {
                add(acc, 1.0f, part_s[k][lane]);
                L += redl[k];
            }
            store(t.x + row, col, acc, L, M);
        }
        __syncthreads();
    }
}

/* the workspace: partial sums | their statistics | the split tiles (each in whole 16 bytes) */
void carve(Shape *p, int grid)
{
    char *w = static_cast<char *>(p->d.ws);
    p->step = (unsigned)(((unsigned long long)p->NT * 65536 + 2ull * p->d.heads - 1) / (2ull * p->d.heads));
    p->part_ld = (p->d.kl + 3) & ~3;
    p->part = reinterpret_cast<float *>(w);
    w += (size_t)2 * grid * p->NT * p->part_ld * sizeof(float);
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
    p.kt_log = 5;
    carve(&p, sms);
    const int D = p.d.kl + p.d.rope, ld = gen_ld(D);
    /* bit 0: the cache's rows are copied asynchronously, bit 1: the queries' */
    int async = 0;
    if (sizeof(T) == 4 && D % 4 == 0) {
        async |= p.d.row_stride % 4 == 0 && ((uintptr_t)p.d.cache & 15) == 0;
        async |= p.d.q_token_stride % 4 == 0 && p.d.q_head_stride % 4 == 0 && ((uintptr_t)p.d.q & 15) == 0 ? 2 : 0;
    }
    size_t smem = sizeof(GenSmem) + (size_t)3 * kGenRows * ld * sizeof(float);
    const int bufs = smem <= 227 * 1024 ? 2 : 1;
    if (bufs == 1) smem -= (size_t)kGenRows * ld * sizeof(float);
    cudaError_t e = cudaFuncSetAttribute(mla_gen_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)smem);
    if (e != cudaSuccess) return e;
    mla_gen_kernel<T><<<sms, kGenThreads, smem, s>>>(p, bufs, async);
    wc_count_launches(1);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    e = wc_pdl::launch(mla_combine_kernel<T, 0>, dim3(4 * sms), dim3(kCombThreads), 0, s, true, p, sms);
    wc_count_launches(1);
    return e;
}

template <typename T, int N, bool TMA>
cudaError_t tc_launch(Shape &p, const CUtensorMap &map, int box_rows, int sms, cudaStream_t s)
{
    p.NT = N;
    p.KT = kTcKeys;
    p.kt_log = 7;
    carve(&p, sms);
    const size_t smem = TcCfg<N>::off_ctl + sizeof(TcCtl<N>) + 1024;
    static_assert(TcCfg<N>::off_ctl + sizeof(TcCtl<N>) + 1024 <= 227 * 1024, "attention tile exceeds shared memory");
    cudaError_t e = cudaFuncSetAttribute(mla_tc_kernel<T, N, TMA>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)smem);
    if (e != cudaSuccess) return e;
    mla_tc_kernel<T, N, TMA><<<sms, kTcThreads, smem, s>>>(p, map, box_rows);
    wc_count_launches(1);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    e = wc_pdl::launch(mla_combine_kernel<T, 1>, dim3(4 * sms), dim3(kCombThreads), 0, s, true, p, sms);
    wc_count_launches(1);
    return e;
}

template <typename T>
cudaError_t tc_launch(Shape &p, const CUtensorMap &map, int box_rows, int sms, cudaStream_t s)
{
    const bool few = (long long)p.d.T * p.d.heads <= 32ll * p.d.B;
    if (box_rows > 1)
        return few ? tc_launch<T, 32, true>(p, map, box_rows, sms, s) : tc_launch<T, 64, true>(p, map, box_rows, sms, s);
    return few ? tc_launch<T, 32, false>(p, map, box_rows, sms, s) : tc_launch<T, 64, false>(p, map, box_rows, sms, s);
}

} /* namespace */

extern "C" {

/* Whether the tensor-core kernel takes the call: a 16-bit cache of whole
 * 64-column chunks, a rope part of at most one, and rows that 16-byte copies
 * can start at (0: the other kernel's). Where pages are whole 8-row swizzle
 * groups TMA loads them, in boxes of 64 columns by the returned number of
 * rows; 1: they are copied row by row, which takes two to three times as long
 * (64 tokens over up to 4096 rows each: 61 us by TMA, 140 by rows; 512 tokens
 * over 8192 rows: 433 and 1330). */
int wc_mla_tree_box(const waste_cuda_mla_tree_desc *d)
{
    const uintptr_t addr = (uintptr_t)d->q | (uintptr_t)d->cache;
    if (d->dtype == WASTE_CUDA_F32 || d->kl % 64 || d->rope > 64 || d->rope % 8 || (addr & 15) ||
        d->row_stride % 8 || d->q_token_stride % 8 || d->q_head_stride % 8)
        return 0;
    if (d->page % 8 || d->n_blocks < 1 || d->n_blocks > 0x7fffffff ||
        d->row_stride * 2 * d->page >= ((size_t)1 << 40))
        return d->n_blocks < 0xffffffffll / d->page ? 1 : 0;
    int r = 8;
    while (r < kTcKeys && d->page % (2 * r) == 0) r *= 2;
    return r;
}

size_t wc_mla_tree_ws_bytes(int kl, int sms)
{
    return (size_t)2 * sms * kTileMax * (((kl + 3) & ~3) + 2) * sizeof(float) + (size_t)sms * sizeof(int4);
}

int wc_mla_tree_launch(const waste_cuda_mla_tree_desc *d, const CUtensorMap *map, int box_rows,
                       unsigned int *err, int sms, void *stream)
{
    Shape p = {};
    p.d = *d;
    p.err = err;
    const cudaStream_t s = (cudaStream_t)stream;
    if (sms > kCombMax) sms = kCombMax;
    if (box_rows > 0)
        return (int)(d->dtype == WASTE_CUDA_F16 ? tc_launch<__half>(p, *map, box_rows, sms, s)
                                                : tc_launch<__nv_bfloat16>(p, *map, box_rows, sms, s));
    if (d->dtype == WASTE_CUDA_F32) return (int)gen_launch<float>(p, sms, s);
    if (d->dtype == WASTE_CUDA_F16) return (int)gen_launch<__half>(p, sms, s);
    return (int)gen_launch<__nv_bfloat16>(p, sms, s);
}

} /* extern "C" */
