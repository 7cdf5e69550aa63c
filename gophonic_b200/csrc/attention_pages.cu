// Attention over listed pages of the cache: every (row, kv head) has a list of logical pages, and the row attends to the keys of
// those pages at positions up to its own.  Entries that name no page of the row's past are passed over; a row whose list holds
// nothing it can see leaves zeros.
//
// Single rows.  A cluster of CTAs owns one (row, kv head): the CTAs take equal stretches of the list's pages, each with a running
// softmax of its own, and join their results through distributed shared memory, so there is neither scratch memory nor a second
// kernel.  The query heads of the group are the rows of the tiles and share every key and value that is read.
//   bfloat16: both products on mma.sync, a page of 64 keys at a time, 16 keys a warp, pages asked for three deep by cp.async;
//   float32:  CUDA cores, half a page a stage, three deep by cp.async.
// Neither these kernels nor the selection ahead of them let the kernel behind them start early: its CTAs took the SMs that clusters
// were waiting for (36 layers of one token behind 32768, 64 pages: 5.2 ms a step with early starts, 3.7 without).
// Scores, the softmax and the sums are float32; with bfloat16 the probabilities are rounded to bfloat16 for the second product, as
// the values are (tensor cores take both operands in one type): 0.0021 to 0.0023 of the result's size against 64 bits, where rounding
// the result alone leaves 0.0017.
#include "mma.cuh"
#include "api.h"

#include <cooperative_groups.h>
#include <math.h>

int gb_attention_pages_tc5_accepts(const PagesParams& p);
int gb_attention_pages_tc5(const PagesParams& p, cudaStream_t stream);

namespace {

namespace cg = cooperative_groups;
typedef __nv_bfloat16 bf16;
constexpr float LOG2E = 1.4426950408889634f;
constexpr int THREADS = 128;
constexpr int MAX_TOP = 1024;     // entries of a list
// Rows times key heads from which on runs of rows go to tcgen05 (attention_pages_tc5.cu), us here / there, 32 pages behind 20000: 8
// key heads, one sequence of 4 rows 11.7 / 14.0, of 8 rows 16.8 / 15.6, of 16 rows 28 / 18; eight sequences of 2 rows 28 / 20; two
// key heads, one sequence of 16 rows 13 / 18, of 32 rows 18 / 19, of 48 rows 28 / 21.  Rows are counted as the longest sequence's times
// the sequences, of which the launch is made.
constexpr int TC5_MIN_UNITS = 64;

// The row's listed pages that it can see, in the list's order, packed into `to`, and behind them (from to[p.top] on) where they are in
// the planes; how many there are.  Every thread of the CTA.  (Looked up page by page, the block table's latency stood ahead of
// every page's copies: some 600 cycles of 2000.)
__device__ __forceinline__ int pack_list(const PagesParams& p, const int* bt, const int* list, int own_page, int* to, int* counts) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int n = 0;
    for (int base = 0; base < p.top; base += THREADS) {
        const int i = base + tid;
        const int lp = i < p.top ? list[i] : -1;
        const bool ok = lp >= 0 && lp <= own_page && lp < p.bt_stride;
        const int place = ok ? (int)page_of(bt, lp * GB_PAGE, p.bt_stride, p.pages) : 0;
        const unsigned who = __ballot_sync(0xffffffffu, ok);
        if (lane == 0) counts[warp] = __popc(who);
        __syncthreads();
        int at = n + __popc(who & ((1u << lane) - 1u));
        for (int w = 0; w < THREADS / 32; w++) {
            if (w < warp) at += counts[w];
            n += counts[w];
        }
        if (ok) {
            to[at] = lp;
            to[p.top + at] = place;
        }
        __syncthreads();
    }
    return n;
}

// What the CTAs of a cluster leave for one another: per head of the chunk its maximum, sum and weighted values.  Joined by all of them:
// CTA r of the cluster writes every PIECES-th four channels.  All pieces' values are asked for before the first is used: one
// trip through the cluster's shared memory instead of two dozen.  saw: the row's list names a page it can see.
template <typename T, int PIECES>
__device__ __forceinline__ void join_pieces(const float* ml, const float* os, int nh, int hd, T* out, bool saw) {
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = PIECES == 1 ? 0 : (int)cluster.block_rank();
    const int quads = hd / 4;
    for (int idx = threadIdx.x * PIECES + rank; idx < nh * quads; idx += THREADS * PIECES) {
        const int r = idx / quads, c = (idx - r * quads) * 4;
        float2 v[PIECES];
        float4 x[PIECES];
#pragma unroll
        for (int w = 0; w < PIECES; w++) {
            const float* m = PIECES == 1 ? ml : cluster.map_shared_rank(ml, w);
            const float* o = PIECES == 1 ? os : cluster.map_shared_rank(os, w);
            v[w] = *reinterpret_cast<const float2*>(m + 2 * r);
            x[w] = *reinterpret_cast<const float4*>(o + (size_t)r * hd + c);
        }
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < PIECES; w++) M = fmaxf(M, v[w].x);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        const float base = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int w = 0; w < PIECES; w++) {
            const float e = exp2f(v[w].x - base);        // a NaN score leaves no maximum but a NaN sum, which stays one
            L += e * v[w].y;
            acc.x += e * x[w].x;
            acc.y += e * x[w].y;
            acc.z += e * x[w].z;
            acc.w += e * x[w].w;
        }
        T* op = out + (int64_t)r * hd + c;
        const float inv = L != 0.f ? 1.f / L : saw ? NAN : 0.f;     // nothing seen: zeros; scores that are all -inf: 0 / 0
        op[0] = from_f32<T>(acc.x * inv);
        op[1] = from_f32<T>(acc.y * inv);
        op[2] = from_f32<T>(acc.z * inv);
        op[3] = from_f32<T>(acc.w * inv);
    }
}

template <typename T>
__device__ __forceinline__ void join(const float* ml, const float* os, int nh, int hd, T* out, bool saw) {
    cg::cluster_group cluster = cg::this_cluster();
    const int pieces = (int)cluster.num_blocks();
    if (pieces == 1) {
        __syncthreads();
        join_pieces<T, 1>(ml, os, nh, hd, out, saw);
        return;
    }
    cluster.sync();
    switch (pieces) {
        case 2: join_pieces<T, 2>(ml, os, nh, hd, out, saw); break;
        case 4: join_pieces<T, 4>(ml, os, nh, hd, out, saw); break;
        case 8: join_pieces<T, 8>(ml, os, nh, hd, out, saw); break;
        default: join_pieces<T, 16>(ml, os, nh, hd, out, saw); break;
    }
    cluster.sync();     // a CTA's shared memory outlives its readers
}

// The place of a CTA: its row, kv head, first head and number of heads; false: nothing to do (for the whole cluster).
struct Place {
    int row, pos, kvh, h0, nh;
    const int* bt;
    __device__ __forceinline__ bool find(const PagesParams& p, int GC) {
        const int pieces = (int)cg::this_cluster().num_blocks();
        const int unit = (int)blockIdx.x / pieces, seq = unit / p.max_q_len, qi = unit % p.max_q_len;
        const int q_len = p.seq_q_len[seq];
        if (qi >= q_len) return false;
        const int G = p.heads / p.kv_heads, chunks = (G + GC - 1) / GC;
        kvh = (int)blockIdx.y / chunks;
        const int chunk = (int)blockIdx.y % chunks;
        row = p.seq_q_start[seq] + qi;
        pos = p.seq_kv_len[seq] - q_len + qi;
        h0 = kvh * G + chunk * GC;
        nh = min(GC, G - chunk * GC);
        bt = block_table_row(p.block_table, p.bt_stride, p.seq_slot[seq], p.max_slots);
        return true;
    }
};

// ---- bfloat16 ------------------------------------------------------------------------------------
constexpr int STAGES = 3;

template <int HD>
__global__ void __launch_bounds__(THREADS) attn_pages_mma_kernel(PagesParams p) {
    constexpr bool QREG = HD <= 128;
    constexpr int SD = HD + 8, KS = HD / 16, NF = HD / 8, CH = HD / 8;
    constexpr int STAGE = 2 * 64 * SD;   // elements: keys, then values
    extern __shared__ __align__(16) unsigned char raw[];
    bf16* Qs = reinterpret_cast<bf16*>(raw);       // [16][SD]
    bf16* KV = Qs + 16 * SD;                       // [STAGES][2][64][SD]
    int* pages = reinterpret_cast<int*>(KV + STAGES * STAGE);   // [2][top]: their numbers, their places
    __shared__ int counts[THREADS / 32];
    __shared__ alignas(8) float ml[16][2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    pdl_wait();
    Place at;
    const int G = p.heads / p.kv_heads, GC = G < 16 ? G : 16;
    if (!at.find(p, GC)) return;
    const int pieces = (int)cg::this_cluster().num_blocks(), piece = (int)cg::this_cluster().block_rank();
    {
        const bf16* qsrc = (const bf16*)p.q + (int64_t)at.row * p.q_row_stride + (int64_t)at.h0 * HD;
        for (int idx = tid; idx < 16 * CH; idx += THREADS) {
            const int r = idx / CH, c = idx - r * CH;
            const bool ok = r < at.nh;
            cp_async16(Qs + r * SD + c * 8, ok ? qsrc + (int64_t)r * HD + c * 8 : qsrc, ok ? 16 : 0);
        }
        cp_async_commit();
    }
    const int n_all = pack_list(p, at.bt, p.list + ((int64_t)at.row * p.kv_heads + at.kvh) * p.top, at.pos / GB_PAGE, pages, counts);
    const int lo = (int)((int64_t)n_all * piece / pieces), n = (int)((int64_t)n_all * (piece + 1) / pieces) - lo;

    const bf16* kbase = (const bf16*)p.k_plane;
    const bf16* vbase = (const bf16*)p.v_plane;
    auto load_tile = [&](int i) {
        const int64_t off = ((int64_t)pages[p.top + lo + i] * p.kv_heads + at.kvh) * (GB_PAGE * HD);
        bf16* st = KV + (i % STAGES) * STAGE;
        for (int idx = tid; idx < 64 * CH; idx += THREADS) {
            const int r = idx / CH, c = idx - r * CH;
            cp_async16(st + r * SD + c * 8, kbase + off + r * HD + c * 8, 16);
        }
        for (int idx = tid; idx < 64 * CH; idx += THREADS) {
            const int r = idx / CH, c = idx - r * CH;
            cp_async16(st + 64 * SD + r * SD + c * 8, vbase + off + r * HD + c * 8, 16);
        }
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; s++) {
        if (s < n) load_tile(s);
        cp_async_commit();
    }
    const float sc = p.scale * LOG2E;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    float o[NF][4];
#pragma unroll
    for (int j = 0; j < NF; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[j][e] = 0.f;
    uint32_t qf[QREG ? KS : 1][4];
    for (int i = 0; i < n; i++) {
        cp_async_wait<STAGES - 2>();   // page i has landed, and the queries before it
        __syncthreads();
        if (i + STAGES - 1 < n) load_tile(i + STAGES - 1);
        cp_async_commit();
        if (QREG && i == 0) {
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
                ldmatrix_x4(qf[QREG ? ks : 0], Qs + ((lane & 7) + ((lane >> 3) & 1) * 8) * SD + ks * 16 + (lane >> 4) * 8);
        }
        const bf16* kt = KV + (i % STAGES) * STAGE;
        const bf16* vt = kt + 64 * SD;
        const int key0 = pages[lo + i] * GB_PAGE + warp * 16;
        if (pages[lo + i] * GB_PAGE + GB_PAGE - 1 > at.pos) {
            // The row's own page: what stands behind its position gets probabilities of zero, and zero times an Inf or NaN
            // that was left there would not be zero.
            const int seen = at.pos + 1 - pages[lo + i] * GB_PAGE;
            for (int idx = tid; idx < (64 - seen) * CH; idx += THREADS)
                *reinterpret_cast<uint4*>(KV + (i % STAGES) * STAGE + (64 + seen + idx / CH) * SD + idx % CH * 8) = make_uint4(0, 0, 0, 0);
            __syncthreads();
        }
        float s[2][4];
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) s[j][e] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            uint32_t a[4], b[4];
            if (QREG) {
#pragma unroll
                for (int e = 0; e < 4; e++) a[e] = qf[QREG ? ks : 0][e];
            } else {
                ldmatrix_x4(a, Qs + ((lane & 7) + ((lane >> 3) & 1) * 8) * SD + ks * 16 + (lane >> 4) * 8);
            }
            ldmatrix_x4(b, kt + (warp * 16 + (lane & 7) + (lane >> 4) * 8) * SD + ks * 16 + ((lane >> 3) & 1) * 8);
            mma_bf16_16816(s[0], a[0], a[1], a[2], a[3], b[0], b[1]);
            mma_bf16_16816(s[1], a[0], a[1], a[2], a[3], b[2], b[3]);
        }
        float mx0 = m0, mx1 = m1;
#pragma unroll
        for (int j = 0; j < 2; j++) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const bool ok = key0 + j * 8 + t4 * 2 + (e & 1) <= at.pos;
                const float v = ok ? s[j][e] * sc : -INFINITY;
                s[j][e] = v;
                if (e & 2) mx1 = fmaxf(mx1, v); else mx0 = fmaxf(mx0, v);
            }
        }
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
        const float base0 = mx0 == -INFINITY ? 0.f : mx0, base1 = mx1 == -INFINITY ? 0.f : mx1;
        const float c0 = exp2f(m0 - base0), c1 = exp2f(m1 - base1);
        m0 = mx0;
        m1 = mx1;
        l0 *= c0;
        l1 *= c1;
#pragma unroll
        for (int j = 0; j < NF; j++) {
            o[j][0] *= c0;
            o[j][1] *= c0;
            o[j][2] *= c1;
            o[j][3] *= c1;
        }
        uint32_t pa[4];
        {
            const float p00 = exp2f(s[0][0] - base0), p01 = exp2f(s[0][1] - base0), p02 = exp2f(s[0][2] - base1), p03 = exp2f(s[0][3] - base1);
            const float p10 = exp2f(s[1][0] - base0), p11 = exp2f(s[1][1] - base0), p12 = exp2f(s[1][2] - base1), p13 = exp2f(s[1][3] - base1);
            l0 += p00 + p01 + p10 + p11;
            l1 += p02 + p03 + p12 + p13;
            pa[0] = pack_bf16(p00, p01);
            pa[1] = pack_bf16(p02, p03);
            pa[2] = pack_bf16(p10, p11);
            pa[3] = pack_bf16(p12, p13);
        }
#pragma unroll
        for (int c = 0; c < KS; c++) {
            uint32_t b[4];
            ldmatrix_x4_trans(b, vt + (warp * 16 + (lane & 7) + ((lane >> 3) & 1) * 8) * SD + c * 16 + (lane >> 4) * 8);
            mma_bf16_16816(o[c * 2], pa[0], pa[1], pa[2], pa[3], b[0], b[1]);
            mma_bf16_16816(o[c * 2 + 1], pa[0], pa[1], pa[2], pa[3], b[2], b[3]);
        }
    }
    cp_async_wait<0>();
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    __syncthreads();   // every warp is done with the pages: their memory takes the warps' results

    float* Ms = reinterpret_cast<float*>(KV);   // [4][16]
    float* Ls = Ms + 64;                        // [4][16]
    float* Os = Ls + 64;                        // [4][16][HD]; the CTA's own over the first warp's
    if (t4 == 0) {
        Ms[warp * 16 + g] = m0;
        Ms[warp * 16 + g + 8] = m1;
        Ls[warp * 16 + g] = l0;
        Ls[warp * 16 + g + 8] = l1;
    }
#pragma unroll
    for (int j = 0; j < NF; j++) {
        float* o0 = Os + ((size_t)warp * 16 + g) * HD + j * 8 + t4 * 2;
        if (g < at.nh) *reinterpret_cast<float2*>(o0) = make_float2(o[j][0], o[j][1]);
        if (g + 8 < at.nh) *reinterpret_cast<float2*>(o0 + 8 * HD) = make_float2(o[j][2], o[j][3]);
    }
    __syncthreads();
    for (int idx = tid; idx < at.nh * HD / 4; idx += THREADS) {
        const int r = idx / (HD / 4), c = (idx - r * (HD / 4)) * 4;
        const float M = fmaxf(fmaxf(Ms[r], Ms[16 + r]), fmaxf(Ms[32 + r], Ms[48 + r]));
        float L = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        const float base = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float e = exp2f(Ms[w * 16 + r] - base);
            const float4 x = *reinterpret_cast<const float4*>(Os + ((size_t)w * 16 + r) * HD + c);
            L += e * Ls[w * 16 + r];
            acc.x += e * x.x;
            acc.y += e * x.y;
            acc.z += e * x.z;
            acc.w += e * x.w;
        }
        *reinterpret_cast<float4*>(Os + (size_t)r * HD + c) = acc;
        if (c == 0) {
            ml[r][0] = M;
            ml[r][1] = L;
        }
    }
    join<bf16>(&ml[0][0], Os, at.nh, HD, (bf16*)p.out + (int64_t)at.row * p.out_row_stride + (int64_t)at.h0 * HD, n_all > 0);
}

// ---- float32 -------------------------------------------------------------------------------------
// Half a page of keys and values a stage.  A tile's scores: each warp takes a quarter of the channels, a lane a key; the quarters are
// added where a warp has the softmax of a head; then a thread sums its channels over the tile's keys.
constexpr int F_KEYS = 32, F_STAGES = 3;
constexpr int F_CH = 2;          // channels a thread sums at most: head_dim up to 256

__host__ __device__ constexpr int f32_stage(int d) { return F_KEYS * (2 * d + 4); }   // floats: key rows start four banks further each
__host__ __device__ constexpr int f32_floats(int d, int nh) { return nh * d * 2 + nh * F_KEYS * 5 + F_STAGES * f32_stage(d); }

template <int NH>
__global__ void __launch_bounds__(THREADS) attn_pages_f32_kernel(PagesParams p) {
    extern __shared__ __align__(16) float sm[];
    const int d = p.d, sd = d + 4;
    float* KV = sm;                                // [F_STAGES][32][sd], then [32][d]
    float* Qs = KV + F_STAGES * f32_stage(d);      // [NH][d], scaled
    float* Os = Qs + NH * d;                       // [NH][d]
    float* Part = Os + NH * d;                     // [4 warps][NH][32]
    float* Ps = Part + 4 * NH * F_KEYS;            // [NH][32]
    int* pages = reinterpret_cast<int*>(Ps + NH * F_KEYS);
    __shared__ int counts[THREADS / 32];
    __shared__ alignas(8) float ml[NH][2];
    __shared__ float corr[NH];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();
    Place at;
    const int G = p.heads / p.kv_heads, GC = G < NH ? G : NH;
    if (!at.find(p, GC)) return;
    const int pieces = (int)cg::this_cluster().num_blocks(), piece = (int)cg::this_cluster().block_rank();
    const float* qsrc = (const float*)p.q + (int64_t)at.row * p.q_row_stride + (int64_t)at.h0 * d;
    const float sc = p.scale * LOG2E;
    for (int i = tid; i < NH * d; i += THREADS) Qs[i] = i < at.nh * d ? qsrc[i] * sc : 0.f;
    if (tid < NH) {
        ml[tid][0] = -INFINITY;
        ml[tid][1] = 0.f;
    }
    const int n_all = pack_list(p, at.bt, p.list + ((int64_t)at.row * p.kv_heads + at.kvh) * p.top, at.pos / GB_PAGE, pages, counts);
    const int lo = (int)((int64_t)n_all * piece / pieces), n = 2 * ((int)((int64_t)n_all * (piece + 1) / pieces) - lo);   // half pages
    const int CH = d / 4;
    auto load_tile = [&](int i) {
        const int64_t off = (((int64_t)pages[p.top + lo + i / 2] * p.kv_heads + at.kvh) * GB_PAGE + (i & 1) * F_KEYS) * d;
        const float *k = (const float*)p.k_plane + off, *v = (const float*)p.v_plane + off;
        float* st = KV + (i % F_STAGES) * f32_stage(d);
        for (int r = warp; r < F_KEYS; r += THREADS / 32)      // a warp a key
            for (int c = lane * 4; c < d; c += 128) {
                cp_async16(st + r * sd + c, k + r * d + c, 16);
                cp_async16(st + F_KEYS * sd + r * d + c, v + r * d + c, 16);
            }
    };
#pragma unroll
    for (int s = 0; s < F_STAGES - 1; s++) {
        if (s < n) load_tile(s);
        cp_async_commit();
    }
    float o[NH][F_CH];
#pragma unroll
    for (int h = 0; h < NH; h++)
#pragma unroll
        for (int c = 0; c < F_CH; c++) o[h][c] = 0.f;
    const int quarter = (CH + 3) / 4, c_lo = warp * quarter, c_hi = min(CH, c_lo + quarter);    // the warp's chunks of four channels
    for (int i = 0; i < n; i++) {
        cp_async_wait<F_STAGES - 2>();
        __syncthreads();               // the tile has landed, and the one before is done with
        if (i + F_STAGES - 1 < n) load_tile(i + F_STAGES - 1);
        cp_async_commit();
        const float *Ks = KV + (i % F_STAGES) * f32_stage(d), *Vs = Ks + F_KEYS * sd;
        const int key0 = pages[lo + i / 2] * GB_PAGE + (i & 1) * F_KEYS, keys = min(F_KEYS, at.pos + 1 - key0);   // keys the row sees
        if (keys <= 0) continue;
        {
            float s[NH];
#pragma unroll
            for (int h = 0; h < NH; h++) s[h] = 0.f;
#pragma unroll 4
            for (int c = c_lo; c < c_hi; c++) {
                const float4 kk = *reinterpret_cast<const float4*>(Ks + lane * sd + c * 4);
#pragma unroll
                for (int h = 0; h < NH; h++) {
                    const float4 qq = *reinterpret_cast<const float4*>(Qs + h * d + c * 4);
                    s[h] = fmaf(qq.x, kk.x, fmaf(qq.y, kk.y, fmaf(qq.z, kk.z, fmaf(qq.w, kk.w, s[h]))));
                }
            }
#pragma unroll
            for (int h = 0; h < NH; h++) Part[(warp * NH + h) * F_KEYS + lane] = s[h];
        }
        __syncthreads();
        for (int h = warp; h < at.nh; h += THREADS / 32) {
            float s = 0.f;
#pragma unroll
            for (int w = 0; w < 4; w++) s += Part[(w * NH + h) * F_KEYS + lane];
            if (lane >= keys) s = -INFINITY;       // also where the key holds Inf or NaN
            const float old = ml[h][0], m = fmaxf(old, warp_max(s)), base = m == -INFINITY ? 0.f : m;
            const float w = exp2f(s - base), sum = warp_sum(w);
            Ps[h * F_KEYS + lane] = w;
            __syncwarp();
            if (lane == 0) {
                corr[h] = exp2f(old - base);
                ml[h][0] = m;
                ml[h][1] = ml[h][1] * corr[h] + sum;
            }
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < F_CH; c++) {
            const int ch = tid + c * THREADS;
            if (ch < d) {
#pragma unroll
                for (int h = 0; h < NH; h++) o[h][c] *= corr[h];
                if (keys == F_KEYS) {
#pragma unroll 4
                    for (int key = 0; key < F_KEYS; key += 4) {
                        float v[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) v[e] = Vs[(key + e) * d + ch];
#pragma unroll
                        for (int h = 0; h < NH; h++) {
                            const float4 w = *reinterpret_cast<const float4*>(Ps + h * F_KEYS + key);
                            o[h][c] = fmaf(w.x, v[0], fmaf(w.y, v[1], fmaf(w.z, v[2], fmaf(w.w, v[3], o[h][c]))));
                        }
                    }
                } else {
                    // values behind the row's position are not touched: they may be Inf or NaN
                    for (int key = 0; key < keys; key++) {
                        const float v = Vs[key * d + ch];
#pragma unroll
                        for (int h = 0; h < NH; h++) o[h][c] = fmaf(Ps[h * F_KEYS + key], v, o[h][c]);
                    }
                }
            }
        }
    }
    cp_async_wait<0>();
#pragma unroll
    for (int h = 0; h < NH; h++)
#pragma unroll
        for (int c = 0; c < F_CH; c++)
            if (h < at.nh && tid + c * THREADS < d) Os[h * d + tid + c * THREADS] = o[h][c];
    __syncthreads();
    join<float>(&ml[0][0], Os, at.nh, d, (float*)p.out + (int64_t)at.row * p.out_row_stride + (int64_t)at.h0 * d, n_all > 0);
}

// Into how many pieces a row's list is cut: the CTAs of a cluster, a power of two (sixteen where the GPU holds all of the clusters).  As many
// as run at once (one token over eight key heads, 32 pages: 34 us in one piece, 19 in two, 12 in four, 8.4 in eight, 8.1 in
// sixteen); where not even two pieces each do, two if their waves end sooner than those of whole rows (50 sequences over eight key
// heads, 64 pages: 173 us in one piece, 147 in two, 158 in four, 197 in eight; 139 in two since a list's places are looked up at once).
int pieces_for(const PagesParams& p, int chunks, int per_sm, int wide) {
    const int64_t units = (int64_t)p.nseq * p.max_q_len * p.kv_heads * chunks;
    int pieces = 1;
    const int64_t slots = (int64_t)gb_sm_count() * per_sm;
    while (pieces < 8 && units * pieces * 2 <= slots && p.top >= 4 * pieces) pieces *= 2;
    if (pieces == 1 && p.top >= 8 && units <= 4 * slots && (units * 2 + slots - 1) / slots < 2 * ((units + slots - 1) / slots)) pieces = 2;
    if (pieces == 8 && units <= wide && p.top >= 32) pieces = 16;
    return pieces;
}

template <typename K>
int launch(K kernel, const PagesParams& p, int chunks, int pieces, int smem, cudaStream_t stream) {
    const int64_t x = (int64_t)p.nseq * p.max_q_len * pieces;
    if (x > 0x7fffffff || p.kv_heads * chunks > 65535)
        GB_REFUSE("attention_pages: %d sequences of up to %d rows, %d kv heads exceed one launch", p.nseq, p.max_q_len, p.kv_heads);
    launch_pdl_cluster(kernel, dim3((unsigned)x, p.kv_heads * chunks), dim3(THREADS), (size_t)smem, stream, pieces, 1, p);
    GB_CHECK_LAUNCH("attention_pages");
    return 0;
}

// Shared memory and clusters of 16 for a kernel on the current device; how many of those clusters it holds at once (0: none, or not
// allowed).  known: one number a device, one more than that.
template <typename K>
int configure(K kernel, int smem, int (&known)[64], int& wide) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || dev < 0 || dev >= 64) GB_REFUSE("attention_pages: no current device");
    if (!known[dev]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) GB_REFUSE("attention_pages: cannot reserve %d bytes of shared memory: %s", smem, cudaGetErrorString(e));
        int most = 0;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(16);
            cfg.blockDim = dim3(THREADS);
            cfg.dynamicSmemBytes = smem;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = 16;
            attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            if (cudaOccupancyMaxActiveClusters(&most, kernel, &cfg) != cudaSuccess) most = 0;
        }
        cudaGetLastError();     // what was not possible is no error of the call
        known[dev] = 1 + (most > 0 ? most : 0);
    }
    wide = known[dev] - 1;
    return 0;
}

template <int HD>
int launch_mma(const PagesParams& p, cudaStream_t stream) {
    constexpr int SD = HD + 8;
    constexpr int base = (16 * SD + STAGES * 2 * 64 * SD) * 2;
    static_assert(base >= (128 + 64 * HD) * 4 + 16 * SD * 2, "the warps' results fit where the pages were");
    static int known[64];
    int wide = 0;
    if (int rc = configure(attn_pages_mma_kernel<HD>, base + MAX_TOP * 8, known, wide)) return rc;
    const int G = p.heads / p.kv_heads, chunks = (G + 15) / 16;
    return launch(attn_pages_mma_kernel<HD>, p, chunks, pieces_for(p, chunks, HD <= 128 ? 2 : 1, wide), base + p.top * 8, stream);
}

template <int NH>
int launch_f32(const PagesParams& p, cudaStream_t stream) {
    static int known[64];
    int wide = 0;
    constexpr int most = f32_floats(256, NH) * 4 + MAX_TOP * 8;
    static_assert(most <= 231000, "the widest heads' stages fit");
    if (int rc = configure(attn_pages_f32_kernel<NH>, most, known, wide)) return rc;
    const int G = p.heads / p.kv_heads, chunks = (G + NH - 1) / NH;
    return launch(attn_pages_f32_kernel<NH>, p, chunks, pieces_for(p, chunks, p.d <= 128 ? 2 : 1, wide), f32_floats(p.d, NH) * 4 + p.top * 8, stream);
}

}  // namespace

GB_API int gb_attention_pages(const PagesParams* pp, int dtype, cudaStream_t stream) {
    const PagesParams p = *pp;
    const char* who = "attention_pages";
    if (p.nseq <= 0 || p.max_q_len <= 0) return 0;
    if (dtype != GB_F32 && dtype != GB_BF16) GB_REFUSE("%s: dtype code %d", who, dtype);
    if (p.heads <= 0 || p.kv_heads <= 0 || p.heads % p.kv_heads) GB_REFUSE("%s: %d heads over %d kv heads", who, p.heads, p.kv_heads);
    if (p.top <= 0 || p.top > MAX_TOP) GB_REFUSE("%s: lists of %d pages; this kernel takes 1 to %d", who, p.top, MAX_TOP);
    if (p.pages <= 0 || p.bt_stride <= 0 || p.max_slots <= 0) GB_REFUSE("%s: %d pages, block table %d x %d", who, p.pages, p.max_slots, p.bt_stride);
    if (((uintptr_t)p.k_plane | (uintptr_t)p.v_plane) & 15) GB_REFUSE("%s: the planes must be 16-byte aligned", who);
    if (dtype == GB_F32) {
        if (p.d <= 0 || p.d % 4 || p.d > 256) GB_REFUSE("%s: head_dim %d is not a multiple of 4 up to 256", who, p.d);
        const int G = p.heads / p.kv_heads;
        return G <= 1 ? launch_f32<1>(p, stream) : G <= 2 ? launch_f32<2>(p, stream) : G <= 4 ? launch_f32<4>(p, stream) : launch_f32<8>(p, stream);
    }
    if (((uintptr_t)p.q & 15) || (p.q_row_stride & 7)) GB_REFUSE("%s: query rows must be 16-byte aligned", who);
    if (p.max_q_len > 1 && (int64_t)p.nseq * p.max_q_len * p.kv_heads >= TC5_MIN_UNITS && gb_attention_pages_tc5_accepts(p)) return gb_attention_pages_tc5(p, stream);
    switch (p.d) {
        case 16: return launch_mma<16>(p, stream);
        case 32: return launch_mma<32>(p, stream);
        case 48: return launch_mma<48>(p, stream);
        case 64: return launch_mma<64>(p, stream);
        case 80: return launch_mma<80>(p, stream);
        case 96: return launch_mma<96>(p, stream);
        case 112: return launch_mma<112>(p, stream);
        case 128: return launch_mma<128>(p, stream);
        case 256: return launch_mma<256>(p, stream);
    }
    GB_REFUSE("%s: bfloat16 heads of %d are not one of 16, 32, ..., 128, 256", who, p.d);
}

// the checked build's record of the first index this file's kernels found out of bounds
GB_CHECK_READER(gb_checked_status_attention_pages)
