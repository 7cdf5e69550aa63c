// Attention over listed pages for runs of rows, on the fifth-generation tensor cores (bfloat16, head_dim 128).
//
// Every row has a list of pages of its own, but rows that follow one another list nearly the same ones.  A CTA owns a tile of one
// sequence and kv head, 128 rows of (token, query head of the group), and walks the pages that any of its tokens lists, each
// once: its keys and values are fetched once for the tile.  For each of these pages a word of bits says which tokens list it.  A
// warp none of whose tokens lists the page writes zero weights without looking at the scores; a row that does not list it
// takes none of what its warp finds.
//     S = Q K^T   (M 128, N 64 keys, K 128)   -> two S buffers of 64 columns
//     O += P V    (M 128, N 128, K 64 keys)    -> 128 columns
// Roles by warp: warp 0 loads queries and keys by TMA, the last one the values, two pages deep each; one thread each of warps 1 and
// 2 issues the scores and the values products; warps 3-6 are the softmax (a thread a row, probabilities back into tensor memory
// over the scores as the second product's A operand, O rescaled only when a row's maximum has grown by more than 2^8 since the
// scale in use was chosen).
//
// Two CTAs share an SM (110 KB, half of the tensor memory each).  A page takes a CTA some 2000 cycles, of which the softmax has 900,
// and the chain probabilities - values product - next scores in the same buffer most of the rest; two CTAs overlap.  2000 rows of
// 32 heads over 8 behind 30700, 32 pages each (113 in a tile): 237 us; with two groups of 128 rows in one CTA of four stages,
// whose tiles list 163 pages, 279; with one group in a CTA of three or four stages, which has the SM to itself, 394.
//
// The heads of a group are rows of the tile (a group of G heads takes the next power of two: a tensor map of three dimensions
// brings token after token, head after head), so that they share every page too.
//
// The probabilities are rounded to bfloat16 for the second product, whose operands have one type.  A weight of zero times an infinite or
// NaN value is NaN, and stays one in the row's sums: a row whose sums are not all finite is computed once more at the end, over
// its own keys alone, which gives what it gives if the value was the row's own.
// (A warp that looked through every page's values instead cost 11 %.)
//
// Where there are few tiles, a cluster of CTAs shares one: each takes a stretch of the pages, and they join their rows through
// distributed shared memory.  All barrier waits are bounded; one that gives up sets a status word and the CTA runs out.
#include "mma.cuh"
#include "tc5.cuh"
#include "api.h"

#include <cooperative_groups.h>
#include <math.h>

namespace {

namespace cg = cooperative_groups;

__device__ int g_status;

typedef __nv_bfloat16 bf16;
constexpr int HD = 128, BKV = 64;
constexpr int QPANEL = 128 * 128;               // 128 rows of 128 bytes (64 channels)
constexpr int KPANEL = 64 * 128;                // 64 keys of 128 bytes
constexpr int Q_BYTES = 2 * QPANEL, K_BYTES = 2 * KPANEL, V_BYTES = 2 * KPANEL, STAGE_BYTES = K_BYTES + V_BYTES;
constexpr int ROWS = 128, STAGES = 2;
constexpr int FIRST_SOFTMAX_WARP = 3, VALUE_LOADER_WARP = FIRST_SOFTMAX_WARP + 4, WARPS = VALUE_LOADER_WARP + 1, THREADS = WARPS * 32;
constexpr int TILE_BYTES = Q_BYTES + STAGES * STAGE_BYTES;
constexpr int LIST_BYTES = 232448 - 4 * 1024 - TILE_BYTES;   // most for the tile's pages and their bits, beside the static part and the alignment
constexpr int TMEM_COLS = 256, O_COL = 128;                     // two buffers of 64 columns for S, then O
static_assert(ROWS * HD * 4 <= STAGES * STAGE_BYTES, "a tile's sums fit where the pages were");
constexpr int MAX_TABLE = 32768;                // pages of a sequence: their bitmap is made where the pages will go
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE_AT = 8.0f;
constexpr int MAX_PIECES = 8;
// The tile: tokens, bits of a page's entry.
__host__ __device__ inline int padded_group(int G) {
    int gp = 1;
    while (gp < G) gp *= 2;
    return gp;
}
__host__ __device__ inline int mask_words(int tokens) { return tokens > 32 ? tokens / 32 : 1; }

// One (token, head) over its own keys alone, by a warp: the way of rows whose sums are not finite.
__device__ __noinline__ void row_alone(const PagesParams& p, const int* bt, int row, int pos, int head, int kvh, int lane) {
    const int* list = p.list + ((int64_t)row * p.kv_heads + kvh) * p.top;
    const bf16* q = (const bf16*)p.q + (int64_t)row * p.q_row_stride + (int64_t)head * HD;
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    bool saw = false;
    for (int i = 0; i < p.top; i++) {
        const int lp = list[i];
        if (lp < 0 || lp > pos / BKV || lp >= p.bt_stride) continue;
        saw = true;
        const int64_t off = (page_of(bt, lp * BKV, p.bt_stride, p.pages) * p.kv_heads + kvh) * (int64_t)(BKV * HD);
        const bf16 *k = (const bf16*)p.k_plane + off, *v = (const bf16*)p.v_plane + off;
        const int n = min(BKV, pos + 1 - lp * BKV);
        for (int half = 0; half < n; half += 32) {
            float s = -INFINITY;
            if (half + lane < n) {
                s = 0.f;
                for (int c = 0; c < HD; c++) s = fmaf(__bfloat162float(q[c]), __bfloat162float(k[(half + lane) * HD + c]), s);
                s *= p.scale * LOG2E;
            }
            // A maximum that does not lose a NaN score.
            float big = s;
            for (int d = 16; d > 0; d >>= 1) {
                const float other = __shfl_xor_sync(0xffffffffu, big, d);
                big = other != other || big != big ? NAN : fmaxf(big, other);
            }
            const float now = big != big || m != m ? NAN : fmaxf(m, big);
            const float base = now == -INFINITY ? 0.f : now, corr = exp2f(m - base), w = exp2f(s - base);
            l = l * corr + warp_sum(w);
            for (int e = 0; e < 4; e++) o[e] *= corr;
            for (int t = 0; t < min(32, n - half); t++) {
                const float wt = __shfl_sync(0xffffffffu, w, t);
                for (int e = 0; e < 4; e++) o[e] = fmaf(wt, __bfloat162float(v[(half + t) * HD + lane * 4 + e]), o[e]);
            }
            m = now;
        }
    }
    bf16* to = (bf16*)p.out + (int64_t)row * p.out_row_stride + (int64_t)head * HD + lane * 4;
    const float inv = m != -INFINITY ? 1.f / l : saw ? NAN : 0.f;
    for (int e = 0; e < 4; e++) to[e] = __float2bfloat16_rn(o[e] * inv);
}

__global__ void __launch_bounds__(THREADS, 2) attn_pages_tc5_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                                 const __grid_constant__ CUtensorMap map_v,
                                                                 const __grid_constant__ PagesParams p) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* base = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    unsigned char* Qs = base;                 // two panels of 64 channels
    unsigned char* KVs = Qs + Q_BYTES;        // [STAGES][K | V]
    __shared__ uint64_t q_full, k_full[STAGES], v_full[STAGES], k_empty[STAGES], v_empty[STAGES];
    __shared__ uint64_t s_full[2], p_full[2], o_done[2];
    __shared__ uint32_t tmem_base_s;
    __shared__ int abort_s, n_s;
    __shared__ float row_m[ROWS], row_l[ROWS];         // of a tile that several CTAs share

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    pdl_trigger();
    const cg::cluster_group cluster = cg::this_cluster();
    const int pieces = (int)cluster.num_blocks(), piece = (int)cluster.block_rank();
    const int G = p.heads / p.kv_heads, GP = padded_group(G), TOK = ROWS / GP, MW = mask_words(TOK);
    const int seq = blockIdx.z, kvh = blockIdx.y;
    const int q_len = p.seq_q_len[seq], kv_len = p.seq_kv_len[seq];
    const int q0 = ((int)blockIdx.x / pieces) * TOK;
    if (q0 >= q_len) return;                           // the whole cluster leaves before anything is allocated
    const int past = kv_len - q_len, q_start = p.seq_q_start[seq];
    const int tokens = min(TOK, q_len - q0);
    const int* bt = block_table_row(p.block_table, p.bt_stride, p.seq_slot[seq], p.max_slots);
    int* entry = reinterpret_cast<int*>(KVs + STAGES * STAGE_BYTES);    // the tile's pages
    const int cap = min(TOK * p.top, p.bt_stride);
    uint32_t* bits = reinterpret_cast<uint32_t*>(entry + cap);          // [entry][MW]: the tokens that list it

    if (threadIdx.x == 0) {
        mbar_init(&q_full, 1);
        for (int s = 0; s < STAGES; s++) {
            mbar_init(&k_full[s], 1);
            mbar_init(&v_full[s], 1);
            mbar_init(&k_empty[s], 1);
            mbar_init(&v_empty[s], 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(&s_full[b], 1);
            mbar_init(&p_full[b], 4);
            mbar_init(&o_done[b], 1);
        }
        abort_s = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
        mbar_expect_tx(&q_full, Q_BYTES);
#pragma unroll
        for (int h = 0; h < 2; h++) tma_load_3d(Qs + h * QPANEL, &map_q, h * 64, kvh * G, q_start + q0, &q_full);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(s32(&tmem_base_s)), "n"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    // The tile's pages in ascending order, and who lists them: a bitmap of the sequence's pages, the number of pages ahead of
    // each of its words, then every list once more to set its token's bit.  The bitmap stands where the pages will go.
    {
        uint32_t* map = reinterpret_cast<uint32_t*>(KVs);
        int* ahead = reinterpret_cast<int*>(map + MAX_TABLE / 32);
        const int words = (p.bt_stride + 31) / 32;
        const int* lists = p.list + ((int64_t)(q_start + q0) * p.kv_heads + kvh) * p.top;
        constexpr int KEPT = 8;        // entries of the lists a thread keeps, all asked for at once; longer lists are read twice
        const bool kept = tokens * p.top <= KEPT * THREADS;
        auto place = [&](int i) -> int {      // token and page of entry i of the tile's lists, -1 for one that names nothing
            const int tok = i / p.top;
            const int lp = lists[(int64_t)tok * p.kv_heads * p.top + (i - tok * p.top)];
            return lp >= 0 && lp <= (past + q0 + tok) / BKV && lp < p.bt_stride ? tok << 16 | lp : -1;
        };
        int mine[KEPT];
#pragma unroll
        for (int e = 0; e < KEPT; e++) mine[e] = kept && (int)threadIdx.x + e * THREADS < tokens * p.top ? place(threadIdx.x + e * THREADS) : -1;
        auto each = [&](auto use) {
            if (kept) {
#pragma unroll
                for (int e = 0; e < KEPT; e++)
                    if (mine[e] >= 0) use(mine[e] >> 16, mine[e] & 0xffff);
            } else {
                for (int i = threadIdx.x; i < tokens * p.top; i += THREADS) {
                    const int v = place(i);
                    if (v >= 0) use(v >> 16, v & 0xffff);
                }
            }
        };
        for (int i = threadIdx.x; i < words; i += THREADS) map[i] = 0;
        __syncthreads();
        each([&](int, int lp) { atomicOr(&map[lp >> 5], 1u << (lp & 31)); });
        __syncthreads();
        if (warp == 0) {
            const int per = (words + 31) / 32, a = min(words, lane * per), b = min(words, a + per);
            int own = 0;
            for (int i = a; i < b; i++) own += __popc(map[i]);
            int to = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, to, o);
                if (lane >= o) to += v;
            }
            if (lane == 31) n_s = to;
            to -= own;
            for (int i = a; i < b; i++) {
                ahead[i] = to;
                to += __popc(map[i]);
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < n_s * MW; i += THREADS) bits[i] = 0;
        for (int i = threadIdx.x; i < words; i += THREADS) {
            int at = ahead[i];
            for (uint32_t m = map[i]; m; m &= m - 1) entry[at++] = i * 32 + __ffs(m) - 1;
        }
        __syncthreads();
        each([&](int tok, int lp) {
            const int at = ahead[lp >> 5] + __popc(map[lp >> 5] & ((1u << (lp & 31)) - 1u));
            atomicOr(&bits[at * MW + (tok >> 5)], 1u << (tok & 31));
        });
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    const uint32_t tmem_base = tmem_base_s;
    const int lo = (int)((int64_t)n_s * piece / pieces), n = (int)((int64_t)n_s * (piece + 1) / pieces) - lo;
    entry += lo;
    bits += lo * MW;

    if (warp == 0 || warp == VALUE_LOADER_WARP) {
        if (lane == 0) {
            const bool keys = warp == 0;
            uint64_t *full = keys ? k_full : v_full, *empty = keys ? k_empty : v_empty;
            int issued = 0;
            auto row_of = [&](int j) { return j < n ? ((int)page_of(bt, entry[j] * BKV, p.bt_stride, p.pages) * p.kv_heads + kvh) * BKV : 0; };
            int next = row_of(0);      // looked up a page ahead
            for (int j = 0; j < n; j++) {
                const int s = j % STAGES, row = next;
                next = row_of(j + 1);
                if (!mbar_wait_relaxed(&empty[s], ((uint32_t)(j / STAGES) & 1u) ^ 1u)) {
                    atomicCAS(&g_status, 0, 1);
                    abort_s = 1;
                }
                if (*(volatile int*)&abort_s) break;
                mbar_expect_tx(&full[s], K_BYTES);
                unsigned char* to = KVs + (size_t)s * STAGE_BYTES + (keys ? 0 : K_BYTES);
#pragma unroll
                for (int h = 0; h < 2; h++) tma_load_2d(to + h * KPANEL, keys ? &map_k : &map_v, h * 64, row, &full[s]);
                issued = j + 1;
            }
            if (*(volatile int*)&abort_s) {
                for (int j = issued > STAGES ? issued - STAGES : 0; j < issued; j++) mbar_wait(&full[j % STAGES], (uint32_t)(j / STAGES) & 1u);
                if (keys) mbar_wait(&q_full, 0);
            }
        }
    } else if (warp < FIRST_SOFTMAX_WARP) {
        if (lane == 0) {
            bool ok = true;
            if (warp == 1) {
                const uint32_t idesc = instr_desc(ROWS, BKV);
                ok = mbar_wait(&q_full, 0);
                const uint64_t q_desc = smem_desc(s32(Qs)), k_desc = smem_desc(s32(KVs));
                for (int j = 0; j < n && ok; j++) {
                    const int b = j & 1;
                    ok = mbar_wait(&k_full[j % STAGES], (uint32_t)(j / STAGES) & 1u);
                    // the probabilities of the page before last lie in this buffer's columns until their product has read them
                    if (ok && j >= 2) ok = mbar_wait(&o_done[b], (uint32_t)((j - 2) >> 1) & 1u);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                    const uint64_t kd = k_desc + (uint64_t)((j % STAGES) * (STAGE_BYTES >> 4));
#pragma unroll
                    for (int ks = 0; ks < 8; ks++)
                        umma(tmem_base + (uint32_t)(b * 64), q_desc + (uint64_t)((ks >> 2) * (QPANEL >> 4) + (ks & 3) * 2),
                             kd + (uint64_t)((ks >> 2) * (KPANEL >> 4) + (ks & 3) * 2), idesc, ks > 0 ? 1u : 0u);
                    umma_commit(&s_full[b]);
                    umma_commit(&k_empty[j % STAGES]);
                }
            } else {
                const uint32_t idesc = instr_desc(ROWS, HD) | (1u << 16);  // values enter MN-major
                const uint64_t v_desc = smem_desc_mn(s32(KVs + K_BYTES), KPANEL);
                for (int j = 0; j < n && ok; j++) {
                    const int b = j & 1;
                    ok = mbar_wait(&v_full[j % STAGES], (uint32_t)(j / STAGES) & 1u) && mbar_wait(&p_full[b], (uint32_t)(j >> 1) & 1u);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                    const uint64_t vd = v_desc + (uint64_t)((j % STAGES) * (STAGE_BYTES >> 4));
#pragma unroll
                    for (int kk = 0; kk < BKV / 16; kk++)
                        umma_ta(tmem_base + O_COL, tmem_base + (uint32_t)(b * 64 + kk * 8), vd + (uint64_t)(kk * ((16 * 128) >> 4)), idesc,
                                (j > 0 || kk > 0) ? 1u : 0u);
                    umma_commit(&o_done[b]);
                    umma_commit(&v_empty[j % STAGES]);
                }
            }
            if (!ok) {
                atomicCAS(&g_status, 0, 3);
                abort_s = 1;
            }
        }
    }
    const bool softmax = warp >= FIRST_SOFTMAX_WARP && warp < VALUE_LOADER_WARP;
    const int r = (warp & 3) * 32 + lane, tok = r / GP, h = r % GP;       // a softmax thread's row: the warp's quarter of tensor memory
    const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16, o_addr = tmem_base + lane_addr + O_COL;
    const bool row_ok = softmax && tok < tokens && h < G;
    float m_used = -INFINITY, l = 0.f;
    if (softmax) {
        const int pos = past + q0 + tok;
        const float sc = p.scale * LOG2E;    // > 0
        float m_run = -INFINITY;
        bool ok = true, saw = false;
        for (int j = 0; j < n && ok; j++) {
            const int b = j & 1, key0 = entry[j] * BKV;
            const bool mine = (bits[j * MW + (tok >> 5)] >> (tok & 31)) & 1u;
            const bool any = __any_sync(0xffffffffu, mine);
            if (!mbar_wait(&s_full[b], (uint32_t)(j >> 1) & 1u)) {
                ok = false;
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            const uint32_t s_addr = tmem_base + lane_addr + (uint32_t)(b * 64);
            uint32_t pw[32];
            uint64_t sum2[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
            if (!any) {
                // scores of this buffer were issued behind the product of two pages ago: it may be written
#pragma unroll
                for (int e = 0; e < 32; e++) pw[e] = 0u;
                tmem_st32(s_addr, pw);
            } else {
                uint32_t v0[32], v1[32];
                tmem_ld32_nowait(s_addr, v0);
                tmem_ld32_nowait(s_addr + 32u, v1);
                tmem_wait_ld();
                if (mine && key0 + BKV - 1 > pos) {      // (0 times -inf, where the row does not list the page, would be NaN)
#pragma unroll
                    for (int e = 0; e < 32; e++) {
                        if (key0 + e > pos) v0[e] = 0xff800000u;  // -inf
                        if (key0 + 32 + e > pos) v1[e] = 0xff800000u;
                    }
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < 32; e += 4)
#pragma unroll
                    for (int f = 0; f < 4; f++) mx[f] = max3_nan(mx[f], __uint_as_float(v0[e + f]), __uint_as_float(v1[e + f]));
                const float tile_max = max_nan(max3_nan(mx[0], mx[1], mx[2]), mx[3]) * sc;
                if (mine) m_run = max_nan(m_run, tile_max);
                saw = saw || mine;
                const bool grow = m_run > m_used + RESCALE_AT || (m_used == -INFINITY && m_run != -INFINITY);
                if (__any_sync(0xffffffffu, grow && j > 0)) {
                    // O may only be touched between products: wait for the previous page's
                    if (!mbar_wait(&o_done[(j - 1) & 1], (uint32_t)((j - 1) >> 1) & 1u)) {
                        ok = false;
                        break;
                    }
                    const float f = (grow && j > 0) ? fast_exp2(m_used - m_run) : 1.f;  // m_used = -inf gives 0: O is all zeros then
                    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
#pragma unroll 1
                    for (int c0 = 0; c0 < HD; c0 += 32) {
                        uint32_t o[32];
                        tmem_ld32(o_addr + (uint32_t)c0, o);
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_st32(o_addr + (uint32_t)c0, o);
                    }
                    l *= f;
                }
                if (grow) m_used = m_run;
                const float mbase = m_used == -INFINITY ? 0.f : m_used;
                // a row that does not list the page: 2^-inf, which is 0; a score of it that is not finite makes the row's sums NaN, and
                // they are made anew
                const uint64_t sc2 = mine ? pack2(sc, sc) : pack2(0.f, 0.f), nmb2 = mine ? pack2(-mbase, -mbase) : pack2(-INFINITY, -INFINITY);
#pragma unroll
                for (int c = 0; c < 32; c++) {
                    const uint32_t a = c < 16 ? v0[(c & 15) * 2] : v1[(c & 15) * 2], bb = c < 16 ? v0[(c & 15) * 2 + 1] : v1[(c & 15) * 2 + 1];
                    const uint64_t t = fma2(pack2(__uint_as_float(a), __uint_as_float(bb)), sc2, nmb2);
                    float p0, p1;
                    if (c % 4 == 3) {
                        unpack2(exp2_poly_x2(t), p0, p1);
                    } else {
                        unpack2(t, p0, p1);
                        p0 = fast_exp2(p0);
                        p1 = fast_exp2(p1);
                    }
                    sum2[c & 1] = add2(sum2[c & 1], pack2(p0, p1));
                    const __nv_bfloat162 h2 = __floats2bfloat162_rn(p0, p1);
                    pw[c] = *reinterpret_cast<const uint32_t*>(&h2);
                }
                tmem_st32(s_addr, pw);
            }
            asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[b]);
            float sum[4];
            unpack2(sum2[0], sum[0], sum[1]);
            unpack2(sum2[1], sum[2], sum[3]);
            if (mine) l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        }
        // A NaN score's weight is 0 where the polynomial has it; and of a score of +inf, beside which the others weigh nothing, so is its
        // own, inf - inf.
        if (!(m_run < INFINITY)) l = NAN;
        // Scores that are all -inf: 0 / 0, but other CTAs of the tile may have found better ones for the row.
        if (saw && l == 0.f) l = pieces == 1 ? NAN : -1.f;
        if (ok && n > 0 && !mbar_wait(&o_done[(n - 1) & 1], (uint32_t)((n - 1) >> 1) & 1u)) ok = false;
        if (!ok) {
            atomicCAS(&g_status, 0, 4);
            abort_s = 1;
        }
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    }
    __syncthreads();      // every role is done with the pages
    const bool aborted = *(volatile int*)&abort_s != 0;
    if (pieces == 1) {
        if (softmax && !aborted) {
            const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;       // nothing seen: zeros; a NaN stays one
            bf16* op = (bf16*)p.out + (int64_t)(q_start + q0 + tok) * p.out_row_stride + (int64_t)(kvh * G + h) * HD;
            uint32_t most = 0;     // of the sums' exponents
#pragma unroll 1
            for (int c0 = 0; c0 < HD; c0 += 32) {
                uint32_t o[32];
                if (n > 0) {
                    tmem_ld32(o_addr + (uint32_t)c0, o);
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = 0u;
                }
#pragma unroll
                for (int e = 0; e < 32; e++) most = max(most, o[e] & 0x7fffffffu);
                if (row_ok) {
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        uint32_t w[4];
#pragma unroll
                        for (int f = 0; f < 4; f++) {
                            const __nv_bfloat162 a = __floats2bfloat162_rn(__uint_as_float(o[e + 2 * f]) * inv, __uint_as_float(o[e + 2 * f + 1]) * inv);
                            w[f] = *reinterpret_cast<const uint32_t*>(&a);
                        }
                        *reinterpret_cast<uint4*>(op + c0 + e) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
            for (unsigned again = __ballot_sync(0xffffffffu, row_ok && most >= 0x7f800000u); again; again &= again - 1) {
                const int rr = (warp & 3) * 32 + __ffs(again) - 1, tk = rr / GP;
                row_alone(p, bt, q_start + q0 + tk, past + q0 + tk, kvh * G + rr % GP, kvh, lane);
            }
        }
    } else {
        // A row's 32 chunks of four channels stand in an order of their own (the chunk's number xor the row's), so that the
        // threads of a warp, a row each, write to different banks.
        float* sums = reinterpret_cast<float*>(KVs);
        if (softmax) {
            const int at = r;
            row_m[at] = m_used;
            row_l[at] = l;
            if (n > 0) {
#pragma unroll 1
                for (int c0 = 0; c0 < HD; c0 += 32) {
                    uint32_t o[32];
                    tmem_ld32(o_addr + (uint32_t)c0, o);
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        *reinterpret_cast<uint4*>(sums + (size_t)at * HD + (((c0 >> 2) + e) ^ (at & 31)) * 4) =
                            make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                }
            }
        }
        cluster.sync();
        // (A CTA that gave up has left a status and whatever its rows held: the results are not valid, but they are written.)
        for (int at = piece + warp * pieces; at < ROWS; at += WARPS * pieces) {
            const int tk = at / GP, hh = at % GP;
            if (tk >= tokens || hh >= G) continue;
            // a lane a piece: its maximum and sum; all pieces' values are asked for before the first is used
            float m = -INFINITY, l_w = 0.f;
            if (lane < pieces) {
                m = *cluster.map_shared_rank(&row_m[at], lane);
                l_w = *cluster.map_shared_rank(&row_l[at], lane);
            }
            float4 x[MAX_PIECES];
#pragma unroll
            for (int w = 0; w < MAX_PIECES; w++)
                if (w < pieces) x[w] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(sums, w) + (size_t)at * HD + (lane ^ (at & 31)) * 4);
            const float M = warp_max(m);
            // this row saw nothing there, or scores of -inf alone: no maximum, and a sum of 0 or -1 (a NaN score has a NaN sum)
            const bool none = m == -INFINITY && l_w <= 0.f, lost = __any_sync(0xffffffffu, l_w < 0.f);
            const float f_w = none ? 0.f : m == -INFINITY ? 1.f : fast_exp2(m - M);
            const float L = warp_sum(none ? 0.f : f_w * l_w);
            float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < MAX_PIECES; w++) {
                const float f = __shfl_sync(0xffffffffu, f_w, w);
                if (w >= pieces || __shfl_sync(0xffffffffu, (int)none, w)) continue;      // its sums may be anything
                o[0] += f * x[w].x;
                o[1] += f * x[w].y;
                o[2] += f * x[w].z;
                o[3] += f * x[w].w;
            }
            if (__any_sync(0xffffffffu, !(fabsf(o[0]) + fabsf(o[1]) + fabsf(o[2]) + fabsf(o[3]) < INFINITY))) {
                row_alone(p, bt, q_start + q0 + tk, past + q0 + tk, kvh * G + hh, kvh, lane);
                continue;
            }
            const float inv = L > 0.f ? 1.f / L : L == 0.f && !lost ? 0.f : NAN;
            const __nv_bfloat162 a = __floats2bfloat162_rn(o[0] * inv, o[1] * inv), b = __floats2bfloat162_rn(o[2] * inv, o[3] * inv);
            bf16* op = (bf16*)p.out + (int64_t)(q_start + q0 + tk) * p.out_row_stride + (int64_t)(kvh * G + hh) * HD + lane * 4;
            *reinterpret_cast<uint2*>(op) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
        }
        cluster.sync();     // a CTA's shared memory outlives its readers
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "n"(TMEM_COLS) : "memory");
    }
}

int make_map(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
    Tc5EncodeTiledFn fn = tc5_encode_fn();
    if (!fn) GB_REFUSE("attention_pages: the driver offers no cuTensorMapEncodeTiled");
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) GB_REFUSE("attention_pages: cuTensorMapEncodeTiled failed with code %d", (int)r);
    return 0;
}

int list_bytes(const PagesParams& p) {
    const int tokens = ROWS / padded_group(p.heads / p.kv_heads);
    const int64_t most = (int64_t)tokens * p.top;
    const int cap = (int)(most < p.bt_stride ? most : p.bt_stride);
    return cap * 4 * (1 + mask_words(tokens));
}

}  // namespace

// Whether this kernel takes the call: heads of 128 in groups of up to 128, 16-byte aligned rows, a positive scale, and a tile's
// pages (those its tokens can list together) within the shared memory there is for them.
int gb_attention_pages_tc5_accepts(const PagesParams& p) {
    return p.d == HD && p.heads / p.kv_heads <= ROWS && p.scale > 0.f && !((uintptr_t)p.q & 15) && !(p.q_row_stride & 7) && !((uintptr_t)p.out & 15) &&
           !(p.out_row_stride & 7) && p.rows > 0 && p.bt_stride <= MAX_TABLE && (int64_t)p.pages * p.kv_heads * BKV <= 0x7fffffff &&
           list_bytes(p) <= LIST_BYTES;
}

int gb_attention_pages_tc5(const PagesParams& p, cudaStream_t stream) {
    static bool done[64];
    constexpr int most = TILE_BYTES + 1024 + LIST_BYTES;
    if (const cudaError_t e = gb_allow_smem(attn_pages_tc5_kernel, most, done))
        GB_REFUSE("attention_pages: cannot reserve %d bytes of shared memory: %s", most, cudaGetErrorString(e));
    const int G = p.heads / p.kv_heads, gp = padded_group(G), tok = ROWS / gp;
    CUtensorMap map_q, map_k, map_v;
    {
        const cuuint64_t dims[3] = {HD, (cuuint64_t)p.heads, (cuuint64_t)p.rows}, strides[2] = {HD * 2, (cuuint64_t)p.q_row_stride * 2};
        const cuuint32_t box[3] = {64, (cuuint32_t)gp, (cuuint32_t)tok};
        if (int rc = make_map(&map_q, p.q, 3, dims, strides, box)) return rc;
    }
    {
        const cuuint64_t dims[2] = {HD, (cuuint64_t)p.pages * p.kv_heads * BKV}, strides[1] = {HD * 2};
        const cuuint32_t box[2] = {64, 64};
        if (int rc = make_map(&map_k, p.k_plane, 2, dims, strides, box)) return rc;
        if (int rc = make_map(&map_v, p.v_plane, 2, dims, strides, box)) return rc;
    }
    // As many CTAs to a tile as run at once, two an SM (24 tiles of 90 rows behind 20000, us: 106 in one piece, 64 in two, 37 in four, 35 in
    // six, 31 in eight).
    const int64_t tiles = (int64_t)p.nseq * ceil_div(p.max_q_len, tok) * p.kv_heads;
    int pieces = (int)(2 * gb_sm_count() / tiles);
    pieces = pieces < 1 ? 1 : pieces > MAX_PIECES ? MAX_PIECES : pieces;
    const dim3 grid(ceil_div(p.max_q_len, tok) * pieces, p.kv_heads, p.nseq);
    if (grid.y > 65535 || grid.z > 65535) GB_REFUSE("attention_pages: grid (%u, %u, %u) exceeds one launch", grid.x, grid.y, grid.z);
    const cudaError_t e = launch_pdl_cluster(attn_pages_tc5_kernel, grid, dim3(THREADS), (size_t)(TILE_BYTES + 1024 + list_bytes(p)), stream,
                                             pieces, 1, map_q, map_k, map_v, p);
    if (e != cudaSuccess) GB_REFUSE("attention_pages: launch failed: %s", cudaGetErrorString(e));
    return 0;
}

GB_API int gb_attention_pages_status() {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_status, sizeof(int)) != cudaSuccess) return -1;
    if (v != 0) cudaMemcpyToSymbol(g_status, &zero, sizeof(int));
    return v;
}

// the checked build's record of the first index this file's kernels found out of bounds
GB_CHECK_READER(gb_checked_status_attention_pages_tc5)
