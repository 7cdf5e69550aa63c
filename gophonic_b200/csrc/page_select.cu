// Which pages of the cache a row of a step should read.
//
// page_bounds keeps, beside the keys, the lowest and the highest value of every channel of each full page of 64 keys:
//     lo[c] = min_t k[t][c],  hi[c] = max_t k[t][c].
// For a query q no key of the page can score more than sum_c max(q_c lo_c, q_c hi_c).  select_pages takes that bound, summed over
// the G query heads that share a key head, as the page's score:
//     s = sum_h sum_c max(q_hc lo_c, q_hc hi_c) = sum_c (P_c hi_c + N_c lo_c),   P = sum_h max(q_h, 0), N = sum_h min(q_h, 0),
// (a head takes hi where q > 0 and lo where q < 0), one product of 2 d channels a page whatever G is, and chooses for every (row,
// key head) the first `first` pages, the last `last` up to the row's own, and of the others those that score highest, `top` in all.
//
// The choice is the one of 64-bit arithmetic.  Scores are float32 sums with a bound e on their error; with tau the k-th highest
// of them, a page above tau + 2 e is among the k best and one below tau - 2 e is not, whatever the errors were, and only the
// pages between (as a rule the one at the border) are summed again in 64 bits, where a product of two bfloat16 values and
// most of their sums are exact.  Pages that tie go by their number.
#include "mma.cuh"
#include "api.h"

#include <cooperative_groups.h>
#include <math.h>

#include <utility>

namespace {

namespace cg = cooperative_groups;
typedef __nv_bfloat16 bf16;

__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

template <typename T>
struct Chunk {   // 16 bytes of a row
    static constexpr int E = 16 / sizeof(T);
};
__device__ __forceinline__ void unpack(const uint4& v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void unpack(const uint4& v, float (&x)[4]) {
    x[0] = __uint_as_float(v.x);
    x[1] = __uint_as_float(v.y);
    x[2] = __uint_as_float(v.z);
    x[3] = __uint_as_float(v.w);
}

// ---- bounds ------------------------------------------------------------------------------------
// A warp takes one page of one key head of one plane: the page whose last position is among the step's new rows.  A key is CH chunks
// of 16 bytes; LPR lanes (a power of two) have one key's chunks, so the warp reads 32 / LPR keys with one copy, and asks for 32
// copies (16 KB, a whole page of 128 bfloat16 channels) before it looks at any: by cp.async, each lane into places of its own
// that only it reads.  Bound by the read of the keys.
constexpr int BOUND_WARPS = 4, BOUND_LOADS = 32;

__device__ __forceinline__ uint32_t low2(uint32_t a, uint32_t b, bf16) {
    const __nv_bfloat162 v = __hmin2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t high2(uint32_t a, uint32_t b, bf16) {
    const __nv_bfloat162 v = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t low2(uint32_t a, uint32_t b, float) { return __float_as_uint(min_nan(__uint_as_float(a), __uint_as_float(b))); }
__device__ __forceinline__ uint32_t high2(uint32_t a, uint32_t b, float) { return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b))); }

template <typename T, int LPR, int CPL>
__global__ void __launch_bounds__(BOUND_WARPS * 32) page_bounds_kernel(PagesParams p) {
    constexpr int KEYS = 32 / LPR, TIMES = GB_PAGE / KEYS, STEP = BOUND_LOADS / CPL < TIMES ? BOUND_LOADS / CPL : TIMES;   // keys a copy; of each chunk at once
    extern __shared__ __align__(16) unsigned char raw[];
    uint4* mine = reinterpret_cast<uint4*>(raw) + (threadIdx.x >> 5) * BOUND_LOADS * 32 + (threadIdx.x & 31);
    pdl_wait();                     // the keys, and the step's metadata
    pdl_trigger();
    const int seq = blockIdx.z, lane = threadIdx.x & 31;
    const int unit = (int)blockIdx.x * BOUND_WARPS + (int)(threadIdx.x >> 5), kvh = unit % p.kv_heads, plane = unit / p.kv_heads;
    const int kv_len = p.seq_kv_len[seq], past = kv_len - p.seq_q_len[seq];
    const int lp = past / GB_PAGE + (int)blockIdx.y;
    if (lp >= kv_len / GB_PAGE || lp >= p.bt_stride || plane >= p.planes) return;
    const int* bt = block_table_row(p.block_table, p.bt_stride, p.seq_slot[seq], p.max_slots);
    const int64_t at = ((int64_t)plane * p.pages + page_of(bt, lp * GB_PAGE, p.bt_stride, p.pages)) * p.kv_heads + kvh;
    const int CH = p.d * (int)sizeof(T) / 16, sub = lane / LPR, l = lane % LPR;
    const uint4* k = reinterpret_cast<const uint4*>((const T*)p.k_plane + at * GB_PAGE * p.d) + sub * CH;
    uint4* to = reinterpret_cast<uint4*>((T*)p.bounds + at * 2 * p.d);
    uint32_t lo[CPL][4], hi[CPL][4];
    for (int r0 = 0; r0 < TIMES; r0 += STEP) {
#pragma unroll
        for (int r = 0; r < STEP; r++)
#pragma unroll
            for (int c = 0; c < CPL; c++) cp_async16(mine + (r * CPL + c) * 32, l + c * LPR < CH ? k + (r0 + r) * KEYS * CH + l + c * LPR : k, l + c * LPR < CH ? 16 : 0);
        cp_async_commit();
        cp_async_wait<0>();
#pragma unroll
        for (int r = 0; r < STEP; r++)
#pragma unroll
            for (int c = 0; c < CPL; c++) {
                const uint4 x = mine[(r * CPL + c) * 32];
                const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const bool first = r0 == 0 && r == 0;
                    lo[c][e] = first ? w[e] : low2(lo[c][e], w[e], T());
                    hi[c][e] = first ? w[e] : high2(hi[c][e], w[e], T());
                }
            }
    }
#pragma unroll
    for (int o = LPR; o < 32; o *= 2)
#pragma unroll
        for (int c = 0; c < CPL; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                lo[c][e] = low2(lo[c][e], __shfl_xor_sync(0xffffffffu, lo[c][e], o), T());
                hi[c][e] = high2(hi[c][e], __shfl_xor_sync(0xffffffffu, hi[c][e], o), T());
            }
    if (sub == 0)
#pragma unroll
        for (int c = 0; c < CPL; c++)
            if (l + c * LPR < CH) {
                to[l + c * LPR] = make_uint4(lo[c][0], lo[c][1], lo[c][2], lo[c][3]);
                to[CH + l + c * LPR] = make_uint4(hi[c][0], hi[c][1], hi[c][2], hi[c][3]);
            }
}

// ---- selection ---------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t order_key(float s) {
    const uint32_t b = __float_as_uint(s);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ uint64_t order_key(double s) {
    const uint64_t b = (uint64_t)__double_as_longlong(s == 0.0 ? 0.0 : s);   // the two zeros are one score
    return b ^ ((b >> 63) ? 0xffffffffffffffffull : 0x8000000000000000ull);
}

// A row's candidates: pages c0 .. c0 + nc - 1 of its sequence, of which the k highest are wanted.
template <typename T>
struct Row {
    const T* q;              // the group's heads
    int* list;
    const int* bt;
    int n, c0, nc, k;        // pages the row sees; candidates; wanted of them (fewer)
    int kvh;
    __device__ __forceinline__ const T* bounds(const PagesParams& p, int i) const {
        return (const T*)p.bounds + (page_of(bt, (c0 + i) * GB_PAGE, p.bt_stride, p.pages) * p.kv_heads + kvh) * (2 * p.d);
    }
    // false: the row sees no more than `top` pages
    __device__ __forceinline__ bool find(const PagesParams& p, const int* table_row, int row, int pos, int head) {
        kvh = head;
        list = p.list + ((int64_t)row * p.kv_heads + kvh) * p.top;
        q = (const T*)p.q + (int64_t)row * p.q_row_stride + (int64_t)kvh * (p.heads / p.kv_heads) * p.d;
        bt = table_row;
        n = min(pos / GB_PAGE + 1, p.bt_stride);      // (a sequence is no longer than its row of the table)
        c0 = p.first;
        nc = n - p.first - p.last;
        k = p.top - p.first - p.last;
        return n > p.top;
    }
};

// P and N in 64 bits, in the registers of a warp: lane l holds channels l, l + 32, ...
struct Coef64 {
    double up[8], down[8];
    template <typename T>
    __device__ __forceinline__ void load(const PagesParams& p, const T* q, int lane) {
        const int G = p.heads / p.kv_heads;
#pragma unroll
        for (int j = 0; j < 8; j++) up[j] = down[j] = 0.0;
        for (int h0 = 0; h0 < G; h0 += 4) {      // four heads' values are asked for together
            T v[4][8];
#pragma unroll
            for (int h = 0; h < 4; h++)
#pragma unroll
                for (int j = 0; j < 8; j++) v[h][j] = h0 + h < G && lane + 32 * j < p.d ? q[(int64_t)(h0 + h) * p.d + lane + 32 * j] : from_f32<T>(0.f);
#pragma unroll
            for (int h = 0; h < 4; h++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    if (32 * j >= p.d) break;
                    const float x = to_f32<T>(v[h][j]);
                    up[j] += (double)(x <= 0.f ? 0.f : x);      // a NaN is in both
                    down[j] += (double)(x >= 0.f ? 0.f : x);
                }
        }
    }
    // Two pages' scores, the same in every lane; NaN counts as the lowest.  Where no head looks one way there is nothing to add, also
    // where the bound is infinite.
    template <typename T>
    __device__ __forceinline__ void scores(const T* b0, const T* b1, int d, int lane, double& s0, double& s1) const {
        T lo[2][8], hi[2][8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int c = lane + 32 * j;
            lo[0][j] = c < d ? b0[c] : from_f32<T>(0.f);
            hi[0][j] = c < d ? b0[d + c] : from_f32<T>(0.f);
            lo[1][j] = c < d ? b1[c] : from_f32<T>(0.f);
            hi[1][j] = c < d ? b1[d + c] : from_f32<T>(0.f);
        }
        double s[2] = {0.0, 0.0};
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if (32 * j >= d) break;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                if (down[j] != 0.0) s[e] += down[j] * (double)to_f32<T>(lo[e][j]);
                if (up[j] != 0.0) s[e] += up[j] * (double)to_f32<T>(hi[e][j]);
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            s[0] += __shfl_xor_sync(0xffffffffu, s[0], o);
            s[1] += __shfl_xor_sync(0xffffffffu, s[1], o);
        }
        s0 = s[0] == s[0] ? s[0] : -INFINITY;
        s1 = s[1] == s[1] ? s[1] : -INFINITY;
    }
    template <typename T>
    __device__ __forceinline__ double score(const T* b, int d, int lane) const {
        double s0, s1;
        scores(b, b, d, lane, s0, s1);
        return s0;
    }
};

// The choice from float32 scores, by a group of W warps.  key[i] is the ordered float32 score of candidate i, off by no more than
// `err`.  Warp w has the candidates from w * seg on, 32 at a time; where there are few enough (R > 0: up to 32 R a warp) they stay in
// registers: every step of the search for the border is a loop over them, and from shared memory it took 670 cycles for 500
// scores where it takes a tenth.
template <int W, int BAND, int FEW, int MORE>
struct Chooser {
    union {
        struct {
            double band_s[BAND];
            int band_i[BAND];          // pages near the border, kept with their 64-bit scores
        };
        alignas(8) int hist[256];      // of the slow way; and what the fast one packs, before it has a border
    };
    int warp_a[W], warp_b[W];
    int digit, rest;

    static __device__ __forceinline__ void sync() {
        if (W == 1) __syncwarp(); else __syncthreads();
    }
    // Sums over the group.  `at` alternates between two arrays, so that one barrier a call is enough.
    __device__ __forceinline__ int total(int v, int* at, int warp, int lane) {
        v = __reduce_add_sync(0xffffffffu, v);
        if (W > 1) {
            if (lane == 0) at[warp] = v;
            sync();
            v = 0;
#pragma unroll
            for (int w = 0; w < W; w++) v += at[w];
        }
        return v;
    }
    __device__ __forceinline__ uint32_t least(uint32_t v, int* at, int warp, int lane) {
        v = __reduce_min_sync(0xffffffffu, v);
        if (W > 1) {
            if (lane == 0) at[warp] = (int)v;
            sync();
#pragma unroll
            for (int w = 0; w < W; w++) v = min(v, (uint32_t)at[w]);
        }
        return v;
    }
    // hist holds how many keys have each digit: the digit of the `want`-th highest key, and how many are wanted of those that have it
    __device__ __forceinline__ void pick(int want, int lane) {
        int v[8], own = 0;      // each lane: 8 digits, from the highest down
#pragma unroll
        for (int j = 0; j < 8; j++) own += v[j] = hist[255 - (lane * 8 + j)];
        int before = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += x;
        }
        before -= own;
        if (before < want && want <= before + own) {
            int left = want - before;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if (left > 0 && left <= v[j]) {
                    digit = 255 - (lane * 8 + j);
                    rest = left;
                }
                left -= v[j];
            }
        }
    }

    // The choice among scores at(j) of candidates id(j), `steps` a lane (N of them if N > 0: registers), in the candidates' order lane by
    // lane and step by step; scores of 0 are none.  `lo` and `hi`: as many as k or more keys from lo on, fewer from hi on.  false: too
    // many pages near the border.
    template <typename T, int N, class At, class Id>
    __device__ __forceinline__ bool choose(const PagesParams& p, const Row<T>& r, uint32_t* key, float err, int steps, At at, Id id, uint32_t lo, uint32_t hi,
                                           int warp, int lane) {
        const int k = r.k;
        auto each = [&](auto use) {
            if constexpr (N > 0) {
#pragma unroll
                for (int j = 0; j < N; j++) use(j, at(j));
            } else {
                for (int j = 0; j < steps; j++) use(j, at(j));
            }
        };
        // tau, the k-th highest float32 score: [lo, hi) is halved until a border parts exactly k keys (some ten steps), or one value is
        // left
        for (bool odd = false; hi - lo > 1u; odd = !odd) {
            const uint32_t mid = lo + (hi - lo) / 2u;
            int c = 0;
            each([&](int, uint32_t v) { c += v >= mid; });
            c = total(c, odd ? warp_b : warp_a, warp, lane);
            if (c >= k) lo = mid; else hi = mid;
            if (c == k) break;
        }
        uint32_t border = 0xffffffffu;      // the least key that is `lo` or more
        each([&](int, uint32_t v) {
            if (v >= lo) border = min(border, v);
        });
        sync();
        border = least(border, warp_a, warp, lane);
        const float tau = of_key(border);
        const uint32_t sure_from = order_key(tau + 2.f * err + fabsf(tau) * 2.4e-7f) + 1u, near_from = lowest_near(border, err);
        int sure = 0, near = 0;
        each([&](int, uint32_t v) {
            sure += v >= sure_from;
            near += v >= near_from && v < sure_from;
        });
        const int near_mine = near;
        const int wanted = k - total(sure, warp_b, warp, lane), m = total(near, warp_a, warp, lane);
        if (m > BAND && m > wanted) return false;
        const bool settle = m > wanted;
        if (settle) {
            // the pages near the border, in any order: their 64-bit scores, and which are among the best of them
            if (W > 1) sync();
            if (warp == 0 && lane == 0) rest = 0;
            sync();
            if (__any_sync(0xffffffffu, near_mine > 0))
                each([&](int j, uint32_t v) {
                    if (v >= near_from && v < sure_from) band_i[atomicAdd(&rest, 1)] = id(j);
                });
            sync();
            Coef64 c;
            c.load(p, r.q, lane);
            for (int j = 2 * warp; j < m; j += 2 * W) {
                double v0, v1;
                c.scores(r.bounds(p, band_i[j]), r.bounds(p, band_i[min(j + 1, m - 1)]), p.d, lane, v0, v1);
                if (lane == 0) {
                    band_s[j] = v0;
                    if (j + 1 < m) band_s[j + 1] = v1;
                }
            }
            sync();
            for (int j = warp * 32 + lane; j < m; j += W * 32) {
                int better = 0;
                for (int o = 0; o < m; o++) better += band_s[o] > band_s[j] || (band_s[o] == band_s[j] && band_i[o] < band_i[j]);
                key[band_i[j]] = better < wanted ? 0xffffffffu : 0u;
            }
            sync();
        }
        auto taken = [&](int j, uint32_t v) -> bool {
            if (settle && v >= near_from && v < sure_from) v = key[id(j)];
            return v >= (settle ? sure_from : near_from);
        };
        int before = 0;
        if (W > 1) {
            int mine = 0;
            each([&](int j, uint32_t v) { mine += taken(j, v); });
            mine = __reduce_add_sync(0xffffffffu, mine);
            if (lane == 0) warp_b[warp] = mine;
            sync();
            for (int w = 0; w < warp; w++) before += warp_b[w];
        }
        int* list = r.list + r.c0;
        each([&](int j, uint32_t v) {
            const bool yes = taken(j, v);
            const unsigned who = __ballot_sync(0xffffffffu, yes);
            if (yes) list[before + __popc(who & ((1u << lane) - 1u))] = r.c0 + id(j);
            before += __popc(who);
        });
        return true;
    }

    // The least key that a score can have and still be within 2 err of that of `border`, or above it.
    static __device__ __forceinline__ uint32_t lowest_near(uint32_t border, float err) {
        const float v = of_key(border), lower = v - 2.f * err - fabsf(v) * 2.4e-7f;
        return order_key(lower == 0.f ? -0.f : lower);
    }

    template <typename T, int R>
    __device__ __forceinline__ bool fast(const PagesParams& p, const Row<T>& r, uint32_t* key, float err, int warp, int lane) {
        const int nc = r.nc, k = r.k;
        const int steps = R > 0 ? R : (nc + 32 * W - 1) / (32 * W), from = warp * steps * 32 + lane;
        auto id = [&](int j) { return from + j * 32; };
        if constexpr (R > 0) {
            uint32_t reg[R];
#pragma unroll
            for (int j = 0; j < R; j++) reg[j] = from + j * 32 < nc ? key[from + j * 32] : 0u;     // no finite score's key is 0
            if (W == 1 && k <= 32) {
                // One warp, and no more wanted than lanes there are: of the lanes' highest scores the k-th is no higher than tau, and only
                // some dozens of all are as high or near it.  They are packed and the rest forgotten.  (2000 rows 100 -> 88 us.  With
                // half lanes for up to 64 wanted too many are left: 50 sequences that want 61 took 31 us instead of 26.)
                uint32_t a = 0;
#pragma unroll
                for (int j = 0; j < R; j++) a = max(a, reg[j]);
                uint32_t lo = max(1u, __reduce_min_sync(0xffffffffu, a));
                const uint32_t end = __reduce_max_sync(0xffffffffu, a) + 1u;
                for (uint32_t hi = end; hi - lo > 1u;) {
                    const uint32_t mid = lo + (hi - lo) / 2u;
                    const int c = __popc(__ballot_sync(0xffffffffu, a >= mid));
                    if (c >= k) lo = mid; else hi = mid;
                    if (c == k) break;
                }
                const uint32_t cut = lowest_near(lo, err);
                uint2* packed = reinterpret_cast<uint2*>(hist);
                constexpr int MOST = sizeof(hist) / sizeof(uint2), N = MOST / 32;
                int m = 0;
#pragma unroll
                for (int j = 0; j < R; j++) {
                    const bool in = reg[j] >= cut && reg[j] != 0u;
                    const unsigned who = __ballot_sync(0xffffffffu, in);
                    const int to = m + __popc(who & ((1u << lane) - 1u));
                    if (in && to < MOST) packed[to] = make_uint2(reg[j], id(j));
                    m += __popc(who);
                }
                __syncwarp();
                if (m <= MOST) {
                    uint2 few[N];
#pragma unroll
                    for (int j = 0; j < N; j++) few[j] = j * 32 + lane < m ? packed[j * 32 + lane] : make_uint2(0u, 0u);
                    return choose<T, N>(p, r, key, err, N, [&](int j) { return few[j].x; }, [&](int j) { return (int)few[j].y; }, lo, end, warp, lane);
                }
            }
            uint32_t lo = 0xffffffffu, most = 0u;
#pragma unroll
            for (int j = 0; j < R; j++) {
                if (reg[j]) lo = min(lo, reg[j]);
                most = max(most, reg[j]);
            }
            lo = least(lo, warp_a, warp, lane);
            const uint32_t hi = ~least(~most, warp_b, warp, lane) + 1u;
            return choose<T, R>(p, r, key, err, R, [&](int j) { return reg[j]; }, id, lo, hi, warp, lane);
        } else {
            auto at = [&](int j) -> uint32_t { return from + j * 32 < nc ? key[from + j * 32] : 0u; };
            uint32_t lo = 0xffffffffu, most = 0u;
            for (int j = 0; j < steps; j++) {
                const uint32_t v = at(j);
                if (v) lo = min(lo, v);
                most = max(most, v);
            }
            lo = least(lo, warp_a, warp, lane);
            const uint32_t hi = ~least(~most, warp_b, warp, lane) + 1u;
            return choose<T, 0>(p, r, key, err, steps, at, id, lo, hi, warp, lane);
        }
    }

    // Scores beyond float32, or hundreds that tie: the k-th highest of the 64-bit scores, which are summed anew for every digit.
    // Rare, and right for any input.
    template <typename T>
    __device__ __noinline__ void slow(const PagesParams& p, const Row<T> r, uint32_t* key, int warp, int lane) {
        const int nc = r.nc, NT = W * 32, tid = warp * 32 + lane;
        Coef64 c;
        c.load(p, r.q, lane);
        uint64_t prefix = 0;
        int want = r.k;
        for (int shift = 56; shift >= 0; shift -= 8) {
            sync();
            for (int i = tid; i < 256; i += NT) hist[i] = 0;
            sync();
            for (int i = warp; i < nc; i += W) {
                const uint64_t v = order_key(c.score(r.bounds(p, i), p.d, lane));
                if (lane == 0 && (shift == 56 || (v >> (shift + 8)) == (prefix >> (shift + 8)))) atomicAdd(&hist[(int)(v >> shift) & 255], 1);
            }
            sync();
            if (warp == 0) pick(want, lane);
            sync();
            prefix |= (uint64_t)digit << shift;
            want = rest;
        }
        for (int i = warp; i < nc; i += W) {
            const uint64_t v = order_key(c.score(r.bounds(p, i), p.d, lane));
            if (lane == 0) key[i] = v > prefix ? 2 : v == prefix ? 1 : 0;
        }
        sync();
        // in order, by one warp; of those that tie the first
        if (warp == 0) {
            int at = 0;
            for (int i0 = 0; i0 < nc; i0 += 32) {
                const uint32_t v = i0 + lane < nc ? key[i0 + lane] : 0u;
                const unsigned sure = __ballot_sync(0xffffffffu, v == 2), tie = __ballot_sync(0xffffffffu, v == 1), below = (1u << lane) - 1u;
                const int ties = __popc(tie & below);
                if (v == 2 || (v == 1 && ties < want)) r.list[r.c0 + at + __popc(sure & below) + min(ties, want)] = r.c0 + i0 + lane;
                at += __popc(sure) + min(__popc(tie), want);
                want -= min(__popc(tie), want);
            }
        }
    }

    // unsafe: the float32 scores cannot be relied on.
    template <typename T>
    __device__ __forceinline__ void run(const PagesParams& p, const Row<T>& r, uint32_t* key, float err, bool unsafe, int tid) {
        const int warp = W == 1 ? 0 : tid >> 5, lane = tid & 31;
        for (int i = tid; i < r.c0; i += W * 32) r.list[i] = i;
        for (int i = tid; i < p.last; i += W * 32) r.list[p.top - p.last + i] = r.n - p.last + i;
        if (r.k > 0) {
            bool done = false;
            if (!unsafe)
                done = r.nc <= FEW * 32 * W    ? fast<T, FEW>(p, r, key, err, warp, lane)
                       : r.nc <= MORE * 32 * W ? fast<T, MORE>(p, r, key, err, warp, lane)
                                               : fast<T, 0>(p, r, key, err, warp, lane);
            if (!done) slow(p, r, key, warp, lane);
        }
        sync();     // before the group's next row
    }
};

// Single rows ----------------------------------------------------------------------------------
// A cluster of CTAs scores one (row, kv head): each takes a stretch of the pages and leaves their scores in the first one's shared
// memory, which then chooses.  A page's 2 d bounds are 16-byte chunks, LP lanes share them, CPL chunks a lane, and hold their
// coefficients in registers.
constexpr int SELECT_THREADS = 256, SELECT_WARPS = SELECT_THREADS / 32;
constexpr int MAX_PIECES = 8;
constexpr int ROW_BAND = 512;
constexpr int RING_CHUNKS = 8;      // 16-byte chunks a lane asks for with one batch: 4 KB a warp

struct SelectSmem {
    union {
        Chooser<SELECT_WARPS, ROW_BAND, 4, 16> all;
        Chooser<1, ROW_BAND, 16, 16> one;       // up to 32 wanted of 512: no barriers between the steps of the search
    } choose;
    float coef[2 * 256];                        // [N | P], in the order of a page's bounds
    float err[MAX_PIECES * SELECT_WARPS];       // of every warp of the cluster; a NaN: unsafe
};

template <int N, int LP>
__device__ __forceinline__ float sum_many(float (&v)[N], int lane) {
    // The sums of N values over LP lanes (both powers of two): half of the values go to the other half of the lanes, until a
    // lane has one; lane l ends with value l / (LP / N) of the group's (N <= LP)
    if constexpr (N == 1) {
#pragma unroll
        for (int o = LP / 2; o > 0; o >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
        return v[0];
    } else {
        float half[N / 2];
        const bool upper = lane & (LP / 2);
#pragma unroll
        for (int j = 0; j < N / 2; j++) {
            const float give = upper ? v[j] : v[j + N / 2], keep = upper ? v[j + N / 2] : v[j];
            half[j] = keep + __shfl_xor_sync(0xffffffffu, give, LP / 2);
        }
        return sum_many<N / 2, LP / 2>(half, lane);
    }
}

template <typename T, int LP, int CPL>
__global__ void __launch_bounds__(SELECT_THREADS, 2) select_row_kernel(const __grid_constant__ PagesParams p, int longest_first, int depth) {
    constexpr int E = Chunk<T>::E, U = 8 / CPL, PER_WARP = 32 / LP;     // pages a group of LP lanes takes at a time
    extern __shared__ __align__(16) unsigned char raw[];
    SelectSmem& s = *reinterpret_cast<SelectSmem*>(raw);
    uint32_t* key = reinterpret_cast<uint32_t*>(raw + sizeof(SelectSmem));   // [candidates]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const cg::cluster_group cluster = cg::this_cluster();
    const int pieces = (int)cluster.num_blocks(), piece = (int)cluster.block_rank();
    pdl_wait();
    const int unit = blockIdx.x / pieces / p.kv_heads, head = blockIdx.x / pieces % p.kv_heads, qi = unit % p.max_q_len;
    int seq = unit / p.max_q_len;
    if (longest_first) {
        // more CTAs than run at once: the sequence that is `seq`-th in length, so that none of the long ones begins last
        int* at = reinterpret_cast<int*>(s.coef);
        for (int i = tid; i < p.nseq; i += SELECT_THREADS) at[i] = p.seq_kv_len[i];
        __syncthreads();
        for (int i = tid; i < p.nseq; i += SELECT_THREADS) {
            int before = 0;
            for (int j = 0; j < p.nseq; j++) before += at[j] > at[i] || (at[j] == at[i] && j < i);
            if (before == seq) s.err[0] = __int_as_float(i);
        }
        __syncthreads();
        seq = __float_as_int(s.err[0]);
        __syncthreads();
    }
    const int q_len = p.seq_q_len[seq];
    if (qi >= q_len) return;                    // the whole cluster
    Row<T> r;
    if (!r.find(p, block_table_row(p.block_table, p.bt_stride, p.seq_slot[seq], p.max_slots), p.seq_q_start[seq] + qi, p.seq_kv_len[seq] - q_len + qi, head)) {
        if (piece == 0)
            for (int i = tid; i < p.top; i += SELECT_THREADS) r.list[i] = i < r.n ? i : -1;
        return;
    }
    auto started = cluster.barrier_arrive();    // waited for before the first CTA's memory is written
    const int d2 = 2 * p.d, G = p.heads / p.kv_heads, NC = d2 / E, sub = lane / LP, l = lane % LP;
    constexpr int BATCH = U * PER_WARP;
    const int first_batch = (piece * SELECT_WARPS + warp) * BATCH, step = pieces * SELECT_WARPS * BATCH;
    const T* plane = (const T*)p.bounds;
    // A lane's page of the batch at i: the numbers are asked for a batch ahead of the bounds.  The bounds of `depth` (two or three)
    // batches are on their way by cp.async, each lane's chunks into places of its own that only it reads.
    auto page_for = [&](int i) -> int { return lane < BATCH && i + lane < r.nc ? (int)page_of(r.bt, (r.c0 + i + lane) * GB_PAGE, p.bt_stride, p.pages) : 0; };
    uint4* ring = reinterpret_cast<uint4*>(raw + ((sizeof(SelectSmem) + (size_t)p.bt_stride * sizeof(uint32_t) + 15) & ~(size_t)15)) + warp * depth * RING_CHUNKS * 32 + lane;
    auto ask = [&](int i, int page, int slot) {
        if (i < r.nc)
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int at = min(sub * U + u, r.nc - 1 - i);     // pages beyond the last are the last once more
                const int64_t pg = __shfl_sync(0xffffffffu, page, at);
                const T* b = plane + (pg * p.kv_heads + r.kvh) * d2;
#pragma unroll
                for (int j = 0; j < CPL; j++)
                    if (l + j * LP < NC) cp_async16(ring + (slot * RING_CHUNKS + u * CPL + j) * 32, b + (l + j * LP) * E, 16);
            }
        cp_async_commit();
    };
    int early[3];
#pragma unroll
    for (int s0 = 0; s0 < 3; s0++) early[s0] = page_for(first_batch + s0 * step);
    int next = depth == 3 ? page_for(first_batch + 3 * step) : early[2];
#pragma unroll
    for (int s0 = 0; s0 < 3; s0++)
        if (s0 < depth) ask(first_batch + s0 * step, early[s0], s0);
    for (int c = tid; c < p.d; c += SELECT_THREADS) {
        float up = 0.f, down = 0.f;
#pragma unroll 4
        for (int h = 0; h < G; h++) {
            const float x = to_f32<T>(r.q[(int64_t)h * p.d + c]);
            up += x <= 0.f ? 0.f : x;      // a NaN is in both
            down += x >= 0.f ? 0.f : x;
        }
        s.coef[c] = down;
        s.coef[p.d + c] = up;
    }
    __syncthreads();
    cluster.barrier_wait(std::move(started));
    float cf[CPL][E], mx[CPL][E];
#pragma unroll
    for (int j = 0; j < CPL; j++)
#pragma unroll
        for (int e = 0; e < E; e++) {
            cf[j][e] = l + j * LP < NC ? s.coef[(l + j * LP) * E + e] : 0.f;
            mx[j][e] = 0.f;
        }
    uint32_t* keys0 = cluster.map_shared_rank(key, 0);
    bool odd = false;
    int slot = 0;
    for (int i0 = first_batch; i0 < r.nc; i0 += step) {
        if (depth == 3) cp_async_wait<2>(); else cp_async_wait<1>();      // this batch has landed
        float acc[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            acc[u] = 0.f;
#pragma unroll
            for (int j = 0; j < CPL; j++) {
                if (l + j * LP >= NC) break;
                float f[E];
                unpack(ring[(slot * RING_CHUNKS + u * CPL + j) * 32], f);
#pragma unroll
                for (int e = 0; e < E; e++) {
                    acc[u] = fmaf(cf[j][e], f[e], acc[u]);
                    mx[j][e] = fmaxf(mx[j][e], fabsf(f[e]));
                }
            }
        }
        const int page = next;
        next = page_for(i0 + (depth + 1) * step);
        ask(i0 + depth * step, page, slot);
        slot = slot + 1 == depth ? 0 : slot + 1;
        const float sum = sum_many<U, LP>(acc, lane);
        constexpr int SHARE = LP / U;                     // lanes that end with the same page
        const int i = i0 + sub * U + l / SHARE;
        odd = odd || !(fabsf(sum) <= 3.0e38f);
        if (l % SHARE == 0 && i < r.nc) keys0[i] = order_key(sum);
    }
    cp_async_wait<0>();
    float most = 0.f;      // the sum of the terms' sizes is no more than that of the coefficients times the channels' largest bounds
#pragma unroll
    for (int j = 0; j < CPL; j++)
#pragma unroll
        for (int e = 0; e < E; e++) most = fmaf(fabsf(cf[j][e]), mx[j][e], most);
    if (odd || !(most <= 3.0e38f)) most = NAN;
#pragma unroll
    for (int o = LP / 2; o > 0; o >>= 1) most += __shfl_xor_sync(0xffffffffu, most, o);
#pragma unroll
    for (int o = 16; o >= LP; o >>= 1) {
        const float other = __shfl_xor_sync(0xffffffffu, most, o);
        most = most <= other || other != other ? other : most;
    }
    if (lane == 0) cluster.map_shared_rank(s.err, 0)[piece * SELECT_WARPS + warp] = most;
    cluster.sync();
    if (piece != 0) return;
    float err = 0.f;
    bool unsafe = false;
    for (int w = lane; w < pieces * SELECT_WARPS; w += 32) {
        err = fmaxf(err, s.err[w]);
        unsafe = unsafe || !(s.err[w] <= 3.0e38f);
    }
    err = warp_max(err);
    unsafe = __any_sync(0xffffffffu, unsafe);
    // A float32 sum of at most 16 products a lane and 5 steps between lanes, of coefficients that are sums of G values: 22 + G half steps
    // of 2^-23 relative to the sum of the terms' sizes, itself known to 2^-18; products below the normal range add next to nothing.
    err = err * ((24.f + (float)G) * 5.9604645e-8f) + 1.0e-42f;
    if (r.nc > 512 || r.k > 32)
        s.choose.all.run(p, r, key, err, unsafe, tid);
    else if (warp == 0)
        s.choose.one.run(p, r, key, err, unsafe, lane);
}

// Runs of rows -----------------------------------------------------------------------------------
// A CTA takes RT rows of one sequence and kv head and scores all their candidate pages as one product on mma.sync: the rows'
// coefficients, each as the sum of two bfloat16 values (2^-17 relative), against the pages' bounds, which come from the cache
// straight into the fragments.  The channels of a block of 32 are dealt to the k steps so that a lane's share of a page is 16
// consecutive bytes; the coefficients are read in the same order.  The scores stand in shared memory, a warp chooses for a row.
constexpr int TILE_BAND = 48;

template <int TILE_WARPS>
struct alignas(16) TileSmem {
    Chooser<1, TILE_BAND, 16, 16> choose[TILE_WARPS];
    float size[32];          // per chunk of 8 channels: their bounds' largest size, over all pages
    int next;                // the row that the next warp to be done takes: rows whose border is close take twice as long
};

__host__ __device__ inline int tile_coef_stride(int d) { return 2 * d + 32; }        // elements: rows 64 bytes of banks apart
__host__ __device__ inline int tile_key_stride(int pages) { return (pages + 31) / 32 * 32 + 8; }

// KB_MAX: blocks of 32 bounds a page has at most, or, with EXACT (KB_MAX even), has: the offsets are then known (2000 rows 74 -> 70 us).
template <int MT, int KB_MAX, bool EXACT, int TILE_WARPS>
__global__ void __launch_bounds__(TILE_WARPS * 32, 16 / TILE_WARPS) select_tile_kernel(const __grid_constant__ PagesParams p) {
    constexpr int RT = MT * 16, TILE_THREADS = TILE_WARPS * 32;
    using TileSmem = TileSmem<TILE_WARPS>;
    extern __shared__ __align__(16) unsigned char raw[];
    TileSmem& s = *reinterpret_cast<TileSmem*>(raw);
    const int d = EXACT ? KB_MAX * 16 : p.d, KB = d / 16;
    const int CS = tile_coef_stride(d), KS = tile_key_stride(p.bt_stride);
    bf16* coef = reinterpret_cast<bf16*>(raw + sizeof(TileSmem));                    // [2][RT][CS]
    uint32_t* keys = reinterpret_cast<uint32_t*>(coef + 2 * RT * CS);                // [RT][KS]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    pdl_wait();
    pdl_trigger();
    const int seq = blockIdx.z, kvh = blockIdx.y, q0 = blockIdx.x * RT;
    const int q_len = p.seq_q_len[seq];
    if (q0 >= q_len) return;
    const int rows = min(RT, q_len - q0), G = p.heads / p.kv_heads;
    const int* bt = block_table_row(p.block_table, p.bt_stride, p.seq_slot[seq], p.max_slots);
    // candidates of the last row, which has the most
    const int past = p.seq_kv_len[seq] - q_len, q_start = p.seq_q_start[seq];
    const int nc = min((past + q0 + rows - 1) / GB_PAGE + 1, p.bt_stride) - p.first - p.last;
    {
        const bf16* q = (const bf16*)p.q + (int64_t)(q_start + q0) * p.q_row_stride + (int64_t)kvh * G * d;
        const bool whole = !(((uintptr_t)p.q & 15) | (p.q_row_stride & 7));     // rows of 16-byte chunks
        const int CH = d / 8;
        for (int i = tid; i < RT * CH; i += TILE_THREADS) {
            const int row = i / CH, c = (i - row * CH) * 8;
            float up[8], down[8];
#pragma unroll
            for (int e = 0; e < 8; e++) up[e] = down[e] = 0.f;
            if (row < rows) {
#pragma unroll 4
                for (int h = 0; h < G; h++) {
                    const bf16* at = q + (int64_t)row * p.q_row_stride + h * d + c;
                    float x[8];
                    if (whole) {
                        unpack(*reinterpret_cast<const uint4*>(at), x);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; e++) x[e] = __bfloat162float(at[e]);
                    }
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        up[e] += x[e] <= 0.f ? 0.f : x[e];
                        down[e] += x[e] >= 0.f ? 0.f : x[e];
                    }
                }
            }
            bf16* to = coef + row * CS + c;
#pragma unroll
            for (int side = 0; side < 2; side++) {
                uint32_t first[4], second[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float x0 = side ? up[2 * e] : down[2 * e], x1 = side ? up[2 * e + 1] : down[2 * e + 1];
                    first[e] = pack_bf16(x0, x1);
                    const float r0 = __uint_as_float(first[e] << 16), r1 = __uint_as_float(first[e] & 0xffff0000u);
                    second[e] = pack_bf16(x0 - r0, x1 - r1);
                }
                *reinterpret_cast<uint4*>(to + side * d) = make_uint4(first[0], first[1], first[2], first[3]);
                *reinterpret_cast<uint4*>(to + RT * CS + side * d) = make_uint4(second[0], second[1], second[2], second[3]);
            }
        }
        for (int i = tid; i < 32; i += TILE_THREADS) s.size[i] = 0.f;
        if (tid == 0) s.next = TILE_WARPS;
    }
    __syncthreads();
    const bf16* plane = (const bf16*)p.bounds;
    // Of each block of bounds, in the lane's chunk of 8: the least of the lowest values, the most of the highest.  As lo <= hi, a channel's
    // bounds are no larger than the larger of the two.
    __nv_bfloat162 reach[KB_MAX];
#pragma unroll
    for (int kb = 0; kb < KB_MAX; kb++) reach[kb] = __floats2bfloat162_rn(0.f, 0.f);
    for (int i0 = warp * 16; i0 < nc; i0 += TILE_WARPS * 16) {
        const bf16* b[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const int i = min(i0 + t * 8 + g, nc - 1);         // pages beyond the last are the last once more
            b[t] = plane + (page_of(bt, (p.first + i) * GB_PAGE, p.bt_stride, p.pages) * p.kv_heads + kvh) * (2 * d) + t4 * 8;
        }
        float acc[2][MT][2][4];      // of the coefficients' first parts and of their second ones, so that the sums of the larger are short
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[0][m][t][e] = acc[1][m][t][e] = 0.f;
#pragma unroll
        for (int half = 0; half < KB_MAX / 4; half++) {        // blocks in fours: what a lane asks for at once
            if (half * 4 >= KB) break;
            uint4 x[4][2];
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int t = 0; t < 2; t++)
                    if (half * 4 + j < KB) x[j][t] = *reinterpret_cast<const uint4*>(b[t] + (half * 4 + j) * 32);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int kb = half * 4 + j;
                if (kb >= KB) break;
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const uint32_t w[4] = {x[j][t].x, x[j][t].y, x[j][t].z, x[j][t].w};
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(&w[e]);
                        reach[kb] = (EXACT ? kb * 2 < KB : kb * 4 + t4 < KB * 2) ? __hmin2_nan(reach[kb], v) : __hmax2_nan(reach[kb], v);
                    }
                }
#pragma unroll
                for (int term = 0; term < 2; term++)
#pragma unroll
                    for (int m = 0; m < MT; m++) {
                        const bf16* a = coef + (term * RT + m * 16 + g) * CS + kb * 32 + t4 * 8;
                        const uint4 a0 = *reinterpret_cast<const uint4*>(a), a1 = *reinterpret_cast<const uint4*>(a + 8 * CS);
#pragma unroll
                        for (int t = 0; t < 2; t++) {
                            mma_bf16_16816(acc[term][m][t], a0.x, a1.x, a0.y, a1.y, x[j][t].x, x[j][t].y);
                            mma_bf16_16816(acc[term][m][t], a0.z, a1.z, a0.w, a1.w, x[j][t].z, x[j][t].w);
                        }
                    }
            }
        }
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int i = i0 + t * 8 + t4 * 2;             // KS has room for whole blocks of 16
                float sum[4];
#pragma unroll
                for (int e = 0; e < 4; e++) sum[e] = acc[0][m][t][e] + acc[1][m][t][e];
                *reinterpret_cast<uint2*>(keys + (m * 16 + g) * KS + i) = make_uint2(order_key(sum[0]), order_key(sum[1]));
                *reinterpret_cast<uint2*>(keys + (m * 16 + g + 8) * KS + i) = make_uint2(order_key(sum[2]), order_key(sum[3]));
            }
    }
#pragma unroll
    for (int kb = 0; kb < KB_MAX; kb++) {
        if (kb >= KB) break;
        const float a = fabsf(__low2float(reach[kb])), b = fabsf(__high2float(reach[kb]));
        float v = a != a || b != b ? INFINITY : fmaxf(a, b);
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
        // (not negative: ordered as integers); a chunk of the lowest values and the same channels' highest share a place
        if (g == 0) {
            const int at = kb * 4 + t4;
            atomicMax(reinterpret_cast<int*>(&s.size[at < KB * 2 ? at : at - KB * 2]), __float_as_int(v));
        }
    }
    __syncthreads();
    for (int row = warp; row < rows; row = __shfl_sync(0xffffffffu, lane == 0 ? atomicAdd(&s.next, 1) : 0, 0)) {
        Row<bf16> r;
        if (!r.find(p, bt, q_start + q0 + row, past + q0 + row, kvh)) {
            for (int i = lane; i < p.top; i += 32) r.list[i] = i < r.n ? i : -1;
            continue;
        }
        // The coefficients are good to 2^-18 (3.9e-6) and G half steps of 2^-23, relative to the sum of the terms' sizes.  The products
        // of their first parts are summed up by 2 KB products of the tensor cores, of which the PTX manual says that they accumulate with at
        // least single precision, in any order and rounding: 17 numbers each, the sum so far among them, so no more than 17 units of
        // 2^-23 of what has been summed up to there, and a block's terms count once for every step from their own on.  (The second parts'
        // products are 2^-8 of that, the two sums' sum half a unit: 18.)  What is below the normal range may count as nothing: a
        // coefficient's second part (let in by 1e-35), a coefficient or a bound (1.2e-38 of the other), a sum.
        float most = 0.f, steps = 0.f;
#pragma unroll 8
        for (int c = lane; c < 2 * d; c += 32) {
            const float size = s.size[(c < d ? c : c - d) >> 3], of = fabsf(__bfloat162float(coef[row * CS + c])), term = (of + 1.0e-35f) * size;
            most += term;
            steps = fmaf(term, (float)(2 * (KB - (c >> 5))), steps);
            steps = fmaf(of + size, 6.0e-33f, steps);      // 1.2e-38 / (18 * 2^-23)
        }
        most = warp_sum(most);
        steps = warp_sum(steps);
        const bool unsafe = !(most <= 1.0e36f);
        const float err = 1.02f * (most * (3.9e-6f + (float)G * 5.9604645e-8f) + steps * (18.f * 1.1920929e-7f)) + 2.0e-35f;
        s.choose[warp].run(p, r, keys + row * KS, err, unsafe, lane);
    }
}

constexpr int MAX_PAGES = 32768;        // of a sequence: their scores stand in shared memory
constexpr int MAX_TILE_SMEM = 232448;   // what a CTA can have
constexpr int HALF_TILE_SMEM = 115712;  // what a CTA can have where two share an SM
// Rows of a sequence from which on they are scored as tiles, us row by row / in tiles, 32 pages behind 20000: 8 key heads, one sequence of
// 4 rows 7.7 / 11.2, of 8 rows 13.9 / 11.4, of 16 rows 18 / 13, of 32 rows 21 / 25 (two tiles of 16 as one of 32); eight sequences of
// 2 rows 17 / 12, of 8 rows 30 / 13; two key heads, one sequence of 8 rows 9.1 / 11.9, of 32 rows 14 / 24, eight of 16 rows 23 / 13.  By the
// longest sequence: 50 single rows beside one of 8, 33 / 32.
constexpr int TILE_MIN_ROWS = 8;

int check(const PagesParams& p, int dtype, const char* who) {
    if (dtype != GB_F32 && dtype != GB_BF16) GB_REFUSE("%s: dtype code %d", who, dtype);
    const int E = dtype == GB_F32 ? 4 : 8;
    if (p.d <= 0 || p.d % E || p.d > 256) GB_REFUSE("%s: head_dim %d is not a multiple of %d up to 256", who, p.d, E);
    if (p.kv_heads <= 0 || p.pages <= 0 || p.bt_stride <= 0 || p.max_slots <= 0)
        GB_REFUSE("%s: %d kv heads, %d pages, block table %d x %d", who, p.kv_heads, p.pages, p.max_slots, p.bt_stride);
    if ((uintptr_t)p.bounds & 15) GB_REFUSE("%s: the page bounds must be 16-byte aligned", who);
    return 0;
}

}  // namespace

GB_API int gb_page_bounds(const PagesParams* pp, int dtype, cudaStream_t stream) {
    const PagesParams p = *pp;
    if (p.nseq <= 0 || p.max_q_len <= 0 || p.planes <= 0) return 0;
    if (int rc = check(p, dtype, "page_bounds")) return rc;
    if ((uintptr_t)p.k_plane & 15) GB_REFUSE("page_bounds: the key plane must be 16-byte aligned");
    constexpr int smem = BOUND_WARPS * BOUND_LOADS * 512;
    const int pages = ceil_div(p.max_q_len, GB_PAGE);
    if ((int64_t)p.kv_heads * p.planes > (1 << 28) || pages > 65535 || p.nseq > 65535)
        GB_REFUSE("page_bounds: %d kv heads x %d planes, %d sequences of up to %d rows exceed one launch", p.kv_heads, p.planes, p.nseq, p.max_q_len);
    const dim3 grid(ceil_div(p.kv_heads * p.planes, BOUND_WARPS), pages, p.nseq);
    const int chunks = p.d * (dtype == GB_F32 ? 4 : 2) / 16;
#define GB_BOUNDS(T, LPR, CPL)                                                                                                          \
    do {                                                                                                                                \
        static bool done[64];                                                                                                           \
        const cudaError_t e = gb_allow_smem(page_bounds_kernel<T, LPR, CPL>, smem, done);                                               \
        if (e != cudaSuccess) GB_REFUSE("page_bounds: cannot reserve %d bytes of shared memory: %s", smem, cudaGetErrorString(e));       \
        launch_pdl(page_bounds_kernel<T, LPR, CPL>, grid, dim3(BOUND_WARPS * 32), (size_t)smem, stream, p);                             \
    } while (0)
    if (dtype == GB_F32) {
        if (chunks <= 16) GB_BOUNDS(float, 16, 1);
        else if (chunks <= 32) GB_BOUNDS(float, 32, 1);
        else GB_BOUNDS(float, 32, 2);
    } else {
        if (chunks <= 8) GB_BOUNDS(bf16, 8, 1);
        else if (chunks <= 16) GB_BOUNDS(bf16, 16, 1);
        else GB_BOUNDS(bf16, 32, 1);
    }
#undef GB_BOUNDS
    GB_CHECK_LAUNCH("page_bounds");
    return 0;
}

template <typename T, int LP, int CPL>
static int launch_rows(const PagesParams& p, cudaStream_t stream) {
    static bool done[64];
    const cudaError_t e = gb_allow_smem(select_row_kernel<T, LP, CPL>, MAX_TILE_SMEM, done);
    if (e != cudaSuccess) GB_REFUSE("select_pages: cannot reserve shared memory: %s", cudaGetErrorString(e));
    // pieces of no fewer pages than the CTA's warps take at a time, while they all run at once
    const int64_t units = (int64_t)p.nseq * p.max_q_len * p.kv_heads;
    int pieces = 1;
    while (pieces < MAX_PIECES && units * pieces * 2 <= 4 * gb_sm_count() && p.bt_stride > pieces * SELECT_WARPS * 8) pieces *= 2;
    if (units * pieces > 0x7fffffff) GB_REFUSE("select_pages: %d sequences of up to %d rows, %d kv heads exceed one launch", p.nseq, p.max_q_len, p.kv_heads);
    const int longest_first = pieces == 1 && p.max_q_len == 1 && p.nseq <= 512 && units > gb_sm_count();    // (the lengths stand where the coefficients will)
    // batches in flight: three, or two beside the scores of more than some 31000 pages
    const size_t scores = (sizeof(SelectSmem) + (size_t)p.bt_stride * sizeof(uint32_t) + 15) & ~(size_t)15, batch = SELECT_WARPS * RING_CHUNKS * 512;
    const int depth = scores + 3 * batch <= (size_t)MAX_TILE_SMEM ? 3 : 2;
    launch_pdl_cluster(select_row_kernel<T, LP, CPL>, dim3((unsigned)(units * pieces)), dim3(SELECT_THREADS), scores + depth * batch, stream, pieces, 1, p, longest_first,
                       depth);
    GB_CHECK_LAUNCH("select_pages");
    return 0;
}

template <int TILE_WARPS>
static int64_t tile_smem(const PagesParams& p, int rt) {
    return (int64_t)sizeof(TileSmem<TILE_WARPS>) + 2 * rt * tile_coef_stride(p.d) * 2 + (int64_t)rt * tile_key_stride(p.bt_stride) * 4;
}

template <int MT, int KB_MAX, bool EXACT, int TILE_WARPS>
static int launch_tiles_of(const PagesParams& p, cudaStream_t stream) {
    static bool done[64];
    const cudaError_t e = gb_allow_smem(select_tile_kernel<MT, KB_MAX, EXACT, TILE_WARPS>, MAX_TILE_SMEM, done);
    if (e != cudaSuccess) GB_REFUSE("select_pages: cannot reserve shared memory: %s", cudaGetErrorString(e));
    const dim3 grid(ceil_div(p.max_q_len, MT * 16), p.kv_heads, p.nseq);
    if (grid.y > 65535 || grid.z > 65535) GB_REFUSE("select_pages: %d kv heads, %d sequences exceed one launch", p.kv_heads, p.nseq);
    launch_pdl(select_tile_kernel<MT, KB_MAX, EXACT, TILE_WARPS>, grid, dim3(TILE_WARPS * 32), (size_t)tile_smem<TILE_WARPS>(p, MT * 16), stream, p);
    GB_CHECK_LAUNCH("select_pages");
    return 0;
}

template <int MT, int TILE_WARPS>
static int launch_tiles(const PagesParams& p, cudaStream_t stream) {
    if (p.d == 128) return launch_tiles_of<MT, 8, true, TILE_WARPS>(p, stream);
    if (p.d == 64) return launch_tiles_of<MT, 4, true, TILE_WARPS>(p, stream);
    return launch_tiles_of<MT, 16, false, TILE_WARPS>(p, stream);
}

GB_API int gb_select_pages(const PagesParams* pp, int dtype, cudaStream_t stream) {
    const PagesParams p = *pp;
    if (p.nseq <= 0 || p.max_q_len <= 0) return 0;
    if (int rc = check(p, dtype, "select_pages")) return rc;
    if (p.heads <= 0 || p.heads % p.kv_heads) GB_REFUSE("select_pages: %d heads over %d kv heads", p.heads, p.kv_heads);
    if (p.first < 0 || p.last < 1 || (int64_t)p.first + p.last > p.top)
        GB_REFUSE("select_pages: %d pages of which the first %d and the last %d are always chosen", p.top, p.first, p.last);
    if (p.bt_stride > MAX_PAGES) GB_REFUSE("select_pages: sequences of up to %d pages; this kernel takes %d", p.bt_stride, MAX_PAGES);
    if (dtype == GB_BF16 && p.max_q_len >= TILE_MIN_ROWS && p.d % 16 == 0) {
        if (p.max_q_len > 16 && tile_smem<8>(p, 32) <= HALF_TILE_SMEM) return launch_tiles<2, 8>(p, stream);
        if (p.max_q_len > 16 && tile_smem<16>(p, 32) <= MAX_TILE_SMEM) return launch_tiles<2, 16>(p, stream);
        if (tile_smem<16>(p, 16) <= MAX_TILE_SMEM) return launch_tiles<1, 16>(p, stream);
    }
    const int chunks = 2 * p.d / (dtype == GB_F32 ? 4 : 8);
    if (dtype == GB_F32) {
        if (chunks <= 16) return launch_rows<float, 16, 1>(p, stream);
        if (chunks <= 32) return launch_rows<float, 32, 1>(p, stream);
        if (chunks <= 64) return launch_rows<float, 32, 2>(p, stream);
        return launch_rows<float, 32, 4>(p, stream);
    }
    if (chunks <= 16) return launch_rows<bf16, 16, 1>(p, stream);
    if (chunks <= 32) return launch_rows<bf16, 32, 1>(p, stream);
    return launch_rows<bf16, 32, 2>(p, stream);
}

// the checked build's record of the first index this file's kernels found out of bounds
GB_CHECK_READER(gb_checked_status_page_select)
