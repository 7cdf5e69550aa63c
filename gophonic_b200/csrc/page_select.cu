// Which pages of the cache a row of a step should read.
//
// page_bounds keeps, beside the keys, the lowest and the highest value of every channel of each full page of 64 keys:
//     lo[c] = min_t k[t][c],  hi[c] = max_t k[t][c].
// For a query q no key of the page can score more than sum_c max(q_c lo_c, q_c hi_c).  select_pages takes that bound, summed over
// the G query heads that share a key head, as the page's score:
//     s = sum_h sum_c max(q_hc lo_c, q_hc hi_c) = sum_c (P_c hi_c + N_c lo_c),   P = sum_h max(q_h, 0), N = sum_h min(q_h, 0),
// (a head takes hi where q > 0 and lo where q < 0), one product of 2 d channels a page whatever G is, and chooses for every (row, key head) the first `first` pages, the last
// `last` up to the row's own, and of the others those that score highest, `top` in all.
//
// The choice is the one of 64-bit arithmetic.  Scores are float32 sums with a bound e on their error; with tau the k-th highest
// of them, a page above tau + 2 e is among the k best and one below tau - 2 e is not, whatever the errors were, and only the
// pages between (as a rule the one at the border) are summed again in 64 bits, where a product of two bfloat16 values and
// most of their sums are exact.  Pages that tie go by their number.
#include "common.cuh"
#include "api.h"

#include <math.h>

namespace {

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
constexpr int BOUND_THREADS = 256;

// A CTA takes one page of one key head: the page whose last position is among the step's new rows.
template <typename T>
__global__ void __launch_bounds__(BOUND_THREADS) page_bounds_kernel(PagesParams p) {
    constexpr int E = Chunk<T>::E;
    extern __shared__ float sm[];   // [row groups][2][d]
    pdl_wait();                     // the keys, and the step's metadata
    const int seq = blockIdx.z, kvh = blockIdx.y % p.kv_heads, plane = blockIdx.y / p.kv_heads;
    const int kv_len = p.seq_kv_len[seq], past = kv_len - p.seq_q_len[seq];
    const int lp = past / GB_PAGE + (int)blockIdx.x;
    if (lp >= kv_len / GB_PAGE) return;
    const int* bt = block_table_row(p.block_table, p.bt_stride, p.seq_slot[seq], p.max_slots);
    const int64_t at = ((int64_t)plane * p.pages + page_of(bt, lp * GB_PAGE, p.bt_stride, p.pages)) * p.kv_heads + kvh;
    const T* k = (const T*)p.k_plane + at * GB_PAGE * p.d;
    T* to = (T*)p.bounds + at * 2 * p.d;
    const int CH = p.d / E, groups = min(GB_PAGE, BOUND_THREADS / CH);
    const int c = threadIdx.x % CH, g = threadIdx.x / CH;
    if (g < groups) {
        float lo[E], hi[E], x[E];
        unpack(*reinterpret_cast<const uint4*>(k + (int64_t)g * p.d + c * E), x);
#pragma unroll
        for (int e = 0; e < E; e++) lo[e] = hi[e] = x[e];
        for (int r = g + groups; r < GB_PAGE; r += groups) {
            unpack(*reinterpret_cast<const uint4*>(k + (int64_t)r * p.d + c * E), x);
#pragma unroll
            for (int e = 0; e < E; e++) {
                lo[e] = min_nan(lo[e], x[e]);
                hi[e] = max_nan(hi[e], x[e]);
            }
        }
        float* row = sm + g * 2 * p.d + c * E;
#pragma unroll
        for (int e = 0; e < E; e++) {
            row[e] = lo[e];
            row[p.d + e] = hi[e];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * p.d; i += BOUND_THREADS) {
        float v = sm[i];
        for (int r = 1; r < groups; r++) v = i < p.d ? min_nan(v, sm[r * 2 * p.d + i]) : max_nan(v, sm[r * 2 * p.d + i]);
        to[i] = from_f32<T>(v);   // one of the page's own values: no rounding
    }
}

// ---- selection ---------------------------------------------------------------------------------
constexpr int SELECT_THREADS = 256, SELECT_WARPS = SELECT_THREADS / 32;
constexpr int BAND = 512;              // pages near the border that are kept with their 64-bit scores

__device__ __forceinline__ uint32_t order_key(float s) {
    const uint32_t b = __float_as_uint(s);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ uint64_t order_key(double s) {
    const uint64_t b = (uint64_t)__double_as_longlong(s == 0.0 ? 0.0 : s);   // the two zeros are one score
    return b ^ ((b >> 63) ? 0xffffffffffffffffull : 0x8000000000000000ull);
}

template <typename T>
struct SelectSmem {
    double coef_d[2 * 256];      // [N | P], in the order of a page's bounds
    double band_s[BAND];
    float coef[2 * 256];
    int band_i[BAND];
    int hist[256];
    int warp_a[SELECT_WARPS], warp_b[SELECT_WARPS];
    float warp_e[SELECT_WARPS];
    int digit, rest, above, n_band, unsafe;
};

// Sum over a page's 2 d bounds in 64 bits by one warp; NaN counts as the lowest score.
template <typename T>
__device__ __forceinline__ double page_score(const T* b, const double* coef, int d2, int lane) {
    double s = 0.0;
    for (int i = lane; i < d2; i += 32)
        if (coef[i] != 0.0) s += coef[i] * (double)to_f32<T>(b[i]);   // no head looks that way: nothing, also where the bound is infinite
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s == s ? s : -INFINITY;
}

// hist holds how many keys have each digit: the digit of the `want`-th highest key, and how many are wanted of those that have it
__device__ __forceinline__ void pick_digit(int* hist, int want, int& digit, int& rest) {
    // by the first warp: each lane sums 8 digits, from the highest down
    const int lane = threadIdx.x;
    int own = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) own += hist[255 - (lane * 8 + j)];
    int before = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
    }
    before -= own;
    if (before < want && want <= before + own) {
        int left = want - before;
        for (int j = 0; j < 8; j++) {
            const int v = hist[255 - (lane * 8 + j)];
            if (left <= v) {
                digit = 255 - (lane * 8 + j);
                rest = left;
                break;
            }
            left -= v;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(SELECT_THREADS) select_pages_kernel(PagesParams p) {
    constexpr int E = Chunk<T>::E, MOST = 16 / E;     // chunks a lane holds: 16 channels at most
    extern __shared__ __align__(16) unsigned char raw[];
    SelectSmem<T>& s = *reinterpret_cast<SelectSmem<T>*>(raw);
    uint32_t* key = reinterpret_cast<uint32_t*>(raw + sizeof(SelectSmem<T>));   // [candidates]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();
    pdl_trigger();
    const int seq = blockIdx.x / p.max_q_len, qi = blockIdx.x % p.max_q_len, kvh = blockIdx.y;
    const int q_len = p.seq_q_len[seq];
    if (qi >= q_len) return;
    const int row = p.seq_q_start[seq] + qi, pos = p.seq_kv_len[seq] - q_len + qi;
    int* list = p.list + ((int64_t)row * p.kv_heads + kvh) * p.top;
    const int n = pos / GB_PAGE + 1;                      // pages that the row can see
    if (n <= p.top) {
        for (int i = tid; i < p.top; i += SELECT_THREADS) list[i] = i < n ? i : -1;
        return;
    }
    const int c0 = p.first, nc = n - p.first - p.last, k = p.top - p.first - p.last;   // candidates; wanted of them: fewer
    const int* bt = block_table_row(p.block_table, p.bt_stride, p.seq_slot[seq], p.max_slots);
    const int d2 = 2 * p.d, G = p.heads / p.kv_heads;
    const T* bounds = (const T*)p.bounds;
    auto bounds_of = [&](int i) { return bounds + (page_of(bt, (c0 + i) * GB_PAGE, p.bt_stride, p.pages) * p.kv_heads + kvh) * d2; };

    const T* q = (const T*)p.q + (int64_t)row * p.q_row_stride + (int64_t)kvh * G * p.d;
    for (int c = tid; c < p.d; c += SELECT_THREADS) {
        double up = 0.0, down = 0.0;
        for (int h = 0; h < G; h++) {
            const double x = (double)to_f32<T>(q[(int64_t)h * p.d + c]);
            up += x <= 0.0 ? 0.0 : x;      // a NaN is in both
            down += x >= 0.0 ? 0.0 : x;
        }
        s.coef_d[c] = down;
        s.coef_d[p.d + c] = up;
        s.coef[c] = (float)down;
        s.coef[p.d + c] = (float)up;
    }
    if (tid == 0) s.n_band = s.unsafe = 0;
    __syncthreads();
    // A page's 2 d values are 16-byte chunks; LP lanes share a page and hold their coefficients in registers.
    {
        const int NC = d2 / E;
        int LP = 1;
        while (LP < 32 && LP < NC) LP *= 2;
        const int sub = lane / LP, l = lane % LP, per_warp = 32 / LP;
        float cf[MOST][E];
#pragma unroll
        for (int j = 0; j < MOST; j++)
#pragma unroll
            for (int e = 0; e < E; e++) cf[j][e] = l + j * LP < NC ? s.coef[(l + j * LP) * E + e] : 0.f;
        float most = 0.f;     // of this lane's share of a page's sum of |terms|
        bool odd = false;
        for (int i0 = warp * per_warp; i0 < nc; i0 += SELECT_WARPS * per_warp) {
            const int i = i0 + sub;
            float acc = 0.f, mag = 0.f;
            if (i < nc) {
                const uint4* b = reinterpret_cast<const uint4*>(bounds_of(i));
#pragma unroll
                for (int j = 0; j < MOST; j++) {
                    if (l + j * LP >= NC) break;
                    float x[E];
                    unpack(b[l + j * LP], x);
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        acc = fmaf(cf[j][e], x[e], acc);
                        mag = fmaf(fabsf(cf[j][e]), fabsf(x[e]), mag);
                    }
                }
            }
            most = fmaxf(most, mag);
            for (int o = LP / 2; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
            odd = odd || !(fabsf(acc) <= 3.0e38f);
            if (i < nc && l == 0) key[i] = order_key(acc);
        }
        for (int o = LP / 2; o > 0; o >>= 1) most += __shfl_xor_sync(0xffffffffu, most, o);
        most = warp_max(most);
        if (lane == 0) s.warp_e[warp] = most;
        if (odd || !(most <= 3.0e38f)) s.unsafe = 1;
    }
    __syncthreads();
    float err = 0.f;
#pragma unroll
    for (int w = 0; w < SELECT_WARPS; w++) err = fmaxf(err, s.warp_e[w]);
    // A float32 sum of at most 16 products a lane and 5 steps between lanes, of coefficients rounded once: 22 half steps of 2^-23
    // relative to the sum of the terms' sizes, itself known to 2^-18; products below the normal range add next to nothing.
    err = err * (24.f * 5.9604645e-8f) + 1.0e-42f;
    const bool unsafe = s.unsafe != 0;
    int ties_wanted = 0;
    if (k > 0 && !unsafe) {
        // tau: the k-th highest float32 score, digit by digit
        uint32_t prefix = 0;
        int want = k;
        for (int shift = 24; shift >= 0; shift -= 8) {
            s.hist[tid] = 0;
            __syncthreads();
            for (int i = tid; i < nc; i += SELECT_THREADS)
                if (shift == 24 || (key[i] >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&s.hist[(key[i] >> shift) & 255], 1);
            __syncthreads();
            if (warp == 0) pick_digit(s.hist, want, s.digit, s.rest);
            __syncthreads();
            prefix |= (uint32_t)s.digit << shift;
            want = s.rest;
        }
        const float tau = __uint_as_float(prefix ^ ((prefix >> 31) ? 0x80000000u : 0xffffffffu));
        const float hi = tau + 2.f * err + fabsf(tau) * 2.4e-7f, lo = tau - 2.f * err - fabsf(tau) * 2.4e-7f;
        if (tid == 0) s.above = 0;
        __syncthreads();
        for (int i = tid; i < nc; i += SELECT_THREADS) {
            const uint32_t kb = key[i];
            const float v = __uint_as_float(kb ^ ((kb >> 31) ? 0x80000000u : 0xffffffffu));
            uint32_t mark = 0;
            if (v > hi) {
                mark = 2;
                atomicAdd(&s.above, 1);
            } else if (v >= lo) {
                const int at = atomicAdd(&s.n_band, 1);
                if (at < BAND) s.band_i[at] = i;
                mark = 2;      // until the band is settled
            }
            key[i] = mark;
        }
        __syncthreads();
        const int m = s.n_band, wanted = k - s.above;
        if (m > wanted && m <= BAND) {
            for (int j = warp; j < m; j += SELECT_WARPS) {
                const double v = page_score<T>(bounds_of(s.band_i[j]), s.coef_d, d2, lane);
                if (lane == 0) s.band_s[j] = v;
            }
            __syncthreads();
            for (int j = tid; j < m; j += SELECT_THREADS) {
                int better = 0;
                for (int o = 0; o < m; o++)
                    better += s.band_s[o] > s.band_s[j] || (s.band_s[o] == s.band_s[j] && s.band_i[o] < s.band_i[j]);
                key[s.band_i[j]] = better < wanted ? 2 : 0;
            }
        }
        __syncthreads();
    }
    if (k > 0 && (unsafe || s.n_band > BAND)) {
        // Scores beyond float32, or hundreds that tie: the k-th highest of the 64-bit scores, which are summed anew for
        // every digit.  Rare, and right for any input.
        uint64_t prefix = 0;
        int want = k;
        for (int shift = 56; shift >= 0; shift -= 8) {
            s.hist[tid] = 0;
            __syncthreads();
            for (int i = warp; i < nc; i += SELECT_WARPS) {
                const uint64_t v = order_key(page_score<T>(bounds_of(i), s.coef_d, d2, lane));
                if (lane == 0 && (shift == 56 || (v >> (shift + 8)) == (prefix >> (shift + 8)))) atomicAdd(&s.hist[(int)(v >> shift) & 255], 1);
            }
            __syncthreads();
            if (warp == 0) pick_digit(s.hist, want, s.digit, s.rest);
            __syncthreads();
            prefix |= (uint64_t)s.digit << shift;
            want = s.rest;
        }
        for (int i = warp; i < nc; i += SELECT_WARPS) {
            const uint64_t v = order_key(page_score<T>(bounds_of(i), s.coef_d, d2, lane));
            if (lane == 0) key[i] = v > prefix ? 2 : v == prefix ? 1 : 0;
        }
        ties_wanted = want;
        __syncthreads();
    }
    // the chosen pages in order: each thread counts a stretch of the pages
    auto kind = [&](int page) -> uint32_t {
        if (page < c0 || page >= c0 + nc) return 2;
        return k > 0 ? key[page - c0] : 0;
    };
    const int per = (n + SELECT_THREADS - 1) / SELECT_THREADS;
    const int a = min(n, tid * per), b = min(n, a + per);
    int sure = 0, tie = 0;
    for (int i = a; i < b; i++) {
        const uint32_t m = kind(i);
        sure += m == 2;
        tie += m == 1;
    }
    int sure_to = sure, tie_to = tie;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, sure_to, o), y = __shfl_up_sync(0xffffffffu, tie_to, o);
        if (lane >= o) {
            sure_to += x;
            tie_to += y;
        }
    }
    if (lane == 31) {
        s.warp_a[warp] = sure_to;
        s.warp_b[warp] = tie_to;
    }
    __syncthreads();
    sure_to -= sure;
    tie_to -= tie;
    for (int w = 0; w < warp; w++) {
        sure_to += s.warp_a[w];
        tie_to += s.warp_b[w];
    }
    for (int i = a; i < b; i++) {
        const uint32_t m = kind(i);
        if (m == 2 || (m == 1 && tie_to < ties_wanted)) list[sure_to + min(tie_to, ties_wanted)] = i;
        sure_to += m == 2;
        tie_to += m == 1;
    }
}

constexpr int MAX_PAGES = 32768;   // of a sequence: their scores stand in shared memory

int check(const PagesParams& p, int dtype, const char* who) {
    if (dtype != GB_F32 && dtype != GB_BF16) GB_REFUSE("%s: dtype code %d", who, dtype);
    const int E = dtype == GB_F32 ? 4 : 8;
    if (p.d <= 0 || p.d % E || p.d > 256) GB_REFUSE("%s: head_dim %d is not a multiple of %d up to 256", who, p.d, E);
    if (p.kv_heads <= 0 || p.pages <= 0 || p.bt_stride <= 0 || p.max_slots <= 0) GB_REFUSE("%s: %d kv heads, %d pages, block table %d x %d", who, p.kv_heads, p.pages, p.max_slots, p.bt_stride);
    if ((uintptr_t)p.bounds & 15) GB_REFUSE("%s: the page bounds must be 16-byte aligned", who);
    return 0;
}

}  // namespace

GB_API int gb_page_bounds(const PagesParams* pp, int dtype, cudaStream_t stream) {
    const PagesParams p = *pp;
    if (p.nseq <= 0 || p.max_q_len <= 0 || p.planes <= 0) return 0;
    if (int rc = check(p, dtype, "page_bounds")) return rc;
    if ((uintptr_t)p.k_plane & 15) GB_REFUSE("page_bounds: the key plane must be 16-byte aligned");
    const dim3 grid(ceil_div(p.max_q_len, GB_PAGE), p.kv_heads * p.planes, p.nseq);
    if ((int64_t)p.kv_heads * p.planes > 65535 || p.nseq > 65535) GB_REFUSE("page_bounds: %d kv heads x %d planes, %d sequences exceed one launch", p.kv_heads, p.planes, p.nseq);
    const int E = dtype == GB_F32 ? 4 : 8, groups = BOUND_THREADS / (p.d / E) < GB_PAGE ? BOUND_THREADS / (p.d / E) : GB_PAGE;
    const size_t smem = (size_t)groups * 2 * p.d * sizeof(float);
    if (dtype == GB_F32)
        launch_pdl(page_bounds_kernel<float>, grid, dim3(BOUND_THREADS), smem, stream, p);
    else
        launch_pdl(page_bounds_kernel<bf16>, grid, dim3(BOUND_THREADS), smem, stream, p);
    GB_CHECK_LAUNCH("page_bounds");
    return 0;
}

template <typename T>
static int launch_select(const PagesParams& p, cudaStream_t stream) {
    const size_t smem = sizeof(SelectSmem<T>) + (size_t)p.bt_stride * sizeof(uint32_t);
    static bool configured = false;
    if (!configured) {
        const cudaError_t e = cudaFuncSetAttribute(select_pages_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   (int)(sizeof(SelectSmem<T>) + MAX_PAGES * sizeof(uint32_t)));
        if (e != cudaSuccess) GB_REFUSE("select_pages: cannot reserve shared memory: %s", cudaGetErrorString(e));
        configured = true;
    }
    if (p.kv_heads > 65535 || (int64_t)p.nseq * p.max_q_len > 0x7fffffff) GB_REFUSE("select_pages: %d sequences of up to %d rows exceed one launch", p.nseq, p.max_q_len);
    launch_pdl(select_pages_kernel<T>, dim3(p.nseq * p.max_q_len, p.kv_heads), dim3(SELECT_THREADS), smem, stream, p);
    GB_CHECK_LAUNCH("select_pages");
    return 0;
}

GB_API int gb_select_pages(const PagesParams* pp, int dtype, cudaStream_t stream) {
    const PagesParams p = *pp;
    if (p.nseq <= 0 || p.max_q_len <= 0) return 0;
    if (int rc = check(p, dtype, "select_pages")) return rc;
    if (p.heads <= 0 || p.heads % p.kv_heads) GB_REFUSE("select_pages: %d heads over %d kv heads", p.heads, p.kv_heads);
    if (p.first < 0 || p.last < 1 || p.first + p.last > p.top) GB_REFUSE("select_pages: %d pages of which the first %d and the last %d are always chosen", p.top, p.first, p.last);
    if (p.bt_stride > MAX_PAGES) GB_REFUSE("select_pages: sequences of up to %d pages; this kernel takes %d", p.bt_stride, MAX_PAGES);
    return dtype == GB_F32 ? launch_select<float>(p, stream) : launch_select<bf16>(p, stream);
}

// the checked build's record of the first index this file's kernels found out of bounds
GB_CHECK_READER(gb_checked_status_page_select)
