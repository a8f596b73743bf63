// Selection over a vocabulary: the largest logits of every row with the row's log-normaliser, and the best continuations of
// beams.  The language-model side of the circuits: a teacher's top logits to learn from, beam search to answer with.
//
// One pass over the logits, which carries the running maximum m and sum s = sum exp((x - m) / T) of a softmax and the n largest
// logits.  Places are part of the keys (a lower place first among equals), keys are unique, and the answer does not depend on
// how rows are cut or in which order logits come.  Two forms, by the number of rows (see `launch_rows`):
//   a warp a row   Its lanes leave the maximum of every four loads of 16 bytes in shared memory.  After (at most) 16 tiles of 4
//                  KB a threshold is bisected over these maxima that n, or a few more, of them reach: so do n logits, and the
//                  n largest are among the logits of those maxima, which alone are read again.
//   CTAs a row     The CTA keeps the n largest so far; rows are cut into parts until the device is full, and a second kernel
//                  joins their lists, one CTA per row.
// For beams another kernel joins the rows of a sequence and adds the scores, in 64 bits: a sum of a score and a logit is
// rounded only in the returned score, never before it is compared, and normalisers that leave the order in doubt are taken again.
#include "pcx_common.cuh"
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <algorithm>
#include <cmath>

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxTop = 128;                        // entries of a list
constexpr int kRoom = 4096;                         // candidates a CTA holds besides its list
constexpr int kFew = 512;                           // candidates ranked by counting at once
constexpr int kMaxSplits = 32;                      // parts of a row: their lists fit kRoom

typedef unsigned long long u64;

// What a CTA leaves for the join: the sorted keys of its list, the maximum of its part and the sum of exp((x - m) / T).
struct Part { float m; int count; double s; };

// Unsigned integers in the order of the floats; one zero (-0 counts as 0).
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t k) {
    return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ u64 ordered(double x) {
    const u64 b = (u64)__double_as_longlong(x + 0.0);
    return b ^ ((b >> 63) ? ~0ull : 0x8000000000000000ull);
}
__device__ __forceinline__ double unordered(u64 k) {
    return __longlong_as_double((long long)(k ^ ((k >> 63) ? 0x8000000000000000ull : ~0ull)));
}
__device__ __forceinline__ u64 key_of(float x, uint32_t place) { return ((u64)ordered(x) << 32) | (uint32_t)~place; }
__device__ __forceinline__ float value_of(u64 key) { return unordered((uint32_t)(key >> 32)); }
__device__ __forceinline__ uint32_t place_of(u64 key) { return ~(uint32_t)key; }

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The terms of a sum are 2^(x * scale - r) with r = m * scale rounded once: one fused operation each, and all of them relative to
// the same r.  That is off by up to half a step of r, at most 64 below kNear: far from the range's ends, and put right when the
// sum is read.  Larger r (logits of -1e30, the lowest number of a type) leave nothing of a difference: their terms are 2^((x - m) *
// scale), more slowly.
constexpr float kNear = 2147483648.0f;
__device__ __forceinline__ bool near(float r) { return fabsf(r) < kNear; }
// What the sum relative to (m, r) is multiplied by to be relative to (top, nr): the difference of the r is taken to the last bit.
__device__ __forceinline__ float to_other(float m, float r, float top, float nr, float scale) {
    if (near(r) && near(nr)) {
        const float d = r - nr, z = d - r, rest = (r - (d - z)) - (nr + z);
        const float f = exp2_fast(d);
        return fmaf(f, rest * 0.69314718f, f);
    }
    return exp2_fast((m - top) * scale + (near(r) ? fmaf(-m, scale, r) : 0.0f) - (near(nr) ? fmaf(-top, scale, nr) : 0.0f));
}
// The sum relative to (m, r) as one relative to M >= m itself.
__device__ __forceinline__ double to_own(float s, float m, float r, float M, float scale) {
    if (!(m > PCX_NEG_INF) || !(M < CUDART_INF_F)) return 0.0;
    if (near(r)) return (double)s * exp2((double)r - (double)M * (double)scale);
    return m == M ? (double)s : (double)s * exp2(((double)m - (double)M) * (double)scale);
}
__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
    return x;
}

// 16 bytes of logits: their maximum (NaN skipped) and the logits one by one.
template <typename T> struct Pack;
template <> struct Pack<float> {
    static constexpr int N = 4, UNUSED = 0;                // UNUSED: low bits that all values have alike as 32-bit numbers
    static __device__ __forceinline__ float max(const uint4& v) {
        return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
    }
    static __device__ __forceinline__ float at(const uint4& v, int i) { return __uint_as_float((&v.x)[i]); }
};
template <> struct Pack<__nv_bfloat16> {
    static constexpr int N = 8, UNUSED = 16;
    static __device__ __forceinline__ float max(const uint4& v) {
        const __nv_bfloat162* h = (const __nv_bfloat162*)&v;
        const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
        return fmaxf(__low2float(m), __high2float(m));
    }
    static __device__ __forceinline__ float at(const uint4& v, int i) {
        const uint32_t w = (&v.x)[i >> 1];
        return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
    }
};
template <> struct Pack<__half> {
    static constexpr int N = 8, UNUSED = 13;
    static __device__ __forceinline__ float max(const uint4& v) {
        const __half2* h = (const __half2*)&v;
        const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
        return fmaxf(__low2float(m), __high2float(m));
    }
    static __device__ __forceinline__ float at(const uint4& v, int i) {
        const __half2 h = ((const __half2*)&v)[i >> 1];
        return i & 1 ? __high2float(h) : __low2float(h);
    }
};

// Their terms: three sums one after the other at most.
template <typename T>
__device__ __forceinline__ float group_sum(const uint4& v, float scale, float r) {
    constexpr int VE = Pack<T>::N;
    float t[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) t[i] = exp2_fast(fmaf(Pack<T>::at(v, i), scale, -r));
#pragma unroll
    for (int o = VE / 2; o; o /= 2)
#pragma unroll
        for (int i = 0; i < o; ++i) t[i] += t[i + o];
    return t[0];
}

// The 16 bytes of elements e ... of a row, -inf beyond its ends.  (Out of line, as everything that few tiles need: the warps
// of an SM are in different places of the code, and it has to fit the instruction cache.)
template <typename T>
__device__ __noinline__ uint4 load_edge(const T* x, int e, int vocab) {
    constexpr int VE = Pack<T>::N;
    T edge[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) edge[i] = e + i >= 0 && e + i < vocab ? x[e + i] : (T)PCX_NEG_INF;
    return *(const uint4*)edge;
}
// Group `gi` of a row; whole groups are [whole0, whole1), there is none from g1 on.
template <typename T>
__device__ __forceinline__ uint4 load_group(const T* x, int gi, int off, int whole0, int whole1, int g1, int vocab) {
    constexpr int VE = Pack<T>::N;
    if (gi >= whole0 && gi < whole1) return __ldg((const uint4*)(x + (int64_t)gi * VE - off));
    return load_edge<T>(x, gi < g1 ? gi * VE - off : -VE, vocab);
}

struct RowArgs {
    const void* logits;
    const float* scores;           // beams: [rows], a row whose score is -inf or NaN is skipped; null = none
    const uint8_t* finished;       // beams: [rows], finished rows are skipped; null = none
    u64* keys;                     // [rows * splits][n]
    Part* parts;                   // [rows * splits]
    int64_t* ids;                  // single-part answers go straight to the outputs (null = to keys / parts)
    void* values;
    float* norms;
    int64_t stride0, stride1;      // elements: row r starts at (r / inner) * stride0 + (r % inner) * stride1
    int inner, vocab, n, splits;
    float scale;                   // log2(e) / T
    double inv_t;
};

// log sum exp(x / T) from the maximum and the sum of exp((x - m) / T).
__device__ __forceinline__ double log_norm(float m, double s, double inv_t) {
    if (m == PCX_NEG_INF) return -CUDART_INF;
    if (m == CUDART_INF_F) return CUDART_INF;
    return (double)m * inv_t + log(s);
}

struct Shared {
    alignas(16) u64 keys[kRoom + kMaxTop]; // the list (sorted, first), behind it the candidates of a tile
    u64 list[kMaxTop];
    float red_m[kWarps];
    double red_s[kWarps];
    uint32_t warp_t[kWarps], warp_u[kWarps];
    int count;
};

__device__ __forceinline__ int block_sum(int mine, int* total) {       // every thread gets the sum
    mine = __reduce_add_sync(~0u, mine);
    __syncthreads();
    if (threadIdx.x == 0) *total = 0;
    __syncthreads();
    if ((threadIdx.x & 31) == 0 && mine != 0) atomicAdd(total, mine);
    __syncthreads();
    return *total;
}

// A threshold t with least <= #(keys >= t) <= most, by bisection between the smallest and the largest key; where equal keys
// allow none, the largest t with at least `least`.  `at_least(i, t)`: whether key i < total is t or more.
template <typename F>
__device__ __forceinline__ u64 bisect(int total, int least, int most, u64 lo, u64 hi, F at_least) {
    const int tid = threadIdx.x;
    while (lo < hi) {
        const u64 mid = lo + ((hi - lo) >> 1) + ((hi - lo) & 1);
        int c = 0;
        for (int i0 = 0; i0 < total; i0 += kThreads) c += __syncthreads_count(i0 + tid < total && at_least(i0 + tid, mid));
        if (c >= least) {
            lo = mid;
            if (c <= most) break;
        } else {
            hi = mid - 1;
        }
    }
    return lo;
}

// Smallest and largest of the high halves of keys[0, total), as bounds of all keys.
__device__ __forceinline__ void key_range(const u64* keys, int total, uint32_t* low, uint32_t* high, u64& lo, u64& hi) {
    uint32_t least = ~0u, most = 0;
    for (int i = threadIdx.x; i < total; i += kThreads) {
        const uint32_t v = (uint32_t)(keys[i] >> 32);
        least = min(least, v);
        most = max(most, v);
    }
    least = __reduce_min_sync(~0u, least);
    most = __reduce_max_sync(~0u, most);
    if ((threadIdx.x & 31) == 0) { low[threadIdx.x >> 5] = least; high[threadIdx.x >> 5] = most; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) { least = min(least, low[w]); most = max(most, high[w]); }
    lo = (u64)least << 32;
    hi = ((u64)most << 32) | 0xffffffffu;
}

// Cuts the `total` (more than kFew) unique keys in sh.keys back to n ... kFew / 2 of the largest, at its front.  Returns how
// many are left.
__device__ __noinline__ int trim(Shared& sh, int total, int n) {
    const int tid = threadIdx.x;
    u64 lo, hi;
    key_range(sh.keys, total, sh.warp_t, sh.warp_u, lo, hi);
    lo = bisect(total, n, kFew / 2, lo, hi, [&](int i, u64 mid) { return sh.keys[i] >= mid; });
    // compaction, a block of keys after the other: those of a block are read before any is overwritten
    __syncthreads();
    if (tid == 0) sh.count = 0;
    for (int i0 = 0; i0 < total; i0 += kThreads) {
        const u64 own = i0 + tid < total ? sh.keys[i0 + tid] : 0;
        __syncthreads();
        if (own >= lo && own != 0) sh.keys[atomicAdd(&sh.count, 1)] = own;
    }
    __syncthreads();
    total = sh.count;
    __syncthreads();
    return total;
}

// Keeps the n largest of the `total` unique keys in sh.keys, sorted, at its front.  Returns how many there are.
__device__ int prune(Shared& sh, int total, int n) {
    const int tid = threadIdx.x;
    if (total > kFew) total = trim(sh, total, n);
    const int kept = min(total, n);
    for (int i = tid; i < total; i += kThreads) {
        const u64 k = sh.keys[i];
        int rank = 0;
        for (int j = 0; j < (total & ~1); j += 2) {
            const ulonglong2 o = *(const ulonglong2*)(sh.keys + j);
            rank += (o.x > k) + (o.y > k);
        }
        if (total & 1) rank += sh.keys[total - 1] > k;
        if (rank < n) sh.list[rank] = k;
    }
    __syncthreads();
    for (int i = tid; i < kept; i += kThreads) sh.keys[i] = sh.list[i];
    __syncthreads();
    return kept;
}

// Statistics of a block: maximum and sum of all warps' (m, s), to every thread.
__device__ __forceinline__ void block_stats(Shared& sh, float m, double s, double inv_t, float& M, double& S) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane == 0) { sh.red_m[warp] = m; sh.red_s[warp] = s; }
    __syncthreads();
    M = sh.red_m[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) M = fmaxf(M, sh.red_m[w]);
    S = 0.0;
    if (threadIdx.x == 0 && M > PCX_NEG_INF && M < CUDART_INF_F)
#pragma unroll
        for (int w = 0; w < kWarps; ++w)
            if (sh.red_m[w] > PCX_NEG_INF) S += sh.red_s[w] * exp(((double)sh.red_m[w] - (double)M) * inv_t);
}

// An answer of top logits, or a part of one.
template <typename T>
__device__ __forceinline__ void leave(const RowArgs& a, const Shared& sh, int64_t row, int have, float M, double S) {
    const int tid = threadIdx.x;
    if (a.ids == nullptr) {
        if (tid == 0) a.parts[blockIdx.x] = Part{M, have, S};
        for (int i = tid; i < have; i += kThreads) a.keys[(int64_t)blockIdx.x * a.n + i] = sh.keys[i];
        return;
    }
    if (tid == 0) a.norms[row] = (float)log_norm(M, S, a.inv_t);
    for (int i = tid; i < a.n; i += kThreads) {
        const u64 k = i < have ? sh.keys[i] : 0;
        a.ids[row * a.n + i] = i < have ? (int64_t)place_of(k) : -1;
        ((T*)a.values)[row * a.n + i] = i < have ? (T)value_of(k) : (T)PCX_NEG_INF;
    }
}

constexpr int kRowWarps = 4, kGroups = 8;           // warps of a CTA; groups of 16 bytes a lane and tile
constexpr int kQuad = 4;                            // groups that share a maximum
constexpr int kChunk = 16, kMaxima = kChunk * 32 * (kGroups / kQuad);       // tiles whose maxima a warp holds
constexpr int kSet = 320;                           // keys a warp holds

// Cuts a warp's set of `count` (at least n) unique keys back to n ... n + n / 8 of the largest.  Returns how many are left;
// `bound`: a key that n of them reach.
__device__ __noinline__ int cut(u64* keys, int count, int n, u64* bound) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
    uint32_t least = ~0u, most = 0;
    for (int i = lane; i < count; i += 32) {
        const uint32_t v = (uint32_t)(keys[i] >> 32);
        least = min(least, v);
        most = max(most, v);
    }
    u64 lo = (u64)__reduce_min_sync(~0u, least) << 32;                        // #(keys >= lo) >= n
    if (count > n + n / 8) {
        u64 hi = ((u64)__reduce_max_sync(~0u, most) << 32) | 0xffffffffu;
        while (lo < hi) {
            const u64 mid = lo + ((hi - lo) >> 1) + ((hi - lo) & 1);
            int c = 0;
            for (int i = lane; i < count; i += 32) c += keys[i] >= mid;
            c = __reduce_add_sync(~0u, c);
            if (c >= n) {
                lo = mid;
                if (c <= n + n / 8) break;
            } else {
                hi = mid - 1;
            }
        }
        int kept = 0;
        for (int i0 = 0; i0 < count; i0 += 32) {
            const u64 k = i0 + lane < count ? keys[i0 + lane] : 0;
            __syncwarp();
            const unsigned stays = __ballot_sync(~0u, i0 + lane < count && k >= lo);
            if (stays >> lane & 1) keys[kept + __popc(stays & ((1u << lane) - 1))] = k;
            kept += __popc(stays);
        }
        count = kept;
        __syncwarp();
    }
    *bound = lo;
    return count;
}

// The sum over the lanes before this one; `n` becomes the sum over all.
__device__ __forceinline__ int warp_before(int& n) {
    const int lane = threadIdx.x & 31;
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(~0u, x, o); if (lane >= o) x += y; }
    const int before = x - n;
    n = __shfl_sync(~0u, x, 31);
    return before;
}

// What a lane's part of a tile adds to its sum when the quick way gave no number: NaN, infinities, or a maximum that is not `near`.
template <typename T>
__device__ __noinline__ float careful_sum(const T* x, int first, int groups, int step, int end, float m, float r, float scale) {
    constexpr int VE = Pack<T>::N;
    double s = 0.0;
#pragma unroll 1
    for (int i = 0; i < groups * VE; ++i) {
        const int e = first + i / VE * step + i % VE;
        if (e < 0 || e >= end) continue;
        const float f = fmaxf((float)x[e], PCX_NEG_INF);
        s += (double)exp2_fast(near(r) ? fmaf(f, scale, -r) : f == m ? 0.0f : (f - m) * scale);
    }
    return (float)s;
}

// Many rows, or short ones: a warp a row, sixteen rows under way per SM (128 registers: a tile is on its way while the one
// before is taken).  8192 rows of 32768 bf16, n = 32: 186 us, 595 MB read (2.9 TB/s of the 6.4 that a copy reaches).  The
// walk alone takes 105 us; the bisection and the logits that are read again are 4 K instructions a row of little parallelism,
// and 8192 rows are 3.5 times what the device holds.  Chunks of 8 tiles instead of 16: 237 us.
template <typename T>
__global__ void __launch_bounds__(kRowWarps * 32, 4)
top_rows_warp_kernel(RowArgs a, int64_t n_rows) {
    constexpr int VE = Pack<T>::N, G = kGroups, H = G / kQuad;
    constexpr int SIDE = 32 / (kQuad * VE), AHEAD = 12;                   // maxima whose logits fit the lanes; such steps at once
    __shared__ alignas(16) u64 all_keys[kRowWarps][kSet];
    __shared__ float all_maxima[kRowWarps][kMaxima];
    __shared__ uint16_t all_hot[kRowWarps][kMaxima];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = (int64_t)blockIdx.x * kRowWarps + warp;
    if (row >= n_rows) return;                      // (no barrier of the CTA follows)
    u64* keys = all_keys[warp];                     // the largest so far, keys[0, count), unsorted
    float* maxima = all_maxima[warp];
    uint16_t* hot = all_hot[warp];
    int count = 0;
    u64 bound = 0;                                  // n keys of the set are at least this large; 0 before there are n
    float m = PCX_NEG_INF, r = PCX_NEG_INF, s = 0.0f;
    bool skip = a.finished != nullptr && a.finished[row] != 0;
    if (a.scores != nullptr) skip |= !(a.scores[row] > PCX_NEG_INF);
    if (!skip) {
        const T* x = (const T*)a.logits + (row / a.inner) * a.stride0 + (row % a.inner) * a.stride1;
        // groups begin on 16-byte boundaries; the first and the last may reach over the row's ends
        const int off = (int)(((uintptr_t)x & 15) / sizeof(T));
        const int groups = (int)(((int64_t)off + a.vocab + VE - 1) / VE);
        // whole groups: those of the row's ends are read element by element
        const int whole0 = off != 0 ? 1 : 0, whole1 = (off + a.vocab) / VE;
        for (int chunk = 0; chunk < groups; chunk += 32 * G * kChunk) {
            const int tiles = min(kChunk, (groups - chunk + 32 * G - 1) / (32 * G));
            auto load = [&](uint4 (&v)[G], int t) {
                const int g = chunk + t * 32 * G;
                const T* mine = x + (int64_t)(g + lane) * VE - off;
                if (g >= whole0 && g + 32 * G <= whole1) {
#pragma unroll
                    for (int j = 0; j < G; ++j) v[j] = __ldg((const uint4*)(mine + j * 32 * VE));
                } else {
#pragma unroll
                    for (int j = 0; j < G; ++j) v[j] = load_group<T>(x, g + j * 32 + lane, off, whole0, whole1, groups, a.vocab);
                }
            };
            auto take = [&](const uint4 (&v)[G], int t) {
                float top = PCX_NEG_INF;
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    float f = Pack<T>::max(v[h * kQuad]);
#pragma unroll
                    for (int j = 1; j < kQuad; ++j) f = fmaxf(f, Pack<T>::max(v[h * kQuad + j]));
                    f = fmaxf(f, PCX_NEG_INF);      // (not NaN)
                    maxima[(t * H + h) * 32 + lane] = f;
                    top = fmaxf(top, f);
                }
                if (top > m) {
                    const float nr = top * a.scale;
                    s = m > PCX_NEG_INF ? s * to_other(m, r, top, nr, a.scale) : 0.0f;
                    m = top;
                    r = nr;
                }
                if (m > PCX_NEG_INF) {
                    float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
                    for (int j = 0; j < G; j += 2) {
                        s0 += group_sum<T>(v[j], a.scale, r);
                        s1 += group_sum<T>(v[j + 1], a.scale, r);
                    }
                    s0 += s1;
                    if (!(s0 < CUDART_INF_F) || !near(r))
                        s0 = careful_sum<T>(x, (chunk + t * 32 * G + lane) * VE - off, G, 32 * VE, a.vocab, m, r, a.scale);
                    s += s0;
                }
            };
            uint4 even[G], odd[G];                  // a tile is on its way while the one before is taken
            load(even, 0);
#pragma unroll 1
            for (int t = 0; t < tiles; t += 2) {
                if (t + 1 < tiles) load(odd, t + 1);
                take(even, t);
                if (t + 1 >= tiles) break;
                if (t + 2 < tiles) load(even, t + 2);
                take(odd, t + 1);
            }
            __syncwarp();
            // the threshold: n, or a few more, of the maxima (and of the keys so far) are that large
            const int n_max = tiles * H;            // maxima a lane
            float own[kChunk * H];
            float least = bound != 0 ? value_of(bound) : -3.402823466e38f;
            float most = PCX_NEG_INF;
            int pass = 0;
#pragma unroll
            for (int q = 0; q < kChunk * H; ++q) {
                own[q] = q < n_max ? maxima[q * 32 + lane] : PCX_NEG_INF;
                most = fmaxf(most, own[q]);
                pass += own[q] >= least;
            }
            pass = __reduce_add_sync(~0u, pass);
            if (pass == 0) continue;
            if (pass > 2 * a.n) {
                // (every lane's largest reaches the smallest of them: a start for n up to 32)
                constexpr int BITS = Pack<T>::UNUSED;
                const uint32_t top = ordered(most), all = a.n <= 32 ? __reduce_min_sync(~0u, top) : 0;
                uint32_t lo = max(ordered(least), all) >> BITS, hi = __reduce_max_sync(~0u, top) >> BITS;
#pragma unroll 1
                while (lo < hi) {
                    const uint32_t mid = lo + ((hi - lo) >> 1) + ((hi - lo) & 1);
                    const float f = unordered(mid << BITS);
                    int c = 0;
#pragma unroll
                    for (int q = 0; q < kChunk * H; ++q) c += own[q] >= f;
                    c = __reduce_add_sync(~0u, c);
                    if (c >= a.n) {
                        lo = mid;
                        if (c <= a.n + a.n / 4 + 4) break;
                    } else {
                        hi = mid - 1;
                    }
                }
                least = unordered(lo << BITS);
            }
            int n_hot = 0;
#pragma unroll
            for (int q = 0; q < kChunk * H; ++q) n_hot += own[q] >= least;
            int to = warp_before(n_hot);
#pragma unroll
            for (int q = 0; q < kChunk * H; ++q)
                if (own[q] >= least) hot[to++] = (uint16_t)(q * 32 + lane);
            __syncwarp();
            // their logits, a lane for each
            const int h_own = lane / (kQuad * VE), e_own = chunk * VE - off + lane / VE % kQuad * 32 * VE + lane % VE;
            auto place = [&](int h) { return e_own + (hot[h] / 32 * kQuad * 32 + hot[h] % 32) * VE; };     // (quads lie one after the other)
#pragma unroll 1
            for (int h0 = h_own; h0 - h_own < n_hot; h0 += SIDE * AHEAD) {
                float f[AHEAD];
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) {
                    const int h = h0 + i * SIDE;
                    f[i] = PCX_NEG_INF;
                    if (h < n_hot) {
                        const int e = place(h);
                        if (e >= 0 && e < a.vocab) f[i] = (float)x[e];
                    }
                }
                unsigned wanted = 0;
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) wanted |= (unsigned)(f[i] >= least) << i;
                int n_new = __popc(wanted);
                int at_key = warp_before(n_new);
                if (count + n_new <= kSet) {        // the usual case
#pragma unroll
                    for (int i = 0; i < AHEAD; ++i)
                        if (wanted >> i & 1) keys[count + at_key++] = key_of(f[i], (uint32_t)place(h0 + i * SIDE));
                    count += n_new;
                } else {                            // many equal or ordered logits: a few at a time, the set cut in between
#pragma unroll
                    for (int i = 0; i < AHEAD; ++i) {
                        if (count > kSet - 32) count = cut(keys, count, a.n, &bound);
                        const u64 key = wanted >> i & 1 ? key_of(f[i], (uint32_t)place(h0 + i * SIDE)) : 0;
                        const bool fits = key != 0 && key >= bound;
                        const unsigned lanes = __ballot_sync(~0u, fits);
                        if (fits) keys[count + __popc(lanes & ((1u << lane) - 1))] = key;
                        count += __popc(lanes);
                    }
                }
                __syncwarp();
            }
            if (count >= a.n && chunk + 32 * G * kChunk < groups) count = cut(keys, count, a.n, &bound);
            __syncwarp();
        }
    }
    // the lanes' sums become one in 64 bits
    float M = m;
#pragma unroll
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(~0u, M, o));
    const double S = warp_sum(to_own(s, m, r, M, a.scale));
    // the set in order: a key's place is the number of larger ones
    if (count > a.n + a.n / 2 + 16) count = cut(keys, count, a.n, &bound);
    __syncwarp();
    const int have = min(count, a.n);
    if (lane == 0) {
        if (a.ids == nullptr) a.parts[row] = Part{M, have, S};
        else a.norms[row] = (float)log_norm(M, S, a.inv_t);
    }
#pragma unroll 1
    for (int i = lane; i < count; i += 32) {
        const u64 k = keys[i];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < (count & ~1); j += 2) {
            const ulonglong2 o = *(const ulonglong2*)(keys + j);
            rank += (int)(o.x > k) + (int)(o.y > k);
        }
        if (count & 1) rank += (int)(keys[count - 1] > k);
        if (rank >= a.n) continue;
        if (a.ids == nullptr) {
            a.keys[row * a.n + rank] = k;
        } else {
            a.ids[row * a.n + rank] = (int64_t)place_of(k);
            ((T*)a.values)[row * a.n + rank] = (T)value_of(k);
        }
    }
    if (a.ids != nullptr)
        for (int i = have + lane; i < a.n; i += 32) {
            a.ids[row * a.n + i] = -1;
            ((T*)a.values)[row * a.n + i] = (T)PCX_NEG_INF;
        }
}

// Few rows: a CTA a row or part of one, tiles of G groups of 16 bytes a thread (8; 2 for parts too short for that).  The CTA
// keeps the n largest logits so far, sorted; the last of them is a bound that few later logits pass, so that a tile costs a
// comparison a thread and a barrier.  The first tile's bound comes from its threads' maxima.  1024 rows of 32768 bf16, n = 32:
// 36 us a call (1.9 TB/s); 1001 rows of 50257 fp32, n = 100: 107 us (1.9 TB/s), of which the walk is 41: what bounds it are the
// barriers and the ranking of a tile's candidates, after nearly every tile (up to seven a row here).  (8192 rows with tiles of 4,
// 8 and 16 groups: 271, 235, 250 us.)
template <typename T, int G>
__global__ void __launch_bounds__(kThreads, G > 4 ? 3 : 4)
top_rows_block_kernel(RowArgs a) {
    constexpr int VE = Pack<T>::N;
    __shared__ Shared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.x / a.splits;
    const int part = blockIdx.x % a.splits;
    float m = PCX_NEG_INF, r = PCX_NEG_INF, s = 0.0f;
    int have = 0;
    bool skip = a.finished != nullptr && a.finished[row] != 0;
    if (a.scores != nullptr) skip |= !(a.scores[row] > PCX_NEG_INF);
    if (!skip) {
        const T* x = (const T*)a.logits + (row / a.inner) * a.stride0 + (row % a.inner) * a.stride1;
        // groups begin on 16-byte boundaries; the first and the last may reach over the row's ends
        const int off = (int)(((uintptr_t)x & 15) / sizeof(T));
        const int groups = (int)(((int64_t)off + a.vocab + VE - 1) / VE);
        const int per = (groups + a.splits - 1) / a.splits;
        const int g0 = part * per, g1 = min(groups, g0 + per);
        const int whole0 = off != 0 ? 1 : 0, whole1 = (off + a.vocab) / VE;
        float bound = PCX_NEG_INF;             // value of the last entry of a full list
        for (int g = g0; g < g1; g += kThreads * G) {
            uint4 v[G];
#pragma unroll
            for (int j = 0; j < G; ++j) v[j] = load_group<T>(x, g + j * kThreads + tid, off, whole0, min(g1, whole1), g1, a.vocab);
            float top = PCX_NEG_INF, group_top[G];
#pragma unroll
            for (int j = 0; j < G; ++j) {
                group_top[j] = Pack<T>::max(v[j]);
                top = fmaxf(top, group_top[j]);
            }
            if (top > m) {
                const float nr = top * a.scale;
                s = m > PCX_NEG_INF ? s * to_other(m, r, top, nr, a.scale) : 0.0f;
                m = top;
                r = nr;
            }
            if (m > PCX_NEG_INF) {
                float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
                for (int j = 0; j < G; j += 2) {
                    s0 += group_sum<T>(v[j], a.scale, r);
                    s1 += group_sum<T>(v[j + 1], a.scale, r);
                }
                s0 += s1;
                if (!(s0 < CUDART_INF_F) || !near(r))
                    s0 = careful_sum<T>(x, (g + tid) * VE - off, G, kThreads * VE, min(a.vocab, g1 * VE - off), m, r, a.scale);
                s += s0;
            }
            const int over = __syncthreads_count(top > bound);
            if (over == 0) continue;
            float least = PCX_NEG_INF;
            if (over > 2 * a.n) {
                // A lower bound of the tile's n-th largest logit: every warp's (n / warps)-th largest thread maximum, the
                // smallest of them (at least n threads hold one that large)
                uint32_t k = ordered(top);
#pragma unroll
                for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
                    for (int o = size >> 1; o; o >>= 1) {
                        const uint32_t other = __shfl_xor_sync(~0u, k, o);
                        const bool up = ((lane & size) == 0) == ((lane & o) == 0);       // larger first
                        k = up ? max(k, other) : min(k, other);
                    }
                if (lane == (a.n + kWarps - 1) / kWarps - 1) sh.warp_t[warp] = k;
                __syncthreads();
                uint32_t t = sh.warp_t[0];
#pragma unroll
                for (int w = 1; w < kWarps; ++w) t = min(t, sh.warp_t[w]);
                least = unordered(t);
            }
            // every logit that may be among the n largest so far, read again (its group is among the few that hold one);
            // `from`: a key below which none is wanted
            uint32_t hot = 0;
            if (top > bound && top >= least) {
#pragma unroll
                for (int j = 0; j < G; ++j) hot |= (uint32_t)(group_top[j] > bound && group_top[j] >= least) << j;
            }
            auto each = [&](u64 from, auto&& found) {
                for (uint32_t left = hot; left != 0; left &= left - 1) {
                    const int e = (g + (__ffs(left) - 1) * kThreads + tid) * VE - off;
                    const uint4 w = load_group<T>(x, g + (__ffs(left) - 1) * kThreads + tid, off, whole0, min(g1, whole1), g1, a.vocab);
#pragma unroll
                    for (int i = 0; i < VE; ++i) {
                        const float f = Pack<T>::at(w, i);
                        if (f > bound && f >= least) {
                            const u64 key = key_of(f, (uint32_t)(e + i));
                            if (key >= from) found(key);
                        }
                    }
                }
            };
            auto collect = [&](u64 from) {
                if (tid == 0) sh.count = have;
                __syncthreads();
                each(from, [&](u64 key) {
                    const int at = atomicAdd(&sh.count, 1);
                    if (at < kRoom + kMaxTop) sh.keys[at] = key;
                });
                __syncthreads();
                const int total = sh.count;
                __syncthreads();
                return total;
            };
            int total = collect(0);
            if (total > kRoom + kMaxTop) {
                // too many (ordered or equal logits): a key that n to kRoom of them reach
                u64 lo = 0, hi = ~0ull;
                while (lo < hi) {
                    const u64 mid = lo + ((hi - lo) >> 1) + ((hi - lo) & 1);
                    int c = 0;
                    each(mid, [&](u64) { ++c; });
                    c = block_sum(c, &sh.count);
                    if (c >= a.n) {
                        lo = mid;
                        if (c <= kRoom) break;
                    } else {
                        hi = mid - 1;
                    }
                }
                __syncthreads();
                total = collect(lo);
            }
            have = prune(sh, total, a.n);
            if (have == a.n) bound = value_of(sh.keys[a.n - 1]);
        }
    }
    // the lanes' and warps' sums become one in 64 bits
    float wm = m;
#pragma unroll
    for (int o = 16; o; o >>= 1) wm = fmaxf(wm, __shfl_xor_sync(~0u, wm, o));
    float M;
    double S;
    block_stats(sh, wm, warp_sum(to_own(s, m, r, wm, a.scale)), a.inv_t, M, S);
    leave<T>(a, sh, row, have, M, S);
}

// Waits for the kernel before this one in the stream (launch_next).  Nothing that it writes may be read through the read-only
// path, whose loads may be moved up over this.
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---- the join --------------------------------------------------------------------------------------------------------

// (5 us for 13 parts of 8 keys.)  The parts of a row become one: in place of the row's answer (top logits) or as its only part (beams).
template <typename T>
__global__ void __launch_bounds__(kThreads)
join_parts_kernel(RowArgs a, const u64* keys, const Part* parts) {
    __shared__ Shared sh;
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    if (tid == 0) sh.count = 0;
    __syncthreads();
    after_previous();
    float m = PCX_NEG_INF;
    double s = 0.0;
    if (tid < 32) {                                 // (kMaxSplits parts at most)
        if (tid < a.splits) { m = parts[row * a.splits + tid].m; s = parts[row * a.splits + tid].s; }
        float wm = m;
#pragma unroll
        for (int o = 16; o; o >>= 1) wm = fmaxf(wm, __shfl_xor_sync(~0u, wm, o));
        s = m > PCX_NEG_INF && wm < CUDART_INF_F ? s * exp(((double)m - (double)wm) * a.inv_t) : 0.0;
        s = warp_sum(s);
        m = wm;
    }
    for (int i = tid; i < a.splits * a.n; i += kThreads)
        if (i % a.n < parts[row * a.splits + i / a.n].count)
            sh.keys[atomicAdd(&sh.count, 1)] = keys[row * a.splits * a.n + i];
    __syncthreads();
    const int total = sh.count;
    __syncthreads();
    const int have = prune(sh, total, a.n);
    float M;
    double S;
    block_stats(sh, m, s, a.inv_t, M, S);
    leave<T>(a, sh, row, have, M, S);
}

struct BeamArgs {
    const u64* keys;               // [batch * beams][n]
    const Part* parts;             // [batch * beams]
    const float* scores;
    const uint8_t* finished;
    const void* logits;
    int64_t stride_batch, stride_beam;
    float* out_scores;
    int64_t *tokens, *parents;
    int beams, n, vocab, pad_id, normalize, dtype;
    double slack;                  // scores of different beams that are no further apart than this may be in the wrong order
};

constexpr int kBeamTile = 2048;                     // candidates looked at together
constexpr int kBehind = 4;                         // continuations that are kept behind the n best
struct BeamShared {
    u64 score[kBeamTile + kMaxTop];
    uint32_t place[kBeamTile + kMaxTop];            // beam * vocab + token: a lower one first among equal scores
    u64 list_s[kMaxTop + kBehind];
    uint32_t list_p[kMaxTop + kBehind];
    double norm[kMaxTop], red[kWarps];              // what a beam's logits are lowered by
    float own[kMaxTop];                             // its score
    uint8_t exact[kMaxTop], doubt[kMaxTop];
    int any_doubt;                                  // (the first CTA's word to the others of its cluster)
    uint32_t low[kWarps], high[kWarps];
    int count;
};

// Part `seg` of kSegments of sum exp(x - m) over a row, in 64 bits, to thread 0.  The order of the sum goes by the places alone: equal
// rows, wherever they lie, have equal bits.
constexpr int kSegments = 8;
template <int PER_SM, typename T>
__device__ __noinline__ double segment_sum(const T* x, int vocab, int seg, float m, double* red) {
    constexpr int AHEAD = 8;
    constexpr int64_t STEP = kSegments * kThreads;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    double s = 0.0;
    float next[AHEAD];
    int64_t e0 = (int64_t)seg * kThreads + threadIdx.x;
    auto fetch = [&]() {                            // (NaN counts nothing)
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) next[i] = fmaxf(e0 + i * STEP < vocab ? (float)x[e0 + i * STEP] : PCX_NEG_INF, PCX_NEG_INF);
        e0 += AHEAD * STEP;
    };
    fetch();
    for (int64_t left = (int64_t)vocab - seg * kThreads; left > 0; left -= AHEAD * STEP) {
        double t[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) t[i] = (double)next[i] - (double)m;
        fetch();
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) t[i] = exp(t[i]);
#pragma unroll
        for (int o = 1; o < AHEAD; o *= 2)
#pragma unroll
            for (int i = 0; i < AHEAD; i += 2 * o) t[i] += t[i + o];
        s += t[0];
    }
    s = warp_sum(s);
    __syncthreads();
    if (lane == 0) red[warp] = s;
    __syncthreads();
    s = 0.0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += red[w];
    return s;
}

// One CTA per sequence; 64 sequences of 16 lists of 32: 10 us, in which 512 candidates are bisected down to at most 64 before
// they are ranked (ranking them all: 65 us).
// The normalisers of the rows carry the error of their fp32 terms.  Where that leaves two continuations of different beams in
// doubt, among the n best or at their end, those beams' normalisers are taken again in 64 bits and the choice is made again.  Once is
// enough: a score moves by half the slack at most, so that only pairs within the slack can change places.  Few sequences have
// clusters of CTAs that share these sums; the first CTA does all the rest, for which the others wait.  64 sequences of 16 beams over
// 32768 tokens, a call: 43 us, 57 with two beams in doubt (one call in twelve of random rows), 155 with all (350 by one CTA a
// sequence).  What bounds the sums are fp64 instructions; with PER_SM = 2 they have the registers for eight exponentials at a time.
template <int PER_SM>
__global__ void __launch_bounds__(kThreads, PER_SM)
join_beams_kernel(BeamArgs a) {
    __shared__ BeamShared sh;
    namespace cg = cooperative_groups;
    const cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, ctas = cluster.num_blocks(), rank = cluster.block_rank();
    const int64_t sequence = blockIdx.x / ctas, first = sequence * a.beams;
    cluster.sync();                                 // (all CTAs have started: their shared memory may be written)
    after_previous();
    // the sums in doubt: kSegments for every beam, in the first CTA's `score`
    auto take_sums = [&]() {
        double* sums = (double*)cluster.map_shared_rank(sh.score, 0);
        for (int b = 0; b < a.beams; ++b) {
            if (!sh.doubt[b]) continue;
            const char* row = (const char*)a.logits + (sequence * a.stride_batch + b * a.stride_beam) * (a.dtype == 0 ? 4 : 2);
            const float m = a.parts[first + b].m;
            for (int seg = rank; seg < kSegments; seg += ctas) {
                const double s = a.dtype == 0 ? segment_sum<PER_SM>((const float*)row, a.vocab, seg, m, sh.red)
                    : a.dtype == 1 ? segment_sum<PER_SM>((const __nv_bfloat16*)row, a.vocab, seg, m, sh.red)
                                   : segment_sum<PER_SM>((const __half*)row, a.vocab, seg, m, sh.red);
                if (tid == 0) sums[b * kSegments + seg] = s;
            }
        }
        cluster.sync();
    };
    if (rank > 0) {
        cluster.sync();                             // (the first CTA says what is in doubt)
        if (sh.any_doubt) take_sums();
        return;
    }
    for (int b = tid; b < a.beams; b += kThreads) {
        const Part p = a.parts[first + b];
        const bool done = a.finished != nullptr && a.finished[first + b] != 0;
        sh.own[b] = a.scores[first + b];
        sh.norm[b] = a.normalize && !done ? log_norm(p.m, p.s, 1.0) : 0.0;
        sh.exact[b] = done || !a.normalize;
        sh.doubt[b] = 0;
    }
    __syncthreads();
    const int slots = a.beams * a.n;
    // The score of an entry of the lists, its place; not above -inf if there is none (NaN: a row without a normaliser)
    auto candidate = [&](int i, uint32_t& place) {
        const int b = i / a.n;
        if (i % a.n >= a.parts[first + b].count) return -CUDART_INF;
        const u64 k = a.keys[first * a.n + i];
        place = (uint32_t)b * a.vocab + place_of(k);
        return ((double)sh.own[b] + (double)value_of(k)) - sh.norm[b];
    };
    auto is_finished = [&](int b) { return a.finished != nullptr && a.finished[first + b] != 0 && sh.own[b] > PCX_NEG_INF; };
    // to the other CTAs, which wait for it at a barrier
    auto tell = [&](int doubt) {
        for (int r = 1; r < ctas; ++r) {
            BeamShared* other = cluster.map_shared_rank(&sh, r);
            if (tid == 0) other->any_doubt = doubt;
            if (doubt)
                for (int b = tid; b < a.beams; b += kThreads) other->doubt[b] = sh.doubt[b];
        }
    };
    bool any = false;                               // normalisers are taken again
    const int kept = a.n + kBehind;
    int have = 0;
    for (bool again = false;; again = true) {
        if (tid == 0) sh.count = 0;
        __syncthreads();
        for (int b = tid; b < a.beams; b += kThreads)
            if (is_finished(b)) {                   // a finished beam has one continuation, at its own score
                const int at = atomicAdd(&sh.count, 1);
                sh.score[at] = ordered((double)sh.own[b]);
                sh.place[at] = (uint32_t)b * a.vocab + a.pad_id;
            }
        __syncthreads();
        for (int at = 0; at < slots; at += kBeamTile - kMaxTop) {
            for (int i = tid; i < kBeamTile - kMaxTop && at + i < slots; i += kThreads) {
                uint32_t place;
                const double score = candidate(at + i, place);
                if (!(score > -CUDART_INF)) continue;
                const int to = atomicAdd(&sh.count, 1);
                sh.score[to] = ordered(score);
                sh.place[to] = place;
            }
            __syncthreads();
            int total = sh.count;
            __syncthreads();
            const int few = max(64, 2 * a.n);
            if (total > few) {
                u64 t, most;
                key_range(sh.score, total, sh.low, sh.high, t, most);
                t = bisect(total, kept, few, t, most, [&](int i, u64 mid) { return sh.score[i] >= mid; });
                __syncthreads();
                if (tid == 0) sh.count = 0;
                for (int i0 = 0; i0 < total; i0 += kThreads) {
                    const u64 own = i0 + tid < total ? sh.score[i0 + tid] : 0;
                    const uint32_t place = i0 + tid < total ? sh.place[i0 + tid] : 0;
                    __syncthreads();
                    if (own >= t && own != 0) {
                        const int to = atomicAdd(&sh.count, 1);
                        sh.score[to] = own;
                        sh.place[to] = place;
                    }
                }
                __syncthreads();
                total = sh.count;
            }
            for (int i = tid; i < total; i += kThreads) {
                const u64 s = sh.score[i];
                const uint32_t p = sh.place[i];
                int rank = 0;
#pragma unroll 4
                for (int j = 0; j < total; ++j) {
                    const u64 o = sh.score[j];
                    rank += (int)(o > s) | ((int)(o == s) & (int)(sh.place[j] < p));
                }
                if (rank < kept) { sh.list_s[rank] = s; sh.list_p[rank] = p; }
            }
            __syncthreads();
            have = min(total, kept);
            for (int i = tid; i < have; i += kThreads) { sh.score[i] = sh.list_s[i]; sh.place[i] = sh.list_p[i]; }
            if (tid == 0) sh.count = have;
            __syncthreads();
        }
        if (again || a.beams == 1 || !a.normalize) break;
        // pairs of one of the n best and any continuation behind it within the slack
        int seen = 0;                               // 1: such a pair; 2: they reach beyond what is kept
        for (int i = tid; i < min(have, a.n); i += kThreads) {
            const double score = unordered(sh.score[i]);
            int j = i + 1;
            for (; j < have && score - unordered(sh.score[j]) <= a.slack; ++j) {
                const int b = sh.place[i] / (uint32_t)a.vocab, c = sh.place[j] / (uint32_t)a.vocab;
                if (b == c) continue;
                sh.doubt[b] = sh.doubt[c] = 1;
                seen |= 1;
            }
            if (j == kept) seen |= 2;
        }
        if (!__syncthreads_or(seen)) break;
        if (__syncthreads_or(seen & 2)) {           // (rows of equal logits)
            const double least = unordered(sh.score[a.n - 1]) - a.slack;
            auto against = [&](double score, int b) {
                for (int i = 0; i < a.n; ++i) {
                    const int c = sh.place[i] / (uint32_t)a.vocab;
                    if (c != b && fabs(score - unordered(sh.score[i])) <= a.slack) sh.doubt[b] = sh.doubt[c] = 1;
                }
            };
            for (int b = tid; b < a.beams; b += kThreads)
                if (is_finished(b)) against((double)sh.own[b], b);
            for (int i = tid; i < slots; i += kThreads) {
                uint32_t place;
                const double score = candidate(i, place);
                if (score >= least) against(score, i / a.n);
            }
        }
        __syncthreads();
        any = __syncthreads_or(tid < a.beams && sh.doubt[tid] && !sh.exact[tid]);
        if (!any) break;
        for (int b = tid; b < a.beams; b += kThreads) sh.doubt[b] = sh.doubt[b] && !sh.exact[b];
        __syncthreads();
        tell(1);
        cluster.sync();
        take_sums();
        for (int b = tid; b < a.beams; b += kThreads)
            if (sh.doubt[b]) {
                double s = 0.0;
                for (int i = 0; i < kSegments; ++i) s += ((const double*)sh.score)[b * kSegments + i];
                sh.norm[b] = log_norm(a.parts[first + b].m, s, 1.0);
            }
        __syncthreads();
    }
    if (!any) {
        tell(0);
        cluster.sync();
    }
    for (int i = tid; i < a.n; i += kThreads) {
        const int64_t to = sequence * a.n + i;
        const bool is = i < have;
        const uint32_t p = is ? sh.place[i] : 0;
        a.tokens[to] = is ? (int64_t)(p % (uint32_t)a.vocab) : -1;
        a.parents[to] = is ? (int64_t)(p / (uint32_t)a.vocab) : 0;
        a.out_scores[to] = is ? (float)unordered(sh.score[i]) : PCX_NEG_INF;
    }
}

// How far a row's normaliser may be off (temperature 1), in steps of 2^-24 of its sum: an exponential of 2^-22 (4); its argument a, once
// rounded itself and by 0.23 through the scale, ln 2 |a| each, where a is at most max(3/4 b, b - 4) of b = log2(vocab) on average
// under the weights (their entropy, less what the largest term has for itself); 8 sums one after the other in a tile; for every
// further tile of a lane a sum, a product and its exponential (6), for the first a sum; 2 for what is left.
double norm_error(int vocab, int tiles) {
    const double bits = std::log2((double)vocab);
    return (4.0 + 0.7 * 1.23 * std::max(0.75 * bits, bits - 4.0) + 8.0 + 6.0 * (tiles - 1) + 3.0) * 5.9604644775390625e-8;
}

// ---- reordering of states --------------------------------------------------------------------------------------------
constexpr int kStates = 8;                          // tensors moved by one launch
constexpr int kMoveRows = 8, kMoveUnits = 8;        // outer rows, and units of a row, that a thread moves
struct Moved {
    const char* src;
    char* dst;
    int64_t outer, chunks, src_outer, src_beam;     // rows before the beams, units per beam, strides in bytes
    uint32_t first_block, column_blocks, segments;  // blocks: columns, then segments of a beam's units, then outer rows
    uint32_t lanes, unit;                           // threads side by side over a beam's units; bytes of a unit
};
struct MoveArgs {
    Moved t[kStates];
    const void* parents;
    int n_tensors, wide_ids;
    uint32_t beams, n, columns;                     // columns: batch * n
};

// dst[o, b * n + j, i] = src[o, b * beams + parents[b, j], i], in units of sizeof(U) bytes; zeros for a parent that is none
// of the sequence's beams.  A thread looks its parent up once for up to 8 outer rows and 8 units of each, all of which it
// has under way together; neighbours write neighbouring units.  4096 rows of 1024 beams, 4 bytes each: 12 us (2.8 TB/s read and
// written; 25 us with a parent looked up per unit).
template <typename U>
__device__ __forceinline__ void move(const MoveArgs& a, const Moved& t, uint32_t block) {
    const uint32_t c = block % t.column_blocks * (256 / t.lanes) + threadIdx.x / t.lanes;
    block /= t.column_blocks;
    if (c >= a.columns) return;
    const int64_t i0 = (int64_t)(block % t.segments) * (t.lanes * kMoveUnits) + threadIdx.x % t.lanes;
    const int64_t o0 = (int64_t)(block / t.segments) * kMoveRows;
    const int64_t p = a.wide_ids ? ((const int64_t*)a.parents)[c] : (int64_t)((const int32_t*)a.parents)[c];
    const bool is = p >= 0 && p < a.beams;
    const char* src = t.src + o0 * t.src_outer + ((int64_t)(c / a.n) * a.beams + (is ? p : 0)) * t.src_beam;
    const int64_t row = a.columns * t.chunks;
    U* dst = (U*)t.dst + o0 * row + c * t.chunks;
    const int rows = (int)min((int64_t)kMoveRows, t.outer - o0);
    if (t.chunks <= t.lanes) {                      // a unit a row
        if (i0 >= t.chunks) return;
        U u[kMoveRows] = {};
#pragma unroll
        for (int r = 0; r < kMoveRows; ++r)
            if (r < rows && is) u[r] = ((const U*)(src + r * t.src_outer))[i0];
#pragma unroll
        for (int r = 0; r < kMoveRows; ++r)
            if (r < rows) dst[r * row + i0] = u[r];
        return;
    }
    for (int r = 0; r < rows; ++r) {
        U u[kMoveUnits] = {};
#pragma unroll
        for (int k = 0; k < kMoveUnits; ++k)
            if (i0 + k * t.lanes < t.chunks && is) u[k] = ((const U*)(src + r * t.src_outer))[i0 + k * t.lanes];
#pragma unroll
        for (int k = 0; k < kMoveUnits; ++k)
            if (i0 + k * t.lanes < t.chunks) dst[r * row + i0 + k * t.lanes] = u[k];
    }
}

__global__ void __launch_bounds__(256) reorder_kernel(MoveArgs a) {
    int w = 0;
    while (w + 1 < a.n_tensors && blockIdx.x >= a.t[w + 1].first_block) ++w;
    const Moved& t = a.t[w];
    const uint32_t block = blockIdx.x - t.first_block;
    switch (t.unit) {
        case 16: move<uint4>(a, t, block); break;
        case 8: move<uint2>(a, t, block); break;
        case 4: move<uint32_t>(a, t, block); break;
        case 2: move<uint16_t>(a, t, block); break;
        default: move<uint8_t>(a, t, block);
    }
}

// A kernel of `grid` blocks whose start overlaps the end of the one before it in the stream (it waits for that one's results
// itself, after_previous).  64 sequences of 16 beams, three launches: 44.8 -> 42 us a call.
template <typename... P, typename... A>
cudaError_t launch_next(void (*kernel)(P...), unsigned grid, unsigned cluster, cudaStream_t stream, A... args) {
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid); cfg.blockDim = dim3(kThreads); cfg.stream = stream; cfg.attrs = attr; cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

// Groups a thread of a CTA that takes a part of a row, per tile
int block_groups(int vocab, int ve, int splits) { return vocab / ve / splits > 3 * kThreads ? 8 : 2; }

template <typename T>
void launch_rows(const RowArgs& a, int64_t rows, bool warps, cudaStream_t stream) {
    if (warps) {
        top_rows_warp_kernel<T><<<(unsigned)pcx_cdiv(rows, kRowWarps), kRowWarps * 32, 0, stream>>>(a, rows);
        return;
    }
    const unsigned grid = (unsigned)(rows * a.splits);
    if (block_groups(a.vocab, Pack<T>::N, a.splits) == 8) top_rows_block_kernel<T, 8><<<grid, kThreads, 0, stream>>>(a);
    else top_rows_block_kernel<T, 2><<<grid, kThreads, 0, stream>>>(a);
}

// The lists of all rows, one part each when this returns: in the answer's place, or in `keys` and `parts`.
template <typename T>
int select_rows(RowArgs a, void* scratch, int64_t rows, cudaStream_t stream) {
    const bool warps = a.splits == 0;
    if (warps) a.splits = 1;
    const int64_t lists = rows * a.splits;
    u64* keys = (u64*)scratch;
    Part* parts = (Part*)(keys + lists * a.n);
    u64* joined_keys = (u64*)(parts + lists);
    Part* joined_parts = (Part*)(joined_keys + rows * a.n);
    RowArgs rows_args = a;
    rows_args.keys = keys;
    rows_args.parts = parts;
    if (a.splits == 1) {
        if (a.ids == nullptr) { rows_args.keys = joined_keys; rows_args.parts = joined_parts; }
        launch_rows<T>(rows_args, rows, warps, stream);
        PCX_LAUNCH_CHECK();
        return 0;
    }
    rows_args.ids = nullptr;
    launch_rows<T>(rows_args, rows, warps, stream);
    PCX_LAUNCH_CHECK();
    a.keys = joined_keys;
    a.parts = joined_parts;
    return (int)launch_next(join_parts_kernel<T>, (unsigned)rows, 1, stream, a, keys, parts);
}
int select_rows(const RowArgs& a, int dtype, void* scratch, int64_t rows, cudaStream_t stream) {
    switch (dtype) {
        case 0: return select_rows<float>(a, scratch, rows, stream);
        case 1: return select_rows<__nv_bfloat16>(a, scratch, rows, stream);
        case 2: return select_rows<__half>(a, scratch, rows, stream);
        default: return -1;
    }
}

}  // namespace

extern "C" {

int pcx_top_logits(int64_t* ids, void* values, float* norms, void* scratch, const void* logits, int dtype, int64_t rows,
                   int vocab, int64_t row_stride, int n, int splits, double temperature, void* stream) {
    if (rows <= 0 || n <= 0) return 0;
    if (n > kMaxTop || vocab <= 0 || splits < 0 || splits > kMaxSplits || rows * std::max(splits, 1) > 0x7fffffff) return -1;
    RowArgs a{};
    a.logits = logits;
    a.stride1 = row_stride;
    a.inner = 0x7fffffff;
    a.vocab = vocab; a.n = n; a.splits = splits;
    a.inv_t = 1.0 / temperature;
    a.scale = (float)(1.4426950408889634 / temperature);
    a.ids = ids; a.values = values; a.norms = norms;
    return select_rows(a, dtype, scratch, rows, (cudaStream_t)stream);
}

int pcx_beam_select(float* out_scores, int64_t* parents, int64_t* tokens, void* scratch, const void* logits, int dtype,
                    const float* scores, const uint8_t* finished, int64_t batch, int beams, int vocab, int64_t stride_batch,
                    int64_t stride_beam, int n, int pad_id, int normalize, int splits, void* stream) {
    if (batch <= 0 || n <= 0) return 0;
    const int64_t rows = batch * beams;
    if (n > kMaxTop || vocab <= 0 || beams <= 0 || beams > kMaxTop || splits < 0 || splits > kMaxSplits ||
        (int64_t)beams * vocab > 0x7fffffff || rows * std::max(splits, 1) > 0x7fffffff)
        return -1;
    RowArgs a{};
    a.logits = logits; a.scores = scores; a.finished = finished;
    a.stride0 = stride_batch; a.stride1 = stride_beam;
    a.inner = beams; a.vocab = vocab; a.n = n; a.splits = splits;
    a.inv_t = 1.0;
    a.scale = 1.4426950408889634f;
    const int rc = select_rows(a, dtype, scratch, rows, (cudaStream_t)stream);
    if (rc != 0) return rc;
    const int ve = dtype == 0 ? 4 : 8, parts = std::max(splits, 1);
    const int64_t in_tile = splits == 0 ? 32 * kGroups : kThreads * block_groups(vocab, ve, splits);
    BeamArgs j{};
    j.keys = (const u64*)((const char*)scratch + rows * std::max(splits, 1) * ((int64_t)n * 8 + (int64_t)sizeof(Part)));
    j.parts = (const Part*)(j.keys + rows * n);
    j.scores = scores; j.finished = finished;
    j.out_scores = out_scores; j.tokens = tokens; j.parents = parents;
    j.logits = logits; j.stride_batch = stride_batch; j.stride_beam = stride_beam; j.dtype = dtype;
    j.beams = beams; j.n = n; j.vocab = vocab; j.pad_id = pad_id; j.normalize = normalize;
    j.slack = 2.0 * norm_error(vocab, (int)pcx_cdiv(pcx_cdiv(vocab / ve + 2, parts), in_tile));
    // CTAs a sequence: they share the sums that are taken again, and only wait otherwise: two an SM at most.  Many sequences are done
    // sooner where more CTAs fit an SM (512 of 8 beams over 4096 tokens: 26.8 us a call against 29.4)
    unsigned ctas = 1;
    while (ctas < kSegments && normalize && beams > 1 && batch * ctas * 2 <= 148 * 2) ctas *= 2;
    if (ctas == 1) return (int)launch_next(join_beams_kernel<4>, (unsigned)batch, 1, (cudaStream_t)stream, j);
    return (int)launch_next(join_beams_kernel<2>, (unsigned)batch * ctas, ctas, (cudaStream_t)stream, j);
}

// `states`: n_tensors times (source, destination, outer rows, bytes per beam, source strides in bytes of outer rows and
// beams, unit), host memory.
int pcx_reorder(const int64_t* states, int n_tensors, const void* parents, int wide_ids, int64_t batch, int beams, int n,
                void* stream) {
    if (n_tensors <= 0 || batch <= 0 || n <= 0) return 0;
    if (n_tensors > kStates || beams <= 0 || batch * n > 0x7fffffff) return -1;
    MoveArgs a{};
    a.parents = parents;
    a.wide_ids = wide_ids; a.beams = (uint32_t)beams; a.n = (uint32_t)n; a.columns = (uint32_t)(batch * n);
    int64_t blocks = 0;
    for (int i = 0; i < n_tensors; ++i) {
        const int64_t* s = states + 7 * i;
        const int64_t unit = s[6];
        if ((unit != 1 && unit != 2 && unit != 4 && unit != 8 && unit != 16) || s[3] % unit != 0) return -1;
        const int64_t chunks = s[3] / unit;
        if (s[2] == 0 || chunks == 0) continue;
        int lanes = 1;
        while (lanes < 256 && lanes < chunks) lanes *= 2;
        const int64_t column_blocks = pcx_cdiv((int64_t)a.columns, 256 / lanes), segments = pcx_cdiv(chunks, (int64_t)lanes * kMoveUnits);
        const int64_t more = column_blocks * segments * pcx_cdiv(s[2], kMoveRows);
        if (segments > 0x7fffffff || more > 0x7fffffff - blocks) return -1;
        a.t[a.n_tensors++] = Moved{(const char*)s[0], (char*)s[1], s[2], chunks, s[4], s[5], (uint32_t)blocks, (uint32_t)column_blocks,
                                   (uint32_t)segments, (uint32_t)lanes, (uint32_t)unit};
        blocks += more;
    }
    if (blocks == 0) return 0;
    if (blocks > 0x7fffffff) return -1;
    reorder_kernel<<<(unsigned)blocks, 256, 0, (cudaStream_t)stream>>>(a);
    PCX_LAUNCH_CHECK();
    return 0;
}

}  // extern "C"
