// Selection over a vocabulary: the largest logits of every row with the row's log-normaliser, and the best continuations of
// beams.  The language-model side of the circuits: a teacher's top logits to learn from, beam search to answer with.
//
// One pass over the logits.  A CTA walks a part of a row in tiles that stay in registers; its threads carry the running
// maximum m and sum s = sum exp((x - m) / T) of a softmax, and the CTA keeps the n largest logits seen so far, sorted, in
// shared memory.  Once that list is full its smallest entry is a threshold that few later logits pass, so that a tile
// costs one comparison per thread and a barrier.  Places are part of the keys (a lower place first among equals): keys are
// unique, and the answer does not depend on how rows are split over CTAs or in which order threads append.
// A row takes as many CTAs as are needed to fill the device; the lists and the (m, s) of the parts are joined by a second
// kernel, one CTA per answer, which for beams also adds the scores, in 64 bits: a sum of a score and a logit is rounded
// only in the returned score, never before it is compared.
#include "pcx_common.cuh"
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <algorithm>

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kTile = kThreads * 16;     // logits of a tile: 16 per thread
constexpr int kMaxTop = 128;                                                      // entries of a list
constexpr int kFew = 512;                                                         // candidates ranked by counting at once

typedef unsigned long long u64;

// What a CTA leaves for the join: the sorted keys of its list, then the maximum and the sum of its part.
struct Part { float m; int count; double s; };

template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32(float x) { return x; }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }

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
    u64 keys[kTile + kMaxTop];     // the list (sorted, first), behind it the candidates of a tile
    u64 list[kMaxTop];
    float red_m[kWarps];
    double red_s[kWarps];
    uint32_t warp_t[kWarps];
    int count;
};

// Keeps the n largest of the `total` unique keys in sh.keys, sorted, at its front.  Returns how many there are.
__device__ int prune(Shared& sh, int total, int n) {
    const int tid = threadIdx.x;
    if (total > kFew) {
        // bisect over the key's bits until no more than kFew keys (and at least n) are above the threshold
        u64 lo = 0, hi = ~0ull;
        while (true) {
            const u64 mid = lo + ((hi - lo) >> 1) + ((hi - lo) & 1);
            int mine = 0;
            for (int i = tid; i < total; i += kThreads) mine += sh.keys[i] >= mid;
            for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(~0u, mine, o);
            if (tid == 0) sh.count = 0;
            __syncthreads();
            if ((tid & 31) == 0) atomicAdd(&sh.count, mine);
            __syncthreads();
            const int c = sh.count;
            __syncthreads();
            if (c >= n) { lo = mid; if (c <= kFew) break; }
            else hi = mid - 1;
            if (lo >= hi) break;
        }
        // compaction through registers: a thread's keys are read before any is overwritten
        u64 own[(kTile + kMaxTop + kThreads - 1) / kThreads];
#pragma unroll
        for (int j = 0; j < (kTile + kMaxTop + kThreads - 1) / kThreads; ++j) {
            const int i = tid + j * kThreads;
            own[j] = i < total ? sh.keys[i] : 0;
        }
        if (tid == 0) sh.count = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < (kTile + kMaxTop + kThreads - 1) / kThreads; ++j)
            if (own[j] != 0 && own[j] >= lo) sh.keys[atomicAdd(&sh.count, 1)] = own[j];
        __syncthreads();
        total = sh.count;
        __syncthreads();
    }
    const int kept = min(total, n);
    for (int i = tid; i < total; i += kThreads) {
        const u64 k = sh.keys[i];
        int rank = 0;
        for (int j = 0; j < total; ++j) rank += sh.keys[j] > k;
        if (rank < n) sh.list[rank] = k;
    }
    __syncthreads();
    for (int i = tid; i < kept; i += kThreads) sh.keys[i] = sh.list[i];
    __syncthreads();
    return kept;
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
top_rows_kernel(RowArgs a) {
    constexpr int VE = 16 / (int)sizeof(T), G = 16 / VE;
    __shared__ Shared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.x / a.splits;
    const int part = blockIdx.x % a.splits;
    float m = PCX_NEG_INF, s = 0.0f;
    int have = 0;
    bool skip = a.finished != nullptr && a.finished[row] != 0;
    if (a.scores != nullptr) skip |= !(a.scores[row] > PCX_NEG_INF);
    if (!skip) {
        const T* x = (const T*)a.logits + (row / a.inner) * a.stride0 + (row % a.inner) * a.stride1;
        // groups of 16 bytes that begin on 16-byte boundaries; the first and the last may reach over the row's ends
        const int off = (int)(((uintptr_t)x & 15) / sizeof(T));
        const int groups = (int)(((int64_t)off + a.vocab + VE - 1) / VE);
        const int per = (groups + a.splits - 1) / a.splits;
        const int g0 = part * per, g1 = min(groups, g0 + per);
        float bound = PCX_NEG_INF;             // value of the last entry of a full list
        for (int g = g0; g < g1; g += kThreads * G) {
            T v[G][VE];
#pragma unroll
            for (int j = 0; j < G; ++j) {
                const int gi = g + j * kThreads + tid;
                const int e = gi * VE - off;
                if (gi < g1 && e >= 0 && e + VE <= a.vocab) {
                    *(uint4*)v[j] = __ldg((const uint4*)(x + e));
                } else {
#pragma unroll
                    for (int i = 0; i < VE; ++i)
                        v[j][i] = gi < g1 && e + i >= 0 && e + i < a.vocab ? x[e + i] : (T)PCX_NEG_INF;
                }
            }
            float top = PCX_NEG_INF;
#pragma unroll
            for (int j = 0; j < G; ++j)
#pragma unroll
                for (int i = 0; i < VE; ++i) top = fmaxf(top, to_f32(v[j][i]));       // (skips NaN)
            if (top > m) {
                s *= exp2f((m - top) * a.scale);
                m = top;
            }
            if (m > PCX_NEG_INF) {
#pragma unroll
                for (int j = 0; j < G; ++j)
#pragma unroll
                    for (int i = 0; i < VE; ++i)
                        s += exp2f((fmaxf(to_f32(v[j][i]), PCX_NEG_INF) - m) * a.scale);
            }
            if (!__syncthreads_or(top > bound)) continue;
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
            const int nth = (a.n + kWarps - 1) / kWarps - 1;
            if (lane == nth) sh.warp_t[warp] = k;
            if (tid == 0) sh.count = have;
            __syncthreads();
            uint32_t t = sh.warp_t[0];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) t = min(t, sh.warp_t[w]);
            const float least = unordered(t);
            if (top > bound && top >= least) {
#pragma unroll
                for (int j = 0; j < G; ++j)
#pragma unroll
                    for (int i = 0; i < VE; ++i) {
                        const float f = to_f32(v[j][i]);
                        if (f > bound && f >= least)
                            sh.keys[atomicAdd(&sh.count, 1)] =
                                key_of(f, (uint32_t)((g + j * kThreads + tid) * VE - off + i));
                    }
            }
            __syncthreads();
            const int total = sh.count;
            __syncthreads();
            have = prune(sh, total, a.n);
            if (have == a.n) bound = unordered((uint32_t)(sh.keys[a.n - 1] >> 32));
        }
    }
    // the part's maximum and sum
    float M = m;
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(~0u, M, o));
    if (lane == 0) sh.red_m[warp] = M;
    __syncthreads();
    M = sh.red_m[0];
    for (int w = 1; w < kWarps; ++w) M = fmaxf(M, sh.red_m[w]);
    double S = m > PCX_NEG_INF && M < CUDART_INF_F ? (double)s * exp((double)(m - M) * a.inv_t) : 0.0;
    for (int o = 16; o; o >>= 1) S += __shfl_xor_sync(~0u, S, o);
    if (lane == 0) sh.red_s[warp] = S;
    __syncthreads();
    if (a.ids != nullptr) {
        if (tid == 0 && a.norms != nullptr) {
            S = 0.0;
            for (int w = 0; w < kWarps; ++w) S += sh.red_s[w];
            a.norms[row] = (float)log_norm(M, S, a.inv_t);
        }
        for (int i = tid; i < a.n; i += kThreads) {
            const u64 k = i < have ? sh.keys[i] : 0;
            a.ids[row * a.n + i] = i < have ? (int64_t)(uint32_t)~(uint32_t)k : -1;
            ((T*)a.values)[row * a.n + i] = i < have ? (T)unordered((uint32_t)(k >> 32)) : (T)PCX_NEG_INF;
        }
        return;
    }
    if (tid == 0) {
        S = 0.0;
        for (int w = 0; w < kWarps; ++w) S += sh.red_s[w];
        a.parts[blockIdx.x] = Part{M, have, S};
    }
    for (int i = tid; i < have; i += kThreads) a.keys[(int64_t)blockIdx.x * a.n + i] = sh.keys[i];
}

// ---- the join --------------------------------------------------------------------------------------------------------

struct JoinArgs {
    const u64* keys;
    const Part* parts;
    const float* scores;           // null: logits themselves are compared (top logits)
    const uint8_t* finished;
    float* out_scores;             // beams
    int64_t* ids;                  // beams: tokens
    int64_t* parents;              // beams
    void* values;                  // top logits, in their type
    float* norms;                  // top logits
    int rows, splits, n, vocab, pad_id, normalize, elsize;       // rows: beams of an answer
    double inv_t;
};

constexpr int kJoinTile = 2048;                     // candidates looked at together
struct JoinShared {
    u64 score[kJoinTile + kMaxTop];
    uint32_t place[kJoinTile + kMaxTop];            // beam * vocab + token: a lower one first among equal scores
    u64 list_s[kMaxTop];
    uint32_t list_p[kMaxTop];
    int count;
};

__device__ __forceinline__ void store_value(void* out, int elsize, int64_t i, float x) {
    if (elsize == 4) ((float*)out)[i] = x;
    else if (elsize == 2) ((__nv_bfloat16*)out)[i] = __float2bfloat16(x);
    else ((__half*)out)[i] = __float2half(x);       // elsize 3 stands for fp16
}

__global__ void __launch_bounds__(kThreads)
join_kernel(JoinArgs a) {
    __shared__ JoinShared sh;
    extern __shared__ double base[];                // [rows] what a row's logits are raised by
    const int tid = threadIdx.x;
    const int64_t first = (int64_t)blockIdx.x * a.rows;
    for (int r = tid; r < a.rows; r += kThreads) {
        const Part* p = a.parts + (first + r) * a.splits;
        float M = PCX_NEG_INF;
        for (int i = 0; i < a.splits; ++i) M = fmaxf(M, p[i].m);
        double S = 0.0;
        for (int i = 0; i < a.splits; ++i)
            if (p[i].m > PCX_NEG_INF && M < CUDART_INF_F) S += p[i].s * exp((double)(p[i].m - M) * a.inv_t);
        const double norm = log_norm(M, S, a.inv_t);
        if (a.norms != nullptr) a.norms[first + r] = (float)norm;
        base[r] = a.scores == nullptr ? 0.0 : (double)a.scores[first + r] - (a.normalize ? norm : 0.0);
    }
    if (tid == 0) sh.count = 0;
    __syncthreads();
    const int64_t slots = (int64_t)a.rows * a.splits * a.n;
    int have = 0;
    if (a.finished != nullptr) {                    // a finished beam has one continuation, at its own score
        for (int r = tid; r < a.rows; r += kThreads)
            if (a.finished[first + r] != 0) {
                const float sc = a.scores[first + r];
                if (sc > PCX_NEG_INF) {
                    const int at = atomicAdd(&sh.count, 1);
                    sh.score[at] = ordered((double)sc);
                    sh.place[at] = (uint32_t)r * a.vocab + a.pad_id;
                }
            }
        __syncthreads();
    }
    for (int64_t at = 0; at < slots || at == 0; at += kJoinTile - kMaxTop) {
        for (int i = tid; i < kJoinTile - kMaxTop; i += kThreads) {
            const int64_t slot = at + i;
            if (slot >= slots) continue;
            const int list = (int)(slot / a.n), entry = (int)(slot % a.n);
            if (entry >= a.parts[first * a.splits + list].count) continue;
            const u64 k = a.keys[(first * a.splits + list) * a.n + entry];
            const int r = list / a.splits;
            const double score = base[r] + (double)unordered((uint32_t)(k >> 32));
            if (!(score > -CUDART_INF)) continue;   // NaN: a row without a normaliser
            const int to = atomicAdd(&sh.count, 1);
            sh.score[to] = ordered(score);
            sh.place[to] = (uint32_t)r * a.vocab + ~(uint32_t)k;
        }
        __syncthreads();
        const int total = sh.count;
        for (int i = tid; i < total; i += kThreads) {
            const u64 s = sh.score[i];
            const uint32_t p = sh.place[i];
            int rank = 0;
            for (int j = 0; j < total; ++j) {
                const u64 o = sh.score[j];
                rank += o > s || (o == s && sh.place[j] < p);
            }
            if (rank < a.n) { sh.list_s[rank] = s; sh.list_p[rank] = p; }
        }
        __syncthreads();
        have = min(total, a.n);
        for (int i = tid; i < have; i += kThreads) { sh.score[i] = sh.list_s[i]; sh.place[i] = sh.list_p[i]; }
        if (tid == 0) sh.count = have;
        __syncthreads();
    }
    for (int i = tid; i < a.n; i += kThreads) {
        const int64_t to = (int64_t)blockIdx.x * a.n + i;
        const bool is = i < have;
        const uint32_t p = is ? sh.place[i] : 0;
        if (a.parents == nullptr) {
            a.ids[to] = is ? (int64_t)p : -1;
            store_value(a.values, a.elsize, to, is ? (float)unordered(sh.score[i]) : PCX_NEG_INF);
        } else {
            a.ids[to] = is ? (int64_t)(p % (uint32_t)a.vocab) : -1;
            a.parents[to] = is ? (int64_t)(p / (uint32_t)a.vocab) : 0;
            a.out_scores[to] = is ? (float)unordered(sh.score[i]) : PCX_NEG_INF;
        }
    }
}

// ---- reordering of states --------------------------------------------------------------------------------------------
constexpr int kStates = 8;                          // tensors moved by one launch
struct Moved {
    const char* src;
    char* dst;
    int64_t outer, chunks, src_outer, src_beam;     // rows before the beams, units per beam, strides in bytes
    int64_t first_block;
};
struct MoveArgs {
    Moved t[kStates];
    const void* parents;
    int n_tensors, wide_ids, beams, n;
    int64_t columns;                                // batch * n
};

// dst[o, b * n + j, i] = src[o, b * beams + parents[b, j], i], in units of sizeof(U) bytes; zeros for a parent that is none
// of the sequence's beams.  A thread moves one unit; neighbours write neighbouring units.
template <typename U>
__global__ void __launch_bounds__(256) reorder_kernel(MoveArgs a) {
    int w = 0;
    while (w + 1 < a.n_tensors && (int64_t)blockIdx.x >= a.t[w + 1].first_block) ++w;
    const Moved& t = a.t[w];
    const int64_t at = ((int64_t)blockIdx.x - t.first_block) * 256 + threadIdx.x;
    if (at >= t.outer * a.columns * t.chunks) return;
    const int64_t i = at % t.chunks, r = at / t.chunks;
    const int64_t c = r % a.columns, o = r / a.columns;
    const int64_t p = a.wide_ids ? ((const int64_t*)a.parents)[c] : (int64_t)((const int32_t*)a.parents)[c];
    U u = {};
    if (p >= 0 && p < a.beams)
        u = *(const U*)(t.src + o * t.src_outer + (c / a.n * a.beams + p) * t.src_beam + i * (int64_t)sizeof(U));
    ((U*)t.dst)[at] = u;
}

int sm_count() {
    static int counts[64] = {};
    int d = 0;
    if (cudaGetDevice(&d) != cudaSuccess || d < 0 || d >= 64) return 148;
    if (counts[d] == 0 && cudaDeviceGetAttribute(&counts[d], cudaDevAttrMultiProcessorCount, d) != cudaSuccess) counts[d] = 148;
    return counts[d];
}

int launch_rows(const RowArgs& a, int dtype, int64_t rows, cudaStream_t stream) {
    const unsigned grid = (unsigned)(rows * a.splits);
    switch (dtype) {
        case 0: top_rows_kernel<float><<<grid, kThreads, 0, stream>>>(a); break;
        case 1: top_rows_kernel<__nv_bfloat16><<<grid, kThreads, 0, stream>>>(a); break;
        case 2: top_rows_kernel<__half><<<grid, kThreads, 0, stream>>>(a); break;
        default: return -1;
    }
    PCX_LAUNCH_CHECK();
    return 0;
}

}  // namespace

extern "C" {

// CTAs per row: enough to give every SM four, none of less than one tile.
int pcx_vocab_splits(int64_t rows, int64_t vocab) {
    if (rows <= 0 || vocab <= 0) return 1;
    const int64_t want = pcx_cdiv((int64_t)sm_count() * 4, rows);
    return (int)std::max<int64_t>(1, std::min<int64_t>(want, pcx_cdiv(vocab, kTile)));
}

int64_t pcx_vocab_scratch_bytes(int64_t rows, int splits, int n) {
    return rows * splits * ((int64_t)n * 8 + (int64_t)sizeof(Part));
}

int pcx_top_logits(int64_t* ids, void* values, float* norms, void* scratch, const void* logits, int dtype, int64_t rows,
                   int vocab, int64_t row_stride, int n, int splits, double temperature, void* stream) {
    if (rows <= 0 || n <= 0) return 0;
    if (n > kMaxTop || vocab <= 0 || splits < 1 || rows * splits > 0x7fffffff) return -1;
    RowArgs a{};
    a.logits = logits;
    a.stride0 = 0;
    a.stride1 = row_stride;
    a.inner = 0x7fffffff;
    a.vocab = vocab; a.n = n; a.splits = splits;
    a.inv_t = 1.0 / temperature;
    a.scale = (float)(1.4426950408889634 / temperature);
    if (splits == 1) { a.ids = ids; a.values = values; a.norms = norms; }
    a.keys = (u64*)scratch;
    a.parts = (Part*)((char*)scratch + rows * splits * n * 8);
    const int rc = launch_rows(a, dtype, rows, (cudaStream_t)stream);
    if (rc != 0 || splits == 1) return rc;
    JoinArgs j{};
    j.keys = a.keys; j.parts = a.parts;
    j.ids = ids; j.values = values; j.norms = norms;
    j.rows = 1; j.splits = splits; j.n = n; j.vocab = vocab; j.inv_t = a.inv_t;
    j.elsize = dtype == 0 ? 4 : dtype == 1 ? 2 : 3;
    join_kernel<<<(unsigned)rows, kThreads, 8, (cudaStream_t)stream>>>(j);
    PCX_LAUNCH_CHECK();
    return 0;
}

int pcx_beam_select(float* out_scores, int64_t* parents, int64_t* tokens, void* scratch, const void* logits, int dtype,
                    const float* scores, const uint8_t* finished, int64_t batch, int beams, int vocab, int64_t stride_batch,
                    int64_t stride_beam, int n, int pad_id, int normalize, int splits, void* stream) {
    if (batch <= 0 || n <= 0) return 0;
    if (n > kMaxTop || vocab <= 0 || beams <= 0 || beams > kMaxTop || splits < 1 || (int64_t)beams * vocab > 0x7fffffff ||
        batch * beams * splits > 0x7fffffff)
        return -1;
    RowArgs a{};
    a.logits = logits; a.scores = scores; a.finished = finished;
    a.stride0 = stride_batch; a.stride1 = stride_beam;
    a.inner = beams; a.vocab = vocab; a.n = n; a.splits = splits;
    a.inv_t = 1.0;
    a.scale = 1.4426950408889634f;
    const int64_t rows = batch * beams;
    a.keys = (u64*)scratch;
    a.parts = (Part*)((char*)scratch + rows * splits * a.n * 8);
    const int rc = launch_rows(a, dtype, rows, (cudaStream_t)stream);
    if (rc != 0) return rc;
    JoinArgs j{};
    j.keys = a.keys; j.parts = a.parts; j.scores = scores; j.finished = finished;
    j.out_scores = out_scores; j.ids = tokens; j.parents = parents;
    j.rows = beams; j.splits = splits; j.n = n; j.vocab = vocab; j.pad_id = pad_id; j.normalize = normalize; j.inv_t = 1.0;
    join_kernel<<<(unsigned)batch, kThreads, beams * 8, (cudaStream_t)stream>>>(j);
    PCX_LAUNCH_CHECK();
    return 0;
}

// `states`: n_tensors times (source, destination, outer rows, bytes per beam, source strides in bytes of outer rows and
// beams), host memory.
int pcx_reorder(const int64_t* states, int n_tensors, const void* parents, int wide_ids, int64_t batch, int beams, int n,
                int unit, void* stream) {
    if (n_tensors <= 0 || batch <= 0 || n <= 0) return 0;
    if (n_tensors > kStates || beams <= 0) return -1;
    MoveArgs a{};
    a.parents = parents;
    a.wide_ids = wide_ids; a.beams = beams; a.n = n; a.columns = batch * n;
    int64_t blocks = 0;
    for (int i = 0; i < n_tensors; ++i) {
        const int64_t* s = states + 6 * i;
        if (s[3] % unit != 0) return -1;
        a.t[a.n_tensors] = Moved{(const char*)s[0], (char*)s[1], s[2], s[3] / unit, s[4], s[5], blocks};
        const int64_t units = s[2] * a.columns * (s[3] / unit);
        if (units == 0) continue;
        a.n_tensors += 1;
        blocks += pcx_cdiv(units, 256);
    }
    if (blocks == 0) return 0;
    if (blocks > 0x7fffffff) return -1;
    cudaStream_t st = (cudaStream_t)stream;
    switch (unit) {
        case 16: reorder_kernel<uint4><<<(unsigned)blocks, 256, 0, st>>>(a); break;
        case 8: reorder_kernel<uint2><<<(unsigned)blocks, 256, 0, st>>>(a); break;
        case 4: reorder_kernel<uint32_t><<<(unsigned)blocks, 256, 0, st>>>(a); break;
        case 2: reorder_kernel<uint16_t><<<(unsigned)blocks, 256, 0, st>>>(a); break;
        case 1: reorder_kernel<uint8_t><<<(unsigned)blocks, 256, 0, st>>>(a); break;
        default: return -1;
    }
    PCX_LAUNCH_CHECK();
    return 0;
}

}  // extern "C"
