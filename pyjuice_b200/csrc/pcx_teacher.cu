// Leaf tables under a teacher's top logits.
//
//   forward    out[m, b]    = sum_k q[b, k] log p_m(id[b, k])          for every leaf vector (table) and position
//   backward   F_m(c)       = sum_{b, k: id[b, k] = c} q[b, k] g[m, b]  for every category c of the table
//
// with weights q[b, k] = softmax of the teacher's logits over the slots of a position.  A product of a table with a matrix of
// K entries per column, and of its transpose.  Both move 4 bytes per (slot, node): what bounds them is how those reach the
// SM, so that the nodes of one category lie side by side wherever a table is read often (in shared memory for a table of
// one position, in a transposed copy for a table that many positions share).  The backward pass sorts the slots by category
// first; a category's sum then has one owner and one order, whatever the schedule, and every flow is written once.
#include "pcx_common.cuh"
#include "../../include/pcx_b200.h"
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <algorithm>

namespace {

constexpr int kTh = 256, kW = kTh / 32;

// A leaf vector: M nodes over categories [0, C) of variable `var`, values in rows row0 ... of the value buffers.
struct Seg {
    int32_t var, M, C, col;        // col: its first column in a transposed table
    int64_t row0, table;           // table: its first parameter, [M][C]
    int64_t gcol;                  // its place in the turned flows: gcol * W + b * pad4(M) + m
};
// The vectors that share one table, in the order of the variables of `set`.
struct Grp {
    int32_t set, M, C, col;
    int64_t out, gbase;
};
// Tables of a circuit, or (segs null) `T` positions of M nodes, with one table for all (tied) or one each.
struct Geo {
    const Seg* segs;
    const Grp* grps;
    const int32_t* set_first;      // [n_sets + 1] into set_vars
    const int32_t* set_vars;
    int T, M, C, tied, n_segs, n_grps, n_sets, W, K, max_vars;
};

__host__ __device__ __forceinline__ int pad4(int m) { return (m + 3) & ~3; }

__device__ __forceinline__ Seg seg_of(const Geo& g, int s) {
    if (g.segs != nullptr) return g.segs[s];
    return Seg{s, g.M, g.C, g.tied ? 0 : s * g.M, (int64_t)s * g.M, g.tied ? 0 : (int64_t)s * g.M * g.C, (int64_t)s * pad4(g.M)};
}
__device__ __forceinline__ Grp grp_of(const Geo& g, int i) {
    if (g.grps != nullptr) return g.grps[i];
    return Grp{i, g.M, g.C, i * g.M, (int64_t)i * g.M * g.C, (int64_t)i * pad4(g.M)};      // (tied: i = 0)
}
__device__ __forceinline__ int set_begin(const Geo& g, int u) { return g.set_first != nullptr ? g.set_first[u] : u * (g.tied ? g.T : 1); }
__device__ __forceinline__ int set_size(const Geo& g, int u) {
    return g.set_first != nullptr ? g.set_first[u + 1] - g.set_first[u] : g.tied ? g.T : 1;
}
__device__ __forceinline__ int set_var(const Geo& g, int at) { return g.set_vars != nullptr ? g.set_vars[at] : at; }

// ---- weights -----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float load_logit(const void* p, int dtype, int64_t i) {
    if (dtype == 0) return ((const float*)p)[i];
    if (dtype == 1) return __bfloat162float(((const __nv_bfloat16*)p)[i]);
    return __half2float(((const __half*)p)[i]);
}

struct PrepArgs {
    int2* ent;                     // [var][W][K]: category (-1: none), weight
    const void* ids;
    const void* logits;
    const float* norms;
    int64_t ib, iv, ik, lb, lv, lk, nb, nv;            // strides in elements
    int wide_ids, dtype, B, W, V, K;
    float inv_t;
    double inv_t64;
};

// One warp per position.
__global__ void __launch_bounds__(kTh) teacher_prep_kernel(PrepArgs a) {
    const int64_t at = (int64_t)blockIdx.x * kW + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (at >= (int64_t)a.V * a.W) return;
    const int v = (int)(at / a.W), b = (int)(at % a.W);
    int2* out = a.ent + at * a.K;
    if (b >= a.B) {                                    // padding columns
        for (int k = lane; k < a.K; k += 32) out[k] = make_int2(-1, 0);
        return;
    }
    auto slot = [&](int k, int& id, float& x) {
        const int64_t i = b * a.ib + v * a.iv + k * a.ik;
        const int64_t wide = a.wide_ids ? ((const int64_t*)a.ids)[i] : (int64_t)((const int32_t*)a.ids)[i];
        x = load_logit(a.logits, a.dtype, b * a.lb + v * a.lv + k * a.lk);
        if (wide < 0 || !(x > PCX_NEG_INF)) { id = -1; x = PCX_NEG_INF; }
        else id = (int)min(wide, (int64_t)0x7fffffff);
    };
    float m = PCX_NEG_INF;
    for (int k = lane; k < a.K; k += 32) {
        int id; float x;
        slot(k, id, x);
        m = fmaxf(m, x);
    }
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    const float norm = a.norms != nullptr ? a.norms[b * a.nb + v * a.nv] : CUDART_INF_F;
    const bool given = fabsf(norm) < CUDART_INF_F;
    auto raw = [&](float x) {
        if (x == PCX_NEG_INF) return 0.0f;
        if (given) return expf((float)((double)x * a.inv_t64 - (double)norm));
        return x == m ? 1.0f : expf((x - m) * a.inv_t);          // (+inf logits share the weight)
    };
    float sum = 0.0f;
    if (!given) {
        for (int k = lane; k < a.K; k += 32) {
            int id; float x;
            slot(k, id, x);
            sum += raw(x);
        }
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    }
    for (int k = lane; k < a.K; k += 32) {
        int id; float x;
        slot(k, id, x);
        const float q = given ? raw(x) : sum > 0.0f ? raw(x) / sum : 0.0f;
        out[k] = make_int2(q > 0.0f ? id : -1, __float_as_int(q));
    }
}

// ---- forward -----------------------------------------------------------------------------------------------------------
struct FwdArgs {
    Geo g;
    float* out;
    const float* table;            // [M][C] per vector, or turned: [C][R]
    const int2* ent;
    int64_t R;
    int take_log, m_tiles, per_b;
};

// Few slots, or tables of a single node: the table is read where it lies.  Eight lanes share an output.
__global__ void __launch_bounds__(kTh) teacher_fwd_direct_kernel(FwdArgs a) {
    const int s = blockIdx.x / a.m_tiles;
    const Seg seg = seg_of(a.g, s);
    const int64_t o = (int64_t)(blockIdx.x % a.m_tiles) * (kTh / 8) + (threadIdx.x >> 3);
    if (o >= (int64_t)seg.M * a.g.W) return;
    const int sub = threadIdx.x & 7;
    const int m = (int)(o / a.g.W), b = (int)(o % a.g.W);
    const float* row = a.table + seg.table + (int64_t)m * seg.C;
    const int2* e = a.ent + ((int64_t)seg.var * a.g.W + b) * a.g.K;
    float acc = 0.0f;
#pragma unroll 4
    for (int k = sub; k < a.g.K; k += 8) {
        const int2 x = __ldg(e + k);
        if (x.x >= 0) {
            float v = x.x < seg.C ? __ldg(row + x.x) : a.take_log ? 0.0f : PCX_NEG_INF;
            if (a.take_log) v = logf(v);
            acc = fmaf(__int_as_float(x.y), v, acc);
        }
    }
    const unsigned mask = 0xffu << (threadIdx.x & 24);
    for (int off = 4; off; off >>= 1) acc += __shfl_xor_sync(mask, acc, off);
    if (sub == 0) a.out[(seg.row0 + m) * a.g.W + b] = acc;
}

// NM * 32 nodes of one vector; a warp takes one position at a time, its lanes the nodes.  SRC 0: the turned table, four
// neighbouring nodes per lane; 1: the turned table, any alignment; 2: the table's part in shared memory.
template <int SRC, int NM>
__global__ void __launch_bounds__(kTh) teacher_fwd_kernel(FwdArgs a) {
    constexpr int MT = 32 * NM;
    extern __shared__ float sm[];
    float* tile = sm;                                  // [MT][33]
    float* part = sm + MT * 33;                        // [C][MT + 1]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const Seg seg = seg_of(a.g, blockIdx.x / a.m_tiles);
    const int m0 = (blockIdx.x % a.m_tiles) * MT;
    if (m0 >= seg.M) return;
    const int W = a.g.W, K = a.g.K;
    if constexpr (SRC == 2) {
        for (int m = warp; m < MT; m += kW) {
            const float* row = a.table + seg.table + (int64_t)(m0 + m) * seg.C;
            for (int c = lane; c < seg.C; c += 32) {
                float v = m0 + m < seg.M ? row[c] : 1.0f;
                if (a.take_log) v = logf(v);
                part[c * (MT + 1) + m] = v;
            }
        }
        __syncthreads();
    }
    const float* base = a.table + seg.col + m0;
    const int b_end = min(W, (int)(blockIdx.y + 1) * a.per_b);
    for (int b0 = blockIdx.y * a.per_b; b0 < b_end; b0 += 32) {
        for (int j = 0; j < 4; ++j) {
            const int b = b0 + warp * 4 + j;
            if (b >= b_end) break;
            const int2* e = a.ent + ((int64_t)seg.var * W + b) * K;
            float acc[NM] = {};
#pragma unroll 8
            for (int k = 0; k < K; ++k) {
                const int2 x = __ldg(e + k);
                if (x.x < 0) continue;
                const float q = __int_as_float(x.y);
                if (x.x >= seg.C) {
#pragma unroll
                    for (int i = 0; i < NM; ++i) acc[i] = PCX_NEG_INF;
                    continue;
                }
                if constexpr (SRC == 0) {
                    if (m0 + lane * 4 < seg.M) {
                        const float4 v = __ldg((const float4*)(base + (int64_t)x.x * a.R) + lane);
                        acc[0] = fmaf(q, v.x, acc[0]); acc[1] = fmaf(q, v.y, acc[1]);
                        acc[2] = fmaf(q, v.z, acc[2]); acc[3] = fmaf(q, v.w, acc[3]);
                    }
                } else if constexpr (SRC == 1) {
#pragma unroll
                    for (int i = 0; i < NM; ++i)
                        if (m0 + lane + 32 * i < seg.M) acc[i] = fmaf(q, __ldg(base + (int64_t)x.x * a.R + lane + 32 * i), acc[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < NM; ++i) acc[i] = fmaf(q, part[x.x * (MT + 1) + lane + 32 * i], acc[i]);
                }
            }
#pragma unroll
            for (int i = 0; i < NM; ++i) tile[(SRC == 0 ? lane * 4 + i : lane + 32 * i) * 33 + warp * 4 + j] = acc[i];
        }
        __syncthreads();
        for (int m = warp; m < MT; m += kW)
            if (m0 + m < seg.M && b0 + lane < b_end) a.out[(seg.row0 + m0 + m) * W + b0 + lane] = tile[m * 33 + lane];
        __syncthreads();
    }
}

// ---- turning -----------------------------------------------------------------------------------------------------------
// [R][C] -> [C][stride], of logarithms if asked.
__global__ void __launch_bounds__(kTh) teacher_turn_kernel(float* __restrict__ out, const float* __restrict__ in, int64_t R, int C,
                                                          int64_t stride, int64_t r_tiles) {
    __shared__ float tile[32][33];
    const int64_t r0 = (int64_t)(blockIdx.x % r_tiles) * 32;
    const int c0 = (int)(blockIdx.x / r_tiles) * 32;
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    for (int k = ty; k < 32; k += kW) tile[k][tx] = r0 + k < R && c0 + tx < C ? in[(r0 + k) * C + c0 + tx] : 0.0f;
    __syncthreads();
    for (int k = ty; k < 32; k += kW)
        if (c0 + k < C && r0 + tx < stride) out[(c0 + k) * stride + r0 + tx] = tile[tx][k];
}

// Flows [node][sample] -> [sample][node] of every vector, exponentials if they are logarithms; padding nodes are 0.
__global__ void __launch_bounds__(kTh) teacher_turn_flows_kernel(float* __restrict__ out, const float* __restrict__ flows, Geo g,
                                                                int m_tiles, int logspace) {
    __shared__ float tile[32][33];
    const Seg seg = seg_of(g, blockIdx.x / m_tiles);
    const int m0 = (blockIdx.x % m_tiles) * 32, b0 = blockIdx.y * 32, mp = pad4(seg.M);
    if (m0 >= seg.M) return;
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    for (int k = ty; k < 32; k += kW) {
        float v = 0.0f;
        if (m0 + k < seg.M && b0 + tx < g.W) {
            v = flows[(seg.row0 + m0 + k) * g.W + b0 + tx];
            if (logspace) v = expf(v);
        }
        tile[k][tx] = v;
    }
    __syncthreads();
    for (int k = ty; k < 32; k += kW)
        if (b0 + k < g.W && m0 + tx < mp) out[seg.gcol * g.W + (int64_t)(b0 + k) * mp + m0 + tx] = tile[tx][k];
}

// ---- sorting the slots by category -------------------------------------------------------------------------------------
// Per set of variables: keys (category; C for empty slots) with the slot's place (position in the set * W + sample) and
// weight, in the order of categories, the slots of a category in their own order.
constexpr int kSmallSort = 4096, kSortTile = 4096, kDigits = 256, kMaxCats = 1000000;

struct SortArgs {
    Geo g;
    const int2* ent;
    int32_t* keys;                 // sorted
    int2* slots;                   // sorted: place, weight
    int32_t *key_a, *key_b, *idx_a, *idx_b, *hist;
    int C, tiles, shift;
};

__device__ __forceinline__ int2 set_entry(const Geo& g, const int2* ent, int first, int j) {
    const int wk = g.W * g.K;
    return ent[(int64_t)set_var(g, first + j / wk) * wk + j % wk];
}
__device__ __forceinline__ int key_of_entry(int2 e, int C) { return e.x < 0 || e.x >= C ? C : e.x; }

__global__ void __launch_bounds__(1024) teacher_sort_small_kernel(SortArgs a, int P) {
    extern __shared__ uint32_t comp[];
    const int u = blockIdx.x, first = set_begin(a.g, u), N = set_size(a.g, u) * a.g.W * a.g.K;
    for (int j = threadIdx.x; j < P; j += blockDim.x)
        comp[j] = j < N ? ((uint32_t)key_of_entry(set_entry(a.g, a.ent, first, j), a.C) << 12) | (uint32_t)j : ~0u;
    __syncthreads();
    for (int size = 2; size <= P; size <<= 1)
        for (int step = size >> 1; step; step >>= 1) {
            for (int i = threadIdx.x; i < P / 2; i += blockDim.x) {
                const int x = 2 * i - (i & (step - 1)), y = x + step;
                const uint32_t p = comp[x], q = comp[y];
                if ((p > q) == ((x & size) == 0)) { comp[x] = q; comp[y] = p; }
            }
            __syncthreads();
        }
    const int64_t base = (int64_t)first * a.g.W * a.g.K;
    for (int j = threadIdx.x; j < N; j += blockDim.x) {
        const int at = comp[j] & 4095;
        a.keys[base + j] = (int)(comp[j] >> 12);
        a.slots[base + j] = make_int2(at / a.g.K, set_entry(a.g, a.ent, first, at).y);
    }
}

// One pass of a stable radix sort over 8 bits: digit counts of every tile, their running sums, the move.
template <bool FIRST>
__global__ void __launch_bounds__(kTh) teacher_hist_kernel(SortArgs a) {
    __shared__ int count[kDigits];
    const int u = blockIdx.x / a.tiles, tile = blockIdx.x % a.tiles;
    const int first = set_begin(a.g, u), N = set_size(a.g, u) * a.g.W * a.g.K;
    const int64_t base = (int64_t)first * a.g.W * a.g.K;
    for (int d = threadIdx.x; d < kDigits; d += kTh) count[d] = 0;
    __syncthreads();
    for (int j = tile * kSortTile + threadIdx.x; j < min(N, (tile + 1) * kSortTile); j += kTh) {
        const int k = FIRST ? key_of_entry(set_entry(a.g, a.ent, first, j), a.C) : a.key_a[base + j];
        atomicAdd(&count[(k >> a.shift) & (kDigits - 1)], 1);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < kDigits; d += kTh) a.hist[((int64_t)u * kDigits + d) * a.tiles + tile] = count[d];
}

__global__ void __launch_bounds__(1024) teacher_scan_kernel(int32_t* hist, int n) {
    __shared__ int warp_sum[32];
    int32_t* h = hist + (int64_t)blockIdx.x * n;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int carry = 0;
    for (int i0 = 0; i0 < n; i0 += 1024) {
        const int i = i0 + threadIdx.x;
        const int v = i < n ? h[i] : 0;
        int x = v;
        for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(~0u, x, o); if (lane >= o) x += y; }
        if (lane == 31) warp_sum[warp] = x;
        __syncthreads();
        if (warp == 0) {
            int w = warp_sum[lane];
            for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(~0u, w, o); if (lane >= o) w += y; }
            warp_sum[lane] = w;
        }
        __syncthreads();
        const int before = carry + (warp > 0 ? warp_sum[warp - 1] : 0) + x - v;
        carry += warp_sum[31];
        if (i < n) h[i] = before;
        __syncthreads();
    }
}

template <bool FIRST, bool LAST>
__global__ void __launch_bounds__(kTh) teacher_move_kernel(SortArgs a) {
    __shared__ int count[kW][kDigits];
    const int u = blockIdx.x / a.tiles, tile = blockIdx.x % a.tiles;
    const int first = set_begin(a.g, u), N = set_size(a.g, u) * a.g.W * a.g.K;
    if (tile * kSortTile >= N) return;
    const int64_t base = (int64_t)first * a.g.W * a.g.K;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int ROUNDS = kSortTile / kTh;
    for (int i = threadIdx.x; i < kW * kDigits; i += kTh) (&count[0][0])[i] = 0;
    __syncthreads();
    const int j0 = tile * kSortTile + warp * (kSortTile / kW);
    int key[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int j = j0 + r * 32 + lane;
        key[r] = -1;
        if (j < N) {
            key[r] = FIRST ? key_of_entry(set_entry(a.g, a.ent, first, j), a.C) : a.key_a[base + j];
            atomicAdd(&count[warp][(key[r] >> a.shift) & (kDigits - 1)], 1);
        }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < kDigits; d += kTh) {
        int at = a.hist[((int64_t)u * kDigits + d) * a.tiles + tile];
        for (int w = 0; w < kW; ++w) { const int c = count[w][d]; count[w][d] = at; at += c; }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int j = j0 + r * 32 + lane;
        const int d = key[r] < 0 ? kDigits : (key[r] >> a.shift) & (kDigits - 1);
        const unsigned same = __match_any_sync(~0u, d);
        int to = 0;
        if (key[r] >= 0) to = count[warp][d] + __popc(same & ((1u << lane) - 1));
        __syncwarp();
        if (key[r] >= 0 && lane == __ffs(same) - 1) count[warp][d] += __popc(same);
        __syncwarp();
        if (key[r] < 0) continue;
        const int idx = FIRST ? j : a.idx_a[base + j];
        if constexpr (LAST) {
            a.keys[base + to] = key[r];
            a.slots[base + to] = make_int2(idx / a.g.K, set_entry(a.g, a.ent, first, idx).y);
        } else {
            a.key_b[base + to] = key[r];
            a.idx_b[base + to] = idx;
        }
    }
}

// first[u][c] = the first sorted slot of set u with a category of at least c
__global__ void __launch_bounds__(kTh) teacher_first_kernel(int32_t* first, const int32_t* keys, Geo g, int C, int blocks) {
    const int u = blockIdx.x / blocks;
    const int N = set_size(g, u) * g.W * g.K;
    const int64_t base = (int64_t)set_begin(g, u) * g.W * g.K;
    const int j = (blockIdx.x % blocks) * kTh + threadIdx.x;
    if (j > N) return;
    const int lo = j == 0 ? 0 : keys[base + j - 1] + 1, hi = j == N ? C : keys[base + j];
    for (int c = lo; c <= hi; ++c) first[(int64_t)u * (C + 1) + c] = j;
}

// ---- backward ----------------------------------------------------------------------------------------------------------
struct BwdArgs {
    Geo g;
    float* out;                    // [M][C] per group; mode 2: [C][R]
    int32_t* touched;              // mode 2
    const float* flows;            // turned
    const int32_t* keys;
    const int2* slots;
    const int32_t* first;
    int64_t R;
    int C, mode, c_tiles, m_tiles; // mode 0: written, all of it; 1: added; 2: added to the turned table
};

constexpr int kHeavy = 128;        // slots of a category that all warps of a CTA share

// 32 categories x 128 nodes of one group.  A warp sums a category's slots in their order, lanes over the nodes; a category
// with many slots is split over the CTA's warps, whose parts are added in order.
__global__ void __launch_bounds__(kTh) teacher_bwd_kernel(BwdArgs a) {
    __shared__ float acc[32][129];
    __shared__ float part[kW][128];
    __shared__ int from[33];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int64_t at = blockIdx.x;
    const int c0 = (int)(at % a.c_tiles) * 32;
    at /= a.c_tiles;
    const int m0 = (int)(at % a.m_tiles) * 128;
    const Grp grp = grp_of(a.g, (int)(at / a.m_tiles));
    if (m0 >= grp.M || c0 >= grp.C) return;
    const int nc = min(32, grp.C - c0);
    if (tid <= nc) from[tid] = a.first[(int64_t)grp.set * (a.C + 1) + c0 + tid];
    __syncthreads();
    const bool none = from[0] == from[nc];
    if (none && a.mode != 0) return;
    const int mp = pad4(grp.M);
    const float* flows = a.flows + grp.gbase * a.g.W + m0 + lane * 4;
    const int2* slots = a.slots + (int64_t)set_begin(a.g, grp.set) * a.g.W * a.g.K;
    const bool in = m0 + lane * 4 < mp;
    auto sum = [&](int lo, int hi) {
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        if (in) {
#pragma unroll 8
            for (int j = lo; j < hi; ++j) {
                const int2 e = __ldg(slots + j);
                const float q = __int_as_float(e.y);
                const float4 v = __ldg((const float4*)(flows + (int64_t)e.x * mp));
                s.x = fmaf(q, v.x, s.x); s.y = fmaf(q, v.y, s.y); s.z = fmaf(q, v.z, s.z); s.w = fmaf(q, v.w, s.w);
            }
        }
        return s;
    };
    if (!none) {
        for (int cc = warp; cc < nc; cc += kW) {
            const int lo = from[cc], hi = from[cc + 1];
            if (hi - lo > kHeavy) continue;
            const float4 s = sum(lo, hi);
            acc[cc][lane * 4] = s.x; acc[cc][lane * 4 + 1] = s.y; acc[cc][lane * 4 + 2] = s.z; acc[cc][lane * 4 + 3] = s.w;
        }
        for (int cc = 0; cc < nc; ++cc) {
            const int lo = from[cc], hi = from[cc + 1];
            if (hi - lo <= kHeavy) continue;
            const int per = (hi - lo + kW - 1) / kW;
            const float4 s = sum(lo + warp * per, min(hi, lo + (warp + 1) * per));
            *(float4*)&part[warp][lane * 4] = s;
            __syncthreads();
            if (tid < 128) {
                float t = part[0][tid];
                for (int w = 1; w < kW; ++w) t += part[w][tid];
                acc[cc][tid] = t;
            }
            __syncthreads();
        }
        __syncthreads();
    }
    if (a.mode == 2) {
        for (int cc = warp; cc < nc; cc += kW) {
            if (from[cc] == from[cc + 1]) continue;
            float* row = a.out + (int64_t)(c0 + cc) * a.R + grp.col + m0;
            for (int m = lane; m < 128 && m0 + m < grp.M; m += 32) row[m] += acc[cc][m];
            if (lane == 0) a.touched[c0 + cc] = 1;
        }
        return;
    }
    for (int m = warp; m < 128 && m0 + m < grp.M; m += kW) {
        if (lane >= nc) continue;
        float* p = a.out + grp.out + (int64_t)(m0 + m) * grp.C + c0 + lane;
        if (a.mode == 0) *p = none ? 0.0f : acc[lane][m];
        else if (from[lane] != from[lane + 1]) *p += acc[lane][m];
    }
}

// Few slots in large tables: only the categories that occur are visited, one warp each (mode 0: the caller has cleared the
// output).
__global__ void __launch_bounds__(kTh) teacher_bwd_runs_kernel(BwdArgs a, int blocks) {
    const Grp grp = grp_of(a.g, blockIdx.x / blocks);
    const int N = set_size(a.g, grp.set) * a.g.W * a.g.K, lane = threadIdx.x & 31;
    const int64_t base = (int64_t)set_begin(a.g, grp.set) * a.g.W * a.g.K;
    const int j = (blockIdx.x % blocks) * kW + (threadIdx.x >> 5);
    if (j >= N) return;
    const int32_t* keys = a.keys + base;
    const int c = keys[j];
    if (c >= grp.C || (j > 0 && keys[j - 1] == c)) return;
    int end = j + 1;
    while (end < N && keys[end] == c) ++end;
    const int mp = pad4(grp.M);
    const float* flows = a.flows + grp.gbase * a.g.W;
    for (int m = lane; m < grp.M; m += 32) {
        float s = 0.0f;
#pragma unroll 4
        for (int i = j; i < end; ++i) {
            const int2 e = __ldg(a.slots + base + i);
            s = fmaf(__int_as_float(e.y), __ldg(flows + (int64_t)e.x * mp + m), s);
        }
        if (a.mode == 2) a.out[(int64_t)c * a.R + grp.col + m] += s;
        else if (a.mode == 1) a.out[grp.out + (int64_t)m * grp.C + c] += s;
        else a.out[grp.out + (int64_t)m * grp.C + c] = s;
    }
    if (a.mode == 2 && lane == 0) a.touched[c] = 1;
}

Geo make_geo(const PcxTeacherGeo* p) {
    return Geo{(const Seg*)p->segs, (const Grp*)p->groups, p->set_first, p->set_vars, p->positions, p->nodes, p->cats, p->tied,
               p->n_segs, p->n_groups, p->n_sets, p->width, p->slots, p->max_vars};
}

int64_t align(int64_t n) { return (n + 255) & ~(int64_t)255; }

// What the backward pass keeps in its scratch.
struct Layout {
    int64_t flows, keys, slots, first, key_a, key_b, idx_a, idx_b, hist, total;
    int64_t n_max;                 // slots of the largest set
    bool small;
    int tiles;
};
Layout layout(const PcxTeacherGeo* p, bool runs) {
    Layout l{};
    const int64_t E = (int64_t)p->total_vars * p->width * p->slots;
    l.n_max = (int64_t)p->max_vars * p->width * p->slots;
    l.small = l.n_max <= kSmallSort;
    l.tiles = (int)pcx_cdiv(std::max<int64_t>(l.n_max, 1), kSortTile);
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t here = at; at += align(bytes); return here; };
    l.flows = take(p->flow_cols * p->width * 4);
    l.keys = take(E * 4);
    l.slots = take(E * 8);
    l.first = take(runs ? 0 : (int64_t)p->n_sets * (p->cats + 1) * 4);
    if (!l.small) {
        l.key_a = take(E * 4); l.key_b = take(E * 4); l.idx_a = take(E * 4); l.idx_b = take(E * 4);
        l.hist = take((int64_t)p->n_sets * kDigits * l.tiles * 4);
    }
    l.total = at;
    return l;
}

bool fits(const PcxTeacherGeo* p) {
    const int64_t wk = (int64_t)p->width * p->slots;
    return p->width > 0 && p->slots > 0 && p->cats > 0 && p->cats <= kMaxCats && p->n_segs > 0 && wk * p->max_vars <= 0x7fffffff / 2;
}

}  // namespace

extern "C" {

int pcx_teacher_prep(void* entries, const void* ids, int wide_ids, int64_t ids_b, int64_t ids_v, int64_t ids_k, const void* logits,
                     int dtype, int64_t logits_b, int64_t logits_v, int64_t logits_k, const float* norms, int64_t norms_b,
                     int64_t norms_v, int batch, int vars, int slots, int width, double temperature, void* stream) {
    if (vars <= 0 || width <= 0 || slots <= 0) return 0;
    const int64_t blocks = pcx_cdiv((int64_t)vars * width, kW);
    if (blocks > 0x7fffffff || dtype < 0 || dtype > 2) return -1;
    PrepArgs a{(int2*)entries, ids, logits, norms, ids_b, ids_v, ids_k, logits_b, logits_v, logits_k, norms_b, norms_v, wide_ids,
               dtype, batch, width, vars, slots, (float)(1.0 / temperature), 1.0 / temperature};
    teacher_prep_kernel<<<(unsigned)blocks, kTh, 0, (cudaStream_t)stream>>>(a);
    PCX_LAUNCH_CHECK();
    return 0;
}

int pcx_teacher_turn(float* out, const float* table, int64_t rows, int cats, int64_t stride, void* stream) {
    if (rows <= 0 || cats <= 0) return 0;
    const int64_t r_tiles = pcx_cdiv(stride, 32), blocks = r_tiles * pcx_cdiv(cats, 32);
    if (blocks > 0x7fffffff) return -1;
    teacher_turn_kernel<<<(unsigned)blocks, kTh, 0, (cudaStream_t)stream>>>(out, table, rows, cats, stride, r_tiles);
    PCX_LAUNCH_CHECK();
    return 0;
}

// Nodes per CTA of the staged form; 0 = the tables do not fit shared memory
int pcx_teacher_staged_nodes(int cats, int nodes) {
    for (int nm = 4; nm; nm >>= 1) {
        if (nm > 1 && nodes <= 16 * nm) continue;
        if ((int64_t)4 * (32 * nm * 33 + (int64_t)cats * (32 * nm + 1)) <= (nm > 1 ? 110 : 220) * 1024) return 32 * nm;
    }
    return 0;
}

int pcx_teacher_fwd(float* out, const float* table, const void* entries, const PcxTeacherGeo* geo, int form, int64_t turned_stride,
                    int take_log, void* stream) {
    if (!fits(geo)) return -1;
    FwdArgs a{};
    a.g = make_geo(geo);
    a.out = out; a.table = table; a.ent = (const int2*)entries; a.R = turned_stride; a.take_log = take_log;
    cudaStream_t st = (cudaStream_t)stream;
    if (form == 0) {
        const int64_t blocks = pcx_cdiv((int64_t)geo->nodes * geo->width, kTh / 8);
        if (blocks * geo->n_segs > 0x7fffffff) return -1;
        a.m_tiles = (int)blocks;
        teacher_fwd_direct_kernel<<<(unsigned)(blocks * geo->n_segs), kTh, 0, st>>>(a);
        PCX_LAUNCH_CHECK();
        return 0;
    }
    int mt = 128;
    if (form == 2 && (mt = pcx_teacher_staged_nodes(geo->cats, geo->nodes)) == 0) return -1;
    a.m_tiles = (int)pcx_cdiv(geo->nodes, mt);
    if ((int64_t)a.m_tiles * geo->n_segs > 0x7fffffff) return -1;
    // positions per CTA: all of them where the table has to be staged first, unless few CTAs would be left
    const int64_t tiles = (int64_t)a.m_tiles * geo->n_segs;
    const int64_t splits = std::max<int64_t>(1, std::min(pcx_cdiv(geo->width, 32), form == 2 ? pcx_cdiv(148, tiles) : (int64_t)65535));
    a.per_b = (int)(pcx_cdiv(pcx_cdiv(geo->width, splits), 32) * 32);
    const dim3 grid((unsigned)tiles, (unsigned)pcx_cdiv(geo->width, a.per_b));
    const int tile_bytes = mt * 33 * 4;
    if (form == 1) {
        teacher_fwd_kernel<1, 4><<<grid, kTh, tile_bytes, st>>>(a);
    } else if (form == 3) {
        teacher_fwd_kernel<0, 4><<<grid, kTh, tile_bytes, st>>>(a);
    } else {
        const int bytes = tile_bytes + geo->cats * (mt + 1) * 4;
        static PcxOnce done;
        if (!done) {
            for (const void* k : {(const void*)teacher_fwd_kernel<2, 4>, (const void*)teacher_fwd_kernel<2, 2>, (const void*)teacher_fwd_kernel<2, 1>}) {
                const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024);
                if (e != cudaSuccess) return (int)e;
            }
            done = true;
        }
        if (mt == 128) teacher_fwd_kernel<2, 4><<<grid, kTh, bytes, st>>>(a);
        else if (mt == 64) teacher_fwd_kernel<2, 2><<<grid, kTh, bytes, st>>>(a);
        else teacher_fwd_kernel<2, 1><<<grid, kTh, bytes, st>>>(a);
    }
    PCX_LAUNCH_CHECK();
    return 0;
}

int64_t pcx_teacher_bwd_scratch_bytes(const PcxTeacherGeo* geo, int runs) { return layout(geo, runs != 0).total; }

int pcx_teacher_bwd(float* out, int32_t* touched, void* scratch, const float* flows, const void* entries, const PcxTeacherGeo* geo,
                    int mode, int runs, int64_t turned_stride, int logspace, void* stream) {
    if (!fits(geo)) return -1;
    cudaStream_t st = (cudaStream_t)stream;
    const Layout l = layout(geo, runs != 0);
    const Geo g = make_geo(geo);
    char* base = (char*)scratch;
    float* turned = (float*)(base + l.flows);
    {
        const int m_tiles = (int)pcx_cdiv(geo->nodes, 32);
        if ((int64_t)m_tiles * geo->n_segs > 0x7fffffff || pcx_cdiv(geo->width, 32) > 65535) return -1;
        teacher_turn_flows_kernel<<<dim3((unsigned)(m_tiles * geo->n_segs), (unsigned)pcx_cdiv(geo->width, 32)), kTh, 0, st>>>(
            turned, flows, g, m_tiles, logspace);
        PCX_LAUNCH_CHECK();
    }
    SortArgs s{};
    s.g = g; s.ent = (const int2*)entries; s.C = geo->cats;
    s.keys = (int32_t*)(base + l.keys); s.slots = (int2*)(base + l.slots);
    if (l.small) {
        int P = 2;
        while (P < l.n_max) P <<= 1;
        teacher_sort_small_kernel<<<geo->n_sets, std::min(1024, std::max(32, P / 2)), P * 4, st>>>(s, P);
        PCX_LAUNCH_CHECK();
    } else {
        s.key_a = (int32_t*)(base + l.key_a); s.key_b = (int32_t*)(base + l.key_b);
        s.idx_a = (int32_t*)(base + l.idx_a); s.idx_b = (int32_t*)(base + l.idx_b);
        s.hist = (int32_t*)(base + l.hist);
        s.tiles = l.tiles;
        if ((int64_t)l.tiles * geo->n_sets > 0x7fffffff || (int64_t)l.tiles * kDigits > 0x7fffffff) return -1;
        const unsigned grid = (unsigned)(l.tiles * geo->n_sets);
        int bits = 1;
        while ((geo->cats >> bits) != 0) ++bits;
        for (int shift = 0; shift < bits; shift += 8) {
            const bool first = shift == 0, last = shift + 8 >= bits;
            s.shift = shift;
            if (first) teacher_hist_kernel<true><<<grid, kTh, 0, st>>>(s); else teacher_hist_kernel<false><<<grid, kTh, 0, st>>>(s);
            PCX_LAUNCH_CHECK();
            teacher_scan_kernel<<<geo->n_sets, 1024, 0, st>>>(s.hist, kDigits * l.tiles);
            PCX_LAUNCH_CHECK();
            if (first && last) teacher_move_kernel<true, true><<<grid, kTh, 0, st>>>(s);
            else if (first) teacher_move_kernel<true, false><<<grid, kTh, 0, st>>>(s);
            else if (last) teacher_move_kernel<false, true><<<grid, kTh, 0, st>>>(s);
            else teacher_move_kernel<false, false><<<grid, kTh, 0, st>>>(s);
            PCX_LAUNCH_CHECK();
            std::swap(s.key_a, s.key_b);
            std::swap(s.idx_a, s.idx_b);
        }
    }
    BwdArgs a{};
    a.g = g; a.out = out; a.touched = touched; a.flows = turned; a.keys = s.keys; a.slots = s.slots; a.R = turned_stride;
    a.C = geo->cats; a.mode = mode;
    if (runs) {
        const int64_t blocks = pcx_cdiv(l.n_max, kW);
        if (blocks * geo->n_groups > 0x7fffffff) return -1;
        teacher_bwd_runs_kernel<<<(unsigned)(blocks * geo->n_groups), kTh, 0, st>>>(a, (int)blocks);
        PCX_LAUNCH_CHECK();
        return 0;
    }
    {
        const int64_t blocks = pcx_cdiv(l.n_max + 1, kTh);
        if (blocks * geo->n_sets > 0x7fffffff) return -1;
        teacher_first_kernel<<<(unsigned)(blocks * geo->n_sets), kTh, 0, st>>>((int32_t*)(base + l.first), s.keys, g, geo->cats, (int)blocks);
        PCX_LAUNCH_CHECK();
    }
    a.first = (const int32_t*)(base + l.first);
    a.c_tiles = (int)pcx_cdiv(geo->cats, 32);
    a.m_tiles = (int)pcx_cdiv(geo->nodes, 128);
    const int64_t blocks = (int64_t)a.c_tiles * a.m_tiles * geo->n_groups;
    if (blocks > 0x7fffffff) return -1;
    teacher_bwd_kernel<<<(unsigned)blocks, kTh, 0, st>>>(a);
    PCX_LAUNCH_CHECK();
    return 0;
}

}  // extern "C"
