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
//
// Times below: "large" is a table of 4096 nodes x 32768 categories that 128 positions x 64 samples of 32 slots share (250 K
// slots with weight, 4.1 GB looked up in each direction); "small" is 196 tables of 256 x 256, 100 samples of 16 slots.
#include "pcx_common.cuh"
#include "../../include/pcx_b200.h"
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <algorithm>
#include <type_traits>

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

// L lanes per position, four slots a lane in registers (more are read again).  Slots that say something come first, in their
// order: what reads them stops at the first empty one.  7 us large and small: latency (one warp a position took 13 small).
template <int L>
__global__ void __launch_bounds__(kTh) teacher_prep_kernel(PrepArgs a) {
    constexpr int HELD = 4;
    const int64_t at = (int64_t)blockIdx.x * (kTh / L) + threadIdx.x / L;
    const int lane = threadIdx.x % L;
    const bool here = at < (int64_t)a.V * a.W;         // (all lanes take part in the shuffles)
    const int v = (int)(at / a.W), b = here ? (int)(at % a.W) : a.B;
    int2* out = a.ent + at * a.K;
    auto slot = [&](int k, int& id, float& x) {
        id = -1;
        x = PCX_NEG_INF;
        if (k >= a.K || b >= a.B) return;              // (padding columns are empty)
        const int64_t i = b * a.ib + v * a.iv + k * a.ik;
        const int64_t wide = a.wide_ids ? ((const int64_t*)a.ids)[i] : (int64_t)((const int32_t*)a.ids)[i];
        const float y = load_logit(a.logits, a.dtype, b * a.lb + v * a.lv + k * a.lk);
        if (wide >= 0 && y > PCX_NEG_INF) { id = (int)min(wide, (int64_t)0x7fffffff); x = y; }
    };
    int ids[HELD];
    float xs[HELD];
#pragma unroll
    for (int i = 0; i < HELD; ++i) slot(lane + L * i, ids[i], xs[i]);
    auto each = [&](auto&& f) {
#pragma unroll
        for (int i = 0; i < HELD; ++i)
            if (L * i < a.K) f(ids[i], xs[i]);
        for (int k0 = L * HELD; k0 < a.K; k0 += L) {
            int id; float x;
            slot(k0 + lane, id, x);
            f(id, x);
        }
    };
    const float norm = a.norms != nullptr && b < a.B ? a.norms[b * a.nb + v * a.nv] : CUDART_INF_F;
    float m = PCX_NEG_INF, sum = 0.0f;
    each([&](int, float x) { m = fmaxf(m, x); });
#pragma unroll
    for (int o = L / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    const bool given = fabsf(norm) < CUDART_INF_F && m < CUDART_INF_F;       // (logits of +inf leave no other normaliser than theirs)
    auto raw = [&](float x) {
        if (x == PCX_NEG_INF) return 0.0f;
        if (given) return expf((float)((double)x * a.inv_t64 - (double)norm));
        return x == m ? 1.0f : expf((x - m) * a.inv_t);          // (+inf logits share the weight)
    };
    each([&](int, float x) { sum += raw(x); });
#pragma unroll
    for (int o = L / 2; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    int count = 0;
    const int first_lane = threadIdx.x % 32 - lane;
    each([&](int id, float x) {
        const float q = given ? raw(x) : sum > 0.0f ? raw(x) / sum : 0.0f;
        const unsigned says = (__ballot_sync(~0u, id >= 0 && q > 0.0f) >> first_lane) & (L == 32 ? ~0u : (1u << (L & 31)) - 1);
        if (id >= 0 && q > 0.0f) out[count + __popc(says & ((1u << lane) - 1))] = make_int2(id, __float_as_int(q));
        count += __popc(says);
    });
    if (here)
        for (int k = count + lane; k < a.K; k += L) out[k] = make_int2(-1, 0);
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

// Few slots, or tables of a single node: the table is read where it lies.  Eight lanes share an output; the outputs of the
// same nodes at all positions run side by side, since their reads meet in the same parts of the table.  1024 nodes x 50257
// categories, 128 positions of 50 slots: 28 us, 148 MB read at 5 TB/s: HBM, whose sectors of 32 bytes bring 4 wanted ones.
__global__ void __launch_bounds__(kTh) teacher_fwd_direct_kernel(FwdArgs a) {
    const int64_t task = (int64_t)blockIdx.x * (kTh / 8) + (threadIdx.x >> 3);
    const int W = a.g.W, s = (int)(task / W % a.g.n_segs), b = (int)(task % W);
    const int m = (int)(task / W / a.g.n_segs);
    if (m >= a.g.M) return;
    const Seg seg = seg_of(a.g, s);
    if (m >= seg.M) return;
    const int sub = threadIdx.x & 7;
    const float* row = a.table + seg.table + (int64_t)m * seg.C;
    const int2* e = a.ent + ((int64_t)seg.var * W + b) * a.g.K;
    float acc = 0.0f;
    for (int k0 = 0; k0 < a.g.K; k0 += 64) {
        int2 x[8];
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = k0 + 8 * i + sub < a.g.K ? __ldg(e + k0 + 8 * i + sub) : make_int2(-1, 0);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = x[i].x >= 0 && x[i].x < seg.C ? __ldg(row + x[i].x) : a.take_log ? 0.0f : PCX_NEG_INF;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (x[i].x >= 0) acc = fmaf(__int_as_float(x[i].y), a.take_log ? logf(v[i]) : v[i], acc);
    }
    const unsigned mask = 0xffu << (threadIdx.x & 24);
    for (int off = 4; off; off >>= 1) acc += __shfl_xor_sync(mask, acc, off);
    if (sub == 0) a.out[(seg.row0 + m) * W + b] = acc;
}

// Row `i` of `stride` bytes from `base`: one multiply-add.
template <typename T>
__device__ __forceinline__ const T* row_at(const char* base, int i, uint32_t stride) {
    return (const T*)(base + (uint64_t)(uint32_t)i * stride);
}
__device__ __forceinline__ void fma4(float q, const float4& v, float* s) {
    s[0] = fmaf(q, v.x, s[0]); s[1] = fmaf(q, v.y, s[1]); s[2] = fmaf(q, v.z, s[2]); s[3] = fmaf(q, v.w, s[3]);
}

// How a lane's NV values lie among the nodes of a tile: four neighbours at a time, or 32 apart.
template <bool VEC>
__device__ __forceinline__ int node_of(int lane, int i) { return VEC ? (i / 4) * 128 + lane * 4 + i % 4 : i * 32 + lane; }

// A warp's results [NV * 32 nodes][32 positions] of all positions of a block go through shared memory to rows of positions.
template <int NV>
__device__ __forceinline__ void store_rows(const float* tile, float* out, int m_left, int b_left, int W) {
    const int lane = threadIdx.x & 31;
    for (int m = threadIdx.x >> 5; m < min(32 * NV, m_left); m += kW)
        if (lane < b_left) out[(int64_t)m * W + lane] = tile[m * 33 + lane];
}

// Turned table: a warp takes one position at a time, its lanes NV nodes each.  The same nodes of all positions run side by
// side, so that their part of the table stays in L2 (all nodes of a position in a row: 379 us large).  Large: 226 us, at which
// L2 delivers 15.6 TB/s to the SMs, which is what bounds it: 64 registers and 4 CTAs per SM beat more loads in flight (80
// registers: 291 us).
template <bool VEC, int NV>
__global__ void __launch_bounds__(kTh, 4) teacher_fwd_turned_kernel(FwdArgs a) {
    constexpr int MT = 32 * NV;
    extern __shared__ float tile[];                    // [MT][33]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Seg seg = seg_of(a.g, blockIdx.x % a.g.n_segs);
    const int m0 = blockIdx.x / a.g.n_segs * MT;
    if (m0 >= seg.M) return;
    const int W = a.g.W, K = a.g.K;
    constexpr int LOADS = VEC ? NV / 4 : NV;
    const uint32_t stride = (uint32_t)a.R * 4;
    const char* at[LOADS];                             // lanes without a node look at the vector's first
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int m = m0 + node_of<VEC>(lane, VEC ? 4 * i : i);
        at[i] = (const char*)(a.table + seg.col + (m < seg.M ? m : 0));
    }
    const int b_end = min(W, (int)(blockIdx.y + 1) * a.per_b);
    for (int b0 = blockIdx.y * a.per_b; b0 < b_end; b0 += 32) {
        for (int j = 0; j < 4; ++j) {
            const int b = b0 + warp * 4 + j;
            if (b >= b_end) break;
            const int2* e = a.ent + ((int64_t)seg.var * W + b) * K;
            float acc[NV] = {};
            for (int k0 = 0; k0 < K; k0 += 32) {
                const int2 own = k0 + lane < K ? __ldg(e + k0 + lane) : make_int2(-1, 0);
                const int n = __popc(__ballot_sync(~0u, own.x >= 0));
                if (__any_sync(~0u, own.x >= seg.C)) { // a category that the table does not have
#pragma unroll
                    for (int i = 0; i < NV; ++i) acc[i] = PCX_NEG_INF;
                    break;
                }
                constexpr int AHEAD = VEC ? 32 / NV : 4;
                auto some = [&](int k, auto whole) {   // the next AHEAD slots, or what is left of them
                    float q[AHEAD];
                    float4 v[AHEAD][LOADS];
#pragma unroll
                    for (int h = 0; h < AHEAD; ++h) {
                        const int c = __shfl_sync(~0u, own.x, k + h);
                        q[h] = __int_as_float(__shfl_sync(~0u, own.y, k + h));
                        if (whole.value || k + h < n) {
#pragma unroll
                            for (int i = 0; i < LOADS; ++i) {
                                if constexpr (VEC) v[h][i] = __ldg(row_at<float4>(at[i], c, stride));
                                else v[h][i].x = __ldg(row_at<float>(at[i], c, stride));
                            }
                        }
                    }
#pragma unroll
                    for (int h = 0; h < AHEAD; ++h) {
                        if (!whole.value && k + h >= n) break;
#pragma unroll
                        for (int i = 0; i < LOADS; ++i) {
                            if constexpr (VEC) fma4(q[h], v[h][i], acc + 4 * i);
                            else acc[i] = fmaf(q[h], v[h][i].x, acc[i]);
                        }
                    }
                };
                int k = 0;
                for (; k + AHEAD <= n; k += AHEAD) some(k, std::true_type());
                if (k < n) some(k, std::false_type());
                if (n < 32) break;
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) tile[node_of<VEC>(lane, i) * 33 + warp * 4 + j] = acc[i];
        }
        __syncthreads();
        store_rows<NV>(tile, a.out + (seg.row0 + m0) * W + b0, seg.M - m0, b_end - b0, W);
        __syncthreads();
    }
}

// A table of its own: NV * 32 nodes of it go through shared memory, the nodes of a category side by side.  Small: 45 us for 54
// MB; 25 M instructions at 57% of the issue slots, seven for each slot and 64 nodes.  32 or 128 nodes a CTA: 60, 64 us.
template <int NV, bool LOG>
__global__ void __launch_bounds__(kTh) teacher_fwd_staged_kernel(FwdArgs a) {
    constexpr int MT = 32 * NV;
    extern __shared__ float tile[];                    // [MT][33], then the table's part [C][MT + 1] and a row of zeros
    float* part = tile + MT * 33;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Seg seg = seg_of(a.g, blockIdx.x / a.m_tiles);
    const int m0 = blockIdx.x % a.m_tiles * MT;
    if (m0 >= seg.M) return;
    const int W = a.g.W, K = a.g.K, C = seg.C;
    const int b_begin = blockIdx.y * a.per_b, b_end = min(W, b_begin + a.per_b);
    int2 next[4];                                      // the first 32 slots of this warp's next four positions
    auto fetch = [&](int b0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int b = b0 + warp * 4 + j;
            next[j] = b < b_end && lane < K ? __ldg(a.ent + ((int64_t)seg.var * W + b) * K + lane) : make_int2(-1, 0);
        }
    };
    fetch(b_begin);
    constexpr int PER = MT / kW, AT_ONCE = 32 / PER;   // a warp's nodes; categories a lane fetches at a time
    for (int c = lane; c < C; c += 32 * AT_ONCE) {
        const float* row = a.table + seg.table + (int64_t)(m0 + warp * PER) * C + c;
        float v[AT_ONCE][PER];
#pragma unroll
        for (int i = 0; i < PER; ++i)
#pragma unroll
            for (int h = 0; h < AT_ONCE; ++h)
                v[h][i] = m0 + warp * PER + i < seg.M && c + 32 * h < C ? __ldg(row + (int64_t)i * C + 32 * h) : 1.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i)
#pragma unroll
            for (int h = 0; h < AT_ONCE; ++h)
                if (c + 32 * h < C) part[(c + 32 * h) * (MT + 1) + warp * PER + i] = LOG ? logf(v[h][i]) : v[h][i];
    }
    if (threadIdx.x < MT) part[C * (MT + 1) + threadIdx.x] = 0.0f;
    __syncthreads();
    for (int b0 = b_begin; b0 < b_end; b0 += 32) {
        int2 now[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) now[j] = next[j];
        fetch(b0 + 32);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int b = b0 + warp * 4 + j;
            if (b >= b_end) break;
            const int2* e = a.ent + ((int64_t)seg.var * W + b) * K;
            float acc[NV] = {};
            for (int k0 = 0; k0 < K; k0 += 32) {
                const int2 own = k0 == 0 ? now[j] : k0 + lane < K ? __ldg(e + k0 + lane) : make_int2(-1, 0);
                const int n = __popc(__ballot_sync(~0u, own.x >= 0));
                if (__any_sync(~0u, own.x >= C)) {     // a category that the table does not have
#pragma unroll
                    for (int i = 0; i < NV; ++i) acc[i] = PCX_NEG_INF;
                    break;
                }
                const int row = (own.x < 0 ? C : own.x) * (MT + 1);          // empty slots look at the row of zeros
                const float weight = __int_as_float(own.y);
                for (int k = 0; k < n; k += 4)
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        const float* v = part + __shfl_sync(~0u, row, k + h) + lane;
                        const float q = __shfl_sync(~0u, weight, k + h);
#pragma unroll
                        for (int i = 0; i < NV; ++i) acc[i] = fmaf(q, v[32 * i], acc[i]);
                    }
                if (n < 32) break;
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) tile[(32 * i + lane) * 33 + warp * 4 + j] = acc[i];
        }
        __syncthreads();
        store_rows<NV>(tile, a.out + (seg.row0 + m0) * W + b0, seg.M - m0, b_end - b0, W);
        __syncthreads();
    }
}

// ---- turning -----------------------------------------------------------------------------------------------------------
// 64 x 64 tiles; a thread reads and writes four neighbours at a time where rows allow it (VEC).  Large: 167 us for the table (1.07
// GB, 6.4 TB/s, as a copy; 32 x 32 tiles of single words: 370), 38 us for the flows.
constexpr int kTurn = 64;

// out[c][r] = value(r, c) for r < n_r, c < n_c of a tile, 0 for n_r <= r < pad_r.  `in` and `out` point at the tile.
template <bool VEC_IN, bool VEC_OUT, typename F>
__device__ __forceinline__ void turn_tile(float (*tile)[kTurn + 1], const float* in, int64_t in_stride, int n_r, int n_c, float* out,
                                          int64_t out_stride, int pad_r, F value) {
    const int q = (threadIdx.x & 15) * 4, y = threadIdx.x >> 4;
    float4 v[kTurn / 16];
#pragma unroll
    for (int i = 0; i < kTurn / 16; ++i) {
        const int r = y + 16 * i;
        const float* p = in + r * in_stride + q;
        v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < n_r) {
            if (VEC_IN && q + 4 <= n_c) v[i] = *(const float4*)p;
            else {
                if (q < n_c) v[i].x = p[0];
                if (q + 1 < n_c) v[i].y = p[1];
                if (q + 2 < n_c) v[i].z = p[2];
                if (q + 3 < n_c) v[i].w = p[3];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kTurn / 16; ++i) {
        const int r = y + 16 * i;
        tile[r][q] = v[i].x; tile[r][q + 1] = v[i].y; tile[r][q + 2] = v[i].z; tile[r][q + 3] = v[i].w;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kTurn / 16; ++i) {
        const int c = y + 16 * i;
        if (c >= n_c || q >= pad_r) continue;
        float o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = q + k < n_r ? value(tile[q + k][c]) : 0.0f;
        float* p = out + c * out_stride + q;
        if (VEC_OUT && q + 4 <= pad_r) *(float4*)p = make_float4(o[0], o[1], o[2], o[3]);
        else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (q + k < pad_r) p[k] = o[k];
        }
    }
}

// [R][C] -> [C][stride], of logarithms if asked.
template <bool VEC_IN, bool VEC_OUT, bool LOG>
__global__ void __launch_bounds__(kTh) teacher_turn_kernel(float* __restrict__ out, const float* __restrict__ in, int64_t R, int C,
                                                          int64_t stride, int64_t r_tiles) {
    __shared__ float tile[kTurn][kTurn + 1];
    const int64_t r0 = (int64_t)(blockIdx.x % r_tiles) * kTurn;
    const int c0 = (int)(blockIdx.x / r_tiles) * kTurn;
    turn_tile<VEC_IN, VEC_OUT>(tile, in + r0 * C + c0, C, (int)max((int64_t)0, min((int64_t)kTurn, R - r0)), min(kTurn, C - c0),
                               out + c0 * stride + r0, stride, (int)min((int64_t)kTurn, stride - r0), [](float v) { return LOG ? logf(v) : v; });
}

// Flows [node][sample] -> [sample][node] of every vector, exponentials if they are logarithms; padding nodes are 0.
template <bool VEC_IN>
__global__ void __launch_bounds__(kTh) teacher_turn_flows_kernel(float* __restrict__ out, const float* __restrict__ flows, Geo g,
                                                                int m_tiles, int logspace) {
    __shared__ float tile[kTurn][kTurn + 1];
    const unsigned tiles = (unsigned)g.n_segs * m_tiles, at = blockIdx.x % tiles;
    const Seg seg = seg_of(g, at / m_tiles);
    const int m0 = at % m_tiles * kTurn, b0 = blockIdx.x / tiles * kTurn, mp = pad4(seg.M);
    if (m0 >= seg.M) return;
    turn_tile<VEC_IN, true>(tile, flows + (seg.row0 + m0) * g.W + b0, g.W, min(kTurn, seg.M - m0), min(kTurn, g.W - b0),
                            out + seg.gcol * g.W + (int64_t)b0 * mp + m0, mp, min(kTurn, mp - m0),
                            [&](float v) { return logspace ? expf(v) : v; });
}

// ---- sorting the slots by category -------------------------------------------------------------------------------------
// Per set of variables: keys (category; C for empty slots) with the slot's place (position in the set * W + sample) and
// weight, in the order of categories, the slots of a category in their own order.
// Radix passes of at most 10 bits: the digit counts of the warps (and tiles), their running sums in the order of digits,
// then every slot moves to its place; slots of one digit keep their order.  Large: 262 K slots in two passes, 37 us (eight rounds a tile: 42); small: 15 us
// for 1600 slots a CTA (a bitonic network: 26).
constexpr int kSmallSort = 4096, kSortRounds = 4, kSortTile = kTh * kSortRounds, kMaxCats = 1000000;

struct SortArgs {
    Geo g;
    const int2* ent;
    int32_t* keys;                 // sorted
    int2* slots;                   // sorted: place, weight
    int32_t* first;                // [n_sets][C + 1], or null
    const int32_t* key_in;         // what a pass over tiles reads (null: the entries) ...
    const int2* slot_in;
    int32_t* key_out;              // ... and writes
    int2* slot_out;
    int32_t *hist, *totals;        // [n_sets][digits][tiles], [n_sets][digits]
    int C, tiles, shift, bits;
};

__device__ __forceinline__ int2 set_entry(const Geo& g, const int2* ent, int first, int j) {
    const int wk = g.W * g.K;
    return ent[(int64_t)set_var(g, first + j / wk) * wk + j % wk];
}
__device__ __forceinline__ int key_of_entry(int2 e, int C) { return e.x < 0 || e.x >= C ? C : e.x; }

// Running sum over the threads of a block (before this thread's own).
__device__ __forceinline__ int scan_before(int v, int* warp_sum) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n_warps = blockDim.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(~0u, x, o); if (lane >= o) x += y; }
    if (lane == 31) warp_sum[warp] = x;
    __syncthreads();
    int before = x - v;
    for (int w = 0; w < n_warps; ++w) before += w < warp ? warp_sum[w] : 0;
    __syncthreads();
    return before;
}

// A set of at most 4096 slots: one CTA, 128 slots a warp; a slot is its key and, in the low 12 bits, its number.
__global__ void __launch_bounds__(1024) teacher_sort_small_kernel(SortArgs a) {
    extern __shared__ uint32_t sm_sort[];
    const int n_warps = blockDim.x >> 5, cap = n_warps * 128, D = 1 << a.bits;
    uint32_t* here = sm_sort;
    uint32_t* there = here + cap;
    uint16_t* count = (uint16_t*)(there + cap);        // [n_warps][D]
    __shared__ int warp_sum[32];
    const int u = blockIdx.x, first = set_begin(a.g, u), N = set_size(a.g, u) * a.g.W * a.g.K;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int j = tid; j < cap; j += blockDim.x)
        here[j] = j < N ? ((uint32_t)key_of_entry(set_entry(a.g, a.ent, first, j), a.C) << 12) | (uint32_t)j : ~0u;
    for (int shift = 12; (a.C >> (shift - 12)) != 0; shift += a.bits) {
        for (int i = tid; i < n_warps * D / 2; i += blockDim.x) ((uint32_t*)count)[i] = 0;
        __syncthreads();
        uint32_t v[4];
        int rank[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            v[r] = here[warp * 128 + r * 32 + lane];
            const int d = v[r] == ~0u ? -1 : (int)((v[r] >> shift) & (D - 1));
            const unsigned same = __match_any_sync(~0u, d);
            rank[r] = d < 0 ? 0 : count[warp * D + d] + __popc(same & ((1u << lane) - 1));
            __syncwarp();
            if (d >= 0 && lane == __ffs(same) - 1) count[warp * D + d] += __popc(same);
            __syncwarp();
        }
        __syncthreads();
        int run = 0;                                   // digits before those of this round
        for (int d0 = 0; d0 < D; d0 += blockDim.x) {
            const int d = d0 + tid;
            int total = 0;
            if (d < D)
                for (int w = 0; w < n_warps; ++w) { const int c = count[w * D + d]; count[w * D + d] = (uint16_t)total; total += c; }
            const int before = run + scan_before(total, warp_sum);
            if (d < D)
                for (int w = 0; w < n_warps; ++w) count[w * D + d] += (uint16_t)before;
            if (tid == blockDim.x - 1) warp_sum[0] = before + total;
            __syncthreads();
            run = warp_sum[0];
            __syncthreads();
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (v[r] != ~0u) there[count[warp * D + ((v[r] >> shift) & (D - 1))] + rank[r]] = v[r];
        __syncthreads();
        for (int j = N + tid; j < cap; j += blockDim.x) there[j] = ~0u;
        uint32_t* t = here; here = there; there = t;
        __syncthreads();
    }
    const int64_t base = (int64_t)first * a.g.W * a.g.K;
    for (int j = tid; j < N; j += blockDim.x) {
        const int at = here[j] & 4095;
        a.keys[base + j] = (int)(here[j] >> 12);
        a.slots[base + j] = make_int2(at / a.g.K, set_entry(a.g, a.ent, first, at).y);
    }
    if (a.first != nullptr)
        for (int c = tid; c <= a.C; c += blockDim.x) {
            int lo = 0, hi = N;                        // the first slot with a key of at least c
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if ((int)(here[mid] >> 12) < c) lo = mid + 1; else hi = mid;
            }
            a.first[(int64_t)u * (a.C + 1) + c] = lo;
        }
}

// A set of at most 256 slots, a thread each: a slot's place is the number of smaller ones.
constexpr int kTinySort = 256;
__global__ void __launch_bounds__(kTinySort) teacher_sort_tiny_kernel(SortArgs a) {
    __shared__ alignas(16) uint32_t comp[kTinySort];
    const int u = blockIdx.x, first = set_begin(a.g, u), N = set_size(a.g, u) * a.g.W * a.g.K, j = threadIdx.x;
    const int2 e = j < N ? set_entry(a.g, a.ent, first, j) : make_int2(0, 0);
    const uint32_t own = j < N ? ((uint32_t)key_of_entry(e, a.C) << 12) | (uint32_t)j : ~0u;
    comp[j] = own;
    __syncthreads();
    int rank = 0;
#pragma unroll 4
    for (int i = 0; i < (int)blockDim.x; i += 4) {
        const uint4 o = *(const uint4*)(comp + i);
        rank += (int)(o.x < own) + (int)(o.y < own) + (int)(o.z < own) + (int)(o.w < own);
    }
    const int64_t base = (int64_t)first * a.g.W * a.g.K;
    if (j < N) {
        a.keys[base + rank] = (int)(own >> 12);
        a.slots[base + rank] = make_int2(j / a.g.K, e.y);
    }
    if (a.first != nullptr)
        for (int c = j; c <= a.C; c += blockDim.x) {   // slots with a smaller key
            int n = 0;
            for (int i = 0; i < N; ++i) n += (int)((int)(comp[i] >> 12) < c);
            a.first[(int64_t)u * (a.C + 1) + c] = n;
        }
}

template <bool FIRST>
__device__ __forceinline__ int sort_key(const SortArgs& a, int first, int64_t base, int j) {
    return FIRST ? key_of_entry(set_entry(a.g, a.ent, first, j), a.C) : a.key_in[base + j];
}

template <bool FIRST>
__global__ void __launch_bounds__(kTh) teacher_hist_kernel(SortArgs a) {
    __shared__ int count[1024];
    const int u = blockIdx.x / a.tiles, tile = blockIdx.x % a.tiles, D = 1 << a.bits;
    const int first = set_begin(a.g, u), N = set_size(a.g, u) * a.g.W * a.g.K;
    const int64_t base = (int64_t)first * a.g.W * a.g.K;
    for (int d = threadIdx.x; d < D; d += kTh) count[d] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
        const int j = tile * kSortTile + r * kTh + threadIdx.x;
        if (j < N) atomicAdd(&count[(sort_key<FIRST>(a, first, base, j) >> a.shift) & (D - 1)], 1);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += kTh) a.hist[((int64_t)u * D + d) * a.tiles + tile] = count[d];
}

// One warp per set and digit: running sums over the tiles, and the digit's total.
__global__ void __launch_bounds__(kTh) teacher_scan_kernel(int32_t* hist, int32_t* totals, int64_t n, int tiles) {
    const int64_t at = (int64_t)blockIdx.x * kW + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (at >= n) return;
    int32_t* h = hist + at * tiles;
    int carry = 0;
    for (int i0 = 0; i0 < tiles; i0 += 32) {
        const int v = i0 + lane < tiles ? h[i0 + lane] : 0;
        int x = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(~0u, x, o); if (lane >= o) x += y; }
        if (i0 + lane < tiles) h[i0 + lane] = carry + x - v;
        carry += __shfl_sync(~0u, x, 31);
    }
    if (lane == 0) totals[at] = carry;
}

template <bool FIRST>
__global__ void __launch_bounds__(kTh) teacher_move_kernel(SortArgs a) {
    extern __shared__ int sm_move[];                   // [kW][D]
    __shared__ int warp_sum[32];
    const int u = blockIdx.x / a.tiles, tile = blockIdx.x % a.tiles, D = 1 << a.bits;
    const int first = set_begin(a.g, u), N = set_size(a.g, u) * a.g.W * a.g.K;
    if (tile * kSortTile >= N) return;
    const int64_t base = (int64_t)first * a.g.W * a.g.K;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int* count = sm_move + warp * D;
    for (int i = threadIdx.x; i < kW * D; i += kTh) sm_move[i] = 0;
    const int j0 = tile * kSortTile + warp * (32 * kSortRounds) + lane;
    int key[kSortRounds], rank[kSortRounds];
    int2 slot[kSortRounds];
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
        const int j = j0 + r * 32;
        key[r] = -1;
        if (j < N) {
            if constexpr (FIRST) {
                const int2 e = set_entry(a.g, a.ent, first, j);
                key[r] = key_of_entry(e, a.C);
                slot[r] = make_int2(j / a.g.K, e.y);
            } else {
                key[r] = a.key_in[base + j];
                slot[r] = a.slot_in[base + j];
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
        const int d = key[r] < 0 ? -1 : (key[r] >> a.shift) & (D - 1);
        const unsigned same = __match_any_sync(~0u, d);
        rank[r] = d < 0 ? 0 : count[d] + __popc(same & ((1u << lane) - 1));
        __syncwarp();
        if (d >= 0 && lane == __ffs(same) - 1) count[d] += __popc(same);
        __syncwarp();
    }
    __syncthreads();
    int run = 0;
    for (int d0 = 0; d0 < D; d0 += kTh) {
        const int d = d0 + threadIdx.x;
        const int total = d < D ? a.totals[(int64_t)u * D + d] : 0;
        const int before = run + scan_before(total, warp_sum);
        if (d < D) {
            if (tile == 0 && a.first != nullptr && d <= a.C) a.first[(int64_t)u * (a.C + 1) + d] = before;
            int at = before + a.hist[((int64_t)u * D + d) * a.tiles + tile];
            for (int w = 0; w < kW; ++w) { const int c = sm_move[w * D + d]; sm_move[w * D + d] = at; at += c; }
        }
        if (threadIdx.x == kTh - 1) warp_sum[0] = before + total;
        __syncthreads();
        run = warp_sum[0];
        __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
        if (key[r] < 0) continue;
        const int64_t to = base + count[(key[r] >> a.shift) & (D - 1)] + rank[r];
        a.key_out[to] = key[r];
        a.slot_out[to] = slot[r];
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
    int C, mode, c_tiles, m_tiles, c_tile;             // mode 0: written, all of it; 1: added; 2: added to the turned table
};

constexpr int kMaxTile = 64;       // categories of a tile

// c_tile categories x NV * 32 nodes of one group.  The slots of the tile's categories, side by side after the sort,
// are dealt out to the warps in equal parts; a warp walks its part in order, lanes over the nodes, and closes a category's
// sum where the next begins.  A category that an earlier warp began is added to that warp's sum afterwards, in order.
// Large: 405 us, of which writing the 537 MB alone takes 147; L2 delivers 10 TB/s, and its 4.1 GB would take 277 at the 15.5 that
// the forward pass reaches.  Neither more rows under way nor balance is what it lacks: rows kept under way without a pause, in
// registers 419, through a ring in shared memory (cp.async) 640; full tiles first 408; flows laid out tile by tile 410.  Tiles
// of 32 categories: 461; three CTAs an SM: 450; a warp a category, long ones shared: 534.  Small: 39 us.  512 nodes, 1000 categories: 35
// us (512 threads a CTA 31, more launched forms for 3% of a call; tiles of 64 or 32 nodes 42, 63).
template <int NV>
__global__ void __launch_bounds__(kTh, 2) teacher_bwd_kernel(BwdArgs a) {
    constexpr int MT = 32 * NV, AHEAD = NV > 4 ? 4 : 8;
    extern __shared__ float acc[];                     // [c_tile][MT + 1], then [kW][MT]
    __shared__ int from[kMaxTile + 1], carry[kW];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int64_t at = blockIdx.x;
    const int c0 = (int)(at % a.c_tiles) * a.c_tile;
    at /= a.c_tiles;
    const int m0 = (int)(at % a.m_tiles) * MT;
    const Grp grp = grp_of(a.g, (int)(at / a.m_tiles));
    if (m0 >= grp.M || c0 >= grp.C) return;
    const int nc = min(a.c_tile, grp.C - c0), nm = min(MT, grp.M - m0);
    float* part = acc + a.c_tile * (MT + 1);
    if (tid <= nc) from[tid] = a.first[(int64_t)grp.set * (a.C + 1) + c0 + tid];
    __syncthreads();
    const int begin = from[0], end = from[nc];
    if (begin == end && a.mode != 0) return;
    if (begin < end) {
        const int mp = pad4(grp.M);
        const int64_t base = (int64_t)set_begin(a.g, grp.set) * a.g.W * a.g.K;
        const int2* slots = a.slots + base;
        const int32_t* keys = a.keys + base;
        const uint32_t stride = (uint32_t)mp * 4;
        const char* flow_at[NV / 4];                   // lanes without a node look at the group's first
#pragma unroll
        for (int i = 0; i < NV / 4; ++i) {
            const int m = m0 + i * 128 + lane * 4;
            flow_at[i] = (const char*)(a.flows + grp.gbase * a.g.W + (m < mp ? m : 0));
        }
        const int per = (end - begin + kW - 1) / kW;
        const int lo = min(end, begin + warp * per), hi = min(end, lo + per);
        if (lane == 0) carry[warp] = -1;
        if (lo < hi) {
            float s[NV] = {};
            int cur = keys[lo] - c0;
            const bool later = lo > from[cur];
            if (later && lane == 0) carry[warp] = cur;
            float* to = later ? part + warp * MT : acc + cur * (MT + 1);
            auto close = [&]() {
#pragma unroll
                for (int i = 0; i < NV; ++i) { to[node_of<true>(lane, i)] = s[i]; s[i] = 0.0f; }
            };
            for (int j0 = lo; j0 < hi; j0 += 32) {
                const int n = min(32, hi - j0);
                const int2 own = lane < n ? __ldg(slots + j0 + lane) : make_int2(0, 0);
                const int key = lane < n ? __ldg(keys + j0 + lane) - c0 : -1;
                int before = __shfl_up_sync(~0u, key, 1);
                if (lane == 0) before = cur;
                const unsigned opens = __ballot_sync(~0u, lane < n && key != before);
                auto some = [&](int k, auto whole) {   // the next AHEAD slots, or what is left of them
                    float q[AHEAD];
                    float4 v[AHEAD][NV / 4];
#pragma unroll
                    for (int h = 0; h < AHEAD; ++h) {
                        const int place = __shfl_sync(~0u, own.x, k + h);
                        q[h] = __int_as_float(__shfl_sync(~0u, own.y, k + h));
                        if (whole.value || k + h < n) {
#pragma unroll
                            for (int i = 0; i < NV / 4; ++i) v[h][i] = __ldg(row_at<float4>(flow_at[i], place, stride));
                        }
                    }
#pragma unroll
                    for (int h = 0; h < AHEAD; ++h) {
                        if (!whole.value && k + h >= n) break;
                        if (opens >> (k + h) & 1) {
                            close();
                            to = acc + __shfl_sync(~0u, key, k + h) * (MT + 1);
                        }
#pragma unroll
                        for (int i = 0; i < NV / 4; ++i) fma4(q[h], v[h][i], s + 4 * i);
                    }
                };
                int k = 0;
                for (; k + AHEAD <= n; k += AHEAD) some(k, std::true_type());
                if (k < n) some(k, std::false_type());
                cur = __shfl_sync(~0u, key, n - 1);
            }
            close();
        }
        __syncthreads();
        if (tid < MT)
            for (int w = 1; w < kW; ++w)
                if (carry[w] >= 0) acc[carry[w] * (MT + 1) + tid] += part[w * MT + tid];
        __syncthreads();
    }
    if (a.mode == 2) {
        for (int cc = warp; cc < nc; cc += kW) {
            if (from[cc] == from[cc + 1]) continue;
            float* row = a.out + (int64_t)(c0 + cc) * a.R + grp.col + m0;
            for (int m = lane; m < nm; m += 32) row[m] += acc[cc * (MT + 1) + m];
            if (lane == 0) a.touched[c0 + cc] = 1;
        }
        return;
    }
    float* out = a.out + grp.out + (int64_t)m0 * grp.C + c0;
    if (a.mode == 0 && grp.C % 4 == 0 && ((uintptr_t)out & 15) == 0) {       // four categories a thread
        const int n_lanes = a.c_tile / 4, cc = tid % n_lanes * 4;
        if (cc >= nc) return;
        bool has[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) has[i] = from[cc + i] != from[cc + i + 1];
        for (int m = tid / n_lanes; m < nm; m += kTh / n_lanes) {
            const float* v = acc + cc * (MT + 1) + m;
            *(float4*)(out + (int64_t)m * grp.C + cc) = make_float4(has[0] ? v[0] : 0.0f, has[1] ? v[MT + 1] : 0.0f,
                                                                   has[2] ? v[2 * (MT + 1)] : 0.0f, has[3] ? v[3 * (MT + 1)] : 0.0f);
        }
        return;
    }
    const int n_lanes = a.c_tile, cc = tid % n_lanes;  // lanes side by side over the categories
    if (cc >= nc) return;
    const bool has = from[cc] != from[cc + 1];
    for (int m = tid / n_lanes; m < nm; m += kTh / n_lanes) {
        float* p = out + (int64_t)m * grp.C + cc;
        if (a.mode == 0) *p = has ? acc[cc * (MT + 1) + m] : 0.0f;
        else if (has) *p += acc[cc * (MT + 1) + m];
    }
}

// (2048 rows of 64 slots: 8 us beside the 42 that clearing 268 MB takes.)
// Few slots in large tables: only the categories that occur are visited, L lanes each, in an output that has been cleared
// (mode 0).
template <int L>
__global__ void __launch_bounds__(kTh) teacher_bwd_runs_kernel(BwdArgs a, int blocks) {
    const Grp grp = grp_of(a.g, blockIdx.x / blocks);
    const int N = set_size(a.g, grp.set) * a.g.W * a.g.K, lane = threadIdx.x % L;
    const int64_t base = (int64_t)set_begin(a.g, grp.set) * a.g.W * a.g.K;
    const int j = (blockIdx.x % blocks) * (kTh / L) + threadIdx.x / L;
    if (j >= N) return;
    const int32_t* keys = a.keys + base;
    const int c = keys[j];
    if (c >= grp.C || (j > 0 && keys[j - 1] == c)) return;
    int end = j + 1;
    while (end < N && keys[end] == c) ++end;
    const int mp = pad4(grp.M);
    const float* flows = a.flows + grp.gbase * a.g.W;
    for (int m = lane; m < grp.M; m += L) {
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
    int64_t flows, keys, slots, first, key_b, slot_b, hist, totals, total;
    int64_t n_max;                 // slots of the largest set
    bool small;
    int tiles, bits, passes;
};
Layout layout(const PcxTeacherGeo* p, bool runs) {
    Layout l{};
    const int64_t E = (int64_t)p->total_vars * p->width * p->slots;
    l.n_max = (int64_t)p->max_vars * p->width * p->slots;
    l.small = l.n_max <= kSmallSort;
    l.tiles = (int)pcx_cdiv(std::max<int64_t>(l.n_max, 1), kSortTile);
    int bits = 1;
    while ((p->cats >> bits) != 0) ++bits;
    l.passes = (int)pcx_cdiv(bits, l.small ? 9 : 10);
    l.bits = (int)pcx_cdiv(bits, l.passes);
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t here = at; at += align(bytes); return here; };
    l.flows = take(p->flow_cols * p->width * 4);
    l.keys = take(E * 4);
    l.slots = take(E * 8);
    l.first = take(runs ? 0 : (int64_t)p->n_sets * (p->cats + 1) * 4);
    if (!l.small) {
        l.key_b = take(E * 4); l.slot_b = take(E * 8);
        l.hist = take(((int64_t)p->n_sets << l.bits) * l.tiles * 4);
        l.totals = take(((int64_t)p->n_sets << l.bits) * 4);
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
    const int lanes = slots <= 32 ? 8 : slots <= 64 ? 16 : 32;
    const int64_t blocks = pcx_cdiv((int64_t)vars * width, kTh / lanes);
    if (blocks > 0x7fffffff || dtype < 0 || dtype > 2) return -1;
    PrepArgs a{(int2*)entries, ids, logits, norms, ids_b, ids_v, ids_k, logits_b, logits_v, logits_k, norms_b, norms_v, wide_ids,
               dtype, batch, width, vars, slots, (float)(1.0 / temperature), 1.0 / temperature};
    cudaStream_t st = (cudaStream_t)stream;
    if (lanes == 8) teacher_prep_kernel<8><<<(unsigned)blocks, kTh, 0, st>>>(a);
    else if (lanes == 16) teacher_prep_kernel<16><<<(unsigned)blocks, kTh, 0, st>>>(a);
    else teacher_prep_kernel<32><<<(unsigned)blocks, kTh, 0, st>>>(a);
    PCX_LAUNCH_CHECK();
    return 0;
}

int pcx_teacher_turn(float* out, const float* table, int64_t rows, int cats, int64_t stride, int take_log, void* stream) {
    if (rows <= 0 || cats <= 0) return 0;
    const int64_t r_tiles = pcx_cdiv(stride, kTurn), blocks = r_tiles * pcx_cdiv(cats, kTurn);
    if (blocks > 0x7fffffff) return -1;
    const bool in4 = cats % 4 == 0 && (uintptr_t)table % 16 == 0, out4 = stride % 4 == 0 && (uintptr_t)out % 16 == 0;
    const unsigned grid = (unsigned)blocks;
    cudaStream_t st = (cudaStream_t)stream;
    auto launch = [&](auto vec_in, auto vec_out) {
        if (take_log) teacher_turn_kernel<vec_in.value, vec_out.value, true><<<grid, kTh, 0, st>>>(out, table, rows, cats, stride, r_tiles);
        else teacher_turn_kernel<vec_in.value, vec_out.value, false><<<grid, kTh, 0, st>>>(out, table, rows, cats, stride, r_tiles);
    };
    if (in4 && out4) launch(std::true_type(), std::true_type());
    else if (out4) launch(std::false_type(), std::true_type());
    else if (in4) launch(std::true_type(), std::false_type());
    else launch(std::false_type(), std::false_type());
    PCX_LAUNCH_CHECK();
    return 0;
}

// Nodes per CTA of the staged form; 0 = the tables do not fit shared memory
int pcx_teacher_staged_nodes(int cats, int nodes) {
    for (int nm = 4; nm; nm >>= 1) {
        if (nm > 1 && nodes <= 16 * nm) continue;
        if ((int64_t)4 * (32 * nm * 33 + (int64_t)(cats + 1) * (32 * nm + 1)) <= (nm > 1 ? 110 : 220) * 1024) return 32 * nm;
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
        const int64_t blocks = pcx_cdiv((int64_t)geo->nodes * geo->width * geo->n_segs, kTh / 8);
        if (blocks > 0x7fffffff) return -1;
        teacher_fwd_direct_kernel<<<(unsigned)blocks, kTh, 0, st>>>(a);
        PCX_LAUNCH_CHECK();
        return 0;
    }
    // nodes per CTA: as many as there are, 128 or 256, of a turned table
    const int mt = form == 2 ? pcx_teacher_staged_nodes(geo->cats, geo->nodes) : geo->nodes > 128 && form == 3 ? 256 : 128;
    if (mt == 0) return -1;
    a.m_tiles = (int)pcx_cdiv(geo->nodes, mt);
    const int64_t tiles = (int64_t)a.m_tiles * geo->n_segs;
    if (tiles > 0x7fffffff || turned_stride >= 1 << 30) return -1;
    // positions per CTA: all of them where the table has to be staged first, unless few CTAs would be left
    const int64_t splits = std::max<int64_t>(1, std::min(pcx_cdiv(geo->width, 32), form == 2 ? pcx_cdiv(148, tiles) : (int64_t)65535));
    a.per_b = (int)(pcx_cdiv(pcx_cdiv(geo->width, splits), 32) * 32);
    const dim3 grid((unsigned)tiles, (unsigned)pcx_cdiv(geo->width, a.per_b));
    const int tile_bytes = mt * 33 * 4;
    if (form == 1) {
        teacher_fwd_turned_kernel<false, 4><<<grid, kTh, tile_bytes, st>>>(a);
    } else if (form == 3 && mt == 128) {
        teacher_fwd_turned_kernel<true, 4><<<grid, kTh, tile_bytes, st>>>(a);
    } else if (form == 3) {
        teacher_fwd_turned_kernel<true, 8><<<grid, kTh, tile_bytes, st>>>(a);
    } else {
        const int bytes = tile_bytes + (geo->cats + 1) * (mt + 1) * 4;
        static PcxOnce done;
        if (!done) {
            for (const void* k : {(const void*)teacher_fwd_staged_kernel<4, false>, (const void*)teacher_fwd_staged_kernel<2, false>,
                                  (const void*)teacher_fwd_staged_kernel<1, false>, (const void*)teacher_fwd_staged_kernel<4, true>,
                                  (const void*)teacher_fwd_staged_kernel<2, true>, (const void*)teacher_fwd_staged_kernel<1, true>}) {
                const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024);
                if (e != cudaSuccess) return (int)e;
            }
            done = true;
        }
        auto launch = [&](auto nv) {
            if (take_log) teacher_fwd_staged_kernel<nv.value, true><<<grid, kTh, bytes, st>>>(a);
            else teacher_fwd_staged_kernel<nv.value, false><<<grid, kTh, bytes, st>>>(a);
        };
        if (mt == 128) launch(std::integral_constant<int, 4>());
        else if (mt == 64) launch(std::integral_constant<int, 2>());
        else launch(std::integral_constant<int, 1>());
    }
    PCX_LAUNCH_CHECK();
    return 0;
}

// Preparation, turning (form 1 or 3: `turned` has room for cats rows of turned_stride) and forward pass in one call.
int pcx_teacher_expect(float* out, void* entries, float* turned, const float* table, const void* ids, int wide_ids, int64_t ids_b,
                       int64_t ids_v, int64_t ids_k, const void* logits, int dtype, int64_t logits_b, int64_t logits_v, int64_t logits_k,
                       const float* norms, int64_t norms_b, int64_t norms_v, int batch, double temperature, const PcxTeacherGeo* geo,
                       int form, int64_t turned_stride, void* stream) {
    int rc = pcx_teacher_prep(entries, ids, wide_ids, ids_b, ids_v, ids_k, logits, dtype, logits_b, logits_v, logits_k, norms, norms_b,
                              norms_v, batch, geo->positions, geo->slots, geo->width, temperature, stream);
    if (rc != 0) return rc;
    if (form == 1 || form == 3) {
        rc = pcx_teacher_turn(turned, table, (int64_t)geo->n_groups * geo->nodes, geo->cats, turned_stride, 0, stream);
        if (rc != 0) return rc;
        table = turned;
    }
    return pcx_teacher_fwd(out, table, entries, geo, form, turned_stride, 0, stream);
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
        const int m_tiles = (int)pcx_cdiv(geo->nodes, kTurn);
        const int64_t blocks = (int64_t)m_tiles * geo->n_segs * pcx_cdiv(geo->width, kTurn);
        if (blocks > 0x7fffffff) return -1;
        const unsigned grid = (unsigned)blocks;
        if (geo->width % 4 == 0 && (uintptr_t)flows % 16 == 0) teacher_turn_flows_kernel<true><<<grid, kTh, 0, st>>>(turned, flows, g, m_tiles, logspace);
        else teacher_turn_flows_kernel<false><<<grid, kTh, 0, st>>>(turned, flows, g, m_tiles, logspace);
        PCX_LAUNCH_CHECK();
    }
    SortArgs s{};
    s.g = g; s.ent = (const int2*)entries; s.C = geo->cats; s.bits = l.bits;
    s.keys = (int32_t*)(base + l.keys); s.slots = (int2*)(base + l.slots);
    s.first = runs ? nullptr : (int32_t*)(base + l.first);
    if (l.n_max <= kTinySort) {
        teacher_sort_tiny_kernel<<<geo->n_sets, (unsigned)(pcx_cdiv(l.n_max, 32) * 32), 0, st>>>(s);
        PCX_LAUNCH_CHECK();
    } else if (l.small) {
        const int warps = (int)std::max<int64_t>(1, pcx_cdiv(l.n_max, 128));
        const int bytes = warps * (2 * 128 * 4 + (2 << l.bits));
        static PcxOnce done;
        if (!done) {
            const cudaError_t e = cudaFuncSetAttribute((const void*)teacher_sort_small_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 96 * 1024);
            if (e != cudaSuccess) return (int)e;
            done = true;
        }
        teacher_sort_small_kernel<<<geo->n_sets, warps * 32, bytes, st>>>(s);
        PCX_LAUNCH_CHECK();
    } else {
        s.hist = (int32_t*)(base + l.hist); s.totals = (int32_t*)(base + l.totals);
        s.tiles = l.tiles;
        if (l.passes > 1) s.first = nullptr;            // (one pass: the categories are the digits)
        const int64_t digits = (int64_t)geo->n_sets << l.bits;
        if ((int64_t)l.tiles * geo->n_sets > 0x7fffffff || pcx_cdiv(digits, kW) > 0x7fffffff) return -1;
        const unsigned grid = (unsigned)(l.tiles * geo->n_sets);
        // the last of an odd number of passes ends in place; of an even number, the first goes to the other buffer too
        int32_t* key_to[2] = {s.keys, (int32_t*)(base + l.key_b)};
        int2* slot_to[2] = {s.slots, (int2*)(base + l.slot_b)};
        for (int pass = 0; pass < l.passes; ++pass) {
            const int to = (l.passes - 1 - pass) & 1;
            s.shift = pass * l.bits;
            s.key_in = key_to[to ^ 1]; s.slot_in = slot_to[to ^ 1];
            s.key_out = key_to[to]; s.slot_out = slot_to[to];
            if (pass == 0) teacher_hist_kernel<true><<<grid, kTh, 0, st>>>(s); else teacher_hist_kernel<false><<<grid, kTh, 0, st>>>(s);
            PCX_LAUNCH_CHECK();
            teacher_scan_kernel<<<(unsigned)pcx_cdiv(digits, kW), kTh, 0, st>>>(s.hist, s.totals, digits, l.tiles);
            PCX_LAUNCH_CHECK();
            if (pass == 0) teacher_move_kernel<true><<<grid, kTh, (kW << l.bits) * 4, st>>>(s);
            else teacher_move_kernel<false><<<grid, kTh, (kW << l.bits) * 4, st>>>(s);
            PCX_LAUNCH_CHECK();
        }
    }
    BwdArgs a{};
    a.g = g; a.out = out; a.touched = touched; a.flows = turned; a.keys = s.keys; a.slots = s.slots; a.R = turned_stride;
    a.C = geo->cats; a.mode = mode;
    if (runs) {
        if (mode == 0) {
            const cudaError_t e = cudaMemsetAsync(out, 0, (size_t)geo->n_groups * geo->nodes * geo->cats * 4, st);
            if (e != cudaSuccess) return (int)e;
        }
        const int lanes = geo->nodes >= 32 ? 32 : geo->nodes >= 8 ? 8 : 1;
        const int64_t blocks = pcx_cdiv(l.n_max, kTh / lanes);
        if (blocks * geo->n_groups > 0x7fffffff) return -1;
        const unsigned grid = (unsigned)(blocks * geo->n_groups);
        if (lanes == 32) teacher_bwd_runs_kernel<32><<<grid, kTh, 0, st>>>(a, (int)blocks);
        else if (lanes == 8) teacher_bwd_runs_kernel<8><<<grid, kTh, 0, st>>>(a, (int)blocks);
        else teacher_bwd_runs_kernel<1><<<grid, kTh, 0, st>>>(a, (int)blocks);
        PCX_LAUNCH_CHECK();
        return 0;
    }
    if (!l.small && l.passes > 1) {
        const int64_t blocks = pcx_cdiv(l.n_max + 1, kTh);
        if (blocks * geo->n_sets > 0x7fffffff) return -1;
        teacher_first_kernel<<<(unsigned)(blocks * geo->n_sets), kTh, 0, st>>>((int32_t*)(base + l.first), s.keys, g, geo->cats, (int)blocks);
        PCX_LAUNCH_CHECK();
    }
    a.first = (const int32_t*)(base + l.first);
    // nodes and categories per CTA: as many as leave every SM four CTAs
    int mt = geo->nodes > 128 ? 256 : 128;
    a.c_tile = kMaxTile;
    auto ctas = [&]() { return pcx_cdiv(geo->cats, a.c_tile) * pcx_cdiv(geo->nodes, mt) * geo->n_groups; };
    while (a.c_tile > 8 && ctas() < 148 * 4) a.c_tile /= 2;
    if (ctas() < 148 * 4) mt = 128;
    a.c_tiles = (int)pcx_cdiv(geo->cats, a.c_tile);
    a.m_tiles = (int)pcx_cdiv(geo->nodes, mt);
    if (ctas() > 0x7fffffff) return -1;
    const int bytes = (a.c_tile * (mt + 1) + kW * mt) * 4;
    static PcxOnce done;
    if (!done) {
        for (const void* k : {(const void*)teacher_bwd_kernel<4>, (const void*)teacher_bwd_kernel<8>}) {
            const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, 76 * 1024);
            if (e != cudaSuccess) return (int)e;
        }
        done = true;
    }
    if (mt == 256) teacher_bwd_kernel<8><<<(unsigned)ctas(), kTh, bytes, st>>>(a);
    else teacher_bwd_kernel<4><<<(unsigned)ctas(), kTh, bytes, st>>>(a);
    PCX_LAUNCH_CHECK();
    return 0;
}

}  // extern "C"
