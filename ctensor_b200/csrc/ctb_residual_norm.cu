// The norms on both sides of a residual block, fused with the block's gate and residual scale, and
// the gradient of that step.
//
// Forward, row by row (x the residual stream, f the block's output, C columns):
//     n = N_post(f)                       (or f)
//     y = x + scale * gate * n
//     h = N_pre(y)                        (or nothing)
// with N(v) = (v - mean) * rstd * weight + bias, rstd = (var + eps)^-1/2 for a LayerNorm (biased
// variance) and mean = 0, var = mean(v^2) for an RMS norm.
//
// Backward, from dy and dh (the gradients of both results):
//     a  = dh * w_pre,  dx = dy + rstd_y * (a - mean(a) - yhat * mean(a * yhat))       (no mean(a) for RMS)
//     dn = scale * gate * dx,  dgate = fold(scale * n * dx)
//     c  = dn * w_post, df = rstd_f * (c - mean(c) - fhat * mean(c * fhat))
//     dw_pre = sum_rows dh * yhat, db_pre = sum_rows dh, dw_post = sum_rows dn * fhat, db_post = sum_rows dn
//
// Both directions are bound by HBM: 16 bytes per element forward (x, f in; y, h out), 24 backward
// (f, y, dy, dh in; dx, df out), 4 / 8 more with a gate for every element.  A row is owned by a team of
// T threads (a warp to a CTA; for wide rows a cluster of CTAs that hold a slice of the columns each and
// exchange their sums through distributed shared memory); every operand is read once.
#include "ctb_residual_norm.cuh"
#include "ctb_team.cuh"

namespace ctb {

namespace {

// ---- a thread's share of a row: E columns, as 16-byte vectors (VEC = 4) or one by one (VEC = 1: row
// lengths or row starts that are no multiple of 16 bytes) ---------------------------------------------------
template <int T, int VEC> __device__ __forceinline__ int col_of(int group, int tid) { return (group * T + tid) * VEC; }

template <int T, int E, int VEC>
__device__ __forceinline__ void load_share(float (&v)[E], const float* row, int width, int tid) {
#pragma unroll
    for (int i = 0; i < E / VEC; ++i) {
        const int c = col_of<T, VEC>(i, tid);
        if (c < width) {
            if constexpr (VEC == 4) {
                const Vec<float, 4> q = ldg_stream(reinterpret_cast<const Vec<float, 4>*>(row + c));
#pragma unroll
                for (int k = 0; k < 4; ++k) v[i * 4 + k] = q.v[k];
            } else {
                v[i] = row[c];
            }
        } else {
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[i * VEC + k] = 0.0f;
        }
    }
}
template <int T, int VEC>
__device__ __forceinline__ void load_part(float (&v)[VEC], const float* row, int c) {
    if constexpr (VEC == 4) {
        const Vec<float, 4> q = *reinterpret_cast<const Vec<float, 4>*>(row + c);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = q.v[k];
    } else {
        v[0] = row[c];
    }
}
template <int VEC>
__device__ __forceinline__ void store_part(float* row, int c, const float (&v)[VEC]) {
    if constexpr (VEC == 4) {
        Vec<float, 4> q;
#pragma unroll
        for (int k = 0; k < 4; ++k) q.v[k] = v[k];
        stg_stream(reinterpret_cast<Vec<float, 4>*>(row + c), q);
    } else {
        row[c] = v[0];
    }
}

// ---- forward ------------------------------------------------------------------------------------------
// mean and rstd of a row from fp64 sums of v and v^2: one sum over the team instead of two, and no
// cancellation that fp64 would notice until |mean| / sigma is about 1e6.
template <int THREADS, int T, int E>
__device__ __forceinline__ void row_statistics(const float (&v)[E], int kind, float eps, double inv_cols, TeamSlots<THREADS, 2, double>& sh,
                                               int& turn, int cs, float* mean, float* rstd) {
    double s[2] = {0.0, 0.0}, odd[2] = {0.0, 0.0};
#pragma unroll
    for (int e = 0; e < E; e += 2) {
        const double a = v[e], b = v[e + 1];
        s[0] = s[0] + a;
        odd[0] = odd[0] + b;
        s[1] = fma(a, a, s[1]);
        odd[1] = fma(b, b, odd[1]);
    }
    s[0] = s[0] + odd[0];
    s[1] = s[1] + odd[1];
    team_fold<FoldSum, THREADS, T>(s, sh, turn, cs);
    double var = s[1] * inv_cols;
    *mean = 0.0f;
    if (kind == CTB_NORM_LAYER) {
        const double m = s[0] * inv_cols;
        *mean = (float)m;
        var = fma(-m, m, var);
        if (var < 0.0) var = 0.0;
    }
    *rstd = __frsqrt_rn((float)(var + (double)eps));
}

template <int THREADS, int T, int E, int VEC>
__global__ void __launch_bounds__(THREADS)
residual_norm_kernel(ResidualNormGeom g, RowsIn x, RowsIn f, float* __restrict__ y, float* __restrict__ h, float* __restrict__ stats, int cs) {
    __shared__ TeamSlots<THREADS, 2, double> sh;
    const int tid = threadIdx.x % T;
    const uint32_t rank = cs > 1 ? cluster_rank() : 0;
    const int64_t row = (int64_t)(blockIdx.x / cs) * (THREADS / T) + threadIdx.x / T;
    if (row >= g.rows) return;                           // whole teams leave together; never in a cluster
    const int64_t slice = cs > 1 ? ((g.cols + cs - 1) / cs + 3) / 4 * 4 : g.cols;
    const int64_t begin = slice * rank;
    const int width = (int)(begin >= g.cols ? 0 : (g.cols - begin < slice ? g.cols - begin : slice));
    int turn = 0;
    float v[E], fv[E];
    load_share<T, E, VEC>(v, x.p + row * x.stride + begin, width, tid);
    float4 st = make_float4(0.0f, 1.0f, 0.0f, 1.0f);
    if (f.p) {
        load_share<T, E, VEC>(fv, f.p + row * f.stride + begin, width, tid);
        if (g.post_kind != CTB_NORM_NONE) row_statistics<THREADS, T, E>(fv, g.post_kind, g.post_eps, g.inv_cols, sh, turn, cs, &st.x, &st.y);
        const int64_t group = g.gate_mode == kGateNone ? 0 : row / g.gate_rows;
        const float* gate = g.gate.p + group * g.gate.stride;
        const float one_gate = g.gate_mode == kGateScalar ? gate[0] * g.scale : g.scale;
#pragma unroll
        for (int i = 0; i < E / VEC; ++i) {
            const int c = col_of<T, VEC>(i, tid);
            if (c < width) {
                float n[VEC], out[VEC];
#pragma unroll
                for (int k = 0; k < VEC; ++k) n[k] = fv[i * VEC + k];
                if (g.post_kind != CTB_NORM_NONE) {
#pragma unroll
                    for (int k = 0; k < VEC; ++k) n[k] = (n[k] - st.x) * st.y;
                    if (g.post_weight) {
                        float w[VEC];
                        load_part<T, VEC>(w, g.post_weight + begin, c);
#pragma unroll
                        for (int k = 0; k < VEC; ++k) n[k] = n[k] * w[k];
                    }
                    if (g.post_bias) {
                        float w[VEC];
                        load_part<T, VEC>(w, g.post_bias + begin, c);
#pragma unroll
                        for (int k = 0; k < VEC; ++k) n[k] = n[k] + w[k];
                    }
                }
                if (g.gate_mode == kGateRow) {
                    float w[VEC];
                    load_part<T, VEC>(w, gate + begin, c);
#pragma unroll
                    for (int k = 0; k < VEC; ++k) n[k] = n[k] * w[k];
                }
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    out[k] = fmaf(one_gate, n[k], v[i * VEC + k]);
                    v[i * VEC + k] = out[k];
                }
                store_part<VEC>(y + row * g.cols + begin, c, out);
            }
        }
    }
    if (g.pre_kind != CTB_NORM_NONE) {
        row_statistics<THREADS, T, E>(v, g.pre_kind, g.pre_eps, g.inv_cols, sh, turn, cs, &st.z, &st.w);
#pragma unroll
        for (int i = 0; i < E / VEC; ++i) {
            const int c = col_of<T, VEC>(i, tid);
            if (c < width) {
                float n[VEC];
#pragma unroll
                for (int k = 0; k < VEC; ++k) n[k] = (v[i * VEC + k] - st.z) * st.w;
                if (g.pre_weight) {
                    float w[VEC];
                    load_part<T, VEC>(w, g.pre_weight + begin, c);
#pragma unroll
                    for (int k = 0; k < VEC; ++k) n[k] = n[k] * w[k];
                }
                if (g.pre_bias) {
                    float w[VEC];
                    load_part<T, VEC>(w, g.pre_bias + begin, c);
#pragma unroll
                    for (int k = 0; k < VEC; ++k) n[k] = n[k] + w[k];
                }
                store_part<VEC>(h + row * g.cols + begin, c, n);
            }
        }
    }
    if (stats && tid == 0 && rank == 0) *reinterpret_cast<float4*>(stats + row * 4) = st;
}

// ---- backward -------------------------------------------------------------------------------------------
// Teams walk consecutive rows.  While a row is being worked on, the next one's operands are on their way
// into shared memory (cp.async): each thread copies and later reads its own columns only, so there is
// nothing to synchronise but the thread's own copies.  Column sums (weights, biases, a gate shared by
// rows) stay in registers until the team's last row — a shared gate's until its last row in the team —
// and are then written as partials; a second launch adds the partials in order.
template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
    const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(d), "l"(src) : "memory");
}

enum { kInF = 0, kInY = 1, kInDy = 2, kInDh = 3, kInGate = 4, kInCount = 5 };

struct ResidualBwd {
    ResidualNormGeom g;
    RowsIn in[kInCount];            // p == NULL: not read; [kInGate] only where the gate has a row for every row
    const float* stats;
    ResidualNormGrads out;
    int32_t shared_gate;            // the gate's gradient is summed over rows (kGateRow, gate_rows > 1)
    int64_t teams;
    float* part;                    // [pre_weight, pre_bias, post_weight, post_bias][teams][cols]
    float* gate_part;               // [teams + groups][cols or 1]: slot team + group
};

template <int E, int VEC>
__device__ __forceinline__ void read_staged(float (&v)[VEC], const float* stage, int threads, int i) {
    if constexpr (VEC == 4) {
        const float4 q = reinterpret_cast<const float4*>(stage)[i * threads + threadIdx.x];
        v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
        v[0] = stage[i * threads + threadIdx.x];
    }
}

// POST: sums for the post norm's weight and bias; BIAS: sums for biases; GATE: sums for a gate row shared by rows.
template <int THREADS, int T, int E, int VEC, bool POST, bool BIAS, bool GATE>
__global__ void __launch_bounds__(THREADS, 512 / THREADS)
residual_norm_backward_kernel(const __grid_constant__ ResidualBwd a, int cs) {
    extern __shared__ __align__(16) float staged[];      // [2][kInCount][E][THREADS]
    __shared__ TeamSlots<THREADS, 3, float> sh;
    constexpr int STAGE = E * THREADS;
    const ResidualNormGeom& g = a.g;
    const int tid = threadIdx.x % T;
    const uint32_t rank = cs > 1 ? cluster_rank() : 0;
    const int64_t team = (int64_t)(blockIdx.x / cs) * (THREADS / T) + threadIdx.x / T;
    if (team >= a.teams) return;                         // whole teams leave together; never in a cluster
    const int64_t lo = g.rows * team / a.teams, hi = g.rows * (team + 1) / a.teams;
    const int64_t slice = cs > 1 ? ((g.cols + cs - 1) / cs + 3) / 4 * 4 : g.cols;
    const int64_t begin = slice * rank;
    const int width = (int)(begin >= g.cols ? 0 : (g.cols - begin < slice ? g.cols - begin : slice));
    const float inv = (float)g.inv_cols;
    int turn = 0;

    float pre_w[E], pre_b[BIAS ? E : 1], post_w[POST ? E : 1], post_b[POST && BIAS ? E : 1], gate_sum[GATE ? E : 1];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        pre_w[e] = 0.0f;
        if (BIAS) pre_b[e] = 0.0f;
        if (POST) post_w[e] = 0.0f;
        if (POST && BIAS) post_b[e] = 0.0f;
        if (GATE) gate_sum[e] = 0.0f;
    }
    float scalar_gate_sum = 0.0f;
    const bool shared_gate = GATE && a.shared_gate;
    const bool scalar_gate = g.gate_mode == kGateScalar && a.out.gate;
    const bool want_n = g.gate_mode != kGateNone && a.out.gate;

    auto fetch = [&](int64_t row, int which) {
#pragma unroll
        for (int q = 0; q < kInCount; ++q) {
            if (!a.in[q].p) continue;
            const float* src = a.in[q].p + row * a.in[q].stride + begin;
            float* dst = staged + (which * kInCount + q) * STAGE;
#pragma unroll
            for (int i = 0; i < E / VEC; ++i) {
                const int c = col_of<T, VEC>(i, tid);
                if (c < width) copy_async<VEC * 4>(dst + (i * THREADS + threadIdx.x) * VEC, src + c);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const float4* stats = reinterpret_cast<const float4*>(a.stats);
    float4 next_st = make_float4(0.0f, 1.0f, 0.0f, 1.0f);
    if (lo < hi) {
        fetch(lo, 0);
        next_st = stats[lo];
    }
    for (int64_t row = lo; row < hi; ++row) {
        const int which = (int)((row - lo) & 1);
        const float4 st = next_st;
        if (row + 1 < hi) {
            fetch(row + 1, which ^ 1);
            next_st = stats[row + 1];
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        const float* in = staged + which * (kInCount * STAGE);
        float dx[E];                                     // first a = dh * w, then the gradient of y and x
        float hat[E];
        float m1 = 0.0f, m2 = 0.0f;
        if (g.pre_kind != CTB_NORM_NONE) {
            float s[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < E / VEC; ++i) {
                const int c = col_of<T, VEC>(i, tid);
                float yv[VEC], dh[VEC], w[VEC];
#pragma unroll
                for (int k = 0; k < VEC; ++k) { yv[k] = st.z; dh[k] = 0.0f; w[k] = 1.0f; }
                if (c < width) {
                    read_staged<E, VEC>(yv, in + kInY * STAGE, THREADS, i);
                    read_staged<E, VEC>(dh, in + kInDh * STAGE, THREADS, i);
                    if (g.pre_weight) load_part<T, VEC>(w, g.pre_weight + begin, c);
                }
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    const int e = i * VEC + k;
                    hat[e] = (yv[k] - st.z) * st.w;
                    pre_w[e] = fmaf(dh[k], hat[e], pre_w[e]);
                    if (BIAS) pre_b[e] = pre_b[e] + dh[k];
                    dx[e] = dh[k] * w[k];
                    s[0] = s[0] + dx[e];
                    s[1] = fmaf(dx[e], hat[e], s[1]);
                }
            }
            team_fold<FoldSum, THREADS, T>(s, sh, turn, cs);
            m1 = g.pre_kind == CTB_NORM_LAYER ? s[0] * inv : 0.0f;
            m2 = s[1] * inv;
        }
        const int64_t group = g.gate_mode == kGateNone ? 0 : row / g.gate_rows;
        const float* gate = g.gate.p + group * g.gate.stride;
        const float one_gate = g.gate_mode == kGateScalar ? gate[0] * g.scale : g.scale;
        float s[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < E / VEC; ++i) {
            const int c = col_of<T, VEC>(i, tid);
            if (c < width) {
                float dy[VEC], fv[VEC], part[VEC], w[VEC];
#pragma unroll
                for (int k = 0; k < VEC; ++k) dy[k] = 0.0f;
                if (a.in[kInDy].p) read_staged<E, VEC>(dy, in + kInDy * STAGE, THREADS, i);
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    const int e = i * VEC + k;
                    part[k] = dy[k];
                    if (g.pre_kind != CTB_NORM_NONE) part[k] = fmaf(st.w, dx[e] - m1 - hat[e] * m2, dy[k]);
                }
                if (a.out.x) store_part<VEC>(a.out.x + row * g.cols + begin, c, part);
#pragma unroll
                for (int k = 0; k < VEC; ++k) { fv[k] = 0.0f; w[k] = 1.0f; }
                if (a.in[kInF].p) read_staged<E, VEC>(fv, in + kInF * STAGE, THREADS, i);
                // fhat, and n where the gate's gradient wants it
                if (POST && g.post_kind != CTB_NORM_NONE) {
#pragma unroll
                    for (int k = 0; k < VEC; ++k) fv[k] = (fv[k] - st.x) * st.y;
                    if (g.post_weight) load_part<T, VEC>(w, g.post_weight + begin, c);
                }
                float gv[VEC];
#pragma unroll
                for (int k = 0; k < VEC; ++k) gv[k] = one_gate;
                if (g.gate_mode == kGateRow) {
                    float q[VEC];
                    if (a.in[kInGate].p) read_staged<E, VEC>(q, in + kInGate * STAGE, THREADS, i);
                    else load_part<T, VEC>(q, gate + begin, c);
#pragma unroll
                    for (int k = 0; k < VEC; ++k) gv[k] = q[k] * g.scale;
                }
                if (want_n) {
                    float b[VEC], n[VEC];
#pragma unroll
                    for (int k = 0; k < VEC; ++k) b[k] = 0.0f;
                    if (POST && g.post_bias) load_part<T, VEC>(b, g.post_bias + begin, c);
#pragma unroll
                    for (int k = 0; k < VEC; ++k) n[k] = fmaf(fv[k], w[k], b[k]) * (g.scale * part[k]);
                    if (g.gate_mode == kGateScalar) {
#pragma unroll
                        for (int k = 0; k < VEC; ++k) s[2] = s[2] + n[k];
                    } else if (shared_gate) {
#pragma unroll
                        for (int k = 0; k < VEC; ++k) gate_sum[GATE ? i * VEC + k : 0] += n[k];
                    } else {
                        store_part<VEC>(a.out.gate + row * g.cols + begin, c, n);
                    }
                }
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    const int e = i * VEC + k;
                    const float dn = part[k] * gv[k];
                    if (POST) {
                        post_w[e] = fmaf(dn, fv[k], post_w[e]);
                        if (BIAS) post_b[e] = post_b[e] + dn;
                    }
                    dx[e] = dn * w[k];                   // from here on: c = dn * w_post
                    hat[e] = fv[k];
                    if (POST) {
                        s[0] = s[0] + dx[e];
                        s[1] = fmaf(dx[e], fv[k], s[1]);
                    }
                }
            }
        }
        if ((POST && g.post_kind != CTB_NORM_NONE) || scalar_gate) team_fold<FoldSum, THREADS, T>(s, sh, turn, cs);
        if (a.out.f) {
            const float c1 = POST && g.post_kind == CTB_NORM_LAYER ? s[0] * inv : 0.0f, c2 = s[1] * inv;
#pragma unroll
            for (int i = 0; i < E / VEC; ++i) {
                const int c = col_of<T, VEC>(i, tid);
                if (c < width) {
                    float part[VEC];
#pragma unroll
                    for (int k = 0; k < VEC; ++k) {
                        const int e = i * VEC + k;
                        part[k] = POST && g.post_kind != CTB_NORM_NONE ? st.y * (dx[e] - c1 - hat[e] * c2) : dx[e];
                    }
                    store_part<VEC>(a.out.f + row * g.cols + begin, c, part);
                }
            }
        }
        // a gate that rows share: its sum so far goes out when the next row belongs to another gate row
        if (scalar_gate || shared_gate) {
            scalar_gate_sum = scalar_gate_sum + s[2];
            if (row + 1 == hi || (row + 1) / g.gate_rows != group) {
                if (shared_gate) {
#pragma unroll
                    for (int i = 0; i < E / VEC; ++i) {
                        const int c = col_of<T, VEC>(i, tid);
                        float part[VEC];
#pragma unroll
                        for (int k = 0; k < VEC; ++k) {
                            part[k] = gate_sum[GATE ? i * VEC + k : 0];
                            gate_sum[GATE ? i * VEC + k : 0] = 0.0f;
                        }
                        if (c < width) store_part<VEC>(a.gate_part + (team + group) * g.cols + begin, c, part);
                    }
                } else if (tid == 0 && rank == 0) {
                    a.gate_part[team + group] = scalar_gate_sum;
                }
                scalar_gate_sum = 0.0f;
            }
        }
    }
    // column sums of the team
    auto put = [&](int at, const float* sum) {
        float* part_row = a.part + ((int64_t)at * a.teams + team) * g.cols + begin;
#pragma unroll
        for (int i = 0; i < E / VEC; ++i) {
            const int c = col_of<T, VEC>(i, tid);
            float part[VEC];
#pragma unroll
            for (int k = 0; k < VEC; ++k) part[k] = sum[i * VEC + k];
            if (c < width) store_part<VEC>(part_row, c, part);
        }
    };
    if (a.out.pre_weight) put(0, pre_w);
    if (BIAS && a.out.pre_bias) put(1, pre_b);
    if (POST && a.out.post_weight) put(2, post_w);
    if (POST && BIAS && a.out.post_bias) put(3, post_b);
}

// out[c] = sum over partial rows [first, last] of part[row][c], added in row order within eight runs that
// are joined in order, in fp64.  Jobs: the weight vectors, then one for every gate group.
struct FoldJobs {
    const float* part[4];
    float* out[4];
    int32_t vectors;
    int64_t teams, cols;
    const float* gate_part;
    float* gate;
    int64_t groups, gate_width, gate_rows, rows;
    int64_t vector_blocks, tiles, gate_tiles;
};

constexpr int kFoldCols = 32, kFoldRuns = 8;

__global__ void __launch_bounds__(kFoldCols * kFoldRuns)
residual_norm_fold_kernel(const __grid_constant__ FoldJobs j) {
    __shared__ double sums[kFoldRuns][kFoldCols];
    const float* part;
    float* out;
    int64_t first = 0, last = j.teams - 1, width = j.cols, tile;
    const int64_t b = blockIdx.x;
    if (b < j.vector_blocks) {
        const int v = (int)(b / j.tiles);
        tile = b % j.tiles;
        part = j.part[v];
        out = j.out[v];
    } else {
        const int64_t group = (b - j.vector_blocks) / j.gate_tiles;
        tile = (b - j.vector_blocks) % j.gate_tiles;
        // the teams whose rows meet the group's: team t has rows [rows * t / teams, rows * (t + 1) / teams)
        const int64_t r0 = group * j.gate_rows, r1 = r0 + j.gate_rows - 1;
        first = ((r0 + 1) * j.teams - 1) / j.rows + group;
        last = ((r1 + 1) * j.teams - 1) / j.rows + group;
        width = j.gate_width;
        part = j.gate_part;
        out = j.gate + group * width;
    }
    const int64_t c = tile * kFoldCols + threadIdx.x;
    const int64_t run = (last - first + kFoldRuns) / kFoldRuns;
    double sum = 0.0;
    if (c < width)
        for (int64_t r = first + threadIdx.y * run; r < first + (threadIdx.y + 1) * run && r <= last; ++r) sum = sum + (double)part[r * width + c];
    sums[threadIdx.y][threadIdx.x] = sum;
    __syncthreads();
    if (threadIdx.y == 0 && c < width) {
#pragma unroll
        for (int i = 1; i < kFoldRuns; ++i) sum = sum + sums[i][threadIdx.x];
        out[c] = (float)sum;
    }
}

// ---- host -----------------------------------------------------------------------------------------------
bool rows_aligned(const RowsIn& r) { return !r.p || (is_aligned(r.p, 16) && r.stride % 4 == 0); }

// CTAs of a cluster for `cols` columns when one CTA holds `per_cta`.
int cluster_for(int64_t cols, int64_t per_cta) {
    int cs = 1;
    while ((int64_t)cs * per_cta < cols) cs *= 2;
    // slices are rounded up to four columns
    if (cs > 1 && ((cols + cs - 1) / cs + 3) / 4 * 4 > per_cta) cs *= 2;
    return cs;
}

template <int THREADS, int T, int E, int VEC>
int forward_as(const ResidualNormGeom& g, RowsIn x, RowsIn f, float* y, float* h, float* stats, cudaStream_t st) {
    const int cs = T == THREADS ? cluster_for(g.cols, (int64_t)T * E) : 1;
    return launch_clusters("residual_norm", residual_norm_kernel<THREADS, T, E, VEC>, ceil_div(g.rows, (int64_t)(THREADS / T)) * cs, THREADS, 0, cs, st,
                           g, x, f, y, h, stats, cs);
}

template <int THREADS, int T, int E, int VEC, bool POST, bool BIAS, bool GATE>
int backward_as(const ResidualBwd& a, int cs, cudaStream_t st) {
    return launch_clusters("residual_norm", residual_norm_backward_kernel<THREADS, T, E, VEC, POST, BIAS, GATE>, ceil_div(a.teams, (int64_t)(THREADS / T)) * cs,
                           THREADS, (size_t)2 * kInCount * E * THREADS * sizeof(float), cs, st, a, cs);
}

constexpr int kBwdShare = 8;                             // columns per thread

template <int THREADS, int T>
int backward_select(const ResidualBwd& a, bool vec, bool post, bool bias, bool gate, int cs, cudaStream_t st) {
    // rows that cannot be read in 16-byte vectors: one instantiation with every sum
    if (!vec) return backward_as<THREADS, T, kBwdShare, 1, true, true, true>(a, cs, st);
    if (post) {
        if (bias) return gate ? backward_as<THREADS, T, kBwdShare, 4, true, true, true>(a, cs, st) : backward_as<THREADS, T, kBwdShare, 4, true, true, false>(a, cs, st);
        return gate ? backward_as<THREADS, T, kBwdShare, 4, true, false, true>(a, cs, st) : backward_as<THREADS, T, kBwdShare, 4, true, false, false>(a, cs, st);
    }
    if (bias) return gate ? backward_as<THREADS, T, kBwdShare, 4, false, true, true>(a, cs, st) : backward_as<THREADS, T, kBwdShare, 4, false, true, false>(a, cs, st);
    return gate ? backward_as<THREADS, T, kBwdShare, 4, false, false, true>(a, cs, st) : backward_as<THREADS, T, kBwdShare, 4, false, false, false>(a, cs, st);
}

int bwd_team_threads(int64_t cols) { return cols <= 32 * kBwdShare ? 32 : cols <= 128 * kBwdShare ? 128 : cols <= 256 * kBwdShare ? 256 : 512; }
// Teams that walk the rows: as many as the machine holds at once (512 threads per SM), at most one per row.
int64_t bwd_teams(int64_t rows, int64_t cols, int sm_count) {
    const int t = bwd_team_threads(cols);
    int64_t teams = (int64_t)sm_count * (512 / t) / cluster_for(cols, (int64_t)t * kBwdShare);
    if (teams > rows) teams = rows;
    return teams < 1 ? 1 : teams;
}
constexpr int kMaxSms = 256;                             // what the size query, which names no device, allows for

}  // namespace

size_t residual_norm_workspace_bytes(int64_t rows, int64_t cols, int64_t gate_groups, int64_t gate_width) {
    const int64_t teams = bwd_teams(rows, cols, kMaxSms);
    return ((size_t)(4 * teams) * (size_t)cols + (size_t)(gate_groups > 0 ? teams + gate_groups : 0) * (size_t)gate_width) * sizeof(float);
}

int launch_residual_norm(const ResidualNormGeom& geom, RowsIn x, RowsIn f, float* y, float* h, float* stats, cudaStream_t st) {
    if (geom.rows == 0 || geom.cols == 0) return CTB_OK;
    ResidualNormGeom g = geom;
    g.inv_cols = 1.0 / (double)g.cols;
    const bool vec = g.cols % 4 == 0 && rows_aligned(x) && rows_aligned(f) && (!y || is_aligned(y, 16)) && (!h || is_aligned(h, 16)) &&
                     is_aligned(g.post_weight, 16) && is_aligned(g.post_bias, 16) && is_aligned(g.pre_weight, 16) && is_aligned(g.pre_bias, 16) &&
                     (g.gate_mode != kGateRow || rows_aligned(g.gate));
    if (!vec) {
        if (g.cols <= 256) return forward_as<256, 32, 8, 1>(g, x, f, y, h, stats, st);
        if (g.cols <= 2048) return forward_as<256, 128, 16, 1>(g, x, f, y, h, stats, st);
        return forward_as<512, 512, 16, 1>(g, x, f, y, h, stats, st);
    }
    if (g.cols <= 256) return forward_as<256, 32, 8, 4>(g, x, f, y, h, stats, st);
    if (g.cols <= 512) return forward_as<256, 32, 16, 4>(g, x, f, y, h, stats, st);
    if (g.cols <= 1024) return forward_as<256, 32, 32, 4>(g, x, f, y, h, stats, st);
    if (g.cols <= 2048) return forward_as<256, 128, 16, 4>(g, x, f, y, h, stats, st);
    if (g.cols <= 4096) return forward_as<256, 256, 16, 4>(g, x, f, y, h, stats, st);
    return forward_as<512, 512, 16, 4>(g, x, f, y, h, stats, st);
}

int launch_residual_norm_backward(const ResidualNormGeom& g, RowsIn f, RowsIn y, const float* stats, RowsIn grad_y, RowsIn grad_h,
                                  const ResidualNormGrads& out, void* workspace, cudaStream_t st) {
    const int64_t groups = g.rows / g.gate_rows;
    const int64_t gate_width = g.gate_mode == kGateRow ? g.cols : 1;
    if (g.rows == 0 || g.cols == 0) return CTB_OK;
    DeviceInfo di;
    if (int rc = current_device_info(&di)) return rc;
    ResidualBwd a{};
    a.g = g;
    a.g.inv_cols = 1.0 / (double)g.cols;
    const bool want_gate = out.gate && g.gate_mode != kGateNone;
    const bool post = g.post_kind != CTB_NORM_NONE;
    const bool shared_gate = want_gate && g.gate_mode == kGateRow && g.gate_rows > 1;
    if (f.p && (post || want_gate)) a.in[kInF] = f;
    if (g.pre_kind != CTB_NORM_NONE) { a.in[kInY] = y; a.in[kInDh] = grad_h; }
    a.in[kInDy] = grad_y;
    if (g.gate_mode == kGateRow && g.gate_rows == 1) a.in[kInGate] = g.gate;
    a.stats = stats;
    a.out = out;
    a.shared_gate = shared_gate;
    a.teams = bwd_teams(g.rows, g.cols, di.sm_count < kMaxSms ? di.sm_count : kMaxSms);
    a.part = (float*)workspace;
    a.gate_part = a.part + 4 * a.teams * g.cols;
    bool vec = g.cols % 4 == 0 && (!out.x || is_aligned(out.x, 16)) && (!out.f || is_aligned(out.f, 16)) && (!out.gate || is_aligned(out.gate, 16)) &&
               is_aligned(g.post_weight, 16) && is_aligned(g.post_bias, 16) && is_aligned(g.pre_weight, 16) &&
               (g.gate_mode != kGateRow || rows_aligned(g.gate));
    for (const RowsIn& r : a.in) vec = vec && rows_aligned(r);
    const int t = bwd_team_threads(g.cols), cs = cluster_for(g.cols, (int64_t)t * kBwdShare);
    const bool bias = out.pre_bias || out.post_bias;
    int rc;
    if (t == 32) rc = backward_select<256, 32>(a, vec, post, bias, shared_gate, cs, st);
    else if (t == 128) rc = backward_select<256, 128>(a, vec, post, bias, shared_gate, cs, st);
    else if (t == 256) rc = backward_select<256, 256>(a, vec, post, bias, shared_gate, cs, st);
    else rc = backward_select<512, 512>(a, vec, post, bias, shared_gate, cs, st);
    if (rc) return rc;

    FoldJobs j{};
    float* const sums[4] = {out.pre_weight, out.pre_bias, out.post_weight, out.post_bias};
    for (int v = 0; v < 4; ++v)
        if (sums[v]) {
            j.part[j.vectors] = a.part + (int64_t)v * a.teams * g.cols;
            j.out[j.vectors++] = sums[v];
        }
    j.teams = a.teams;
    j.cols = g.cols;
    j.tiles = ceil_div(g.cols, kFoldCols);
    j.vector_blocks = j.vectors * j.tiles;
    const bool fold_gate = want_gate && (g.gate_mode == kGateScalar || g.gate_rows > 1);
    if (fold_gate) {
        j.gate_part = a.gate_part;
        j.gate = out.gate;
        j.groups = groups;
        j.gate_width = gate_width;
        j.gate_rows = g.gate_rows;
        j.rows = g.rows;
        j.gate_tiles = ceil_div(gate_width, kFoldCols);
    }
    const int64_t blocks = j.vector_blocks + (fold_gate ? groups * j.gate_tiles : 0);
    if (blocks == 0) return CTB_OK;
    if (blocks > 0x7FFFFFFFll) return set_error(CTB_ERR_LIMIT, "residual_norm_backward: too many gate rows for one launch");
    residual_norm_fold_kernel<<<(unsigned)blocks, dim3(kFoldCols, kFoldRuns), 0, st>>>(j);
    return cuda_error(cudaGetLastError(), "residual_norm_backward launch");
}

}  // namespace ctb
