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
// exchange their sums through distributed shared memory); every operand is read once.  Measured (share of the
// 6.54 TB/s of a copy, four sets of buffers in turn): forward with one norm [4096, 8192] 82 us, 6.5 TB/s (1.00), with RMS
// norms on both sides [32768, 768] 65 us (0.95), [4096, 8192] 86 us (0.96), [4096, 5120] 61 us (0.85: two folds one behind the
// other); backward with one norm [16384, 1536] 84 us (0.92), RMS on both sides [4096, 5120] 87 us (0.88), with a gate for every
// element 116 us (0.89), [4096, 8192] in clusters 189 us (0.65); LayerNorms on both sides [16384, 1024] 70 us (0.88),
// [8192, 4096] 177 us (0.69), registers for four sums per column leave 12 warps on an SM; rows of odd length go element by
// element: [16000, 1999] with one norm forward 97 us (0.80), backward 137 us (0.72), two LayerNorms 0.53 and 0.36.
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

template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
    const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(d), "l"(src) : "memory");
}

// The thread's own four (or one) values of a stage slot.
template <int VEC>
__device__ __forceinline__ void read_own(float (&v)[VEC], const float* p) {
    if constexpr (VEC == 4) {
        const float4 q = *reinterpret_cast<const float4*>(p);
        v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
        v[0] = *p;
    }
}

// ---- forward ------------------------------------------------------------------------------------------
// v^-1/2, also where v is beyond Float32 or subnormal there (rows of 1e20, or of 1e-20 without an eps).
__device__ __forceinline__ float inverse_root(double v) {
    if (v > 1e-37 && v < 1e38) return __frsqrt_rn((float)v);
    return (float)rsqrt(v);
}
// mean and rstd of a row from fp64 sums of v and v^2: one sum over the team instead of two, and no
// cancellation that fp64 would notice until |mean| / sigma is about 1e6.
template <int THREADS, int T, int E>
__device__ __forceinline__ void row_statistics(const float (&v)[E], int kind, float eps, double inv_cols, TeamSlots<THREADS, 2, double>& sh,
                                               FoldTurn& turn, float* mean, float* rstd) {
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
    team_fold<FoldSum, THREADS, T>(s, sh, turn);
    double var = s[1] * inv_cols;
    *mean = 0.0f;
    if (kind == CTB_NORM_LAYER) {
        const double m = s[0] * inv_cols;
        *mean = (float)m;
        var = fma(-m, m, var);
        if (var < 0.0) var = 0.0;
    }
    *rstd = inverse_root(var + (double)eps);
}

// Wide rows keep x in shared memory (each thread its own columns) until it is needed: 40 registers instead of
// 59, so three CTAs of 512 threads share an SM and one row's folds hide behind the loads of two others.
template <int THREADS, int T, int E, int VEC> constexpr bool kStageX = T == THREADS && E == 16 && VEC == 4;
template <int THREADS, int T, int E, int VEC> constexpr int kForwardCtas = kStageX<THREADS, T, E, VEC> ? 1536 / THREADS : T == THREADS ? 2 : 4;

template <int THREADS, int T, int E, int VEC>
__global__ void __launch_bounds__(THREADS, (kForwardCtas<THREADS, T, E, VEC>))
residual_norm_kernel(ResidualNormGeom g, RowsIn x, RowsIn f, float* __restrict__ y, float* __restrict__ h, float* __restrict__ stats, int cs) {
    __shared__ TeamSlots<THREADS, 2, double> sh;
    const TeamEntry entry(cs);
    const int tid = threadIdx.x % T;
    const uint32_t rank = cs > 1 ? cluster_rank() : 0;
    const int64_t row = (int64_t)(blockIdx.x / cs) * (THREADS / T) + threadIdx.x / T;
    if (row >= g.rows) return;                           // whole teams leave together; never in a cluster
    const int64_t slice = cs > 1 ? ((g.cols + cs - 1) / cs + 3) / 4 * 4 : g.cols;
    const int64_t begin = slice * rank;
    const int width = (int)(begin >= g.cols ? 0 : (g.cols - begin < slice ? g.cols - begin : slice));
    constexpr bool STAGED = kStageX<THREADS, T, E, VEC>;
    __shared__ __align__(16) float staged[STAGED ? E * THREADS : 1];
    float v[E], fv[E];
    if (STAGED && f.p) {
#pragma unroll
        for (int i = 0; i < E / VEC; ++i) {
            const int c = col_of<T, VEC>(i, tid);
            if (c < width) copy_async<VEC * 4>(staged + (i * THREADS + threadIdx.x) * VEC, x.p + row * x.stride + begin + c);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    } else {
        load_share<T, E, VEC>(v, x.p + row * x.stride + begin, width, tid);
    }
    FoldTurn turn = entry.met();
    float4 st = make_float4(0.0f, 1.0f, 0.0f, 1.0f);
    if (f.p) {
        load_share<T, E, VEC>(fv, f.p + row * f.stride + begin, width, tid);
        if (g.post_kind != CTB_NORM_NONE) row_statistics<THREADS, T, E>(fv, g.post_kind, g.post_eps, g.inv_cols, sh, turn, &st.x, &st.y);
        const float* gate = g.gate.p + (int64_t)fast_div((uint32_t)row, g.by_gate_rows) * g.gate.stride;
        const float one_gate = g.gate_mode == kGateScalar ? gate[0] * g.scale : g.scale;
        if (STAGED) asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
        for (int i = 0; i < E / VEC; ++i) {
            const int c = col_of<T, VEC>(i, tid);
            if (STAGED) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) v[i * VEC + k] = 0.0f;
            }
            if (c < width) {
                float n[VEC], out[VEC], xv[VEC];
                if (STAGED) read_own<VEC>(xv, staged + (i * THREADS + threadIdx.x) * VEC);
                else {
#pragma unroll
                    for (int k = 0; k < VEC; ++k) xv[k] = v[i * VEC + k];
                }
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
                    out[k] = fmaf(one_gate, n[k], xv[k]);
                    v[i * VEC + k] = out[k];
                }
                store_part<VEC>(y + row * g.cols + begin, c, out);
            }
        }
    }
    if (g.pre_kind != CTB_NORM_NONE) {
        row_statistics<THREADS, T, E>(v, g.pre_kind, g.pre_eps, g.inv_cols, sh, turn, &st.z, &st.w);
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

// A row of residual_rms_kernel (below) that is near the ends of Float32, normed before it is scaled, from memory.  A call of
// its own: inlined, it took registers from all other rows ([1000000,128] 381 us, 428 so).
template <int THREADS, int T, int VEC>
__device__ __noinline__ void residual_rms_extreme_row(const ResidualNormGeom& g, const float* x, const float* f, float* y, float* h, float* stats, int64_t row,
                                                      float rf, TeamSlots<THREADS, 4, double>& sh, FoldTurn turn) {
    const int tid = threadIdx.x % T, width = (int)g.cols;
    const float* gate = g.gate.p + (int64_t)fast_div((uint32_t)row, g.by_gate_rows) * g.gate.stride;
    const float one_gate = g.gate_mode == kGateScalar ? gate[0] * g.scale : g.scale;
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    for (int c = tid * VEC; c < width; c += T * VEC) {
        float n[VEC], k[VEC];
        load_part<T, VEC>(n, f, c);
#pragma unroll
        for (int q = 0; q < VEC; ++q) n[q] = n[q] * rf;
        if (g.post_weight) {
            load_part<T, VEC>(k, g.post_weight, c);
#pragma unroll
            for (int q = 0; q < VEC; ++q) n[q] = n[q] * k[q];
        }
        if (g.gate_mode == kGateRow) {
            load_part<T, VEC>(k, gate, c);
#pragma unroll
            for (int q = 0; q < VEC; ++q) n[q] = n[q] * k[q];
        }
        load_part<T, VEC>(k, x, c);
#pragma unroll
        for (int q = 0; q < VEC; ++q) {
            n[q] = fmaf(one_gate, n[q], k[q]);
            s[0] = fma((double)n[q], (double)n[q], s[0]);
        }
        store_part<VEC>(y, c, n);
    }
    team_fold<FoldSum, THREADS, T>(s, sh, turn);
    const float ry = inverse_root(s[0] * g.inv_cols + (double)g.pre_eps);
    for (int c = tid * VEC; c < width; c += T * VEC) {
        float n[VEC], k[VEC];
        load_part<T, VEC>(n, y, c);                      // what this thread stored
#pragma unroll
        for (int q = 0; q < VEC; ++q) n[q] = n[q] * ry;
        if (g.pre_weight) {
            load_part<T, VEC>(k, g.pre_weight, c);
#pragma unroll
            for (int q = 0; q < VEC; ++q) n[q] = n[q] * k[q];
        }
        if (g.pre_bias) {
            load_part<T, VEC>(k, g.pre_bias, c);
#pragma unroll
            for (int q = 0; q < VEC; ++q) n[q] = n[q] + k[q];
        }
        store_part<VEC>(h, c, n);
    }
    if (stats && tid == 0) *reinterpret_cast<float4*>(stats) = make_float4(0.0f, rf, 0.0f, ry);
}

// RMS norms on both sides need one fold per row instead of two: with u = scale * gate * w_post * f the stream is
// y = x + rstd_f * u, so
//     sum(y^2) = sum(x^2) + 2 rstd_f sum(x u) + rstd_f^2 sum(u^2)
// and all four sums (fp64) are known after one pass over x and f.  (A bias behind the first norm would have to be
// rounded into x before that norm is known, one rounding more; such rows take the general kernel.)  Where the block's output cancels the stream to
// less than a thousandth, those sums would lose what the norm magnifies: such a row takes the second fold; so does a row near
// the ends of Float32, whose u overflows or is subnormal where n itself is neither, and it is normed before it is scaled.  For
// rows of up to 2048 columns: [16384, 1536] 69 us against 74; wider rows, which hold more of it per thread, lose ([4096, 4096]
// 60 against 52).
template <int THREADS, int T, int E, int VEC>
__global__ void __launch_bounds__(THREADS, E == 2 ? 6 : E == 4 ? 5 : 4)
residual_rms_kernel(const __grid_constant__ ResidualNormGeom g, RowsIn x, RowsIn f, float* __restrict__ y, float* __restrict__ h, float* __restrict__ stats) {
    __shared__ TeamSlots<THREADS, 4, double> sh;
    const int tid = threadIdx.x % T;
    const int64_t row = (int64_t)blockIdx.x * (THREADS / T) + threadIdx.x / T;
    if (row >= g.rows) return;                           // whole teams leave together
    const int width = (int)g.cols;
    FoldTurn turn = TeamEntry(1).met();
    float xv[E], u[E];
    load_share<T, E, VEC>(xv, x.p + row * x.stride, width, tid);
    load_share<T, E, VEC>(u, f.p + row * f.stride, width, tid);
    const float* gate = g.gate.p + (int64_t)fast_div((uint32_t)row, g.by_gate_rows) * g.gate.stride;
    const float one_gate = g.gate_mode == kGateScalar ? gate[0] * g.scale : g.scale;
    double s[4] = {0.0, 0.0, 0.0, 0.0};                  // f^2, x^2, x u, u^2
#pragma unroll
    for (int i = 0; i < E / VEC; ++i) {
        const int c = col_of<T, VEC>(i, tid);
        if (c < width) {
            float k[VEC];
#pragma unroll
            for (int q = 0; q < VEC; ++q) k[q] = one_gate;
            if (g.gate_mode == kGateRow) {
                load_part<T, VEC>(k, gate, c);
#pragma unroll
                for (int q = 0; q < VEC; ++q) k[q] = k[q] * g.scale;
            }
            if (g.post_weight) {
                float w[VEC];
                load_part<T, VEC>(w, g.post_weight, c);
#pragma unroll
                for (int q = 0; q < VEC; ++q) k[q] = k[q] * w[q];
            }
#pragma unroll
            for (int q = 0; q < VEC; ++q) {
                const double fd = u[i * VEC + q], xd = xv[i * VEC + q];
                u[i * VEC + q] = u[i * VEC + q] * k[q];
                const double ud = u[i * VEC + q];
                s[0] = fma(fd, fd, s[0]);
                s[1] = fma(xd, xd, s[1]);
                s[2] = fma(xd, ud, s[2]);
                s[3] = fma(ud, ud, s[3]);
            }
        }
    }
    team_fold<FoldSum, THREADS, T>(s, sh, turn);
    const float rf = inverse_root(s[0] * g.inv_cols + (double)g.post_eps);
    const double r = rf;
    double sy = fma(r, fma(r, s[3], 2.0 * s[2]), s[1]);
    // (both conditions are the same in every thread of the team)
    if (s[0] < INFINITY && (!(s[3] < INFINITY) || rf > 1048576.0f)) {
        residual_rms_extreme_row<THREADS, T, VEC>(g, x.p + row * x.stride, f.p + row * f.stride, y + row * g.cols, h + row * g.cols,
                                                  stats ? stats + row * 4 : nullptr, row, rf, sh, turn);
        return;
    }
    if (!(sy >= 1e-6 * s[1])) {                          // also where infinities in x and f leave no number
        double square = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const double d = col_of<T, VEC>(e / VEC, tid) < width ? fmaf(rf, u[e], xv[e]) : 0.0f;
            square = fma(d, d, square);
        }
        s[0] = square;
        s[1] = s[2] = s[3] = 0.0;
        team_fold<FoldSum, THREADS, T>(s, sh, turn);
        sy = s[0];
    }
    const float ry = inverse_root(sy * g.inv_cols + (double)g.pre_eps);
#pragma unroll
    for (int i = 0; i < E / VEC; ++i) {
        const int c = col_of<T, VEC>(i, tid);
        if (c < width) {
            float out[VEC];
#pragma unroll
            for (int q = 0; q < VEC; ++q) out[q] = fmaf(rf, u[i * VEC + q], xv[i * VEC + q]);
            store_part<VEC>(y + row * g.cols, c, out);
#pragma unroll
            for (int q = 0; q < VEC; ++q) out[q] = out[q] * ry;
            if (g.pre_weight) {
                float w[VEC];
                load_part<T, VEC>(w, g.pre_weight, c);
#pragma unroll
                for (int q = 0; q < VEC; ++q) out[q] = out[q] * w[q];
            }
            if (g.pre_bias) {
                float w[VEC];
                load_part<T, VEC>(w, g.pre_bias, c);
#pragma unroll
                for (int q = 0; q < VEC; ++q) out[q] = out[q] + w[q];
            }
            store_part<VEC>(h + row * g.cols, c, out);
        }
    }
    if (stats && tid == 0) *reinterpret_cast<float4*>(stats + row * 4) = make_float4(0.0f, rf, 0.0f, ry);
}

// ---- backward -------------------------------------------------------------------------------------------
// Teams walk consecutive rows.  While a row is being worked on, the next ones' operands are on their way
// into shared memory (cp.async, a ring of two to four rows): each thread copies and later reads its own columns
// only, so there is nothing to synchronise but the thread's own copies.
//
// One fold over the team per row.  The sums that df needs contain dx, which needs sums itself; but dx is
// linear in them, dx = e - rstd_y * (m1 + yhat * m2) with e = dy + rstd_y * a, so with k = scale * gate * w_post
//     sum(k dx)      = sum(k e)      - rstd_y * (m1 * sum(k)      + m2 * sum(k yhat))
//     sum(k dx fhat) = sum(k e fhat) - rstd_y * (m1 * sum(k fhat) + m2 * sum(k fhat yhat))
// and all eight sums are taken together.  Without a LayerNorm (m1 and the mean of k dx drop out) three remain.  (As
// differences these sums are as exact as dx itself, whose elements are differences of the same size.)
//
// Column sums (weights, biases, a gate shared by rows) stay in registers, as Float32, until the team's last row — a shared
// gate's until its last row in the team — and go out as partials, which a second launch adds in order, in fp64.  A
// team has at most kTeamRows rows and a CTA at most 16 teams, so that a sum is off by no more than 256 half steps however many
// rows there are: beyond it there are several times as many CTAs as run at once ([1000000,128] 487 us, 481 with teams of 422 rows).
// (Sums of a CTA's teams in fp64 would add 0.7 us to [8192,768]'s 30.8.)
enum { kInY = 0, kInDh = 1, kInDy = 2, kInF = 3, kInGate = 4, kInCount = 5 };

struct ResidualBwd {
    ResidualNormGeom g;
    RowsIn in[kInCount];            // p == NULL: not read; [kInGate] only where the gate has a row for every row
    int32_t stages;                 // rows in the ring, 2..4
    const float* stats;
    ResidualNormGrads out;
    int32_t shared_gate;            // the gate's gradient is summed over rows (kGateRow, gate_rows > 1)
    int64_t teams;
    int64_t parts;                  // rows of partial column sums: one per CTA (column slice)
    float* part;                    // [pre_weight, pre_bias, post_weight, post_bias, gate][parts][cols]
    float* gate_part;               // [teams + groups][cols or 1]: slot team + group; gate rows that lie in one team go out directly
    int32_t one_gate_row;           // all rows share one gate row: its sums go to `part`
};

// What a launch is specialised for.  A specialised kernel (FAST) has a pre norm with a weight, the gradient of y
// and, if POST, a post norm with a weight; all of its gradients are wanted, the gate's for GATE != 0: 1 = a row
// that rows share, 2 = a row for every row, 3 = single values.  Otherwise every one of these is looked up at run time, the
// flags then only say that the sums have a place: that took 640 instructions per warp and row where the
// specialised kernel takes 360, and instructions, not bytes, bound narrow rows.
// FULL: there may be LayerNorms and biases.
template <bool FAST_, bool POST_, bool FULL_, int GATE_>
struct BwdFlags {
    static constexpr bool FAST = FAST_, POST = POST_, FULL = FULL_;
    static constexpr int GATE = GATE_;
    static constexpr int SLOTS = !FAST ? kInCount : 3 + (POST || GATE) + (GATE == 2);       // operands in a stage of the ring
};

template <int THREADS, int T, int E, int VEC, typename F>
__global__ void __launch_bounds__(THREADS, THREADS <= 320 ? 2 : 1)
residual_norm_backward_kernel(const __grid_constant__ ResidualBwd a, int cs) {
    extern __shared__ __align__(16) float staged[];      // [stages][SLOTS][E][THREADS]
    constexpr bool FAST = F::FAST, POST = F::POST, FULL = F::FULL, GATE = F::GATE == 1 || !FAST, SCALAR = F::GATE == 3;
    constexpr int SUMS = POST ? (FULL ? 8 : 4) : (FULL ? 2 : 1);
    __shared__ TeamSlots<THREADS, SUMS, float> sh;
    __shared__ TeamSlots<THREADS, 1, float> sh_gate;
    constexpr int SLOT = E * THREADS;
    constexpr int TEAMS = THREADS / T;
    const TeamEntry entry(cs);
    const ResidualNormGeom& g = a.g;
    const int tid = threadIdx.x % T;
    const uint32_t rank = cs > 1 ? cluster_rank() : 0;
    const int64_t team = (int64_t)(blockIdx.x / cs) * TEAMS + threadIdx.x / T;
    const bool present = team < a.teams;
    // (rows are fewer than 2^31, offsets are not)
    const int lo = present ? (int)(g.rows * team / a.teams) : 0, hi = present ? (int)(g.rows * (team + 1) / a.teams) : 0;
    const int64_t slice = cs > 1 ? ((g.cols + cs - 1) / cs + 3) / 4 * 4 : g.cols;
    const int64_t begin = slice * rank;
    const int width = (int)(begin >= g.cols ? 0 : (g.cols - begin < slice ? g.cols - begin : slice));
    const float inv = (float)g.inv_cols;

    float pre_w[E], pre_b[FULL ? E : 1], post_w[POST ? E : 1], post_b[POST && FULL ? E : 1], gate_sum[GATE ? E : 1];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        pre_w[e] = 0.0f;
        if (FULL) pre_b[e] = 0.0f;
        if (POST) post_w[e] = 0.0f;
        if (POST && FULL) post_b[e] = 0.0f;
        if (GATE) gate_sum[e] = 0.0f;
    }
    float scalar_gate_sum = 0.0f;
    // single gate values: a row's sum is left in shared memory by every warp (of the cluster) and added up by one
    // thread after the next row's fold, whose barrier lies in between
    auto leave = [&](float v, int parity) {
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) v = v + __shfl_xor_sync(0xffffffffu, v, off);
        const int warp = threadIdx.x >> 5;
        if ((threadIdx.x & 31) == 0) {
            float* at = &sh_gate.warps[parity][rank * (THREADS / 32) + warp][0];
            if (T == THREADS && cs > 1) store_peer(peer_shared(at, 0), v);
            else *at = v;
        }
    };
    // its sum goes to the gate's gradient when a gate value's last row (in this team) has been added
    auto collect = [&](int64_t row, int64_t of_group, int parity) {
        if (tid != 0 || rank != 0) return;
        const int first = T == THREADS ? 0 : (int)threadIdx.x / 32, count = (T == THREADS ? cs : 1) * (T / 32);
        for (int i = 0; i < count; ++i) scalar_gate_sum = scalar_gate_sum + sh_gate.warps[parity][first + i][0];
        const int64_t from = of_group * g.gate_rows, to = from + g.gate_rows;
        if (row + 1 < hi && row + 1 < to) return;
        if (from >= lo && to <= hi) a.out.gate[of_group] = scalar_gate_sum;
        else a.gate_part[team + of_group] = scalar_gate_sum;
        scalar_gate_sum = 0.0f;
    };
    const bool pre = FAST || g.pre_kind != CTB_NORM_NONE, post = FAST ? POST : g.post_kind != CTB_NORM_NONE;
    const bool has_dy = FAST || a.in[kInDy].p, has_f = FAST ? POST || F::GATE != 0 : a.in[kInF].p != nullptr;
    const bool pre_weight = FAST || g.pre_weight, post_weight = FAST ? POST : g.post_weight != nullptr;
    const bool row_gate = FAST ? F::GATE == 1 || F::GATE == 2 : g.gate_mode == kGateRow, staged_gate = FAST ? F::GATE == 2 : a.in[kInGate].p != nullptr;
    const bool want_n = FAST ? F::GATE != 0 : g.gate_mode != kGateNone && a.out.gate;
    const bool shared_gate = FAST ? F::GATE == 1 : a.shared_gate != 0;
    const bool scalar_gate = FAST ? SCALAR : g.gate_mode == kGateScalar && a.out.gate;

    // Weights, and a gate row that rows share, stay in registers where those suffice (beside the sums of two biases only
    // with 170 of them: [16384, 1536] 134 us without, 101 with):
    // with most of the SM's memory given to the ring, L1 is too small to serve them every row.
    constexpr bool HOLD = FAST && (!FULL || !POST || THREADS <= 384);
    float w_pre[HOLD ? E : 1], w_post[HOLD && POST ? E : 1], w_gate[HOLD && F::GATE == 1 ? E : 1];
    auto hold = [&](float* v, const float* row) {
#pragma unroll
        for (int i = 0; i < E / VEC; ++i) {
            const int c = col_of<T, VEC>(i, tid);
            float w[VEC];
#pragma unroll
            for (int q = 0; q < VEC; ++q) w[q] = 0.0f;
            if (c < width) load_part<T, VEC>(w, row + begin, c);
#pragma unroll
            for (int q = 0; q < VEC; ++q) v[i * VEC + q] = w[q];
        }
    };
    if constexpr (HOLD) {
        hold(w_pre, g.pre_weight);
        if constexpr (POST) hold(w_post, g.post_weight);
    }

    // the thread's place in each operand's next row to fetch, and in its own stage slots
    const float* next[kInCount];
#pragma unroll
    for (int q = 0; q < kInCount; ++q) next[q] = a.in[q].p + lo * a.in[q].stride + begin + tid * VEC;
    float* const mine = staged + threadIdx.x * VEC;
    int fetched = lo;
    auto fetch = [&](int stage_at) {                     // always commits, so that groups count rows
        if (fetched < hi) {
#pragma unroll
            for (int q = 0; q < F::SLOTS; ++q) {
                constexpr int kinds[kInCount] = {kInY, kInDh, kInDy, kInF, kInGate};
                const int op = kinds[q];
                if (!FAST && !a.in[op].p) continue;
#pragma unroll
                for (int i = 0; i < E / VEC; ++i)
                    if (col_of<T, VEC>(i, tid) < width) copy_async<VEC * 4>(mine + stage_at + q * SLOT + i * THREADS * VEC, next[op] + i * T * VEC);
                next[op] += a.in[op].stride;
            }
            ++fetched;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    constexpr int STAGE = F::SLOTS * SLOT;
    const int ring = a.stages * STAGE;
    for (int s = 0; s + 1 < a.stages; ++s) fetch(s * STAGE);
    int group = (int)fast_div((uint32_t)lo, g.by_gate_rows);
    int left = (int)((group + 1) * g.gate_rows - lo);    // rows of this gate row that are still to come
    const float4* stats = reinterpret_cast<const float4*>(a.stats) + lo;
    float4 next_st = make_float4(0.0f, 1.0f, 0.0f, 1.0f);
    if (lo < hi) next_st = *stats;
    int stage_at = 0, ahead_at = (a.stages - 1) * STAGE;
    FoldTurn turn = entry.met(), gate_turn = turn;
    for (int row = lo; row < hi; ++row) {
        const float4 st = next_st;
        fetch(ahead_at);                                 // into the place of the row before this one, which is done with
        if (row + 1 < hi) next_st = *++stats;
        float w_row[HOLD ? 1 : E];                       // ahead of the wait for the row
        if constexpr (!HOLD) {
#pragma unroll
            for (int i = 0; i < E / VEC; ++i) {
                float w[VEC];
#pragma unroll
                for (int q = 0; q < VEC; ++q) w[q] = 1.0f;
                if (pre_weight && col_of<T, VEC>(i, tid) < width) load_part<T, VEC>(w, g.pre_weight + begin, col_of<T, VEC>(i, tid));
#pragma unroll
                for (int q = 0; q < VEC; ++q) w_row[i * VEC + q] = w[q];
            }
        }
        if constexpr (HOLD && F::GATE == 1) {
            if (left == g.gate_rows || row == lo) hold(w_gate, g.gate.p + group * g.gate.stride);
        }
        if (a.stages == 4) asm volatile("cp.async.wait_group 3;" ::: "memory");
        else if (a.stages == 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
        else asm volatile("cp.async.wait_group 1;" ::: "memory");
        const float* in = mine + stage_at;
        stage_at = stage_at + STAGE == ring ? 0 : stage_at + STAGE;
        ahead_at = ahead_at + STAGE == ring ? 0 : ahead_at + STAGE;
        const float* gate = g.gate.p + group * g.gate.stride + (row_gate ? begin : 0);
        const float one_gate = (FAST ? SCALAR : g.gate_mode == kGateScalar) ? gate[0] * g.scale : g.scale;
        const float mean_f = FULL ? st.x : 0.0f, mean_y = FULL ? st.z : 0.0f;

        float e_[E], hat[E];                             // e = dy + rstd_y * a, and yhat
        // sums of a yhat, k e fhat, k fhat yhat; and of a, k e, k, k fhat, k yhat
        float s_ay = 0.0f, s_kef = 0.0f, s_kfy = 0.0f, s_a = 0.0f, s_ke = 0.0f, s_k = 0.0f, s_kf = 0.0f, s_ky = 0.0f;
#pragma unroll
        for (int i = 0; i < E / VEC; ++i) {
            const int c = col_of<T, VEC>(i, tid);
            const float* at = in + i * THREADS * VEC;
            if (c < width) {
                float dy[VEC], fv[VEC], k[VEC], w[VEC];
#pragma unroll
                for (int q = 0; q < VEC; ++q) dy[q] = 0.0f;
                if (has_dy) read_own<VEC>(dy, at + kInDy * SLOT);
                if (pre) {
                    float yv[VEC], dh[VEC];
                    read_own<VEC>(yv, at + kInY * SLOT);
                    read_own<VEC>(dh, at + kInDh * SLOT);
#pragma unroll
                    for (int q = 0; q < VEC; ++q) {
                        const int e = i * VEC + q;
                        hat[e] = FULL ? (yv[q] - mean_y) * st.w : yv[q] * st.w;
                        pre_w[e] = fmaf(dh[q], hat[e], pre_w[e]);
                        if (FULL) pre_b[e] = pre_b[e] + dh[q];
                        const float av = dh[q] * (HOLD ? w_pre[HOLD ? e : 0] : w_row[HOLD ? 0 : e]);
                        if (FULL) s_a = s_a + av;
                        s_ay = fmaf(av, hat[e], s_ay);
                        e_[e] = fmaf(st.w, av, dy[q]);
                    }
                } else {
#pragma unroll
                    for (int q = 0; q < VEC; ++q) { hat[i * VEC + q] = 0.0f; e_[i * VEC + q] = dy[q]; }
                }
                if (post) {
                    read_own<VEC>(fv, at + kInF * SLOT);
#pragma unroll
                    for (int q = 0; q < VEC; ++q) k[q] = one_gate;
                    if (row_gate) {
                        float gv[VEC];
                        if (staged_gate) {
                            read_own<VEC>(gv, at + kInGate * SLOT);
                        } else if constexpr (HOLD && F::GATE == 1) {
#pragma unroll
                            for (int q = 0; q < VEC; ++q) gv[q] = w_gate[i * VEC + q];
                        } else {
                            load_part<T, VEC>(gv, gate, c);
                        }
#pragma unroll
                        for (int q = 0; q < VEC; ++q) k[q] = gv[q] * g.scale;
                    }
                    if (post_weight) {
                        if constexpr (HOLD && POST) {
#pragma unroll
                            for (int q = 0; q < VEC; ++q) w[q] = w_post[i * VEC + q];
                        } else {
                            load_part<T, VEC>(w, g.post_weight + begin, c);
                        }
#pragma unroll
                        for (int q = 0; q < VEC; ++q) k[q] = k[q] * w[q];
                    }
#pragma unroll
                    for (int q = 0; q < VEC; ++q) {
                        const int e = i * VEC + q;
                        const float fh = FULL ? (fv[q] - mean_f) * st.y : fv[q] * st.y, ke = k[q] * e_[e], kf = k[q] * fh;
                        s_kef = fmaf(ke, fh, s_kef);
                        s_kfy = fmaf(kf, hat[e], s_kfy);
                        if (FULL) {
                            s_ke = s_ke + ke;
                            s_k = s_k + k[q];
                            s_kf = s_kf + kf;
                            s_ky = fmaf(k[q], hat[e], s_ky);
                        }
                    }
                }
            } else {
#pragma unroll
                for (int q = 0; q < VEC; ++q) { hat[i * VEC + q] = 0.0f; e_[i * VEC + q] = 0.0f; }
            }
        }
        if (POST || pre) {
            float v[SUMS];
            v[0] = s_ay;
            if constexpr (SUMS == 2) v[1] = s_a;
            if constexpr (SUMS >= 4) { v[1] = s_kef; v[2] = s_kfy; v[3] = s_a; }
            if constexpr (SUMS == 8) { v[4] = s_ke; v[5] = s_k; v[6] = s_kf; v[7] = s_ky; }
            team_fold<FoldSum, THREADS, T>(v, sh, turn);
            if (SCALAR && row > lo) collect(row - 1, left == g.gate_rows ? group - 1 : group, (int)(row - 1 - lo) & 1);
            s_ay = v[0];
            if constexpr (SUMS == 2) s_a = v[1];
            if constexpr (SUMS >= 4) { s_kef = v[1]; s_kfy = v[2]; s_a = v[3]; }
            if constexpr (SUMS == 8) { s_ke = v[4]; s_k = v[5]; s_kf = v[6]; s_ky = v[7]; }
        }
        // dx = e - b0 - yhat * b1;  df = rstd_f * (k dx - c0 - fhat * c1)
        const float b0 = FULL && g.pre_kind == CTB_NORM_LAYER ? st.w * (s_a * inv) : 0.0f, b1 = st.w * (s_ay * inv);
        const float c0 = FULL && g.post_kind == CTB_NORM_LAYER ? (s_ke - (b0 * s_k + b1 * s_ky)) * inv : 0.0f;
        const float c1 = (s_kef - (b0 * s_kf + b1 * s_kfy)) * inv;
        float scalar_sum = 0.0f;
        const int64_t out_at = row * g.cols + begin + tid * VEC;
#pragma unroll
        for (int i = 0; i < E / VEC; ++i) {
            const int c = col_of<T, VEC>(i, tid);
            const float* at = in + i * THREADS * VEC;
            const int out = i * T * VEC;
            if (c < width) {
                float dx[VEC], fv[VEC], w[VEC], gv[VEC];
#pragma unroll
                for (int q = 0; q < VEC; ++q) {
                    const int e = i * VEC + q;
                    dx[q] = pre ? e_[e] - fmaf(hat[e], b1, b0) : e_[e];
                    fv[q] = 0.0f;
                    w[q] = 1.0f;
                    gv[q] = one_gate;
                }
                if (FAST || a.out.x) store_part<VEC>(a.out.x + out_at, out, dx);
                if (has_f) read_own<VEC>(fv, at + kInF * SLOT);
                if (post) {
#pragma unroll
                    for (int q = 0; q < VEC; ++q) fv[q] = FULL ? (fv[q] - mean_f) * st.y : fv[q] * st.y;
                    if constexpr (HOLD && POST) {
#pragma unroll
                        for (int q = 0; q < VEC; ++q) w[q] = w_post[i * VEC + q];
                    } else if (post_weight) {
                        load_part<T, VEC>(w, g.post_weight + begin, c);
                    }
                }
                if (row_gate) {
                    if (staged_gate) {
                        read_own<VEC>(gv, at + kInGate * SLOT);
                    } else if constexpr (HOLD && F::GATE == 1) {
#pragma unroll
                        for (int q = 0; q < VEC; ++q) gv[q] = w_gate[i * VEC + q];
                    } else {
                        load_part<T, VEC>(gv, gate, c);
                    }
#pragma unroll
                    for (int q = 0; q < VEC; ++q) gv[q] = gv[q] * g.scale;
                }
                if (want_n) {
                    float n[VEC];
                    if (FULL && post && g.post_bias) {
                        float b[VEC];
                        load_part<T, VEC>(b, g.post_bias + begin, c);
#pragma unroll
                        for (int q = 0; q < VEC; ++q) n[q] = fmaf(fv[q], w[q], b[q]) * (g.scale * dx[q]);
                    } else {
#pragma unroll
                        for (int q = 0; q < VEC; ++q) n[q] = (post ? fv[q] * w[q] : fv[q]) * (g.scale * dx[q]);
                    }
                    if (scalar_gate) {
#pragma unroll
                        for (int q = 0; q < VEC; ++q) scalar_sum = scalar_sum + n[q];
                    } else if (shared_gate) {
#pragma unroll
                        for (int q = 0; q < VEC; ++q) gate_sum[GATE ? i * VEC + q : 0] += n[q];
                    } else {
                        store_part<VEC>(a.out.gate + out_at, out, n);
                    }
                }
                float df[VEC];
#pragma unroll
                for (int q = 0; q < VEC; ++q) {
                    const int e = i * VEC + q;
                    const float dn = dx[q] * gv[q];
                    if (POST) {
                        post_w[e] = fmaf(dn, fv[q], post_w[e]);
                        if (FULL) post_b[e] = post_b[e] + dn;
                    }
                    df[q] = post ? st.y * (dn * w[q] - fmaf(fv[q], c1, c0)) : dn;
                }
                if (FAST || a.out.f) store_part<VEC>(a.out.f + out_at, out, df);
            }
        }
        if constexpr (SCALAR) {
            leave(scalar_sum, (int)(row - lo) & 1);
        } else if (scalar_gate) {
            float one[1] = {scalar_sum};
            team_fold<FoldSum, THREADS, T>(one, sh_gate, gate_turn);
            scalar_gate_sum = scalar_gate_sum + one[0];
        }
        // a gate that rows share: its sum so far goes out when the next row belongs to another gate row
        if (--left == 0 || row + 1 == hi) {
            const bool whole = group * g.gate_rows >= lo && (group + 1) * g.gate_rows <= hi;
            if (shared_gate && !a.one_gate_row) {
                float* to = (whole ? a.out.gate + group * g.cols : a.gate_part + (team + group) * g.cols) + begin;
#pragma unroll
                for (int i = 0; i < E / VEC; ++i) {
                    const int c = col_of<T, VEC>(i, tid);
                    float part[VEC];
#pragma unroll
                    for (int q = 0; q < VEC; ++q) {
                        part[q] = gate_sum[GATE ? i * VEC + q : 0];
                        gate_sum[GATE ? i * VEC + q : 0] = 0.0f;
                    }
                    if (c < width) store_part<VEC>(to, c, part);
                }
            } else if (!SCALAR && scalar_gate && tid == 0 && rank == 0) {
                *(whole ? a.out.gate + group : a.gate_part + team + group) = scalar_gate_sum;
            }
            if (!SCALAR) scalar_gate_sum = 0.0f;
            ++group;
            left = (int)g.gate_rows;
        }
    }
    if constexpr (SCALAR) {
        if (T == THREADS && cs > 1) { __syncwarp(); cluster_barrier(); }
        else if (T == 32) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(1 + (int)threadIdx.x / T), "r"(T) : "memory");
        if (lo < hi) collect(hi - 1, fast_div((uint32_t)(hi - 1), g.by_gate_rows), (int)(hi - 1 - lo) & 1);
    }
    // column sums: the teams of a CTA add theirs in team order (through the ring, which is done with)
    auto put = [&](int at, const float* sum) {
        if (TEAMS > 1) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < E; ++e) staged[e * THREADS + threadIdx.x] = sum[e];
            __syncthreads();
        }
        if (threadIdx.x >= T) return;
        float* part_row = a.part + ((int64_t)at * a.parts + blockIdx.x / cs) * g.cols + begin;
#pragma unroll
        for (int i = 0; i < E / VEC; ++i) {
            const int c = col_of<T, VEC>(i, tid);
            float part[VEC];
#pragma unroll
            for (int q = 0; q < VEC; ++q) {
                part[q] = sum[i * VEC + q];
#pragma unroll
                for (int t = 1; t < TEAMS; ++t) part[q] = part[q] + staged[(i * VEC + q) * THREADS + t * T + tid];
            }
            if (c < width) store_part<VEC>(part_row, c, part);
        }
    };
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    let_next_start();
    if (a.out.pre_weight) put(0, pre_w);
    if (FULL && a.out.pre_bias) put(1, pre_b);
    if (POST && a.out.post_weight) put(2, post_w);
    if (POST && FULL && a.out.post_bias) put(3, post_b);
    if (GATE && a.one_gate_row) put(4, gate_sum);
}

// out[c] = sum over partial rows [first, last] of part[row][c], in fp64: runs of consecutive rows, joined in
// order.  Jobs: the vectors, then one for every gate group.
struct FoldJobs {
    const float* part[5];
    float* out[5];
    int32_t vectors;
    int64_t parts, teams, cols;
    const float* gate_part;
    float* gate;
    int64_t gate_width, gate_rows, rows;
    int32_t by_group;                   // gate jobs: one for every gate row, or (more gate rows than teams) for every two
                                        // neighbouring teams whose rows share one
    int64_t vector_blocks, tiles, gate_tiles;
};

constexpr int kFoldThreads = 512, kFoldCols = 32, kFoldBatch = 8;

__global__ void __launch_bounds__(kFoldThreads)
residual_norm_fold_kernel(const __grid_constant__ FoldJobs j) {
    __shared__ double sums[kFoldThreads];
    const float* part;
    float* out;
    int64_t first = 0, last = j.parts - 1, width = j.cols, tile;
    const int64_t b = blockIdx.x;
    if (b < j.vector_blocks) {
        const int v = (int)(b / j.tiles);
        tile = b % j.tiles;
        part = j.part[v];
        out = j.out[v];
    } else {
        // team t has rows [rows * t / teams, rows * (t + 1) / teams)
        int64_t group = (b - j.vector_blocks) / j.gate_tiles;
        tile = (b - j.vector_blocks) % j.gate_tiles;
        if (!j.by_group) {
            const int64_t t = group + 1, start = j.rows * t / j.teams;
            group = start / j.gate_rows;
            // a gate row begins here, or the one that does not began before the team ahead, whose job it then is
            if (start % j.gate_rows == 0 || j.rows * (t - 1) / j.teams > group * j.gate_rows) {
                wait_for_previous();                     // also with nothing to add: no block of this launch ends ahead of
                return;                                  // the one before it, which later work in the stream relies on
            }
        }
        const int64_t r0 = group * j.gate_rows, r1 = r0 + j.gate_rows - 1;
        first = ((r0 + 1) * j.teams - 1) / j.rows + group;
        last = ((r1 + 1) * j.teams - 1) / j.rows + group;
        if (first == last) {                             // one team's: it wrote the sum itself
            wait_for_previous();
            return;
        }
        width = j.gate_width;
        part = j.gate_part;
        out = j.gate + group * width;
    }
    const int across = width == 1 ? 1 : kFoldCols, runs = kFoldThreads / across;
    const int64_t c = tile * kFoldCols + threadIdx.x % across;
    const int which = threadIdx.x / across;
    const int64_t run = (last - first + runs) / runs;
    const int64_t lo = first + which * run, hi = min(last + 1, lo + run);
    double sum = 0.0;
    wait_for_previous();
    if (c < width) {
        for (int64_t r = lo; r < hi; r += kFoldBatch) {
            float v[kFoldBatch];
#pragma unroll
            for (int u = 0; u < kFoldBatch; ++u) v[u] = r + u < hi ? part[(r + u) * width + c] : 0.0f;
#pragma unroll
            for (int u = 0; u < kFoldBatch; ++u) sum = sum + (double)v[u];
        }
    }
    sums[threadIdx.x] = sum;
    for (int half = runs / 2; half > 0; half >>= 1) {
        __syncthreads();
        if (which < half) sums[threadIdx.x] = sums[threadIdx.x] + sums[threadIdx.x + half * across];
    }
    if (which == 0 && c < width) out[c] = (float)sums[threadIdx.x];
}

// ---- host -----------------------------------------------------------------------------------------------
bool rows_aligned(const RowsIn& r) { return !r.p || (is_aligned(r.p, 16) && r.stride % 4 == 0); }

// CTAs of a cluster for `cols` columns when one CTA holds `per_cta` (slices are multiples of four columns).
int cluster_for(int64_t cols, int64_t per_cta) {
    int cs = (int)ceil_div(cols, per_cta);
    if (cs > 1 && (ceil_div(cols, (int64_t)cs) + 3) / 4 * 4 > per_cta) ++cs;
    return cs;
}

struct ForwardCall {
    ResidualNormGeom g;
    RowsIn x, f;
    float *y, *h, *stats;
    cudaStream_t st;
};
template <int THREADS, int T, int E, int VEC>
int forward_as(const ForwardCall& c) {
    const char* who = "residual_norm";
    const int64_t ctas = ceil_div(c.g.rows, (int64_t)(THREADS / T));
    if constexpr (T < THREADS) {
        if (c.f.p && c.g.post_kind == CTB_NORM_RMS && c.g.pre_kind == CTB_NORM_RMS && !c.g.post_bias)
            return launch_clusters(who, residual_rms_kernel<THREADS, T, E, VEC>, ctas, THREADS, 0, 1, c.st, c.g, c.x, c.f, c.y, c.h, c.stats);
        return launch_clusters(who, residual_norm_kernel<THREADS, T, E, VEC>, ctas, THREADS, 0, 1, c.st, c.g, c.x, c.f, c.y, c.h, c.stats, 1);
    } else {
        const int cs = cluster_for(c.g.cols, (int64_t)T * E);
        return launch_clusters(who, residual_norm_kernel<THREADS, T, E, VEC>, ctas * cs, THREADS, 0, cs, c.st, c.g, c.x, c.f, c.y, c.h, c.stats, cs);
    }
}

// How a row is dealt out in the backward pass: a team of `team` threads with kBwdShare columns each, `threads` to
// a CTA, `cs` CTAs to a row, `ctas` of them on an SM.  The column sums of a row's team live in registers, so
// 384 to 640 threads fit an SM.  Up to 2048 columns a CTA has several teams, so that one works while another
// waits in its fold; a wider row keeps the SM busy by itself (the next ones are on their way into shared
// memory) as long as one CTA holds it.  Beyond that, clusters of small CTAs, two on an SM for the same reason:
// 4096 rows of 8192 columns with RMS norms took 206 us with one cluster per SM pair, 139 with two.
constexpr int kBwdShare = 8;
struct BwdShape {
    int threads, team, cs, ctas;
};
// Specialised: RMS norms without biases; a LayerNorm or a bias before the next block; both norms, one of them such.
// The last two for rows that go element by element.  Everything else.
enum BwdKind { kBwdLean, kBwdFullPre, kBwdFull, kBwdScalarPre, kBwdScalar, kBwdAny };
BwdShape bwd_shape(int64_t cols, BwdKind kind) {
    for (int team : {32, 64, 96, 128, 192, 256}) {
        if (cols > team * kBwdShare || ((kind == kBwdScalarPre || kind == kBwdScalar) && team != 32 && team != 128 && team != 256)) continue;
        // four sums per column and the weights beside them: 170 registers a thread
        if ((kind == kBwdFull || kind == kBwdScalar) && team <= 192) return {384, team, 1, 1};
        return {team == 96 ? 480 : (team == 192 ? 384 : 512), team, 1, 1};
    }
    // (the sums of a LayerNorm and its bias leave a thread 128 registers where the CTA can be that small)
    if (cols <= 512 * kBwdShare && kind != kBwdLean) return {512, 512, 1, 1};
    const bool small = kind == kBwdLean || kind == kBwdFullPre;
    const int alone = small ? 640 : 512, in_cluster = small ? 320 : 256;
    if (cols <= 640 * kBwdShare && (small || kind == kBwdScalarPre)) return {640, 640, 1, 1};
    const int cs = cluster_for(cols, in_cluster * kBwdShare);
    if ((small || kind == kBwdFull) && cs <= kMaxCluster) return {in_cluster, in_cluster, cs, 2};
    return {alone, alone, cluster_for(cols, alone * kBwdShare), 1};
}
// Teams that walk the rows, at most one per row and at most kTeamRows rows each: `ctas` CTAs (clusters) run at once.
constexpr int64_t kTeamRows = 240;
int64_t bwd_teams(int64_t rows, const BwdShape& s, int64_t ctas) {
    const int64_t at_once = ctas * (s.threads / s.team), teams = at_once < 1 ? 1 : at_once;
    return teams > rows ? rows : teams * ceil_div(rows, teams * kTeamRows);
}
constexpr int kMaxSms = 256;                             // what the size query, which names no device, allows for

struct BwdCall {
    ResidualBwd a;
    BwdShape shape;
    bool vec, fast, post, full;
    int gate;                           // of BwdFlags
    int sm_count;
    void* workspace;
    cudaStream_t st;
};

template <int THREADS, int T, int E, int VEC, typename F>
int backward_as(BwdCall& c) {
    auto kernel = residual_norm_backward_kernel<THREADS, T, E, VEC, F>;
    ResidualBwd& a = c.a;
    const int cs = c.shape.cs;
    const size_t stage = (size_t)F::SLOTS * E * THREADS * sizeof(float), room = (size_t)(212 * 1024) / c.shape.ctas;
    a.stages = stage * 4 <= room ? 4 : (stage * 3 <= room ? 3 : 2);
    int ctas = (c.sm_count < kMaxSms ? c.sm_count : kMaxSms) * c.shape.ctas;
    if (cs > 1) {                       // a second wave of a few clusters would double the time
        int most = 0;
        if (int rc = resident_clusters((const void*)kernel, THREADS, stage * a.stages, cs, &most)) return rc;
        ctas = most < ctas / cs ? most : ctas / cs;
    }
    a.teams = bwd_teams(a.g.rows, c.shape, ctas);
    a.parts = ceil_div(a.teams, (int64_t)(THREADS / T));
    a.part = (float*)c.workspace;
    a.gate_part = a.part + 5 * a.parts * a.g.cols;
    return launch_clusters("residual_norm_backward", kernel, a.parts * cs, THREADS, stage * a.stages, cs, c.st, a, cs);
}

template <int THREADS, int T, bool POST, bool FULL, int VEC = 4>
int backward_gate(BwdCall& c) {
    if (c.gate == 0) return backward_as<THREADS, T, kBwdShare, VEC, BwdFlags<true, POST, FULL, 0>>(c);
    if (c.gate == 1) return backward_as<THREADS, T, kBwdShare, VEC, BwdFlags<true, POST, FULL, 1>>(c);
    if (c.gate == 2) return backward_as<THREADS, T, kBwdShare, VEC, BwdFlags<true, POST, FULL, 2>>(c);
    return backward_as<THREADS, T, kBwdShare, VEC, BwdFlags<true, POST, FULL, 3>>(c);
}
template <int THREADS, int T, bool FULL, int VEC = 4>
int backward_fast(BwdCall& c) {
    return c.post ? backward_gate<THREADS, T, true, FULL, VEC>(c) : backward_gate<THREADS, T, false, FULL, VEC>(c);
}
template <int THREADS>
int backward_lean(BwdCall& c) {
    if (c.full) return backward_gate<THREADS, THREADS, false, true>(c);
    return backward_fast<THREADS, THREADS, false>(c);
}
template <int THREADS, int T>
int backward_narrow(BwdCall& c) {
    constexpr int FULL_THREADS = T <= 192 ? 384 : THREADS;
    if (!c.fast) {
        if (c.vec) return backward_as<THREADS, T, kBwdShare, 4, BwdFlags<false, true, true, 1>>(c);
        return backward_as<THREADS, T, kBwdShare, 1, BwdFlags<false, true, true, 1>>(c);
    }
    if (!c.vec) {
        if constexpr (T == 32 || T == 128 || T == 256 || T == 512) return c.post ? backward_gate<FULL_THREADS, T, true, true, 1>(c) : backward_gate<THREADS, T, false, true, 1>(c);
    }
    if (!c.full) return backward_fast<THREADS, T, false>(c);
    return c.post ? backward_gate<FULL_THREADS, T, true, true>(c) : backward_gate<THREADS, T, false, true>(c);
}

}  // namespace

size_t residual_norm_workspace_bytes(int64_t rows, int64_t cols, int64_t gate_groups, int64_t gate_width) {
    int64_t teams = 0, parts = 0;
    for (BwdKind kind : {kBwdLean, kBwdFullPre, kBwdFull, kBwdScalarPre, kBwdScalar, kBwdAny}) {
        const BwdShape shape = bwd_shape(cols, kind);
        // no more than this, however many of them run at once
        const int64_t most = (int64_t)kMaxSms * shape.ctas / shape.cs * (shape.threads / shape.team) + ceil_div(rows, kTeamRows);
        const int64_t t = most > rows ? rows : most, p = ceil_div(t, (int64_t)(shape.threads / shape.team));
        teams = t > teams ? t : teams;
        parts = p > parts ? p : parts;
    }
    return ((size_t)(5 * parts) * (size_t)cols + (size_t)(gate_groups > 0 ? teams + gate_groups : 0) * (size_t)gate_width) * sizeof(float);
}

int launch_residual_norm(const ResidualNormGeom& geom, RowsIn x, RowsIn f, float* y, float* h, float* stats, cudaStream_t st) {
    if (geom.rows == 0 || geom.cols == 0) return CTB_OK;
    ResidualNormGeom g = geom;
    g.inv_cols = 1.0 / (double)g.cols;
    g.by_gate_rows = make_fastdiv((uint32_t)g.gate_rows);
    const bool vec = g.cols % 4 == 0 && rows_aligned(x) && rows_aligned(f) && (!y || is_aligned(y, 16)) && (!h || is_aligned(h, 16)) &&
                     is_aligned(g.post_weight, 16) && is_aligned(g.post_bias, 16) && is_aligned(g.pre_weight, 16) && is_aligned(g.pre_bias, 16) &&
                     (g.gate_mode != kGateRow || rows_aligned(g.gate));
    const ForwardCall c{g, x, f, y, h, stats, st};
    if (!vec) {                                          // a share that fits: [30000, 301] 36 us, 86 with that of 2048 columns
        if (g.cols <= 64) return forward_as<256, 32, 2, 1>(c);
        if (g.cols <= 128) return forward_as<256, 32, 4, 1>(c);
        if (g.cols <= 256) return forward_as<256, 32, 8, 1>(c);
        if (g.cols <= 512) return forward_as<256, 64, 8, 1>(c);
        if (g.cols <= 1024) return forward_as<256, 128, 8, 1>(c);
        if (g.cols <= 2048) return forward_as<256, 128, 16, 1>(c);
        if (g.cols <= 4096) return forward_as<512, 512, 8, 1>(c);
        return forward_as<512, 512, 16, 1>(c);
    }
    if (g.cols <= 128) return forward_as<256, 32, 4, 4>(c);
    if (g.cols <= 256) return forward_as<256, 32, 8, 4>(c);
    if (g.cols <= 512) return forward_as<256, 32, 16, 4>(c);
    if (g.cols <= 768) return forward_as<288, 96, 8, 4>(c);
    if (g.cols <= 1024) return forward_as<256, 128, 8, 4>(c);
    if (g.cols <= 2048) return forward_as<256, 128, 16, 4>(c);
    if (g.cols <= 4096) return forward_as<256, 256, 16, 4>(c);
    return forward_as<512, 512, 16, 4>(c);
}

int launch_residual_norm_backward(const ResidualNormGeom& g, RowsIn f, RowsIn y, const float* stats, RowsIn grad_y, RowsIn grad_h,
                                  const ResidualNormGrads& out, void* workspace, cudaStream_t st) {
    const int64_t groups = g.rows / g.gate_rows;
    const int64_t gate_width = g.gate_mode == kGateRow ? g.cols : 1;
    if (g.rows == 0 || g.cols == 0) return CTB_OK;
    DeviceInfo di;
    if (int rc = current_device_info(&di)) return rc;
    BwdCall call{};
    ResidualBwd& a = call.a;
    a.g = g;
    a.g.inv_cols = 1.0 / (double)g.cols;
    a.g.by_gate_rows = make_fastdiv((uint32_t)g.gate_rows);
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
    a.one_gate_row = shared_gate && groups == 1;
    bool vec = g.cols % 4 == 0 && (!out.x || is_aligned(out.x, 16)) && (!out.f || is_aligned(out.f, 16)) && (!out.gate || is_aligned(out.gate, 16)) &&
               is_aligned(g.post_weight, 16) && is_aligned(g.post_bias, 16) && is_aligned(g.pre_weight, 16) &&
               (g.gate_mode != kGateRow || rows_aligned(g.gate));
    for (const RowsIn& r : a.in) vec = vec && rows_aligned(r);
    call.vec = vec;
    call.post = post;
    call.fast = g.pre_kind != CTB_NORM_NONE && g.pre_weight && out.pre_weight && grad_y.p && f.p && out.x && out.f &&
                (!post || (g.post_weight && out.post_weight)) && (g.gate_mode == kGateNone || out.gate);
    call.full = g.pre_kind == CTB_NORM_LAYER || g.post_kind == CTB_NORM_LAYER || out.pre_bias || out.post_bias || g.post_bias;
    call.gate = g.gate_mode == kGateNone ? 0 : (g.gate_mode == kGateScalar ? 3 : (shared_gate ? 1 : 2));
    call.shape = bwd_shape(g.cols, !call.fast ? kBwdAny : (!vec ? (post ? kBwdScalar : kBwdScalarPre) : (!call.full ? kBwdLean : (post ? kBwdFull : kBwdFullPre))));
    call.sm_count = di.sm_count;
    call.workspace = workspace;
    call.st = st;
    int rc;
    switch (call.shape.team) {
    case 32: rc = backward_narrow<512, 32>(call); break;
    case 64: rc = backward_narrow<512, 64>(call); break;
    case 96: rc = backward_narrow<480, 96>(call); break;
    case 128: rc = backward_narrow<512, 128>(call); break;
    case 192: rc = backward_narrow<384, 192>(call); break;
    case 256: rc = call.shape.threads == 512 ? backward_narrow<512, 256>(call) : backward_gate<256, 256, true, true>(call); break;
    case 320: rc = backward_lean<320>(call); break;
    case 640: rc = vec ? backward_lean<640>(call) : backward_gate<640, 640, false, true, 1>(call); break;
    default: rc = backward_narrow<512, 512>(call);
    }
    if (rc) return rc;

    FoldJobs j{};
    float* const sums[4] = {out.pre_weight, out.pre_bias, out.post_weight, out.post_bias};
    for (int v = 0; v < 4; ++v)
        if (sums[v]) {
            j.part[j.vectors] = a.part + (int64_t)v * a.parts * g.cols;
            j.out[j.vectors++] = sums[v];
        }
    if (a.one_gate_row) {
        j.part[j.vectors] = a.part + 4 * a.parts * g.cols;
        j.out[j.vectors++] = out.gate;
    }
    j.parts = a.parts;
    j.teams = a.teams;
    j.cols = g.cols;
    j.tiles = ceil_div(g.cols, kFoldCols);
    j.vector_blocks = j.vectors * j.tiles;
    const bool fold_gate = want_gate && !a.one_gate_row && g.gate_rows > 1;
    if (fold_gate) {
        j.gate_part = a.gate_part;
        j.gate = out.gate;
        j.by_group = groups < a.teams;
        j.gate_width = gate_width;
        j.gate_rows = g.gate_rows;
        j.rows = g.rows;
        j.gate_tiles = ceil_div(gate_width, kFoldCols);
    }
    const int64_t blocks = j.vector_blocks + (fold_gate ? (j.by_group ? groups : a.teams - 1) * j.gate_tiles : 0);
    if (blocks == 0) return CTB_OK;
    if (blocks > 0x7FFFFFFFll) return set_error(CTB_ERR_LIMIT, "residual_norm_backward: too many gate rows for one launch");
    return launch_early(residual_norm_fold_kernel, (unsigned)blocks, kFoldThreads, st, j);
}

}  // namespace ctb
