// Attention scores to probabilities, and back: softmax over the admitted keys of every query with a scale,
// a tanh cap, a bias that falls with distance, and causal / prefix / document / length masks.
//
//   t_j = cap * tanh(scale * s_j / cap) - slope * |pos - j|,  p_j = exp(t_j - max t) / sum exp(t - max t)
//   D = sum_j p_j * dp_j,  ds_j = scale * (1 - tanh^2) * p_j * (dp_j - D)
//   dslope = -sum_j |pos - j| * p_j * (dp_j - D)
//
// In both directions a row's distances are counted from the nearest of its keys: what they have in common changes no
// probability, and in dslope it is multiplied by sum_j p_j * (dp_j - D) = 0 (left in, it would bring in D's rounding: slopes'
// gradients of queries 3 million keys away were off by 1e-3).
//
// Causal, prefix and length rules admit a run of keys [0, live); only the document rule is decided key by
// key.  Fours of keys without an admitted one are neither read nor evaluated, their results are written as
// zeros ahead of the loads.
//
// Bound by HBM: 4 bytes per admitted score in, 4 per element out; backward 8 (12 with a cap) in, 4 out.
// Rows that fit are held in the registers of part of a warp, a warp or a CTA and read once; longer rows are swept
// twice by one or more CTAs (second sweep from L2), few long ones held by a cluster.  Measured (bytes that
// have to move over time, share of the 6.54 TB/s of a copy): [8,12,1024,1024] causal forward 94 us, 6.4 TB/s (0.98),
// backward 126 us, 6.4 (0.98); capped 100 us (0.93) and 148 us (1.04, a part from L2); five packed documents, capped: 83 us (0.82),
// with slopes 86, instructions bound it (three quarters of the issue slots: a row that is nearly all zeros still looks at
// every document number), gradients 129 and 152 us; [1,12,512,16384] 138 us (0.89); swept rows of 100000: 162 us (0.58),
// gradients 186 (0.76).
#include "ctb_scores.cuh"
#include "ctb_team.cuh"

namespace ctb {

namespace {

struct ScoreArgs {
    ScoreGeom g;
    ScoreRows s, p, dp;
    float* out;
    double* slope_part;                 // one per row; NULL: not wanted
    int64_t rows;
    FastDiv by_queries, by_heads;
};

// The row of a team.  Teams smaller than a warp keep their warp company when there is no row left for them (they then
// see and write nothing).
struct ScoreRow {
    uint32_t row;
    bool present;
};
template <int THREADS, int T>
__device__ __forceinline__ ScoreRow score_row_of(const ScoreArgs& a, int cs) {
    const int64_t row = (int64_t)(T == THREADS ? blockIdx.x / (unsigned)cs : blockIdx.x) * (THREADS / T) + threadIdx.x / T;
    const bool present = row < a.rows;
    return {present ? (uint32_t)row : (uint32_t)(a.rows - 1), present};
}
constexpr int kNoKey = 0x7FFFFFFF;
// Where a row is and what its query may look at.
struct ScorePlace {
    uint32_t row, b, h, i;
    int live;                           // keys [0, live) may be admitted
    int centre;                         // the key position nearest to the query's within [0, live)
    int near;                           // distances from `centre` are counted from here on
    float slope;
    int doc;
};
__device__ __forceinline__ ScorePlace score_place(const ScoreArgs& a, ScoreRow r) {
    const ScoreGeom& g = a.g;
    const int keys = (int)g.keys;
    ScorePlace w;
    const uint32_t bh = fast_div(r.row, a.by_queries);
    w.row = r.row;
    w.i = r.row - bh * a.by_queries.d;
    w.b = fast_div(bh, a.by_heads);
    w.h = bh - w.b * a.by_heads.d;
    int64_t pos = (g.query_start.p ? (int64_t)g.query_start.p[w.b * g.query_start.sb] : g.keys - g.queries) + w.i;
    w.live = keys;
    if (g.key_lengths.p) w.live = min(keys, g.key_lengths.p[w.b * g.key_lengths.sb]);
    if (g.causal) {
        int reach = (int)max(min(pos + 1, (int64_t)keys), (int64_t)0);
        if (g.prefix.p) reach = max(reach, g.prefix.p[w.b * g.prefix.sb]);
        w.live = min(w.live, reach);
    }
    w.live = max(w.live, 0);
    w.centre = 0;
    w.slope = 0.0f;
    w.near = 0;
    if (g.slopes) {
        w.centre = (int)max(min(pos, (int64_t)w.live - 1), (int64_t)0);
        w.slope = g.slopes[w.h * g.slope_stride];
    }
    w.doc = g.query_docs.p ? g.query_docs.p[w.b * g.query_docs.sb + w.i * g.query_docs.si] : 0;
    return w;
}
__device__ __forceinline__ const float* score_row(const ScoreRows& r, const ScorePlace& w) {
    if (r.even >= 0) return r.p + (int64_t)w.row * r.even;
    return r.p + w.b * r.sb + w.h * r.sh + w.i * r.sq;
}

// What of a row a CTA of its cluster has: the fours from `from` on, up to the column `end`.
struct ScoreSpan {
    int from, end;
    __device__ __forceinline__ ScorePlace sees(ScorePlace w) const {
        w.live = min(w.live, end);
        return w;
    }
};
template <int T>
__device__ __forceinline__ ScoreSpan score_span(const ScoreArgs& a, const ScoreRow& r, int keys, int phase, int cs) {
    if (T < 32 && !r.present) return {0, 0};
    if (cs == 1) return {0, keys};
    const int fours = (keys + phase + 3) / 4, share = (fours + cs - 1) / cs, from = share * (int)cluster_rank();
    return {from, min(keys, max((from + share) * 4 - phase, 0))};
}

// Rows start at any multiple of four bytes.  Columns are dealt out in fours counted from the output row's
// address rounded down to 16 bytes, so whole fours of the output are aligned; a four holds the columns
// c0 .. c0 + 3, of which some may lie outside the row.  ALIGNED: every row of every operand starts on 16 bytes
// and has whole fours only (a four with an admitted column may then be read whole).
__device__ __forceinline__ int score_phase(const float* row) { return (int)(((uintptr_t)row >> 2) & 3); }

// The document numbers of a sequence's keys.  `fours`: contiguous, and the row's fours are 16-byte aligned.
struct ScoreDocs {
    const int32_t* p;
    int64_t si;
    bool fours;
};
template <bool DOCS>
__device__ __forceinline__ ScoreDocs score_docs(const ScoreArgs& a, const ScorePlace& w, int phase) {
    ScoreDocs d{nullptr, 0, false};
    if (DOCS) {
        d.p = a.g.key_docs.p + w.b * a.g.key_docs.sb;
        d.si = a.g.key_docs.si;
        d.fours = d.si == 1 && (int)(((uintptr_t)d.p >> 2) & 3) == phase;
    }
    return d;
}

// The admitted ones of the columns c0 .. c0 + 3, as bits.  HELD: for a row in registers (a swept row has none to
// spare: gradients of 16384 keys 141 us, so 203).
template <bool DOCS, bool HELD>
__device__ __forceinline__ uint32_t score_admitted(const ScoreDocs& docs, const ScorePlace& w, int c0) {
    const int hi = min(max(w.live - c0, 0), 4), lo = min(max(-c0, 0), 4);
    uint32_t bits = (15u >> (4 - hi)) & (15u << lo);
    if (DOCS && bits) {
        if (docs.fours && bits == 15u) {
            const int4 d = *reinterpret_cast<const int4*>(docs.p + c0);
            bits = (uint32_t)(d.x == w.doc) | (uint32_t)(d.y == w.doc) << 1 | (uint32_t)(d.z == w.doc) << 2 | (uint32_t)(d.w == w.doc) << 3;
        } else {
            if (HELD) {                                  // loads ahead of comparisons
                int d[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) d[k] = (bits >> k) & 1u ? docs.p[(int64_t)(c0 + k) * docs.si] : w.doc;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (d[k] != w.doc) bits &= ~(1u << k);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if ((bits >> k) & 1u)
                        if (docs.p[(int64_t)(c0 + k) * docs.si] != w.doc) bits &= ~(1u << k);
            }
        }
    }
    return bits;
}

// The admitted values of four columns (0 elsewhere).  `aligned`: the row's fours are 16-byte aligned.
__device__ __forceinline__ void score_load(float (&v)[4], const float* row, int c0, uint32_t bits, bool aligned) {
    if (bits == 15u && aligned) {
        const Vec<float, 4> q = ldg_stream(reinterpret_cast<const Vec<float, 4>*>(row + c0));
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = q.v[k];
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = (bits >> k) & 1u ? row[c0 + k] : 0.0f;
    }
}
__device__ __forceinline__ void score_store_four(float* at, const float (&v)[4]) {
    Vec<float, 4> q;
#pragma unroll
    for (int k = 0; k < 4; ++k) q.v[k] = v[k];
    stg_stream(reinterpret_cast<Vec<float, 4>*>(at), q);
}
__device__ __forceinline__ void score_store(float* row, int c0, int keys, const float (&v)[4]) {
    if (c0 >= 0 && c0 + 4 <= keys) {
        score_store_four(row + c0, v);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (c0 + k >= 0 && c0 + k < keys) row[c0 + k] = v[k];
    }
}

// e^x = 2^(x log2 e).  x is a difference of logits (were the logits themselves kept in units of log 2, a row of
// the type's lowest values would overflow).  Not the most exact form: the product's rounding is |x| half steps of the
// result, as many as the difference x itself brings along, the constant's a quarter of that, and the instruction's relative error
// is below 2^-22 (4 half steps).  Results below 2^-126 are 0.
__device__ __forceinline__ float score_exp(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
    return r;
}
// t of a four's columns.  The bias is taken from the key nearest to the query, which changes no probability
// (a softmax does not see a constant) and keeps t small where the query is far from every key.  Without documents that
// is the centre.  With them the nearest admitted key may be anywhere, and the team looks for it (`near`): a query 100000
// keys behind its document would else have logits of 5e4 at a slope of 1/2, where a step of Float32 is 0.004.
template <bool CAP, bool DOCS>
__device__ __forceinline__ void score_logits(const ScoreGeom& g, const ScorePlace& w, float (&t)[4], int c0) {
#pragma unroll
    for (int k = 0; k < 4; ++k) t[k] = CAP ? g.cap * tanhf(t[k] * g.over_cap) : t[k] * g.scale;
    if (g.slopes) {
        if (DOCS) {
#pragma unroll
            for (int k = 0; k < 4; ++k) t[k] = fmaf(-w.slope, (float)(abs(c0 + k - w.centre) - w.near), t[k]);
        } else {
            const float from = (float)(c0 - w.centre);
#pragma unroll
            for (int k = 0; k < 4; ++k) t[k] = fmaf(-w.slope, fabsf(from + (float)k), t[k]);
        }
    }
}
// Whether the key at the centre is of another document than the query, which is rare: [8,12,1024,1024] with slopes and 5
// documents 79.5 us and its gradients 142, 80.6 and 155 when every row looks for its nearest key; 512 rows of 40000, swept,
// 399 us, 484 far from their documents.  The same in all lanes of a warp.
template <int T>
__device__ __forceinline__ bool score_apart(const ScoreDocs& docs, const ScorePlace& w) {
    const bool apart = docs.p[w.centre * docs.si] != w.doc;
    return T < 32 ? __any_sync(0xFFFFFFFFu, apart) : apart;
}
// The smallest of the team's distances (kNoKey: none), the same in every thread; beyond 2^24 to Float32, which is as good.
template <int THREADS, int T>
__device__ __forceinline__ int score_near(int near, TeamSlots<THREADS, 1, float>& sh, FoldTurn& turn) {
    float most[1] = {near == kNoKey ? -INFINITY : -(float)near};
    team_fold<FoldMax, THREADS, T>(most, sh, turn);
    return most[0] == -INFINITY ? 0 : (int)-most[0];
}
// sum + the distances times r, over a four's columns
template <bool DOCS>
__device__ __forceinline__ float score_slope(const ScorePlace& w, float sum, int c0, const float (&r)[4]) {
    const float from = (float)(c0 - w.centre);
#pragma unroll
    for (int k = 0; k < 4; ++k) sum = fmaf(DOCS ? (float)(abs(c0 + k - w.centre) - w.near) : fabsf(from + (float)k), r[k], sum);
    return sum;
}
// r *= scale * (1 - tanh^2), with 1 - tanh^2 x = 4 q / (1 + q)^2, q = e^(-2 |x|): far beyond the cap, where tanh is next to 1
// and the difference would lose all its bits (at x = 9 it is 0), all of them count.
template <bool CAP>
__device__ __forceinline__ void score_slow(const ScoreGeom& g, float (&r)[4], const float* s) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        r[k] = r[k] * g.scale;
        if (CAP) {
            const float q = score_exp(-2.0f * fabsf(s[k] * g.over_cap));
            float over;                                  // within 2 half steps
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(over) : "f"(1.0f + q));
            r[k] = r[k] * (q * over * (4.0f * over));
        }
    }
}

// A thread's fours of a row: four v has the columns (v * T + tid) * 4 - phase and on.  Which columns are
// admitted is a comparison with `live` where rows are aligned and no documents are given, else kept as bits.
// With documents few fours of a row may have an admitted key, anywhere in it: a warp then goes over those v that
// have one in any of its lanes, the j-th of them held in the j-th registers, instead of over all with a test and a
// branch each ([8,12,1024,1024] causal, capped, five packed documents: 91 us, so 83, gradients 155 and 129; all
// keys in one document 97 and 101).
template <int T, int NV, bool DOCS, bool ALIGNED>
struct ScoreShare {
    static constexpr bool kBits = DOCS || !ALIGNED;
    static constexpr bool kSparse = DOCS && NV > 2;
    struct Four {                                        // of the v in `active`
        int at;
        uint32_t bits;
        __device__ __forceinline__ int column() const { return at; }
        __device__ __forceinline__ uint32_t four() const { return bits & 15u; }
        __device__ __forceinline__ bool has(int k) const { return ((bits >> k) & 1u) != 0; }
    };
    struct FixedFour {
        const ScoreShare& of;
        int v;
        __device__ __forceinline__ int column() const { return of.column(v); }
        __device__ __forceinline__ uint32_t four() const { return (of.bits >> (4 * v)) & 15u; }
        __device__ __forceinline__ bool has(int k) const { return kBits ? ((of.bits >> (4 * v + k)) & 1u) != 0 : of.rest > v * T * 4 + k; }
    };
    int first;                          // column of the first four
    int rest;                           // admissible columns from there on
    uint32_t bits;
    uint32_t active;                    // kSparse: the v with an admitted column in this warp
    // `from`: the first four of this CTA's slice of the row
    __device__ __forceinline__ void init(const ScoreDocs& docs, const ScorePlace& w, int from, int tid, int phase) {
        first = (from + tid) * 4 - phase;
        rest = w.live - first;
        bits = 0;
        if (DOCS && ALIGNED && docs.fours) {             // fours of document numbers may be read whole
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int left = rest - v * T * 4;
                if (left > 0) {
                    const int4 d = *reinterpret_cast<const int4*>(docs.p + column(v));
                    uint32_t four = (d.x == w.doc ? 1u : 0u) + (d.y == w.doc ? 2u : 0u) + (d.z == w.doc ? 4u : 0u) + (d.w == w.doc ? 8u : 0u);
                    if (left < 4) four &= (1u << left) - 1u;
                    bits |= four << (4 * v);
                }
            }
        } else if (kBits) {
#pragma unroll
            for (int v = 0; v < NV; ++v) bits |= score_admitted<DOCS, true>(docs, w, column(v)) << (4 * v);
        }
        if (kSparse) {
            uint32_t all = __reduce_or_sync(0xFFFFFFFFu, bits);
            all |= all >> 1;
            active = (all | all >> 2) & 0x11111111u;     // bit 4 v
        }
    }
    // f(j, four) for the fours worked on, their values being the j-th.
    template <typename F> __device__ __forceinline__ void each(F&& f) const {
        if (kSparse) {
            uint32_t left = active;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                if (!left) break;
                const int at = __ffs(left) - 1;
                left &= left - 1;
                f(j, Four{first + at * T, bits >> at});
            }
        } else {
#pragma unroll
            for (int v = 0; v < NV; ++v)
                if (any(v)) f(v, FixedFour{*this, v});
        }
    }
    __device__ __forceinline__ int column(int v) const { return first + v * T * 4; }
    // The smallest distance from the centre of the thread's admitted keys (with kBits): it is the last one's up to the
    // centre or the first one's behind it.
    __device__ __forceinline__ int nearest(const ScorePlace& w) const {
        const int ahead = w.centre - first, v = ahead / (4 * T);       // v: of the last four that begins up to the centre
        const int count = ahead < 0 ? 0 : min(4 * v + min(ahead - v * 4 * T, 3) + 1, 32);
        const uint32_t upto = (uint32_t)((1ull << count) - 1ull);
        const int below = 31 - __clz(bits & upto), above = __ffs(bits & ~upto) - 1;
        int d = below < 0 ? kNoKey : w.centre - (column(below >> 2) + (below & 3));
        if (above >= 0) d = min(d, column(above >> 2) + (above & 3) - w.centre);
        return d;
    }
    __device__ __forceinline__ bool any(int v) const { return kBits ? ((bits >> (4 * v)) & 15u) != 0 : rest > v * T * 4; }
    // values of the fours that have an admitted column; others are 0 or keep what they held
    __device__ __forceinline__ void load(float (&x)[NV][4], const float* row, bool aligned) const {
        if (!kSparse && !ALIGNED) {                         // a branch round each four more costs 7 % on a row of 4097
#pragma unroll
            for (int v = 0; v < NV; ++v) score_load(x[v], row, column(v), (bits >> (4 * v)) & 15u, aligned);
            return;
        }
        each([&](int j, const auto& o) {
            if (ALIGNED) {
                if (kSparse) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[j][k] = 0.0f;
                }
                if (!kSparse || o.four()) {
                    const Vec<float, 4> q = ldg_stream(reinterpret_cast<const Vec<float, 4>*>(row + o.column()));
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[j][k] = q.v[k];
                }
            } else {
                score_load(x[j], row, o.column(), o.four(), aligned);
            }
        });
    }
    __device__ __forceinline__ void store(float* out, int column, int end, const float (&x)[4]) const {
        if (!ALIGNED) score_store(out, column, end, x);
        else if (!kSparse || column < end) score_store_four(out + column, x);
    }
    // Zeros into the fours not worked on, ahead of the loads: these stores need not wait for them.
    __device__ __forceinline__ void zeros(float* out, int end) const {
        const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1                                         // unrolled, its addresses double the kernel's registers
        for (int v = 0; v < NV; ++v) {
            const int c0 = column(v);
            if (!(kSparse ? (active >> (4 * v)) & 1u : any(v)) && c0 < end) store(out, c0, end, zero);
        }
    }
};

template <int THREADS, int T, int NV, bool CAP, bool DOCS, bool ALIGNED>
__global__ void __launch_bounds__(THREADS, (ALIGNED ? 1280 : 1024) / THREADS)
score_softmax_kernel(const __grid_constant__ ScoreArgs a, int ctas) {
    const int cs = T == 512 ? ctas : 1;                  // only whole CTAs of 512 threads come in clusters
    const TeamEntry entry(cs);
    static_assert(NV <= 8, "admitted columns are kept as 4 * NV bits");
    __shared__ TeamSlots<THREADS, 1, float> sh;
    const int tid = threadIdx.x % T;
    const ScoreRow place = score_row_of<THREADS, T>(a, cs);
    if (T >= 32 && !place.present) return;               // whole teams leave together; never in a cluster
    const int64_t row = place.row;
    ScorePlace w = score_place(a, place);
    const int keys = (int)a.g.keys;
    float* out = a.out + row * (int64_t)keys;
    const float* s = score_row(a.s, w);
    const int phase = ALIGNED ? 0 : score_phase(out);
    ScoreShare<T, NV, DOCS, ALIGNED> mine;
    const ScoreSpan span = score_span<T>(a, place, keys, phase, cs);
    mine.init(score_docs<DOCS>(a, w, phase), span.sees(w), span.from, tid, phase);
    mine.zeros(out, span.end);
    float t[NV][4];
    mine.load(t, s, score_phase(s) == phase);
    FoldTurn turn = entry.met();
    if (DOCS && a.g.slopes && score_apart<T>(score_docs<DOCS>(a, w, phase), w)) w.near = score_near<THREADS, T>(mine.nearest(w), sh, turn);
    float m[1] = {-INFINITY};
    mine.each([&](int j, const auto& o) {
        score_logits<CAP, DOCS>(a.g, w, t[j], o.column());
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            t[j][k] = o.has(k) ? t[j][k] : -INFINITY;
            m[0] = fmaxf(m[0], t[j][k]);
        }
    });
    team_fold<FoldMax, THREADS, T>(m, sh, turn);
    const float top = m[0] == -INFINITY ? 0.0f : m[0];
    float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    mine.each([&](int j, const auto&) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            t[j][k] = score_exp(t[j][k] - top);
            part[k] = part[k] + t[j][k];
        }
    });
    float z[1] = {(part[0] + part[1]) + (part[2] + part[3])};
    team_fold<FoldSum, THREADS, T>(z, sh, turn);
    const float inv = z[0] == 0.0f ? 0.0f : __frcp_rn(z[0]);
    const bool usual = z[0] < INFINITY;                  // else NaN, which must not reach the masked columns
    mine.each([&](int j, const auto& o) {
        float p[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) p[k] = t[j][k] * inv;
        if (!usual) {
#pragma unroll
            for (int k = 0; k < 4; ++k) p[k] = o.has(k) ? p[k] : 0.0f;
        }
        mine.store(out, o.column(), span.end, p);
    });
}

// Registers: 64 with a cap or ragged rows, 48 else; a spilled word or two costs less than a quarter of the rows in
// flight (capped [8,12,1024,1024], when 1 - tanh^2 still took a tanh: 176 us, so 155; CTAs of 512, one or two an SM: [2,8,1024,8192] 420 and 293).
// With documents the compiler's own choice is the better one (0: no bound; 75 us at [64,12,256,256], 91 with one).
template <int THREADS, int T, int NV, bool CAP, bool DOCS, bool ALIGNED>
__global__ void __launch_bounds__(THREADS, THREADS == 512 ? 2 : DOCS ? 0 : CAP || !ALIGNED ? 4 : 5)
score_softmax_backward_kernel(const __grid_constant__ ScoreArgs a, int ctas) {
    const int cs = T == 512 ? ctas : 1;                  // only whole CTAs of 512 threads come in clusters
    const TeamEntry entry(cs);
    static_assert(NV <= 8, "admitted columns are kept as 4 * NV bits");
    __shared__ TeamSlots<THREADS, 1, float> sh;
    __shared__ TeamSlots<THREADS, 1, double> sh_slope;
    const int tid = threadIdx.x % T;
    const ScoreRow place = score_row_of<THREADS, T>(a, cs);
    if (T >= 32 && !place.present) return;
    const int64_t row = place.row;
    ScorePlace w = score_place(a, place);
    const int keys = (int)a.g.keys;
    float* out = a.out + row * (int64_t)keys;
    const float *pr = score_row(a.p, w), *gr = score_row(a.dp, w), *sr = CAP ? score_row(a.s, w) : nullptr;
    const int phase = ALIGNED ? 0 : score_phase(out);
    ScoreShare<T, NV, DOCS, ALIGNED> mine;
    const ScoreSpan span = score_span<T>(a, place, keys, phase, cs);
    mine.init(score_docs<DOCS>(a, w, phase), span.sees(w), span.from, tid, phase);
    mine.zeros(out, span.end);
    float p[NV][4], dp[NV][4], s[CAP ? NV : 1][4];
    mine.load(p, pr, score_phase(pr) == phase);
    mine.load(dp, gr, score_phase(gr) == phase);
    if constexpr (CAP) mine.load(s, sr, score_phase(sr) == phase);
    float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    mine.each([&](int j, const auto& o) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (ALIGNED) {                               // whole fours were read: masked columns hold anything
                p[j][k] = o.has(k) ? p[j][k] : 0.0f;
                dp[j][k] = o.has(k) ? dp[j][k] : 0.0f;
                if constexpr (CAP) s[j][k] = o.has(k) ? s[j][k] : 0.0f;
            }
            part[k] = fmaf(p[j][k], dp[j][k], part[k]);
        }
    });
    float d[1] = {(part[0] + part[1]) + (part[2] + part[3])};
    FoldTurn turn = entry.met();
    if (DOCS && a.slope_part && score_apart<T>(score_docs<DOCS>(a, w, phase), w)) w.near = score_near<THREADS, T>(mine.nearest(w), sh, turn);
    team_fold<FoldSum, THREADS, T>(d, sh, turn);
    const bool usual = fabsf(d[0]) < INFINITY;           // else 0 * (0 - D) is NaN in the masked columns
    float slope_sum = 0.0f;
    mine.each([&](int j, const auto& o) {
        float r[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            r[k] = p[j][k] * (dp[j][k] - d[0]);
            if (!usual && !o.has(k)) r[k] = 0.0f;
        }
        if (a.slope_part) slope_sum = score_slope<DOCS>(w, slope_sum, o.column(), r);
        score_slow<CAP>(a.g, r, s[CAP ? j : 0]);
        mine.store(out, o.column(), span.end, r);
    });
    if (a.slope_part) {
        double sum[1] = {(double)slope_sum};
        team_fold<FoldSum, THREADS, T>(sum, sh_slope, turn);
        if (tid == 0 && place.present && (cs == 1 || cluster_rank() == 0)) a.slope_part[row] = sum[0];
    }
}

// ---- rows swept by a cluster ----------------------------------------------------------------------------
// CTA `rank` of the row's `cs` CTAs has the fours [rank * share, (rank + 1) * share).
constexpr int kSweepThreads = 512;
constexpr int kSweepBatch = 4;                           // fours in flight per thread and operand

struct SweepSpan { int64_t lo, hi; };
__device__ __forceinline__ SweepSpan sweep_span(int64_t keys, int phase, int cs) {
    const int64_t fours = (keys + phase + 3) / 4, share = (fours + cs - 1) / cs;
    const int64_t lo = share * (cs > 1 ? cluster_rank() : 0);
    return {lo, min(fours, lo + share)};
}

// The smaller one of `near` and the distances of a four's admitted keys from the centre.
__device__ __forceinline__ int nearest_of_four(const ScorePlace& w, int near, int c0, uint32_t bits) {
    if (bits) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if ((bits >> k) & 1u) near = min(near, abs(c0 + k - w.centre));
    }
    return near;
}

template <bool CAP, bool DOCS>
__global__ void __launch_bounds__(kSweepThreads)
score_softmax_sweep_kernel(const __grid_constant__ ScoreArgs a, int cs) {
    const TeamEntry entry(cs);
    __shared__ TeamSlots<kSweepThreads, 1, float> sh;
    const int64_t row = blockIdx.x / cs;
    ScorePlace w = score_place(a, {(uint32_t)row, true});
    const int keys = (int)a.g.keys;
    float* out = a.out + row * (int64_t)keys;
    const float* s = score_row(a.s, w);
    const int phase = score_phase(out);
    const bool aligned = score_phase(s) == phase;
    const ScoreDocs docs = score_docs<DOCS>(a, w, phase);
    const SweepSpan span = sweep_span(keys, phase, cs);
    const int64_t live_end = min(span.hi, ((int64_t)w.live + phase + 3) / 4);
    FoldTurn turn = entry.met();
    if (DOCS && a.g.slopes && score_apart<kSweepThreads>(docs, w)) {         // a pass over the documents alone
        int near = kNoKey;
        for (int64_t f = span.lo + threadIdx.x; f < live_end; f += kSweepThreads * kSweepBatch) {
            uint32_t bits[kSweepBatch];
#pragma unroll
            for (int u = 0; u < kSweepBatch; ++u) {
                const int64_t at = f + (int64_t)u * kSweepThreads;
                bits[u] = at < live_end ? score_admitted<DOCS, true>(docs, w, (int)(at * 4) - phase) : 0u;
            }
#pragma unroll
            for (int u = 0; u < kSweepBatch; ++u) near = nearest_of_four(w, near, (int)((f + (int64_t)u * kSweepThreads) * 4) - phase, bits[u]);
        }
        w.near = score_near<kSweepThreads, kSweepThreads>(near, sh, turn);
    }
    // first sweep: the thread's maximum and its sum of exponentials relative to that maximum
    float m = -INFINITY, z = 0.0f;
    for (int64_t f = span.lo + threadIdx.x; f < live_end; f += kSweepThreads * kSweepBatch) {
        float t[kSweepBatch][4];
        uint32_t bits[kSweepBatch];
#pragma unroll
        for (int u = 0; u < kSweepBatch; ++u) {
            const int64_t at = f + (int64_t)u * kSweepThreads;
            bits[u] = at < live_end ? score_admitted<DOCS, false>(docs, w, (int)(at * 4) - phase) : 0u;
        }
#pragma unroll
        for (int u = 0; u < kSweepBatch; ++u) score_load(t[u], s, (int)((f + (int64_t)u * kSweepThreads) * 4) - phase, bits[u], aligned);
        float top = m;
#pragma unroll
        for (int u = 0; u < kSweepBatch; ++u) {
            if (!bits[u]) continue;
            score_logits<CAP, DOCS>(a.g, w, t[u], (int)((f + (int64_t)u * kSweepThreads) * 4) - phase);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                t[u][k] = (bits[u] >> k) & 1u ? t[u][k] : -INFINITY;
                top = fmaxf(top, t[u][k]);
            }
        }
        if (m != -INFINITY) z = z * score_exp(m - top);
        m = top;
        const float from = m == -INFINITY ? 0.0f : m;
        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int u = 0; u < kSweepBatch; ++u)
            if (bits[u]) {
#pragma unroll
                for (int k = 0; k < 4; ++k) part[k] = part[k] + score_exp(t[u][k] - from);
            }
        z = z + ((part[0] + part[1]) + (part[2] + part[3]));
    }
    float top[1] = {m};
    team_fold<FoldMax, kSweepThreads, kSweepThreads>(top, sh, turn);
    const float from = top[0] == -INFINITY ? 0.0f : top[0];
    float sum[1] = {m == -INFINITY ? z : z * score_exp(m - from)};
    team_fold<FoldSum, kSweepThreads, kSweepThreads>(sum, sh, turn);
    const float inv = sum[0] == 0.0f ? 0.0f : __frcp_rn(sum[0]);
    // second sweep
    for (int64_t f = span.lo + threadIdx.x; f < span.hi; f += kSweepThreads * kSweepBatch) {
        float t[kSweepBatch][4];
        uint32_t bits[kSweepBatch];
#pragma unroll
        for (int u = 0; u < kSweepBatch; ++u) {
            const int64_t at = f + (int64_t)u * kSweepThreads;
            bits[u] = at < live_end ? score_admitted<DOCS, false>(docs, w, (int)(at * 4) - phase) : 0u;
        }
#pragma unroll
        for (int u = 0; u < kSweepBatch; ++u) score_load(t[u], s, (int)((f + (int64_t)u * kSweepThreads) * 4) - phase, bits[u], aligned);
#pragma unroll
        for (int u = 0; u < kSweepBatch; ++u) {
            const int64_t at = f + (int64_t)u * kSweepThreads;
            if (at >= span.hi) break;
            const int c0 = (int)(at * 4) - phase;
            float p[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (bits[u]) {
                score_logits<CAP, DOCS>(a.g, w, t[u], c0);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if ((bits[u] >> k) & 1u) p[k] = score_exp(t[u][k] - from) * inv;
            }
            score_store(out, c0, keys, p);
        }
    }
}

template <bool CAP, bool DOCS>
__global__ void __launch_bounds__(kSweepThreads)
score_softmax_backward_sweep_kernel(const __grid_constant__ ScoreArgs a, int cs) {
    const TeamEntry entry(cs);
    __shared__ TeamSlots<kSweepThreads, 1, float> sh;
    __shared__ TeamSlots<kSweepThreads, 1, double> sh_slope;
    const int64_t row = blockIdx.x / cs;
    ScorePlace w = score_place(a, {(uint32_t)row, true});
    const int keys = (int)a.g.keys;
    float* out = a.out + row * (int64_t)keys;
    const float *pr = score_row(a.p, w), *gr = score_row(a.dp, w), *sr = CAP ? score_row(a.s, w) : nullptr;
    const int phase = score_phase(out);
    const bool p_aligned = score_phase(pr) == phase, g_aligned = score_phase(gr) == phase, s_aligned = CAP && score_phase(sr) == phase;
    const ScoreDocs docs = score_docs<DOCS>(a, w, phase);
    const SweepSpan span = sweep_span(keys, phase, cs);
    const int64_t live_end = min(span.hi, ((int64_t)w.live + phase + 3) / 4);
    const bool apart = DOCS && a.slope_part && score_apart<kSweepThreads>(docs, w);
    int near = kNoKey;
    float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int64_t f = span.lo + threadIdx.x; f < live_end; f += kSweepThreads * kSweepBatch) {
        float p[kSweepBatch][4], dp[kSweepBatch][4];
#pragma unroll
        for (int u = 0; u < kSweepBatch; ++u) {
            const int64_t at = f + (int64_t)u * kSweepThreads;
            const int c0 = (int)(at * 4) - phase;
            const uint32_t bits = at < live_end ? score_admitted<DOCS, false>(docs, w, c0) : 0u;
            score_load(p[u], pr, c0, bits, p_aligned);
            score_load(dp[u], gr, c0, bits, g_aligned);
            if (apart) near = nearest_of_four(w, near, c0, bits);
        }
#pragma unroll
        for (int u = 0; u < kSweepBatch; ++u)
#pragma unroll
            for (int k = 0; k < 4; ++k) part[k] = fmaf(p[u][k], dp[u][k], part[k]);
    }
    float d[1] = {(part[0] + part[1]) + (part[2] + part[3])};
    FoldTurn turn = entry.met();
    if (apart) w.near = score_near<kSweepThreads, kSweepThreads>(near, sh, turn);
    team_fold<FoldSum, kSweepThreads, kSweepThreads>(d, sh, turn);
    double slope_sum = 0.0;
    for (int64_t f = span.lo + threadIdx.x; f < span.hi; f += kSweepThreads * kSweepBatch) {
        float p[kSweepBatch][4], dp[kSweepBatch][4], s[kSweepBatch][4];
        uint32_t bits[kSweepBatch];
#pragma unroll
        for (int u = 0; u < kSweepBatch; ++u) {
            const int64_t at = f + (int64_t)u * kSweepThreads;
            const int c0 = (int)(at * 4) - phase;
            bits[u] = at < live_end ? score_admitted<DOCS, false>(docs, w, c0) : 0u;
            score_load(p[u], pr, c0, bits[u], p_aligned);
            score_load(dp[u], gr, c0, bits[u], g_aligned);
            if (CAP) score_load(s[u], sr, c0, bits[u], s_aligned);
        }
        float slope_part = 0.0f;
#pragma unroll
        for (int u = 0; u < kSweepBatch; ++u) {
            const int64_t at = f + (int64_t)u * kSweepThreads;
            if (at >= span.hi) break;
            const int c0 = (int)(at * 4) - phase;
            float r[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (bits[u]) {
#pragma unroll
                for (int k = 0; k < 4; ++k) r[k] = (bits[u] >> k) & 1u ? p[u][k] * (dp[u][k] - d[0]) : 0.0f;
                if (a.slope_part) slope_part = score_slope<DOCS>(w, slope_part, c0, r);
                score_slow<CAP>(a.g, r, s[u]);
            }
            score_store(out, c0, keys, r);
        }
        slope_sum = slope_sum + (double)slope_part;
    }
    if (a.slope_part) {
        double sum[1] = {slope_sum};
        team_fold<FoldSum, kSweepThreads, kSweepThreads>(sum, sh_slope, turn);
        if (threadIdx.x == 0 && (cs == 1 || cluster_rank() == 0)) a.slope_part[row] = sum[0];
    }
}

// grad_slopes[h] = -sum over the head's rows of part, in a fixed order.
__global__ void __launch_bounds__(256)
score_slope_fold_kernel(const double* __restrict__ part, int64_t batch, int64_t heads, int64_t queries, float* __restrict__ out) {
    __shared__ TeamSlots<256, 1, double> sh;
    const int64_t h = blockIdx.x;
    double sum[1] = {0.0};
    wait_for_previous();
    for (int64_t b = 0; b < batch; ++b)
        for (int64_t i = threadIdx.x; i < queries; i += 256) sum[0] = sum[0] + part[(b * heads + h) * queries + i];
    FoldTurn turn = TeamEntry(1).met();
    team_fold<FoldSum, 256, 256>(sum, sh, turn);
    if (threadIdx.x == 0) out[h] = (float)-sum[0];
}

// ---- host -----------------------------------------------------------------------------------------------
struct ScoreCall {
    ScoreArgs a;
    bool backward, cap, docs, aligned;
    int cs;                             // CTAs per row
    int sm_count;
    cudaStream_t st;
};
constexpr const char* kScoreName = "score_softmax";

enum Ways { kForward = 1, kBackward = 2, kBoth = 3 };    // which kernels a shape is compiled for

template <int THREADS, int T, int NV, int WAYS, bool CAP, bool DOCS, bool ALIGNED>
int rows_with(const ScoreCall& c) {
    const int64_t blocks = ceil_div(c.a.rows, (int64_t)(THREADS / T)) * c.cs;
    if constexpr (WAYS & kBackward)
        if (c.backward) return launch_clusters(kScoreName, score_softmax_backward_kernel<THREADS, T, NV, CAP, DOCS, ALIGNED>, blocks, THREADS, 0, c.cs, c.st, c.a, c.cs);
    if constexpr (WAYS & kForward)
        return launch_clusters(kScoreName, score_softmax_kernel<THREADS, T, NV, CAP, DOCS, ALIGNED>, blocks, THREADS, 0, c.cs, c.st, c.a, c.cs);
    return CTB_OK;                                       // not reached: the shapes below are chosen by direction
}
template <int THREADS, int T, int NV, int WAYS>
int rows_as(const ScoreCall& c) {
    if (c.cap) {
        if (c.docs) return c.aligned ? rows_with<THREADS, T, NV, WAYS, true, true, true>(c) : rows_with<THREADS, T, NV, WAYS, true, true, false>(c);
        return c.aligned ? rows_with<THREADS, T, NV, WAYS, true, false, true>(c) : rows_with<THREADS, T, NV, WAYS, true, false, false>(c);
    }
    if (c.docs) return c.aligned ? rows_with<THREADS, T, NV, WAYS, false, true, true>(c) : rows_with<THREADS, T, NV, WAYS, false, true, false>(c);
    return c.aligned ? rows_with<THREADS, T, NV, WAYS, false, false, true>(c) : rows_with<THREADS, T, NV, WAYS, false, false, false>(c);
}

template <bool CAP, bool DOCS>
int sweep_with(const ScoreCall& c, int cs) {
    if (c.backward) return launch_clusters(kScoreName, score_softmax_backward_sweep_kernel<CAP, DOCS>, c.a.rows * cs, kSweepThreads, 0, cs, c.st, c.a, cs);
    return launch_clusters(kScoreName, score_softmax_sweep_kernel<CAP, DOCS>, c.a.rows * cs, kSweepThreads, 0, cs, c.st, c.a, cs);
}
// CTAs per row beyond what one CTA holds: until what the resident CTAs (two per SM) read twice takes half of L2's
// 126 MB, for rows longer than that would be read from HBM twice (12 heads, gradients of 64 queries x 100000 keys: 1
// CTA 229 us, 4 188, 8 219; 512 x 16384: 1 CTA 217, 2 246); or, with few rows, until the last round of CTAs is
// at least four fifths full while each CTA has 4096 keys.
int sweep_ctas(const ScoreCall& c) {
    const int64_t row_bytes = c.a.g.keys * 4 * (c.backward ? (c.cap ? 3 : 2) : 1);
    const int64_t slots = 2 * c.sm_count;
    auto uneven = [&](int64_t ctas) { return ceil_div(ctas, slots) * slots * 4 > ctas * 5; };
    int cs = 1;
    while (cs < kMaxCluster && (row_bytes / cs * slots > (int64_t(64) << 20) || (uneven(c.a.rows * cs) && c.a.g.keys / (2 * cs) >= 4096))) cs *= 2;
    return cs;
}
int sweep(const ScoreCall& c, int cs) {
    if (c.cap) return c.docs ? sweep_with<true, true>(c, cs) : sweep_with<true, false>(c, cs);
    return c.docs ? sweep_with<false, true>(c, cs) : sweep_with<false, false>(c, cs);
}

// Whether all rows of the operand start on 16 bytes; fills in the distance of consecutive rows if there is one.
bool settle_rows(const ScoreGeom& g, ScoreRows* r) {
    if (!r->p) return true;
    const int64_t q = g.queries > 1 ? r->sq : 0, h = g.heads > 1 ? r->sh : 0, b = g.batch > 1 ? r->sb : 0;
    r->even = -1;
    const int64_t even = g.queries > 1 ? q : (g.heads > 1 ? h : b);
    if ((g.heads <= 1 || h == even * g.queries) && (g.batch <= 1 || b == even * g.queries * g.heads)) r->even = even;
    return is_aligned(r->p, 16) && q % 4 == 0 && h % 4 == 0 && b % 4 == 0;
}

int launch_scores(ScoreCall& c) {
    ScoreArgs& a = c.a;
    a.rows = a.g.batch * a.g.heads * a.g.queries;
    if (a.rows == 0 || a.g.keys == 0) return CTB_OK;
    if (a.rows > 0x7FFFFFFFll || a.g.keys > (1ll << 30)) return set_error(CTB_ERR_LIMIT, "score_softmax: more than 2^31 - 1 rows or 2^30 keys");
    DeviceInfo di;
    if (int rc = current_device_info(&di)) return rc;
    c.sm_count = di.sm_count;
    a.by_queries = make_fastdiv((uint32_t)a.g.queries);
    a.by_heads = make_fastdiv((uint32_t)a.g.heads);
    c.cap = a.g.cap > 0.0f;
    c.docs = a.g.key_docs.p != nullptr;
    const bool rows_aligned = settle_rows(a.g, &a.s) & settle_rows(a.g, &a.p) & settle_rows(a.g, &a.dp);
    c.aligned = rows_aligned && a.g.keys % 4 == 0 && is_aligned(a.out, 16);
    // columns to deal out: up to three more than the keys where rows do not start on 16 bytes
    const int64_t n = a.g.keys % 4 == 0 && is_aligned(a.out, 16) ? a.g.keys : a.g.keys + 3;
    // Up to 512 columns a team takes 16 bytes a lane and as few lanes as hold the row four to a lane (rows of 64
    // keys with a warp each spent most instructions on finding their place: 98304 rows 21.8 us, so 8.0);
    // wider forward rows eight fours a lane, backward rows, with two or three operands, four.
    c.cs = 1;
    if (n <= 32) return rows_as<256, 8, 1, kBoth>(c);
    if (n <= 64) return rows_as<256, 8, 2, kBoth>(c);
    if (n <= 128) return rows_as<256, 8, 4, kBoth>(c);
    if (n <= 256) return rows_as<256, 16, 4, kBoth>(c);
    if (n <= 512) return rows_as<256, 32, 4, kBoth>(c);
    if (n <= 1024) return c.backward ? rows_as<256, 64, 4, kBackward>(c) : rows_as<256, 32, 8, kForward>(c);
    if (n <= 2048) return c.backward ? rows_as<256, 128, 4, kBackward>(c) : rows_as<256, 64, 8, kForward>(c);
    // Few long rows: a cluster of CTAs holds each, as many as it takes to occupy the machine while each has 2048
    // columns.  (With rows enough, clusters cost more than they bring: forward, 6144 rows of 16384 keys, 1 CTA
    // 143 us, 2 268, 4 490; gradients 217 swept by one CTA, 361 held by four.)
    const int64_t most = c.backward ? 8192 : 16384;      // columns in the registers of one CTA
    while (c.cs < kMaxCluster && a.rows * c.cs * 2 <= c.sm_count && n / (c.cs * 2) >= 2048) c.cs *= 2;
    if (c.cs > 1 && n <= most * c.cs) return c.backward ? rows_as<512, 512, 4, kBackward>(c) : rows_as<512, 512, 8, kForward>(c);
    c.cs = 1;
    if (n <= 4096) return c.backward ? rows_as<256, 256, 4, kBackward>(c) : rows_as<256, 128, 8, kForward>(c);
    if (n <= 8192 && !c.backward) return rows_as<256, 256, 8, kForward>(c);
    if (n <= most) return c.backward ? rows_as<512, 512, 4, kBackward>(c) : rows_as<512, 512, 8, kForward>(c);
    // Rows that would be swept by clusters are held by them if they fit.
    c.cs = sweep_ctas(c);
    if (c.cs > 1 && n <= most * c.cs) return c.backward ? rows_as<512, 512, 4, kBackward>(c) : rows_as<512, 512, 8, kForward>(c);
    return sweep(c, c.cs);
}

}  // namespace

int launch_score_softmax(const ScoreGeom& g, ScoreRows scores, float* out, cudaStream_t st) {
    ScoreCall c{};
    c.a.g = g;
    c.a.s = scores;
    c.a.out = out;
    c.st = st;
    return launch_scores(c);
}

int launch_score_softmax_backward(const ScoreGeom& g, ScoreRows grad, ScoreRows probs, ScoreRows scores, float* grad_scores,
                                  float* grad_slopes, double* partials, cudaStream_t st) {
    ScoreCall c{};
    ScoreArgs& a = c.a;
    a.g = g;
    a.s = scores;
    a.p = probs;
    a.dp = grad;
    a.out = grad_scores;
    a.slope_part = grad_slopes ? partials : nullptr;
    c.backward = true;
    c.st = st;
    if (int rc = launch_scores(c)) return rc;
    if (!grad_slopes || g.heads == 0) return CTB_OK;
    if (a.rows == 0 || g.keys == 0) {                    // sums over nothing
        CTB_CUDA_TRY(cudaMemsetAsync(grad_slopes, 0, (size_t)g.heads * sizeof(float), st));
        return CTB_OK;
    }
    return launch_early(score_slope_fold_kernel, (unsigned)g.heads, 256, st, partials, g.batch, g.heads, g.queries, grad_slopes);
}

}  // namespace ctb
