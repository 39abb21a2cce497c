// Log probabilities of given tokens with entropy and the likeliest alternatives, and their gradient.
//
// Forward, one pass over a row: with the running maximum m, d = x - m, S = sum e^d and U = sum e^d d,
//   lse = m + ln S     logprob = x_target - lse     entropy = ln S - U / S;
// when m grows to m', S and U become c S and c (U + (m - m') S) with c = e^(m - m').  Partial results of threads,
// wavefronts and parts of a row meet by the same rule.  The alternatives ride along: each wavefront keeps its best `top` values
// sorted over its lanes and looks closer only at elements above the last of them.
//
// Backward, element by element: w (1[j = target] - p_j) - h p_j (x_j - lse + entropy), p_j = e^(x_j - lse).
#include "wk_internal.hpp"

#include <cmath>

using namespace wk;

namespace {

template <typename T> struct stat_of { using type = float; };
template <> struct stat_of<double> { using type = double; };

constexpr uint32_t TOP_MAX = WK_TOKEN_TOP_MAX;
static_assert(TOP_MAX == 64, "one alternative per lane");
constexpr uint32_t MAX_PARTS = 64; // of a row: one per lane when they are joined
constexpr int JOIN_THREADS = 1024;

__device__ __forceinline__ float lowest(float) { return -__builtin_inff(); }
__device__ __forceinline__ double lowest(double) { return -__builtin_inf(); }
// e^d for d <= 0: the base-2 exponential of the hardware (one unit in the last place) on f32
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * 1.44269504088896340736f); }
__device__ __forceinline__ double exp_of(double d) { return exp(d); }
// e * d, 0 for a masked logit, which has e = 0 and d = -inf (a NaN in d is one in e too)
__device__ __forceinline__ float mul0(float e, float d) { return e * fmaxf(d, -3.402823466e38f); }
__device__ __forceinline__ double mul0(double e, double d) { return e * fmax(d, -1.7976931348623157e308); }
__device__ __forceinline__ float max_of(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double max_of(double a, double b) { return fmax(a, b); }

template <typename A> struct Stats {
    A m, s, u;
};

template <typename A> __device__ __forceinline__ Stats<A> no_stats() { return {lowest(A(0)), A(0), A(0)}; }

// a's sums seen from the maximum m (a.m <= m); an empty a stays empty
template <typename A> __device__ __forceinline__ void rebase(Stats<A> &a, A m) {
    const A shift = a.m == m ? A(0) : a.m - m; // (equal infinities have no difference)
    const A c = exp_of(shift);
    a.s *= c; // (first: with c = 0 the shift may be too large to multiply the sum)
    a.u = c * a.u + mul0(a.s, shift);
    a.m = m;
}

template <typename A> __device__ __forceinline__ Stats<A> join(Stats<A> a, Stats<A> b) {
    const A m = max_of(a.m, b.m);
    rebase(a, m);
    rebase(b, m);
    return {m, a.s + b.s, a.u + b.u};
}

__device__ __forceinline__ int lane_of(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ float lane_of(float v, int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane)); }
__device__ __forceinline__ double lane_of(double v, int lane) {
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), lane), __builtin_amdgcn_readlane(__double2loint(v), lane));
}
// each lane's lower neighbour's value (lane 0: its own)
__device__ __forceinline__ int from_below(int v) { return __builtin_amdgcn_update_dpp(v, v, 0x138 /* wave_shr:1 */, 0xf, 0xf, false); }
__device__ __forceinline__ float from_below(float v) { return __int_as_float(from_below(__float_as_int(v))); }
__device__ __forceinline__ double from_below(double v) { return __hiloint2double(from_below(__double2hiint(v)), from_below(__double2loint(v))); }
// A wavefront's best values, lane l the l-th best with its index; lanes without one hold -inf and -1.
template <typename A> struct Best {
    A v;
    int32_t id;
};

// Puts (v, id), the same in every lane and v > -inf, into the list, behind equal values that are in it already.
template <typename A> __device__ __forceinline__ void insert(Best<A> &b, A v, int32_t id, uint32_t lane) {
    const uint32_t pos = (uint32_t)__popcll(__ballot(b.v >= v));
    const A up = from_below(b.v);
    const int32_t up_id = from_below(b.id);
    b.v = lane > pos ? up : lane == pos ? v : b.v;
    b.id = lane > pos ? up_id : lane == pos ? id : b.id;
}

// A value that at least `top` of the wavefront's values are above: just below the top-th largest of the lanes' maxima, whose
// order as a whole number is found bit by bit from above (20 bits; f64: of the upper word), one comparison of all lanes
// each.  -inf where so many lanes have none.
__device__ __forceinline__ uint32_t order_of(uint32_t bits) { return bits >> 31 ? ~bits : bits | 0x80000000u; }
__device__ __forceinline__ uint32_t bar_order(uint32_t order, uint32_t top) {
    uint32_t t = 0;
#pragma unroll
    for (uint32_t bit = 1u << 31; bit >= 1u << 12; bit >>= 1)
        if ((uint32_t)__popcll(__ballot(order >= (t | bit))) >= top) t |= bit;
    t -= 1u << 12; // a value before it (one step before +0 would be -0, its equal)
    return t >> 31 ? t & 0x7fffffffu : ~t;
}
__device__ __forceinline__ float first_bar(float cm, uint32_t top) {
    const float v = __uint_as_float(bar_order(order_of(__float_as_uint(cm)), top));
    return v == v ? v : lowest(v);
}
__device__ __forceinline__ double first_bar(double cm, uint32_t top) {
    const double v = __hiloint2double((int)bar_order(order_of((uint32_t)__double2hiint(cm)), top), 0);
    return v == v ? v : lowest(v);
}

// whether (v, id) comes before (w, id_w) among the alternatives; id < 0: no value there, behind all others
template <typename A> __device__ __forceinline__ bool before(A v, int32_t id, A w, int32_t id_w) {
    return id >= 0 && (id_w < 0 || v > w || (v == w && id < id_w));
}

template <typename T, int N> __device__ __forceinline__ void load_n(const T *p, uint32_t left, T raw[N]) {
    if (left >= (uint32_t)N) {
        __builtin_memcpy(raw, p, sizeof(T) * N);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) raw[e] = (uint32_t)e < left ? p[e] : (T)-__builtin_inff();
    }
}

// `raw` was read at min(c, end - N): puts the elements from c on in front, -inf behind them.
template <typename T, int N> __device__ __forceinline__ void raw_from_end(T raw[N], uint32_t c, uint32_t end) {
    const uint32_t over = c <= end - N ? 0 : c - (end - N) < (uint32_t)N ? c - (end - N) : N; // elements of others in front
    const T none = (T)-__builtin_inff();
#pragma unroll
    for (int s = N; s >= 1; s >>= 1)
#pragma unroll
        for (int e = 0; e < N; ++e) raw[e] = over & s ? (e + s < N ? raw[e + s] : none) : raw[e];
}

// What a row's finished statistics are written to; null pointers are not wanted.
template <typename A> struct Outputs {
    A *logprob, *lse, *entropy, *top_logprobs;
    int32_t *top_ids;
    const void *targets;
    bool wide_targets; // i64
};

__device__ __forceinline__ int64_t target_of(const void *targets, bool wide, uint64_t row) {
    return wide ? static_cast<const int64_t *>(targets)[row] : static_cast<const int32_t *>(targets)[row];
}

template <typename T, typename A>
__device__ __forceinline__ void finish_row(const Outputs<A> &o, const T *x, uint64_t row, uint32_t vocab, Stats<A> st) {
    const A nan = A(__builtin_nanf(""));
    const bool empty = st.m == lowest(A(0)) && st.s == A(0);
    const bool bad = !(st.s < A(__builtin_inff())); // NaN, or the sum over a NaN or +inf
    const A log_s = log(st.s);
    if (o.lse) o.lse[row] = bad ? nan : empty ? lowest(A(0)) : st.m + log_s;
    if (o.entropy) o.entropy[row] = bad ? nan : empty ? A(0) : log_s - st.u / st.s;
    if (o.logprob) {
        const int64_t t = target_of(o.targets, o.wide_targets, row);
        A lp = A(0);
        if (bad || t >= (int64_t)vocab) lp = nan;
        else if (t >= 0) lp = empty ? lowest(A(0)) : ((A)x[t] - st.m) - log_s;
        o.logprob[row] = lp;
    }
}

template <typename A> __device__ __forceinline__ void finish_top(const Outputs<A> &o, uint64_t row, uint32_t top, uint32_t place, A v, int32_t id, Stats<A> st) {
    const bool bad = !(st.s < A(__builtin_inff()));
    const bool none = bad || !(v > lowest(A(0)));
    o.top_ids[row * top + place] = none ? -1 : id;
    o.top_logprobs[row * top + place] = bad ? A(__builtin_nanf("")) : none ? lowest(A(0)) : (v - st.m) - log(st.s);
}

// One row, or a part of one, over the 64 * WAVES threads of a work-group (WAVES = 1: four rows to a work-group).  A part
// leaves its statistics and its alternatives in `ws`; a whole row is finished here.
//
// A lane takes DEEP x 16 bytes a step, all loads issued before any is used.  An alternative enters the list in ~100 cycles of the
// whole wavefront, so few should: in the first step the top-th largest of the lanes' maxima is already a bar
// under which nothing can be among the best (at least `top` values reach it), afterwards the list's last value is.
template <typename T, int WAVES, bool TOP>
__global__ __launch_bounds__(WAVES == 1 ? 256 : WAVES * 64) void logprobs_kernel(const T *__restrict__ logits, uint64_t pitch, uint64_t rows,
                                                                                uint32_t vocab, uint32_t part_len, uint32_t parts,
                                                                                uint32_t top, Outputs<typename stat_of<T>::type> o,
                                                                                typename stat_of<T>::type *ws, int32_t *ws_ids) {
    using A = typename stat_of<T>::type;
    constexpr int VE = 16 / sizeof(T);
    constexpr int DEEP = sizeof(T) == 8 ? 2 : 4;
    constexpr uint32_t CHUNK = WAVES * 64 * VE; // elements that the row's wavefronts load at once
    constexpr int ROWS = WAVES == 1 ? 4 : 1;    // rows of a work-group
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const uint64_t unit = ROWS > 1 ? blockIdx.x * 4ull + wave : blockIdx.x;
    if (ROWS > 1 && unit >= rows * parts) return; // whole wavefronts; no barrier below with one wavefront to a row
    const uint64_t row = parts == 1 ? unit : (uint32_t)unit / parts;
    const uint32_t part = parts == 1 ? 0 : (uint32_t)(unit - row * parts);
    const T *x = logits + row * pitch;
    const uint32_t begin = part * part_len, end = vocab - begin < part_len ? vocab : begin + part_len;
    Stats<A> st = no_stats<A>();
    Best<A> best{lowest(A(0)), -1};
    A bar = lowest(A(0)); // only values above it enter the list
    A floor = bar;        // the bar of the first step
    for (uint32_t c0 = begin + (ROWS > 1 ? 0 : wave * 64 * VE); c0 < end; c0 += CHUNK * DEEP) {
        T raw[DEEP][VE];
        const uint32_t mine = c0 + lane * VE;
        const bool whole = end - c0 >= CHUNK * (DEEP - 1) + 64 * VE;
        if (whole) {
#pragma unroll
            for (int u = 0; u < DEEP; ++u) __builtin_memcpy(raw[u], x + mine + u * CHUNK, 16);
        } else if (vocab >= VE) {
            // the last 16 bytes in place of what reaches beyond them, then masked: nothing waits between the loads
#pragma unroll
            for (int u = 0; u < DEEP; ++u) __builtin_memcpy(raw[u], x + (mine + u * CHUNK <= end - VE ? mine + u * CHUNK : end - VE), 16);
#pragma unroll
            for (int u = 0; u < DEEP; ++u) raw_from_end<T, VE>(raw[u], mine + u * CHUNK, end);
        } else {
#pragma unroll
            for (int u = 0; u < DEEP; ++u) {
                const uint32_t c = mine + u * CHUNK;
                load_n<T, VE>(x + (c < end ? c : begin), c < end ? end - c : 0, raw[u]);
            }
        }
        A cu[DEEP]; // the lane's maxima
#pragma unroll
        for (int u = 0; u < DEEP; ++u) {
            cu[u] = (A)raw[u][0];
#pragma unroll
            for (int e = 1; e < VE; ++e) cu[u] = max_of(cu[u], (A)raw[u][e]);
        }
        A cm = cu[0];
#pragma unroll
        for (int u = 1; u < DEEP; ++u) cm = max_of(cm, cu[u]);
        if (cm > st.m) rebase(st, cm);
        const A m = st.m == lowest(A(0)) ? A(0) : st.m;
#pragma unroll
        for (int u = 0; u < DEEP; ++u)
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const A d = (A)raw[u][e] - m, p = exp_of(d);
                st.s += p;
                st.u += mul0(p, d);
            }
        if (TOP) {
            if (c0 - begin < CHUNK) floor = bar = first_bar(cm, top);
            if (__ballot(cm > bar)) {
#pragma unroll
                for (int u = 0; u < DEEP; ++u) {
                    uint64_t some = __ballot(cu[u] > bar);
                    while (some) { // lanes in order, a lane's elements in order: equal values enter by index
                        const int l = __builtin_ctzll(some);
                        some &= some - 1;
#pragma unroll
                        for (int e = 0; e < VE; ++e) {
                            if (!(__ballot((A)raw[u][e] > bar) >> l & 1)) continue;
                            insert(best, lane_of((A)raw[u][e], l), (int32_t)(c0 + u * CHUNK + l * VE + e), lane);
                            bar = max_of(lane_of(best.v, (int)top - 1), floor);
                        }
                    }
                }
            }
        }
    }
#pragma unroll
    for (int k = 32; k; k >>= 1) {
        Stats<A> other{__shfl_xor(st.m, k), __shfl_xor(st.s, k), __shfl_xor(st.u, k)};
        st = join(st, other);
    }
    if constexpr (WAVES == 1) {
        if (parts == 1) {
            if (lane == 0) finish_row<T, A>(o, x, row, vocab, st);
            if (TOP && lane < top) finish_top<A>(o, row, top, lane, best.v, best.id, st);
        }
    } else {
        __shared__ Stats<A> all[WAVES];
        __shared__ A bv[TOP ? WAVES * TOP_MAX : 1];
        __shared__ int32_t bi[TOP ? WAVES * TOP_MAX : 1];
        if (lane == 0) all[wave] = st;
        if (TOP && lane < top) {
            bv[wave * TOP_MAX + lane] = best.v;
            bi[wave * TOP_MAX + lane] = best.id;
        }
        __syncthreads();
        st = all[0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) st = join(st, all[w]);
        if (parts == 1) {
            if (threadIdx.x == 0) finish_row<T, A>(o, x, row, vocab, st);
        } else if (threadIdx.x == 0) {
            ws[unit * 3] = st.m;
            ws[unit * 3 + 1] = st.s;
            ws[unit * 3 + 2] = st.u;
        }
        if (TOP && lane < top) {
            // place among all lists: the own one's elements in front, and what the others have that is better
            const A v = best.v;
            const int32_t id = best.id;
            uint32_t place = lane;
            for (int w = 0; w < WAVES; ++w) {
                if ((uint32_t)w == wave) continue;
                uint32_t lo = 0, hi = top; // the first entry that is not better
                while (lo < hi) {
                    const uint32_t mid = (lo + hi) / 2;
                    const A q = bv[w * TOP_MAX + mid];
                    const int32_t qi = bi[w * TOP_MAX + mid];
                    // lists' unused ends are equal: by wavefront, so that every place is taken once
                    const bool better = before(q, qi, v, id) || (qi < 0 && id < 0 && (uint32_t)w < wave);
                    if (better) lo = mid + 1;
                    else hi = mid;
                }
                place += lo;
            }
            if (place < top) {
                if (parts == 1) {
                    finish_top<A>(o, row, top, place, v, id, st);
                } else {
                    ws[rows * parts * 3 + unit * top + place] = v;
                    ws_ids[unit * top + place] = id;
                }
            }
        }
    }
}

// Joins the parts of a row, a work-group each.  With q = top / parts rounded up and r = top / q rounded up, the r-th best of
// the parts' q-th alternatives has at least top - 1 others before it: it is a bar, and the few that are not behind it go to
// LDS, where each counts those before it.
template <typename T, bool TOP>
__global__ __launch_bounds__(JOIN_THREADS) void logprobs_join_kernel(const T *__restrict__ logits, uint64_t pitch, uint64_t rows, uint32_t vocab,
                                                            uint32_t parts, uint32_t top, Outputs<typename stat_of<T>::type> o,
                                                            const typename stat_of<T>::type *__restrict__ ws, const int32_t *__restrict__ ws_ids) {
    using A = typename stat_of<T>::type;
    const uint64_t row = blockIdx.x;
    const uint32_t lane = threadIdx.x % 64;
    Stats<A> st = no_stats<A>();
    A bar = lowest(A(0));
    int32_t bar_id = -1;
    const A *v0 = ws + rows * parts * 3 + row * parts * top;
    const int32_t *i0 = ws_ids + row * parts * top;
    const uint32_t each = TOP ? (top + parts - 1) / parts : 1;
    if (lane < parts) { // at most 64 parts
        const A *p = ws + (row * parts + lane) * 3;
        st = {p[0], p[1], p[2]};
        if (TOP) {
            bar = v0[lane * top + each - 1];
            bar_id = i0[lane * top + each - 1];
        }
    }
#pragma unroll
    for (int k = 32; k; k >>= 1) {
        Stats<A> other{__shfl_xor(st.m, k), __shfl_xor(st.s, k), __shfl_xor(st.u, k)};
        st = join(st, other);
    }
    if (threadIdx.x == 0) finish_row<T, A>(o, logits + row * pitch, row, vocab, st);
    if constexpr (TOP) {
        __shared__ A cv[MAX_PARTS * TOP_MAX];
        __shared__ int32_t ci[MAX_PARTS * TOP_MAX];
        __shared__ uint32_t count;
        if (threadIdx.x == 0) count = 0;
        uint32_t above = 0; // parts are in the order of their indexes, and only a part without an alternative has -inf
        for (uint32_t l = 0; l < parts; ++l) {
            const A other = lane_of(bar, l);
            above += other > bar || (other == bar && l < lane);
        }
        const uint64_t at_bar = __ballot(lane < parts && above == (top + each - 1) / each - 1);
        bar_id = lane_of(bar_id, __builtin_ctzll(at_bar));
        bar = lane_of(bar, __builtin_ctzll(at_bar));
        __syncthreads();
        for (uint32_t q = threadIdx.x; q < parts * top; q += JOIN_THREADS) {
            const A v = v0[q];
            const int32_t id = i0[q];
            if (id >= 0 && !before(bar, bar_id, v, id)) { // (a part without so many alternatives: id < 0, no bar)
                const uint32_t at = atomicAdd(&count, 1u); // any order: places are counted
                cv[at] = v;
                ci[at] = id;
            }
        }
        __syncthreads();
        const uint32_t left = count;
        for (uint32_t q = threadIdx.x; q < (left > top ? left : top); q += JOIN_THREADS) {
            if (q >= left) { // fewer alternatives than wanted
                finish_top<A>(o, row, top, q, lowest(A(0)), -1, st);
                continue;
            }
            const A v = cv[q];
            const int32_t id = ci[q];
            uint32_t place = 0;
            for (uint32_t w = 0; w < left; ++w) place += before(cv[w], ci[w], v, id);
            if (place < top) finish_top<A>(o, row, top, place, v, id, st);
        }
    }
}

// Parts that a row is cut into, when the caller gives a workspace: so many that the launch has about four work-groups per
// compute unit, each with at least 2048 elements.
uint32_t row_parts(uint64_t rows, uint64_t vocab) {
    if (rows >= 1024) return 1;
    uint64_t parts = (1024 + rows - 1) / rows, most = vocab / 2048;
    if (parts > most) parts = most;
    if (parts > MAX_PARTS) parts = MAX_PARTS;
    return parts < 2 ? 1 : (uint32_t)parts;
}

size_t parts_bytes(uint64_t rows, uint32_t parts, uint32_t top, size_t stat) {
    return (size_t)rows * parts * (3 * stat + (size_t)top * (stat + 4));
}

template <typename T, int WAVES>
void logprobs_enqueue(hipStream_t st, unsigned grid, const T *x, uint64_t pitch, uint64_t rows, uint32_t vocab, uint32_t part_len,
                      uint32_t parts, uint32_t top, const Outputs<typename stat_of<T>::type> &o, typename stat_of<T>::type *ws, int32_t *ids) {
    const dim3 block(WAVES == 1 ? 256 : WAVES * 64);
    if (top)
        hipLaunchKernelGGL((logprobs_kernel<T, WAVES, true>), dim3(grid), block, 0, st, x, pitch, rows, vocab, part_len, parts, top, o, ws, ids);
    else
        hipLaunchKernelGGL((logprobs_kernel<T, WAVES, false>), dim3(grid), block, 0, st, x, pitch, rows, vocab, part_len, parts, top, o, ws, ids);
}

template <typename T>
int logprobs_launch(wk_stream *s, uint64_t rows, uint32_t vocab, const void *logits, uint64_t pitch, const Outputs<typename stat_of<T>::type> &o,
                    uint32_t top, void *workspace, size_t workspace_bytes) {
    using A = typename stat_of<T>::type;
    const T *x = static_cast<const T *>(logits);
    uint32_t parts = row_parts(rows, vocab);
    if (parts > 1 && (!workspace || workspace_bytes < parts_bytes(rows, parts, top, sizeof(A)))) parts = 1;
    // a part is a whole number of a work-group's steps
    constexpr uint32_t step = 256 * 16 / sizeof(T);
    uint32_t part_len = vocab;
    if (parts > 1) {
        part_len = ((vocab + parts - 1) / parts + step - 1) / step * step;
        parts = (vocab + part_len - 1) / part_len;
        if (parts == 1) part_len = vocab;
    }
    A *ws = static_cast<A *>(workspace);
    int32_t *ids = parts > 1 ? reinterpret_cast<int32_t *>(ws + (size_t)rows * parts * (3 + top)) : nullptr;
    const uint64_t units = rows * parts;
    if (units > 0x7fffffffull) return WK_E_INVALID_VALUE;
    if (parts == 1 && vocab <= 1024) logprobs_enqueue<T, 1>(s->stream, (unsigned)((units + 3) / 4), x, pitch, rows, vocab, part_len, parts, top, o, ws, ids);
    else logprobs_enqueue<T, 4>(s->stream, (unsigned)units, x, pitch, rows, vocab, part_len, parts, top, o, ws, ids);
    if (parts > 1) {
        const int rc = launch_status();
        if (rc) return rc;
        if (top)
            hipLaunchKernelGGL((logprobs_join_kernel<T, true>), dim3((unsigned)rows), dim3(JOIN_THREADS), 0, s->stream, x, pitch, rows, vocab, parts, top, o, ws, ids);
        else
            hipLaunchKernelGGL((logprobs_join_kernel<T, false>), dim3((unsigned)rows), dim3(64), 0, s->stream, x, pitch, rows, vocab, parts, top, o, ws, ids);
    }
    return launch_status();
}

constexpr int GRAD_DEEP = 4;

template <typename A> struct GradArgs {
    const A *lse, *entropy, *w, *h;
    const void *targets;
    bool wide_targets;
};

// One thread takes DEEP x 16 bytes of a row, all loads issued before any is used; blockIdx.x counts a row's segments first.
template <typename T, bool ENTROPY>
__global__ __launch_bounds__(256) void logprobs_grad_kernel(const T *x, uint64_t pitch, T *dx, uint64_t grad_pitch, uint32_t vocab,
                                                            uint32_t segments, GradArgs<typename stat_of<T>::type> a) {
    using A = typename stat_of<T>::type;
    constexpr int VE = 16 / sizeof(T);
    const uint32_t row = blockIdx.x / segments;
    const uint32_t seg = blockIdx.x - row * segments;
    const uint32_t c0 = seg * (256 * VE * GRAD_DEEP) + threadIdx.x * VE;
    const T *xr = x + (uint64_t)row * pitch;
    T *dr = dx + (uint64_t)row * grad_pitch;
    T raw[GRAD_DEEP][VE];
#pragma unroll
    for (int u = 0; u < GRAD_DEEP; ++u) {
        const uint32_t c = c0 + u * 256 * VE;
        load_n<T, VE>(xr + (c < vocab ? c : 0), c < vocab ? vocab - c : 0, raw[u]);
    }
    const A lse = a.lse[row];
    A w = A(0), h = A(0), ent = A(0);
    int64_t t = -1;
    if (a.w) {
        t = target_of(a.targets, a.wide_targets, row);
        if (t >= 0) w = t < (int64_t)vocab ? a.w[row] : A(__builtin_nanf(""));
    }
    if (ENTROPY) {
        h = a.h[row];
        ent = a.entropy[row];
    }
    const bool empty = lse == lowest(A(0));
#pragma unroll
    for (int u = 0; u < GRAD_DEEP; ++u) {
        const uint32_t c = c0 + u * 256 * VE;
        if (c >= vocab) continue;
        const bool here = t >= (int64_t)c && t < (int64_t)c + VE;
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            const A d = (A)raw[u][e] - lse, p = exp_of(d);
            A g = -w * p;
            if (ENTROPY) g -= h * mul0(p, d + ent);
            if (here && t == (int64_t)(c + e)) g += w;
            raw[u][e] = (T)(empty ? A(0) : g);
        }
        if (vocab - c >= (uint32_t)VE) {
            __builtin_memcpy(dr + c, raw[u], 16);
        } else {
#pragma unroll
            for (int e = 0; e < VE; ++e)
                if (c + e < vocab) dr[c + e] = raw[u][e];
        }
    }
}

template <typename T>
int grad_launch(wk_stream *s, uint64_t rows, uint32_t vocab, const void *x, uint64_t pitch, void *dx, uint64_t grad_pitch,
                const GradArgs<typename stat_of<T>::type> &a) {
    constexpr uint32_t step = 256 * GRAD_DEEP * 16 / sizeof(T);
    const uint32_t segments = (vocab + step - 1) / step;
    if (rows * segments > 0x7fffffffull) return WK_E_INVALID_VALUE;
    const dim3 grid((unsigned)(rows * segments));
    if (a.h)
        hipLaunchKernelGGL((logprobs_grad_kernel<T, true>), grid, dim3(256), 0, s->stream, static_cast<const T *>(x), pitch, static_cast<T *>(dx), grad_pitch, vocab, segments, a);
    else
        hipLaunchKernelGGL((logprobs_grad_kernel<T, false>), grid, dim3(256), 0, s->stream, static_cast<const T *>(x), pitch, static_cast<T *>(dx), grad_pitch, vocab, segments, a);
    return launch_status();
}

// f(element type) for the types that logits have
template <typename F> int dispatch_logits(int dtype, F &&f) {
    switch (dtype) {
    case WK_F32: return f.template operator()<float>();
    case WK_F64: return f.template operator()<double>();
    case WK_F16: return f.template operator()<_Float16>();
    case WK_BF16: return f.template operator()<__bf16>();
    default: return WK_E_TYPE_NOT_SUPPORTED;
    }
}

int check_rows(uint64_t rows, uint64_t vocab, const void *logits, uint64_t pitch, const void *targets, int target_dtype) {
    if (!rows || !vocab || !logits || vocab >> 31 || rows >> 31) return WK_E_INVALID_VALUE;
    if (rows > 1 && pitch < vocab) return WK_E_INVALID_VALUE;
    if (targets && target_dtype != WK_I32 && target_dtype != WK_I64) return WK_E_TYPE_NOT_SUPPORTED;
    return WK_OK;
}

} // namespace

extern "C" {

size_t wk_token_logprobs_workspace_bytes(int dtype, uint64_t rows, uint64_t vocab, uint32_t top) {
    if (!rows || !vocab || vocab >> 31 || rows >> 31 || top > TOP_MAX || top > vocab) return 0;
    const uint32_t parts = row_parts(rows, vocab);
    if (parts == 1) return 0;
    size_t bytes = 0;
    (void)dispatch_logits(dtype, [&]<typename T>() -> int {
        bytes = parts_bytes(rows, parts, top, sizeof(typename stat_of<T>::type));
        return WK_OK;
    });
    return bytes;
}

int wk_token_logprobs(wk_stream *s, int dtype, uint64_t rows, uint64_t vocab, const void *logits, uint64_t pitch, const void *targets,
                      int target_dtype, void *logprob, void *lse, void *entropy, uint32_t top, int32_t *top_ids, void *top_logprobs,
                      void *workspace, size_t workspace_bytes) {
    int rc = bind(s);
    if (rc) return rc;
    if ((rc = check_rows(rows, vocab, logits, pitch, targets, target_dtype))) return rc;
    if (top > TOP_MAX || top > vocab || (top && (!top_ids || !top_logprobs))) return WK_E_INVALID_VALUE;
    if ((logprob && !targets) || (!logprob && !lse && !entropy && !top)) return WK_E_INVALID_VALUE;
    if (reinterpret_cast<uintptr_t>(workspace) & 15u) return WK_E_INVALID_VALUE;
    return dispatch_logits(dtype, [&]<typename T>() -> int {
        using A = typename stat_of<T>::type;
        const Outputs<A> o{static_cast<A *>(logprob), static_cast<A *>(lse), static_cast<A *>(entropy), static_cast<A *>(top_logprobs),
                           top_ids, targets, target_dtype == WK_I64};
        return logprobs_launch<T>(s, rows, (uint32_t)vocab, logits, pitch, o, top, workspace, workspace_bytes);
    });
}

int wk_token_logprobs_grad(wk_stream *s, int dtype, uint64_t rows, uint64_t vocab, const void *logits, uint64_t pitch, const void *targets,
                           int target_dtype, const void *lse, const void *entropy, const void *logprob_grad, const void *entropy_grad,
                           void *logits_grad, uint64_t grad_pitch) {
    int rc = bind(s);
    if (rc) return rc;
    if ((rc = check_rows(rows, vocab, logits, pitch, targets, target_dtype))) return rc;
    if (!lse || !logits_grad || (!logprob_grad && !entropy_grad)) return WK_E_INVALID_VALUE;
    if ((logprob_grad && !targets) || (entropy_grad && !entropy)) return WK_E_INVALID_VALUE;
    if (rows > 1 && (grad_pitch < vocab || (logits == logits_grad && grad_pitch != pitch))) return WK_E_INVALID_VALUE;
    return dispatch_logits(dtype, [&]<typename T>() -> int {
        using A = typename stat_of<T>::type;
        const GradArgs<A> a{static_cast<const A *>(lse), static_cast<const A *>(entropy), static_cast<const A *>(logprob_grad),
                            static_cast<const A *>(entropy_grad), targets, target_dtype == WK_I64};
        return grad_launch<T>(s, rows, (uint32_t)vocab, logits, pitch, logits_grad, grad_pitch, a);
    });
}

} // extern "C"
