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
constexpr int JOIN_WAVES = 16;

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
// the value of the lane whose number differs in the bit M, without a way through LDS
template <int M> __device__ __forceinline__ int across(int v) {
    if constexpr (M == 1) return __builtin_amdgcn_mov_dpp(v, 0xb1 /* quad_perm 1, 0, 3, 2 */, 0xf, 0xf, false);
    if constexpr (M == 2) return __builtin_amdgcn_mov_dpp(v, 0x4e /* quad_perm 2, 3, 0, 1 */, 0xf, 0xf, false);
    if constexpr (M == 4) { // groups of four: the even ones from four lanes up, the odd ones from four down
        const int even = __builtin_amdgcn_update_dpp(v, v, 0x104 /* row_shl:4 */, 0xf, 0x5, false);
        return __builtin_amdgcn_update_dpp(even, v, 0x114 /* row_shr:4 */, 0xf, 0xa, false);
    }
    if constexpr (M == 8) return __builtin_amdgcn_mov_dpp(v, 0x128 /* row_ror:8 */, 0xf, 0xf, false);
    if constexpr (M == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
        return (int)(__lane_id() & 16 ? r[0] : r[1]);
    }
    if constexpr (M == 32) {
        const auto r = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
        return (int)(__lane_id() & 32 ? r[0] : r[1]);
    }
}
template <int M> __device__ __forceinline__ float across(float v) { return __int_as_float(across<M>(__float_as_int(v))); }
template <int M> __device__ __forceinline__ double across(double v) {
    return __hiloint2double(across<M>(__double2hiint(v)), across<M>(__double2loint(v)));
}

// the statistics of all lanes, in each
template <int M, typename A> __device__ __forceinline__ void join_lanes(Stats<A> &st) {
    st = join(st, Stats<A>{across<M>(st.m), across<M>(st.s), across<M>(st.u)});
    if constexpr (M > 1) join_lanes<M / 2>(st);
}

// Alternatives of a wavefront, one per lane: a value with its index.  Lanes without one hold -inf and NO_ID, which no masked logit
// becomes: only values above -inf are ever taken.
constexpr int32_t NO_ID = 0x7fffffff;
template <typename A> struct Alt {
    A v;
    int32_t id;
};
template <typename A> __device__ __forceinline__ Alt<A> no_alt() { return {lowest(A(0)), NO_ID}; }
template <typename A> __device__ __forceinline__ bool before(Alt<A> a, Alt<A> b) { return a.v > b.v || (a.v == b.v && a.id < b.id); }

// one step of a bitonic network: of the pair of lanes that differ in M, `best` lanes keep what comes first
template <int M, typename A> __device__ __forceinline__ void exchange(Alt<A> &a, bool best) {
    const Alt<A> o{across<M>(a.v), across<M>(a.id)};
    if (before(o, a) == best) a = o;
}
template <int M, typename A> __device__ __forceinline__ void exchange_down(Alt<A> &a, uint32_t lane, bool first) {
    exchange<M>(a, ((lane & M) == 0) == first);
    if constexpr (M > 1) exchange_down<M / 2>(a, lane, first);
}
// the first 64 of two sorted lists, sorted: `b` comes in reverse
template <typename A> __device__ __forceinline__ void merge_reversed(Alt<A> &a, Alt<A> b, uint32_t lane) {
    if (before(b, a)) a = b;
    exchange_down<32>(a, lane, true);
}
// a and a list in any order
template <typename A> __device__ __forceinline__ void merge_unsorted(Alt<A> &a, Alt<A> b, uint32_t lane) {
    exchange_down<1>(b, lane, (lane & 2) == 0);
    exchange_down<2>(b, lane, (lane & 4) == 0);
    exchange_down<4>(b, lane, (lane & 8) == 0);
    exchange_down<8>(b, lane, (lane & 16) == 0);
    exchange_down<16>(b, lane, (lane & 32) == 0);
    exchange_down<32>(b, lane, false);
    merge_reversed(a, b, lane);
}

// Values in order as whole numbers, and back; what lies two below a value's number (one below +0 is -0, its equal) is less.
__device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t b = __float_as_uint(v);
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t order_of(double v) {
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ float value_of(uint32_t o) { return __uint_as_float(o >> 31 ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ double value_of(uint64_t o) { return __longlong_as_double((long long)(o >> 63 ? o & 0x7fffffffffffffffull : ~o)); }

// The top-th largest of the lanes' values, found bit by bit with one comparison of all lanes each.
template <typename O> __device__ __forceinline__ O nth_order(O order, uint32_t top) {
    O t = 0;
#pragma unroll
    for (O bit = O(1) << (8 * sizeof(O) - 1); bit; bit >>= 1)
        if ((uint32_t)__popcll(__ballot(order >= (t | bit))) >= top) t |= bit;
    return t;
}

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2))); // 16 bytes at any element's address

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

template <typename A> __device__ __forceinline__ void finish_top(const Outputs<A> &o, uint64_t row, uint32_t top, uint32_t place, Alt<A> a, Stats<A> st) {
    const bool bad = !(st.s < A(__builtin_inff()));
    const bool none = bad || a.id == NO_ID;
    o.top_ids[row * top + place] = none ? -1 : a.id;
    o.top_logprobs[row * top + place] = bad ? A(__builtin_nanf("")) : none ? lowest(A(0)) : (a.v - st.m) - log(st.s);
}

// One row, or a part of one, over the 64 * WAVES threads of a work-group (WAVES = 1: four rows to a work-group).  A part
// leaves its statistics and its alternatives in `ws`; a whole row is finished here.
//
// A lane takes DEEP x 16 bytes a step, all loads issued before any is used.  Alternatives: the top-th largest of the lanes' running
// maxima is a value t that the wavefront has seen `top` times or more.  In the step that brings it, only elements not below
// t can be among the best, in later steps (higher indexes) only elements above it; those few are collected in LDS.  Where 64 come
// together they are sorted over the lanes and merged with the best so far; most rows get there once, at their end, with what all
// their wavefronts have collected.  (Putting alternatives into a sorted list one by one cost 0.25 us each where a
// wavefront has a unit for itself: one row of 131072, 64 alternatives 28 us for its parts.)
//
// Bound by memory where rows are many: 8192 x 32000 f32 154 us (6.8 TB/s).  16-bit logits with alternatives are bound by
// the exponentials as much (2048 x 50021 bf16, 5 of them: 48 us, 4.3 TB/s, 45 without); one row of 131072 f32 with 20 alternatives
// takes 8.2 us in 64 parts and 6.0 us to join them, nearly all of it latency.
template <typename T, int WAVES, bool TOP>
__global__ __launch_bounds__(WAVES == 1 ? 256 : WAVES * 64) void logprobs_kernel(const T *__restrict__ logits, uint64_t pitch, uint64_t rows,
                                                                                uint32_t vocab, uint32_t part_len, uint32_t parts,
                                                                                uint32_t top, Outputs<typename stat_of<T>::type> o,
                                                                                typename stat_of<T>::type *ws, int32_t *ws_ids, bool stream) {
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
    Alt<A> best = no_alt<A>();
    A bar = lowest(A(0)); // only values above it are collected
    constexpr int LISTS = TOP ? WAVES * ROWS : 1;
    __shared__ A lv[LISTS][TOP ? 2 * TOP_MAX : 1]; // a wavefront's collection
    __shared__ int32_t li[LISTS][TOP ? 2 * TOP_MAX : 1];
    uint32_t held = 0, taken = 0; // in the collection; since the bar moved
    bool sorted = false; // there is something in `best`
    // takes the first 64 of the collection into the best
    auto absorb = [&]() {
        const uint32_t n = held < 64 ? held : 64;
        Alt<A> b = no_alt<A>();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); // other lanes wrote it: nothing read before may stand for it
        if (lane < n) b = {lv[wave][lane], li[wave][lane]};
        const bool rest = lane + 64 < held;
        const Alt<A> r{rest ? lv[wave][lane + 64] : A(0), rest ? li[wave][lane + 64] : 0};
        merge_unsorted(best, b, lane);
        if (rest) {
            lv[wave][lane] = r.v;
            li[wave][lane] = r.id;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        held -= n;
        sorted = true;
    };
    for (uint32_t c0 = begin + (ROWS > 1 ? 0 : wave * 64 * VE); c0 < end; c0 += CHUNK * DEEP) {
        T raw[DEEP][VE];
        const uint32_t mine = c0 + lane * VE;
        const bool whole = end - c0 >= CHUNK * (DEEP - 1) + 64 * VE;
        if (whole && stream) {
#pragma unroll
            for (int u = 0; u < DEEP; ++u) {
                const u32x4_any v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any *>(x + mine + u * CHUNK));
                __builtin_memcpy(raw[u], &v, 16);
            }
        } else if (whole) {
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
            if (__ballot(cm > bar)) {
                // the bar moves in the first step and after every twelve that came over it
                A seen = bar, gate = bar;
                if (c0 - begin < CHUNK || taken >= 12) {
                    const auto nth = nth_order(order_of(st.m), top);
                    const A under = value_of(nth - 2); // (NaN below -inf)
                    seen = value_of(nth);
                    if (under > bar) gate = under;
                    taken = 0;
                }
#pragma unroll
                for (int u = 0; u < DEEP; ++u) {
                    if (!__ballot(cu[u] > gate)) continue;
#pragma unroll
                    for (int e = 0; e < VE; ++e) {
                        const A v = (A)raw[u][e];
                        const uint64_t some = __ballot(v > gate);
                        if (!some) continue;
                        if (v > gate) {
                            const uint32_t at = held + __builtin_amdgcn_mbcnt_hi((uint32_t)(some >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)some, 0));
                            lv[wave][at] = v;
                            li[wave][at] = (int32_t)(mine + u * CHUNK + e);
                        }
                        held += (uint32_t)__popcll(some);
                        taken += (uint32_t)__popcll(some);
                        if (held >= 64) absorb();
                    }
                }
                bar = seen;
            }
        }
    }
    if (TOP && ROWS > 1 && held) absorb();
    join_lanes<32>(st);
    if constexpr (WAVES == 1) {
        if (parts == 1) {
            if (lane == 0) finish_row<T, A>(o, x, row, vocab, st);
            if (TOP && lane < top) finish_top<A>(o, row, top, lane, best, st);
        }
    } else {
        __shared__ Stats<A> all[WAVES];
        __shared__ A bars[WAVES];
        __shared__ A tv[TOP ? WAVES * 64 : 1]; // what is left of all wavefronts' collections
        __shared__ int32_t ti[TOP ? WAVES * 64 : 1];
        __shared__ uint32_t total;
        if (lane == 0) {
            all[wave] = st;
            if (TOP) bars[wave] = bar;
        }
        if (TOP && threadIdx.x == 0) total = 0;
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
        if constexpr (TOP) {
#pragma unroll
            for (int w = 0; w < WAVES; ++w) bar = max_of(bar, bars[w]); // what any of them has seen `top` times
            const Alt<A> c = lane < held ? Alt<A>{lv[wave][lane], li[wave][lane]} : no_alt<A>();
            const bool stays = lane < held && c.v >= bar;
            const uint64_t some = __ballot(stays);
            uint32_t base = 0;
            if (lane == 0 && some) base = atomicAdd(&total, (uint32_t)__popcll(some)); // in any order: they are sorted
            base = (uint32_t)lane_of((int)base, 0);
            if (stays) {
                const uint32_t at = base + __builtin_amdgcn_mbcnt_hi((uint32_t)(some >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)some, 0));
                tv[at] = c.v;
                ti[at] = c.id;
            }
            if (sorted && wave) {
                lv[wave][127 - lane] = best.v; // in reverse, behind the collection
                li[wave][127 - lane] = best.id;
            }
            __shared__ uint32_t has_list[WAVES];
            if (lane == 0) has_list[wave] = sorted;
            __syncthreads();
            if (wave == 0) {
                for (uint32_t q = 0; q < total; q += 64) {
                    const Alt<A> b = q + lane < total ? Alt<A>{tv[q + lane], ti[q + lane]} : no_alt<A>();
                    merge_unsorted(best, b, lane);
                }
                for (int w = 1; w < WAVES; ++w)
                    if (has_list[w]) merge_reversed(best, Alt<A>{lv[w][64 + lane], li[w][64 + lane]}, lane);
                if (lane < top) {
                    if (parts == 1) {
                        finish_top<A>(o, row, top, lane, best, st);
                    } else {
                        ws[rows * parts * 3 + unit * top + lane] = best.v;
                        ws_ids[unit * top + lane] = best.id;
                    }
                }
            }
        }
    }
}

// Joins the parts of a row, a work-group each: sixteen wavefronts merge up to four lists each, then each other's.
template <typename T, bool TOP>
__global__ __launch_bounds__(TOP ? JOIN_WAVES * 64 : 64) void logprobs_join_kernel(const T *__restrict__ logits, uint64_t pitch, uint64_t rows, uint32_t vocab,
                                                                                   uint32_t parts, uint32_t top, Outputs<typename stat_of<T>::type> o,
                                                                                   const typename stat_of<T>::type *__restrict__ ws, const int32_t *__restrict__ ws_ids) {
    using A = typename stat_of<T>::type;
    const uint64_t row = blockIdx.x;
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    constexpr int LISTS = MAX_PARTS / JOIN_WAVES;
    Stats<A> st = no_stats<A>();
    if (lane < parts && wave == 0) {
        const A *p = ws + (row * parts + lane) * 3;
        st = {p[0], p[1], p[2]};
    }
    Alt<A> list[LISTS];
    if (TOP) {
        const A *v0 = ws + rows * parts * 3 + row * parts * top;
        const int32_t *i0 = ws_ids + row * parts * top;
#pragma unroll
        for (int k = 0; k < LISTS; ++k) { // the first one forwards, the others in reverse
            const uint32_t p = wave + k * JOIN_WAVES, at = k ? 63 - lane : lane;
            list[k] = no_alt<A>();
            if (p < parts && at < top) list[k] = {v0[p * top + at], i0[p * top + at]};
        }
    }
    if (wave == 0) {
        join_lanes<32>(st);
        if (lane == 0) finish_row<T, A>(o, logits + row * pitch, row, vocab, st);
    }
    if constexpr (TOP) {
        __shared__ A lv[JOIN_WAVES][64];
        __shared__ int32_t li[JOIN_WAVES][64];
#pragma unroll
        for (int k = 1; k < LISTS; ++k)
            if (wave + k * JOIN_WAVES < parts) merge_reversed(list[0], list[k], lane);
        uint32_t left = parts < JOIN_WAVES ? parts : JOIN_WAVES; // wavefronts with a list
        while (left > 1) {
            const uint32_t half = (left + 1) / 2;
            if (wave >= half && wave < left) {
                lv[wave][63 - lane] = list[0].v;
                li[wave][63 - lane] = list[0].id;
            }
            __syncthreads();
            if (wave + half < left) merge_reversed(list[0], Alt<A>{lv[wave + half][lane], li[wave + half][lane]}, lane);
            left = half;
        }
        if (wave == 0 && lane < top) finish_top<A>(o, row, top, lane, list[0], st);
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
    // Logits of which the last-level cache (256 MB) would not keep enough until the backward pass go by it: 8192 x 32000 f32
    // 177 -> 154 us, 2048 x 50021 bf16 with alternatives 52 -> 48; below half of the cache what was just written is found there.
    // Two sets of logits in turn, without and with it: f32 96 MB 19.0 and 18.4, 128 MB 23.8 and 23.8, 160 MB 31.4 and 28.7, 256 MB 48.4
    // and 43.7; bf16 128 MB 30.5 and 30.7, 160 MB 38.0 and 37.6, 256 MB 58.6 and 56.5.
    const bool stream = rows * vocab * sizeof(T) > (128ull << 20);
    const dim3 block(WAVES == 1 ? 256 : WAVES * 64);
    if (top)
        hipLaunchKernelGGL((logprobs_kernel<T, WAVES, true>), dim3(grid), block, 0, st, x, pitch, rows, vocab, part_len, parts, top, o, ws, ids, stream);
    else
        hipLaunchKernelGGL((logprobs_kernel<T, WAVES, false>), dim3(grid), block, 0, st, x, pitch, rows, vocab, part_len, parts, top, o, ws, ids, stream);
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
    if ((parts == 1 && vocab <= 1024 ? (units + 3) / 4 : units) > most_groups(256)) return WK_E_INVALID_VALUE;
    if (parts == 1 && vocab <= 1024) logprobs_enqueue<T, 1>(s->stream, (unsigned)((units + 3) / 4), x, pitch, rows, vocab, part_len, parts, top, o, ws, ids);
    else logprobs_enqueue<T, 4>(s->stream, (unsigned)units, x, pitch, rows, vocab, part_len, parts, top, o, ws, ids);
    if (parts > 1) {
        const int rc = launch_status();
        if (rc) return rc;
        if (top)
            hipLaunchKernelGGL((logprobs_join_kernel<T, true>), dim3((unsigned)rows), dim3(JOIN_WAVES * 64), 0, s->stream, x, pitch, rows, vocab, parts, top, o, ws, ids);
        else
            hipLaunchKernelGGL((logprobs_join_kernel<T, false>), dim3((unsigned)rows), dim3(64), 0, s->stream, x, pitch, rows, vocab, parts, top, o, ws, ids);
    }
    return launch_status();
}

constexpr int GRAD_DEEP = 2;

template <typename A> struct GradArgs {
    const A *lse, *entropy, *w, *h;
    const void *targets;
    bool wide_targets;
};

// One thread takes GRAD_DEEP x 16 bytes of a row, all loads issued before any is used; blockIdx.x counts a row's segments first.
// STREAM: both tensors together are more than the last-level cache holds (256 MB), so that neither is kept there: 4096 x 65536 bf16
// 190 -> 167 us (6.4 TB/s), where 1000 x 32003 f32, which it half holds, loses (39 -> 45; two sets of both in turn: 128 MB 21.4 -> 24.6,
// 160 MB 32.5 -> 29.7, 224 MB 43.4 -> 39.8, 320 MB 59.3 -> 54.8).  Two loads in flight per thread did
// better than one, four and eight (171 against 175, 180 and 185).
template <typename T, bool ENTROPY, bool STREAM>
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
        if (STREAM && c < vocab && vocab - c >= (uint32_t)VE) {
            const u32x4_any v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any *>(xr + c));
            __builtin_memcpy(raw[u], &v, 16);
        } else {
            load_n<T, VE>(xr + (c < vocab ? c : 0), c < vocab ? vocab - c : 0, raw[u]);
        }
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
    const A none = t >= (int64_t)vocab ? A(__builtin_nanf("")) : A(0); // an empty row's gradient
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
            raw[u][e] = (T)(empty ? none : g);
        }
        if (vocab - c >= (uint32_t)VE) {
            u32x4_any v;
            __builtin_memcpy(&v, raw[u], 16);
            u32x4_any *to = reinterpret_cast<u32x4_any *>(dr + c);
            if (STREAM) __builtin_nontemporal_store(v, to);
            else *to = v;
        } else {
#pragma unroll
            for (int e = 0; e < VE; ++e)
                if (c + e < vocab) dr[c + e] = raw[u][e];
        }
    }
}

template <typename T, bool ENTROPY, bool STREAM>
void grad_enqueue(hipStream_t st, uint64_t rows, uint32_t vocab, const void *x, uint64_t pitch, void *dx, uint64_t grad_pitch, uint32_t segments,
                  const GradArgs<typename stat_of<T>::type> &a) {
    hipLaunchKernelGGL((logprobs_grad_kernel<T, ENTROPY, STREAM>), dim3((unsigned)(rows * segments)), dim3(256), 0, st,
                       static_cast<const T *>(x), pitch, static_cast<T *>(dx), grad_pitch, vocab, segments, a);
}

template <typename T>
int grad_launch(wk_stream *s, uint64_t rows, uint32_t vocab, const void *x, uint64_t pitch, void *dx, uint64_t grad_pitch,
                const GradArgs<typename stat_of<T>::type> &a) {
    constexpr uint32_t step = 256 * GRAD_DEEP * 16 / sizeof(T);
    const uint32_t segments = (vocab + step - 1) / step;
    if (rows * segments > most_groups(256)) return WK_E_INVALID_VALUE;
    const bool stream = 2 * rows * vocab * sizeof(T) > (256ull << 20);
    if (a.h) (stream ? grad_enqueue<T, true, true> : grad_enqueue<T, true, false>)(s->stream, rows, vocab, x, pitch, dx, grad_pitch, segments, a);
    else (stream ? grad_enqueue<T, false, true> : grad_enqueue<T, false, false>)(s->stream, rows, vocab, x, pitch, dx, grad_pitch, segments, a);
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
