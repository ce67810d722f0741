// lm_beams.hip -- the selection of a beam search and the reordering of its states (gfx950).
#include "lm_tokens.h"

namespace spiky {
namespace lm {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64, kPieces = 4;
constexpr uint32_t kMostBeams = 64;

// ---- selection -----------------------------------------------------------------
// A beam's logits are cut into slices, a workgroup each, which stays in registers: its largest
// value, the sum of exponentials relative to that, and its n first candidates.  A second launch
// joins the slices of each search's beams.
template <typename T>
constexpr uint32_t slice_size() {
    return kThreads * kPieces * (16 / sizeof(T));
}

// A beam's part of the workspace: per slice the largest value and the sum, then n logits and tokens.
struct Parts {
    float2 *stats;      // [rows][slices]
    float *logits;      // [rows][slices][n], from the largest; -infinity where there are fewer
    uint32_t *tokens;
    uint32_t slices, n;
};

// Before which a candidate of the same beam comes: the larger logit, then the lower token.
__device__ __forceinline__ bool before(float x, uint32_t token, float y, uint32_t other) {
    return x > y || (x == y && token < other);
}

// What a beam takes part with.
enum Kind : uint32_t { kNothing, kLive, kFinished };

__device__ __forceinline__ Kind kind_of(const spiky_lm_beams_args &a, uint64_t row) {
    if (a.scores[row] == -INFINITY) return kNothing;
    return a.finished && a.finished[row] ? kFinished : kLive;
}

// Floats as whole numbers in their order, without NaN; both zeros are one.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

__device__ __forceinline__ float from_ordered(uint32_t u) {
    return __uint_as_float(u ^ (~(uint32_t)((int32_t)u >> 31) | 0x80000000u));
}

// A number that at least n of the wave's 64 values reach, in its upper `bits` bits: the largest such.
template <int bits>
__device__ __forceinline__ uint32_t reached_by(uint32_t value, uint32_t n) {
    uint32_t found = 0;
#pragma unroll
    for (int i = 31; i > 31 - bits; i--) {
        const uint32_t more = found | 1u << i;
        if (__popcll(__ballot(value >= more)) >= n) found = more;
    }
    return found;
}

constexpr uint32_t kMostListed = 1024;

// The n first candidates of `size` logits from column `first` on, one round over them for each: for
// lists that too many candidates would be on, as where most logits are equal.
template <typename T>
__device__ __forceinline__ void first_by_rounds(const T *x, uint32_t first, uint32_t size, float *logits,
                                                uint32_t *tokens, uint32_t n) {
    __shared__ float wave_value[2][kWaves];
    __shared__ uint32_t wave_token[2][kWaves];
    const uint32_t wave = threadIdx.x / 64, lane = threadIdx.x & 63;
    float last = INFINITY;
    uint32_t last_token = 0;
    for (uint32_t r = 0; r < n; r++) {
        float best = -INFINITY;
        uint32_t token = ~0u;
        auto take = [&](float y, uint32_t other) {
            if (before(y, other, best, token)) {
                best = y;
                token = other;
            }
        };
#pragma unroll 4
        for (uint32_t i = threadIdx.x; i < size; i += kThreads) {
            const float y = to_f32(x[first + i]);
            if (before(last, last_token, y, first + i) && y > -INFINITY) take(y, first + i);
        }
        for (int k = 32; k >= 1; k /= 2) take(__shfl_xor(best, k), __shfl_xor(token, k));
        if (lane == 0) {
            wave_value[r & 1][wave] = best;
            wave_token[r & 1][wave] = token;
        }
        __syncthreads();
        for (int w = 0; w < kWaves; w++) take(wave_value[r & 1][w], wave_token[r & 1][w]);
        if (threadIdx.x == 0) {
            logits[r] = best;
            tokens[r] = token;
        }
        last = best;
        last_token = token;
    }
}

// The n first candidates are among the values that reach a threshold which n of 64 groups of lanes
// reach with their largest: a few more than n of random logits.  These are listed, and each counts
// those before it.  n rounds over the registers, each with a barrier, took 410 us where this takes KK
// (512 beams of 152000 bf16, n = 16).
template <typename T>
__global__ __launch_bounds__(kThreads) void k_beam_slices(const spiky_lm_beams_args a, const Parts parts) {
    constexpr int N = 16 / sizeof(T);
    __shared__ float group_top[64], wave_sum[kWaves];
    __shared__ uint64_t list[kMostListed];
    __shared__ float threshold;
    __shared__ uint32_t listed;
    const uint32_t row = blockIdx.y + blockIdx.z * 32768, beams = (uint32_t)a.beams;  // searches * beams < 2^24
    if (row >= (uint32_t)a.searches * beams || kind_of(a, row) != kLive) return;
    const uint32_t slice = blockIdx.x, wave = threadIdx.x / 64, lane = threadIdx.x & 63;
    const uint32_t search = row / beams;
    const T *x = static_cast<const T *>(a.logits) + (int64_t)search * a.search_stride +
                 (int64_t)(row - search * beams) * a.beam_stride;
    float v[kPieces][N];
    uint32_t col[kPieces];
    const uint64_t first = (uint64_t)slice * slice_size<T>();
    if (first + slice_size<T>() <= a.vocab) {
        Raw<T, N> raw[kPieces];
#pragma unroll
        for (int p = 0; p < kPieces; p++) {
            col[p] = (uint32_t)first + (p * kThreads + threadIdx.x) * N;
            raw[p].load(x + col[p], N);
        }
#pragma unroll
        for (int p = 0; p < kPieces; p++)
#pragma unroll
            for (int i = 0; i < N; i++) v[p][i] = raw[p][i];
    } else {
#pragma unroll
        for (int p = 0; p < kPieces; p++) {
            Place<N> place;
            place.set(a.vocab, first + (p * kThreads + threadIdx.x) * N);
            load(v[p], x + place.col, place.n);
            col[p] = (uint32_t)place.col;
#pragma unroll
            for (int i = 0; i < N; i++) v[p][i] = place.own >> i & 1 ? v[p][i] : -INFINITY;
        }
    }
    float top = -INFINITY;
#pragma unroll
    for (int p = 0; p < kPieces; p++)
#pragma unroll
        for (int i = 0; i < N; i++) top = fmaxf(top, v[p][i]);
    top = fmaxf(top, __shfl_xor(top, 1));
    top = fmaxf(top, __shfl_xor(top, 2));
    if ((lane & 3) == 0) group_top[threadIdx.x / 4] = top;
    if (threadIdx.x == 0) listed = 0;
    __syncthreads();
    const float of_group = group_top[lane];
    top = of_group;
    for (int k = 32; k >= 1; k /= 2) top = fmaxf(top, __shfl_xor(top, k));
    if (wave == 0) {
        const uint32_t t = reached_by<16>(ordered(of_group), parts.n);
        if (lane == 0) threshold = from_ordered(max(t, ordered(-__FLT_MAX__)));  // -infinity is no candidate
    }
    const float from = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
#pragma unroll
    for (int p = 0; p < kPieces; p++)
#pragma unroll
        for (int i = 0; i < N; i++) sum += __expf(v[p][i] - from);
    for (int k = 32; k >= 1; k /= 2) sum += __shfl_xor(sum, k);
    if (lane == 0) wave_sum[wave] = sum;
    __syncthreads();
    const uint64_t at = (uint64_t)row * parts.slices + slice;
    if (threadIdx.x == 0) {
        sum = 0.f;
        for (int w = 0; w < kWaves; w++) sum += wave_sum[w];
        parts.stats[at] = make_float2(top, sum);
    }
    // bit kPieces * N - 1 of `reached`: the first value's.  Few lanes have one, and read its logit again.
    // NaN reaches nothing: it makes its beam's candidates known without a list.
    const float least = threshold;
    uint32_t reached = 0;
#pragma unroll
    for (int p = 0; p < kPieces; p++)
#pragma unroll
        for (int i = 0; i < N; i++) reached += reached + (v[p][i] >= least);
    while (reached) {
        const uint32_t i = kPieces * N - 1 - __builtin_ctz(reached), p = i / N;
        uint32_t from = col[0];
#pragma unroll
        for (int k = 1; k < kPieces; k++) from = p == k ? col[k] : from;
        const uint32_t c = from + i % N, k = atomicAdd(&listed, 1u);
        if (k < kMostListed) list[k] = (uint64_t)ordered(to_f32(x[c])) << 32 | (uint32_t)~c;
        reached &= reached - 1;
    }
    __syncthreads();
    const uint32_t count = listed;
    float *logits = parts.logits + at * parts.n;
    uint32_t *tokens = parts.tokens + at * parts.n;
    if (count > kMostListed) {
        first_by_rounds(x, (uint32_t)first, (uint32_t)min((uint64_t)slice_size<T>(), a.vocab - first), logits, tokens,
                        parts.n);
        return;
    }
    for (uint32_t i = threadIdx.x; i < max(count, parts.n); i += kThreads) {
        if (i >= count) {
            logits[i] = -INFINITY;
            continue;
        }
        const uint64_t own = list[i];
        uint32_t rank = 0;
        for (uint32_t k = 0; k < count; k++) rank += list[k] > own;
        if (rank < parts.n) {
            logits[rank] = from_ordered((uint32_t)(own >> 32));
            tokens[rank] = ~(uint32_t)own;
        }
    }
}

// A candidate of a search.
struct Candidate {
    double rank, score;
    float logit;
    uint32_t beam, token;

    __device__ __forceinline__ bool before(const Candidate &o) const {
        if (rank != o.rank) return rank > o.rank;
        if (beam != o.beam) return beam < o.beam;
        return lm::before(logit, token, o.logit, o.token);
    }
};

template <typename T>
__device__ __forceinline__ T from_lane_xor(T x, int mask) {
    static_assert(sizeof(T) % 4 == 0, "words");
    uint32_t w[sizeof(T) / 4];
    __builtin_memcpy(w, &x, sizeof(T));
#pragma unroll
    for (uint32_t i = 0; i < sizeof(T) / 4; i++) w[i] = __shfl_xor(w[i], mask);
    __builtin_memcpy(&x, w, sizeof(T));
    return x;
}

// What turns a beam's logits into ranks and scores.
struct Beam {
    double top, log_sum, score, length;
    uint32_t kind;  // of Kind
    bool unknown;   // its scores are NaN
};

constexpr int kJoinThreads = 512, kJoinWaves = kJoinThreads / 64;

// The natural logarithm of a positive normal number: of its mantissa m in [0.7, 1.5), 2 artanh z with
// z = (m - 1) / (m + 1), |z| < 0.2, as its series up to z^21 / 21.  The library's functions of
// doubles are several times as long, and a launch that runs once waits for its instructions.
__device__ __forceinline__ double log_of(double x) {
    uint64_t u = (uint64_t)__double_as_longlong(x);
    const uint64_t half = (u >> 51) & 1;  // m >= 1.5 goes down by 2
    const int64_t e = (int64_t)(u >> 52) - 1023 + (int64_t)half;
    u = (u & 0xfffffffffffffull) | (uint64_t)(1023 - half) << 52;
    const double m = __longlong_as_double((int64_t)u), z = (m - 1.0) / (m + 1.0), w = z * z;
    double p = 1.0 / 21;
#pragma unroll
    for (int k = 19; k >= 1; k -= 2) p = fma(p, w, 1.0 / k);
    return fma((double)e, 0.693147180559945309417, 2.0 * z * p);
}

// exp(x) for |x| < 700: 2^k times the series of what is left, |r| < 0.35, up to r^14 / 14!.  The
// logarithm of 2 is its first 36 bits, whose product with k has no rounding, and the rest.
__device__ __forceinline__ double exp_of(double x) {
    const double k = rint(x * 1.44269504088896340736);
    const double r = fma(k, -0x1.cf79abc9e3b3ap-40, fma(k, -0x1.62e42fefa0000p-1, x));
    double p = 1.0;
#pragma unroll
    for (int i = 14; i >= 1; i--) p = fma(p * (1.0 / i), r, 1.0);
    return __longlong_as_double(__double_as_longlong(p) + ((int64_t)k << 52));
}

// A workgroup a search.  As in a slice, candidates that reach what n groups of candidates reach are
// listed, and each counts those before it; the groups are made of the first candidates of the
// slices' lists.  Bound by latency: what does not hang on anything is read first, the beams' values
// and a thread's first logits.
__global__ __launch_bounds__(kJoinThreads) void k_beam_join(const spiky_lm_beams_args a, const Parts parts) {
    constexpr uint32_t kMost = 512, kAhead = 4;
    __shared__ Beam beams[kMostBeams];
    __shared__ Candidate list[kMost], wave_best[2][kJoinWaves];
    __shared__ uint32_t group_top[64], threshold, listed;
    const uint32_t search = blockIdx.x, row0 = search * (uint32_t)a.beams;  // searches * beams < 2^24
    const uint32_t wave = threadIdx.x / 64, lane = threadIdx.x & 63;
    const uint32_t lists = (uint32_t)a.beams * parts.slices;  // at most 64 * 2^19
    const float *logits = parts.logits + (uint64_t)row0 * parts.slices * parts.n;
    const uint32_t *tokens = parts.tokens + (uint64_t)row0 * parts.slices * parts.n;
    float ahead[kAhead];
    uint32_t ahead_token[kAhead];
#pragma unroll
    for (uint32_t o = 0; o < kAhead; o++) {
        const uint64_t at = (uint64_t)min(threadIdx.x, lists - 1) * parts.n + min(o, parts.n - 1);
        ahead[o] = logits[at];  // of no use where the list's beam is not alive
        ahead_token[o] = tokens[at];
    }
    for (uint32_t k = wave; k < a.beams; k += kJoinWaves) {
        const uint32_t row = row0 + k;
        const float score = a.scores[row];
        const bool done = a.finished && a.finished[row];
        const float2 none = make_float2(-INFINITY, 0.f);
        const float2 *stats = parts.stats + (uint64_t)row * parts.slices;
        const float2 own = lane < parts.slices ? stats[lane] : none;
        double grown = 1.0;
        if (a.lengths && a.length_penalty != 0.0) {
            const int64_t n = a.lengths_i64 ? static_cast<const int64_t *>(a.lengths)[row]
                                            : static_cast<const int32_t *>(a.lengths)[row];
            grown = fmax((double)n + (done ? 0.0 : 1.0), 1.0);
        }
        Beam b;
        b.kind = score == -INFINITY ? kNothing : done ? kFinished : kLive;
        b.score = score;
        b.unknown = false;
        float top = own.x;
        double sum = 0.0;
        if (b.kind == kLive) {
            for (uint32_t s = lane + 64; s < parts.slices; s += 64) top = fmaxf(top, stats[s].x);
            for (int i = 32; i >= 1; i /= 2) top = fmaxf(top, __shfl_xor(top, i));
            auto add = [&](const float2 &part) {
                if (part.x > -INFINITY || part.y != part.y) sum += (double)part.y * (double)__expf(part.x - top);
            };
            add(own);
            for (uint32_t s = lane + 64; s < parts.slices; s += 64) add(stats[s]);
            for (int i = 32; i >= 1; i /= 2) sum += from_lane_xor(sum, i);
            b.unknown = sum != sum || score != score || score == INFINITY;
            if (!b.unknown && top == -INFINITY) b.kind = kNothing;
        }
        b.top = top;
        b.log_sum = log_of(sum);
        b.length = grown == 1.0 ? 1.0 : exp_of(a.length_penalty * log_of(grown));
        if (lane == 0) beams[k] = b;
    }
    if (threadIdx.x == 0) listed = 0;
    if (threadIdx.x < 64) group_top[threadIdx.x] = 0;
    __syncthreads();
    const Candidate none = {-INFINITY, -INFINITY, -INFINITY, ~0u, ~0u};
    // Candidate `o` of list `l`, or none, from its logit and token.
    auto made = [&](uint32_t l, uint32_t o, float logit, uint32_t token) {
        Candidate c = none;
        const uint32_t k = l / parts.slices;
        const Beam &b = beams[k];
        if (b.kind == kNothing) return c;
        if (b.kind == kFinished) {
            if (l != k * parts.slices || o > 0) return c;
            c.token = 0;
            c.score = b.score;
        } else if (b.unknown) {
            if (l != k * parts.slices || o >= a.vocab) return c;
            c.token = o;
            c.score = NAN;
        } else {
            if (logit == -INFINITY) return c;
            c.logit = logit;
            c.token = token;
            c.score = logit - b.top - b.log_sum + b.score;
        }
        c.beam = k;
        c.rank = b.length == 1.0 ? c.score : c.score / b.length;
        if (c.rank != c.rank) c.rank = INFINITY;
        return c;
    };
    auto candidate = [&](uint32_t l, uint32_t o) {
        const uint64_t at = (uint64_t)l * parts.n + o;
        return made(l, o, logits[at], tokens[at]);
    };
    // Calls fn(number, candidate) for the first `most` of the thread's lists, kAhead at a time, up to
    // the first that fn returns false for, since those behind it are no better.
    auto each = [&](uint32_t most, auto fn) {
        for (uint32_t l = threadIdx.x; l < lists; l += kJoinThreads) {
            bool more = true;
#pragma unroll
            for (uint32_t o = 0; o < kAhead; o++)
                if (o < most && more)
                    more = fn(l * most + o, l == threadIdx.x ? made(l, o, ahead[o], ahead_token[o]) : candidate(l, o));
            for (uint32_t o = kAhead; o < most && more; o++) more = fn(l * most + o, candidate(l, o));
        }
    };
    // the first `heads` of each list: n or more in all, so that n of the 64 groups hold one
    each((parts.n + lists - 1) / lists, [&](uint32_t i, const Candidate &c) {
        atomicMax(&group_top[i & 63], ordered((float)c.rank));
        return true;
    });
    __syncthreads();
    if (wave == 0) {
        const uint32_t t = reached_by<20>(group_top[lane], parts.n);
        if (lane == 0) threshold = t;
    }
    __syncthreads();
    const uint32_t least = threshold;
    each(parts.n, [&](uint32_t, const Candidate &c) {
        if (c.beam == ~0u || ordered((float)c.rank) < least) return false;
        const uint32_t k = atomicAdd(&listed, 1u);
        if (k < kMost) list[k] = c;
        return true;
    });
    __syncthreads();
    const uint32_t count = listed;
    auto write = [&](uint32_t r, const Candidate &c) {
        const bool there = c.beam != ~0u;
        const uint64_t at = (uint64_t)search * parts.n + r;
        a.out_scores[at] = there ? (float)c.score : -INFINITY;
        a.out_parents[at] = there ? c.beam : 0;
        a.out_tokens[at] = there && beams[c.beam].kind == kLive ? c.token : a.pad;
    };
    if (count <= kMost) {
        for (uint32_t i = threadIdx.x; i < max(count, parts.n); i += kJoinThreads) {
            if (i >= count) {
                write(i, none);
                continue;
            }
            const Candidate own = list[i];
            uint32_t rank = 0;
            for (uint32_t k = 0; k < count; k++) rank += list[k].before(own);
            if (rank < parts.n) write(rank, own);
        }
        return;
    }
    // too many of one rank: a round for each
    Candidate last = none;
    for (uint32_t r = 0; r < parts.n; r++) {
        Candidate best = none;
        for (uint32_t i = threadIdx.x; i < lists * parts.n; i += kJoinThreads) {  // fewer than 2^31
            const Candidate c = candidate(i / parts.n, i % parts.n);
            if (c.beam != ~0u && (r == 0 || last.before(c)) && c.before(best)) best = c;
        }
        for (int k = 32; k >= 1; k /= 2) {
            const Candidate c = from_lane_xor(best, k);
            if (c.before(best)) best = c;
        }
        if (lane == 0) wave_best[r & 1][wave] = best;
        __syncthreads();
        for (int w = 0; w < kJoinWaves; w++)
            if (wave_best[r & 1][w].before(best)) best = wave_best[r & 1][w];
        if (threadIdx.x == 0) write(r, best);
        last = best;
    }
}

uint32_t slices_of(const spiky_lm_beams_args &a) {
    const uint32_t size = a.dtype == SPIKY_F32 ? slice_size<float>() : slice_size<bf16>();
    return a.vocab ? (uint32_t)((a.vocab + size - 1) / size) : 1;  // a finished beam needs one too
}

// ---- reordering -----------------------------------------------------------------
// A thread takes the same 16 bytes of all beams of a search, loads those that go on and stores
// them: so the result may lie in the place of the input.
constexpr int kMostStates = 16;  // of a launch, by value

struct State {
    spiky_lm_state s;
    Divider pieces;  // of a run
};

struct States {
    State of[kMostStates];
};

template <typename V, int kBeams>
__device__ __forceinline__ void move(const char *in, char *out, int64_t in_beam, int64_t out_beam,
                                     const uint32_t *parents, uint32_t beams, uint32_t n, bool in_place) {
    for (uint32_t j0 = 0; j0 < n; j0 += kBeams) {
        V v[kBeams];
#pragma unroll
        for (int j = 0; j < kBeams; j++) {
            if (j0 + j >= n) break;
            const uint32_t p = parents[j0 + j];
            if (p < beams && !(in_place && p == j0 + j))
                __builtin_memcpy(&v[j], in + (int64_t)p * in_beam, sizeof(V));
            else
                v[j] = V();
        }
#pragma unroll
        for (int j = 0; j < kBeams; j++) {
            if (j0 + j >= n) break;
            if (!(in_place && parents[j0 + j] == j0 + j))
                __builtin_memcpy(out + (int64_t)(j0 + j) * out_beam, &v[j], sizeof(V));
        }
    }
}

typedef uint32_t Words4 __attribute__((ext_vector_type(4)));

template <int kBeams>
__global__ __launch_bounds__(kThreads) void k_reorder(const States states, const void *parents_, bool i64,
                                                      uint32_t beams, uint32_t n, uint64_t first) {
    extern __shared__ uint32_t parents[];  // ~0: none
    const uint64_t search = first + blockIdx.y;
    for (uint32_t j = threadIdx.x; j < n; j += kThreads) {
        const uint64_t at = search * n + j;
        const int64_t p = i64 ? static_cast<const int64_t *>(parents_)[at] : static_cast<const int32_t *>(parents_)[at];
        parents[j] = p >= 0 && p < (int64_t)beams ? (uint32_t)p : ~0u;
    }
    __syncthreads();
    const State &state = states.of[blockIdx.z];
    const spiky_lm_state &s = state.s;
    const bool in_place = s.in == s.out;
    for (uint64_t i = (uint64_t)blockIdx.x * kThreads + threadIdx.x; i < s.runs * state.pieces.d;
         i += (uint64_t)gridDim.x * kThreads) {
        const uint64_t run = i < 0x100000000ull ? state.pieces.divide((uint32_t)i) : i / state.pieces.d;
        const uint64_t at = (i - run * state.pieces.d) * 16;
        const char *in = static_cast<const char *>(s.in) + (int64_t)search * s.in_search + (int64_t)run * s.in_run + at;
        char *out = static_cast<char *>(s.out) + (int64_t)search * s.out_search + (int64_t)run * s.out_run + at;
        const uint64_t left = s.run_bytes - at;
        if (left >= 16) {
            move<Words4, kBeams>(in, out, s.in_beam, s.out_beam, parents, beams, n, in_place);
            continue;
        }
        // the end of a run: other threads' pieces may be written already, so it keeps to its own
        uint32_t o = 0;
        if (left & 8) move<uint64_t, kBeams>(in, out, s.in_beam, s.out_beam, parents, beams, n, in_place), o += 8;
        if (left & 4) move<uint32_t, kBeams>(in + o, out + o, s.in_beam, s.out_beam, parents, beams, n, in_place), o += 4;
        if (left & 2) move<uint16_t, kBeams>(in + o, out + o, s.in_beam, s.out_beam, parents, beams, n, in_place), o += 2;
        if (left & 1) move<uint8_t, kBeams>(in + o, out + o, s.in_beam, s.out_beam, parents, beams, n, in_place);
    }
}

}  // namespace

uint64_t beam_select_workspace(const spiky_lm_beams_args &a) {
    return a.searches * a.beams * slices_of(a) * (sizeof(float2) + a.n * 8);
}

hipError_t launch_beam_select(const spiky_lm_beams_args &a, void *workspace, hipStream_t st) {
    Parts parts;
    const uint64_t rows = a.searches * a.beams;
    parts.slices = slices_of(a);
    parts.n = (uint32_t)a.n;
    parts.stats = static_cast<float2 *>(workspace);
    parts.logits = reinterpret_cast<float *>(parts.stats + rows * parts.slices);
    parts.tokens = reinterpret_cast<uint32_t *>(parts.logits + rows * parts.slices * a.n);
    const dim3 grid(parts.slices, (uint32_t)min(rows, (uint64_t)32768), (uint32_t)((rows + 32767) / 32768));
    if (a.dtype == SPIKY_F32)
        k_beam_slices<float><<<grid, dim3(kThreads), 0, st>>>(a, parts);
    else if (a.dtype == SPIKY_BF16)
        k_beam_slices<bf16><<<grid, dim3(kThreads), 0, st>>>(a, parts);
    else
        k_beam_slices<f16><<<grid, dim3(kThreads), 0, st>>>(a, parts);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    k_beam_join<<<dim3((uint32_t)a.searches), dim3(kJoinThreads), 0, st>>>(a, parts);
    return hipGetLastError();
}

hipError_t launch_reorder(const spiky_lm_state *states, uint64_t count, const void *parents, bool parents_i64,
                          uint64_t searches, uint64_t beams, uint64_t n, hipStream_t st) {
    for (uint64_t at = 0; at < count; at += kMostStates) {
        const uint64_t here = min(count - at, (uint64_t)kMostStates);
        States group = {};
        uint64_t most = 0;
        for (uint64_t i = 0; i < here; i++) {
            const uint64_t pieces = (states[at + i].run_bytes + 15) / 16;
            group.of[i] = {states[at + i], Divider((uint32_t)max(pieces, (uint64_t)1))};
            if (pieces == 0) group.of[i].s.runs = 0;
            most = max(most, group.of[i].s.runs * pieces);
        }
        if (most == 0) continue;
        const uint64_t groups = min((most + kThreads - 1) / kThreads, (uint64_t)16384);
        for (uint64_t first = 0; first < searches; first += 32768) {
            const dim3 grid((uint32_t)groups, (uint32_t)min(searches - first, (uint64_t)32768), (uint32_t)here);
            auto go = [&](auto kernel) {
                kernel<<<grid, dim3(kThreads), n * 4, st>>>(group, parents, parents_i64, (uint32_t)beams, (uint32_t)n,
                                                            first);
                return hipGetLastError();
            };
            const hipError_t e = n <= 4 ? go(k_reorder<4>) : n <= 8 ? go(k_reorder<8>) : n <= 16 ? go(k_reorder<16>)
                                 : n <= 32 ? go(k_reorder<32>) : go(k_reorder<64>);
            if (e != hipSuccess) return e;
        }
    }
    return hipSuccess;
}

}  // namespace lm
}  // namespace spiky
