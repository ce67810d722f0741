// lm_beams.hip -- the selection of a beam search and the reordering of its states (gfx950).
#include <type_traits>

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
    Divider by_n, by_slices, by_beams;
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

// The float of such a number.
__device__ __forceinline__ float from_ordered(uint32_t u) {
    return __uint_as_float(u ^ (~(uint32_t)((int32_t)u >> 31) | 0x80000000u));
}

// The same of doubles.
__device__ __forceinline__ uint64_t ordered(double x) {
    const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
    return u ^ ((uint64_t)((int64_t)u >> 63) | (uint64_t)1 << 63);
}

// Half of how far x lies below the top: finite for all but -infinity, which is no candidate.
__device__ __forceinline__ float below(float top, float x) { return fmaf(x, -0.5f, 0.5f * top); }

// The least distance from the top, to kSteps bits, that at least n of the wave's 64 values are within; the largest
// finite one where fewer are above -infinity.  Steps grow with the distance that is asked about, and not with
// an offset that all values have: by 7 or 8 bits of the values' own mantissas, 64 searches of 8 beams of 152000,
// n = 16, took 38 us with scores near -20 and 103 near -1500, where a thousand candidates reach, and fp32 logits
// near 1000 80 for 61.
constexpr int kSteps = 15;  // of a float without its sign, the exponent and 7
__device__ __forceinline__ float reach_of(float distance, uint32_t n) {
    const uint32_t near = ~__float_as_uint(distance);
    uint32_t found = 1u << 31;
#pragma unroll
    for (int i = 30; i > 30 - kSteps; i--) {
        const uint32_t more = found | 1u << i;
        if (__popcll(__ballot(near >= more)) >= n) found = more;
    }
    return __uint_as_float(min(~found, 0x7f7fffffu));
}

// The lane's value combined with those of its row of 16 lanes and of the rows before: lane 63 has all.
// DPP moves instead of shuffles, which go through LDS and take an address each.
template <typename F>
__device__ __forceinline__ float over_wave(float x, float none, F f) {
    auto step = [&](auto ctrl, auto rows) {
        x = f(x, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(none), __float_as_int(x), decltype(ctrl)::value,
                                                            decltype(rows)::value, 0xf, false)));
    };
    using All = std::integral_constant<int, 0xf>;
    step(std::integral_constant<int, 0x111>(), All());  // row_shr 1, 2, 4, 8
    step(std::integral_constant<int, 0x112>(), All());
    step(std::integral_constant<int, 0x114>(), All());
    step(std::integral_constant<int, 0x118>(), All());
    step(std::integral_constant<int, 0x142>(), std::integral_constant<int, 0xa>());  // row_bcast 15 into rows 1 and 3
    step(std::integral_constant<int, 0x143>(), std::integral_constant<int, 0xc>());  // row_bcast 31 into rows 2 and 3
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

__device__ __forceinline__ float wave_max(float x) {
    return over_wave(x, -INFINITY, [](float a, float b) { return fmaxf(a, b); });
}

__device__ __forceinline__ float wave_sum_of(float x) {
    return over_wave(x, 0.f, [](float a, float b) { return a + b; });
}

// The largest of the lane's four.
__device__ __forceinline__ float quad_max(float x) {
    x = fmaxf(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0xb1, 0xf, 0xf, false)));  // quad_perm 1 0 3 2
    return fmaxf(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x4e, 0xf, 0xf, false)));  // 2 3 0 1
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

constexpr float kLog2E = 1.44269504088896340736f;

// The n first candidates are in units, a lane's logits, whose largest reaches a threshold that n of 64
// groups of lanes reach: few more than n units.  The logits of these that reach it too, of random ones
// few more than n again, are listed, and each counts those before it.  n rounds over the registers,
// each with a barrier, took 550 us where this takes 25 (512 beams of 152000 bf16, n = 16, 30 % of
// them finished, 109 MB).  Slices of a wave each, without barriers and with the next logits in
// flight, take 32: all are at the same point at a time, and what the choice takes at a slice's end
// has nothing beside it.  Per logit a conversion, half a maximum, a product and sum, a power of 2 (four
// times as long) and a sum.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_beam_slices(const spiky_lm_beams_args a, const Parts parts) {
    constexpr int N = 16 / sizeof(T);
    constexpr uint32_t kUnit = kPieces * N;
    __shared__ float group_top[64], wave_sum[kWaves], reach;
    __shared__ uint64_t list[kMostListed];
    __shared__ uint32_t units[kThreads], n_units, listed;
    const uint32_t row = blockIdx.y + blockIdx.z * 32768, beams = (uint32_t)a.beams;  // searches * beams < 2^24
    if (row >= (uint32_t)a.searches * beams || kind_of(a, row) != kLive) return;
    const uint32_t slice = blockIdx.x, wave = threadIdx.x / 64, lane = threadIdx.x & 63;
    const uint32_t vocab = (uint32_t)a.vocab, search = parts.by_beams.divide(row), first = slice * slice_size<T>();
    const T *x = static_cast<const T *>(a.logits) + (int64_t)search * a.search_stride +
                 (int64_t)(row - search * beams) * a.beam_stride;
    float v[kUnit];
    if (vocab - first >= slice_size<T>()) {
        Raw<T, N> raw[kPieces];
#pragma unroll
        for (int p = 0; p < kPieces; p++) raw[p].load(x + first + (p * kThreads + threadIdx.x) * N, N);
#pragma unroll
        for (int p = 0; p < kPieces; p++)
#pragma unroll
            for (int i = 0; i < N; i++) v[p * N + i] = raw[p][i];
    } else {
#pragma unroll
        for (int p = 0; p < kPieces; p++) {
            Place<N> place;
            place.set(vocab, (uint64_t)first + (p * kThreads + threadIdx.x) * N);
            float y[N];
            load(y, x + place.col, place.n);
#pragma unroll
            for (int i = 0; i < N; i++) {
                // the last piece's columns in their places, in front of which it has others'
                v[p * N + i] = place.own >> i & 1 ? y[i] : -INFINITY;
            }
        }
    }
    float here = v[0];
#pragma unroll
    for (uint32_t i = 1; i < kUnit; i++) here = fmaxf(here, v[i]);
    float top = quad_max(here);
    if ((lane & 3) == 0) group_top[threadIdx.x / 4] = top;
    if (threadIdx.x == 0) listed = n_units = 0;
    __syncthreads();
    const float of_group = group_top[lane];
    top = wave_max(of_group);
    if (wave == 0) {
        const float t = reach_of(below(top, of_group), parts.n);
        if (lane == 0) reach = t;
    }
    float sum = 0.f;
    if (fabsf(top) <= 1e6f) {  // relative to 2^power, and in the end to exp(top)
        const float power = rintf(top * kLog2E);
#pragma unroll
        for (uint32_t i = 0; i < kUnit; i++) sum += __builtin_amdgcn_exp2f(fmaf(v[i], kLog2E, -power));
        sum *= __builtin_amdgcn_exp2f(fmaf(-top, kLog2E, power));
    } else {  // whose power of 2 has no fraction left
        const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (uint32_t i = 0; i < kUnit; i++) sum += __builtin_amdgcn_exp2f((v[i] - from) * kLog2E);
    }
    sum = wave_sum_of(sum);
    if (lane == 0) wave_sum[wave] = sum;
    __syncthreads();
    const uint64_t at = (uint64_t)row * parts.slices + slice;
    if (threadIdx.x == 0) {
        sum = 0.f;
        for (int w = 0; w < kWaves; w++) sum += wave_sum[w];
        parts.stats[at] = make_float2(top, sum);
    }
    // NaN reaches nothing: it makes its beam's candidates known without a list
    const float most = reach;
    if (below(top, here) <= most) units[atomicAdd(&n_units, 1u)] = threadIdx.x;
    __syncthreads();
    // a unit's logits are read again, a few by each thread
    constexpr uint32_t kAhead = 4;
    const uint32_t all = n_units * kUnit;
    for (uint32_t i = threadIdx.x; i < all; i += kThreads * kAhead) {
        T y[kAhead];
        uint32_t col[kAhead];
#pragma unroll
        for (uint32_t j = 0; j < kAhead; j++) {
            const uint32_t o = min(i + j * kThreads, all - 1), e = o % kUnit;
            col[j] = first + (e / N * kThreads + units[o / kUnit]) * N + e % N;
            y[j] = x[min(col[j], vocab - 1)];
        }
#pragma unroll
        for (uint32_t j = 0; j < kAhead; j++) {
            if (i + j * kThreads >= all || col[j] >= vocab || !(below(top, to_f32(y[j])) <= most)) continue;
            const uint32_t k = atomicAdd(&listed, 1u);
            if (k < kMostListed) list[k] = (uint64_t)ordered(to_f32(y[j])) << 32 | (uint32_t)~col[j];
        }
    }
    __syncthreads();
    const uint32_t count = listed;
    float *logits = parts.logits + at * parts.n;
    uint32_t *tokens = parts.tokens + at * parts.n;
    if (count > kMostListed) {
        first_by_rounds(x, first, min(slice_size<T>(), vocab - first), logits, tokens, parts.n);
        return;
    }
    for (uint32_t i = threadIdx.x; i < max(count, parts.n); i += kThreads) {
        if (i >= count) {
            logits[i] = -INFINITY;
            continue;
        }
        const uint64_t own = list[i];
        uint32_t rank = 0;
#pragma unroll 4
        for (uint32_t k = 0; k < count; k++) rank += list[k] > own;
        if (rank < parts.n) {
            logits[rank] = from_ordered((uint32_t)(own >> 32));
            tokens[rank] = ~(uint32_t)own;
        }
    }
}

// A candidate of a search, as numbers that it is compared by: the largest `first`, then the smallest
// `second` and the lowest token come first.
struct Candidate {
    uint64_t first;   // the rank, ordered; 0: no candidate
    uint64_t second;  // the beam, and the logit against its order
    uint32_t token;
    float score;

    __device__ __forceinline__ bool before(const Candidate &o) const {
        return (first > o.first) | ((first == o.first) & ((second < o.second) | ((second == o.second) & (token < o.token))));
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
constexpr uint32_t kSearchesX = 1u << 20;  // of a grid's x, whose threads have to stay below 2^32

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
    constexpr uint32_t kMost = 512;
    __shared__ Beam beams[kMostBeams];
    __shared__ Candidate list[kMost], wave_best[2][kJoinWaves];
    __shared__ uint32_t ranks[kMost];
    __shared__ uint32_t group_top[64], open_list[kMost], open, listed;
    __shared__ float2 top_and_reach;
    const uint32_t search = blockIdx.x + blockIdx.y * kSearchesX, row0 = search * (uint32_t)a.beams;  // searches * beams < 2^24
    if (search >= a.searches) return;
    const uint32_t wave = threadIdx.x / 64, lane = threadIdx.x & 63;
    const uint32_t lists = (uint32_t)a.beams * parts.slices;
    const float *logits = parts.logits + (uint64_t)row0 * parts.slices * parts.n;
    const uint32_t *tokens = parts.tokens + (uint64_t)row0 * parts.slices * parts.n;
    // the first `heads` candidates of each list: n or more in all, and enough for the groups
    const uint32_t heads = min(parts.n, (63 + lists) / lists);
    // Where the first heads number i lie: list i / heads, candidate i % heads.
    auto head_at = [&](uint32_t i) { return heads == 1 ? i * parts.n : i / heads * parts.n + i % heads; };
    const uint32_t first_at = head_at(min(threadIdx.x, lists * heads - 1));
    const float first_logit = logits[first_at];  // of no use where the list's beam is not alive
    const uint32_t first_token = tokens[first_at];
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
            b.unknown = sum != sum || top == INFINITY || score != score || score == INFINITY;
            if (!b.unknown && top == -INFINITY) b.kind = kNothing;
        }
        b.top = top;
        b.log_sum = log_of(sum);
        b.length = grown == 1.0 ? 1.0 : exp_of(a.length_penalty * log_of(grown));
        if (lane == 0) beams[k] = b;
    }
    if (threadIdx.x == 0) listed = open = 0;
    if (threadIdx.x < 64) group_top[threadIdx.x] = ordered(-INFINITY);
    __syncthreads();
    const Candidate none = {0, ~(uint64_t)0, ~0u, -INFINITY};
    // Candidate `o` of list `l`, or none, from its logit and token; and its rank in 32 bits, finite, or -infinity for none.
    auto made = [&](uint32_t l, uint32_t o, float logit, uint32_t token, float &coarse) {
        const uint32_t k = parts.by_slices.divide(l);
        const Beam &b = beams[k];
        const bool only = l == k * parts.slices;  // what finished and unknown beams have is in their first list
        bool there = logit > -INFINITY;
        double score = logit - b.top - b.log_sum + b.score;
        if (b.kind != kLive || b.unknown) {
            there = only && b.kind != kNothing && (b.kind == kFinished ? o == 0 : o < a.vocab);
            score = b.kind == kFinished ? b.score : NAN;
            token = b.kind == kFinished ? 0 : o;
            logit = 0.f;
        }
        double rank = b.length == 1.0 ? score : score / b.length;
        rank = rank != rank ? INFINITY : rank;
        coarse = there ? fminf(fmaxf((float)rank, -__FLT_MAX__), __FLT_MAX__) : -INFINITY;
        if (!there) return none;
        return Candidate{ordered(rank), (uint64_t)k << 32 | (uint32_t)~ordered(logit), token, (float)score};
    };
    // The candidate at `at` of the search's part of the workspace, at most 64 * 2^19 * 64 = 2^31 long.
    auto candidate = [&](uint32_t at, float &coarse) {
        const uint32_t l = parts.by_n.divide(at);
        return made(l, at - l * parts.n, logits[at], tokens[at], coarse);
    };
    // The heads are in 64 groups; n or more of these hold one.
    for (uint32_t i = threadIdx.x; i < lists * heads; i += kJoinThreads) {
        const uint32_t at = head_at(i), l = parts.by_n.divide(at);
        float coarse;
        if (i == threadIdx.x)
            made(l, at - l * parts.n, first_logit, first_token, coarse);
        else
            candidate(at, coarse);
        atomicMax(&group_top[i & 63], ordered(coarse));
    }
    __syncthreads();
    if (wave == 0) {
        const float x = from_ordered(group_top[lane]), top = wave_max(x), t = reach_of(below(top, x), parts.n);
        if (lane == 0) top_and_reach = make_float2(top, t);
    }
    __syncthreads();
    // the lists whose first candidate reaches the threshold, and of these the candidates that do
    const float top = top_and_reach.x, most = top_and_reach.y;
    for (uint32_t l = threadIdx.x; l < lists; l += kJoinThreads) {
        float coarse;
        if (l == threadIdx.x && heads == 1)
            made(l, 0, first_logit, first_token, coarse);
        else
            candidate(l * parts.n, coarse);
        if (!(below(top, coarse) <= most)) continue;
        const uint32_t k = atomicAdd(&open, 1u);
        if (k < kMost) open_list[k] = l;
    }
    __syncthreads();
    const bool every = open > kMost;
    for (uint32_t i = threadIdx.x; i < (every ? lists : open) * parts.n; i += kJoinThreads) {
        const uint32_t l = parts.by_n.divide(i);
        float coarse;
        const Candidate c = candidate(every ? i : open_list[l] * parts.n + (i - l * parts.n), coarse);
        if (!(below(top, coarse) <= most)) continue;
        const uint32_t k = atomicAdd(&listed, 1u);
        if (k < kMost) {
            list[k] = c;
            ranks[k] = 0;
        }
    }
    __syncthreads();
    const uint32_t count = listed;
    auto write = [&](uint32_t r, const Candidate &c) {
        const uint64_t at = (uint64_t)search * parts.n + r;
        const uint32_t beam = c.first ? (uint32_t)(c.second >> 32) : 0;
        a.out_scores[at] = c.score;
        a.out_parents[at] = beam;
        a.out_tokens[at] = c.first && beams[beam].kind == kLive ? c.token : a.pad;
    };
    if (count <= kMost) {
        // as many threads to a candidate as there are
        uint32_t shares = 1;
        while (2 * shares * count <= kJoinThreads && shares < 16) shares *= 2;
        const uint32_t i = threadIdx.x / shares;
        if (i < count) {
            const Candidate own = list[i];
            uint32_t rank = 0;
#pragma unroll 4
            for (uint32_t k = threadIdx.x % shares; k < count; k += shares) rank += list[k].before(own);
            atomicAdd(&ranks[i], rank);
        }
        __syncthreads();
        if (threadIdx.x < count && ranks[threadIdx.x] < parts.n) write(ranks[threadIdx.x], list[threadIdx.x]);
        if (threadIdx.x >= count && threadIdx.x < parts.n) write(threadIdx.x, none);
        return;
    }
    // too many of one rank, or as far from the best to 2^-7: a round for each
    Candidate last = {~(uint64_t)0, 0, 0, 0.f};
#pragma unroll 1
    for (uint32_t r = 0; r < parts.n; r++) {
        Candidate best = none;
#pragma unroll 1
        for (uint32_t i = threadIdx.x; i < lists * parts.n; i += kJoinThreads) {
            float coarse;
            const Candidate c = candidate(i, coarse);
            if (c.first && last.before(c) && c.before(best)) best = c;
        }
#pragma unroll 1
        for (int k = 32; k >= 1; k /= 2) {
            const Candidate c = from_lane_xor(best, k);
            if (c.before(best)) best = c;
        }
        if (lane == 0) wave_best[r & 1][wave] = best;
        __syncthreads();
#pragma unroll 1
        for (int w = 0; w < kJoinWaves; w++)
            if (wave_best[r & 1][w].before(best)) best = wave_best[r & 1][w];
        if (threadIdx.x == 0) write(r, best);
        last = best.first ? best : Candidate{0, 0, 0, 0.f};
    }
}

void cut(const spiky_lm_beams_args &a, Parts &parts) {
    const uint64_t size = a.dtype == SPIKY_F32 ? slice_size<float>() : slice_size<bf16>();
    parts.slices = (uint32_t)max((a.vocab + size - 1) / size, (uint64_t)1);  // a finished beam needs a list too
    parts.n = (uint32_t)a.n;
    parts.by_n = Divider(parts.n);
    parts.by_slices = Divider(parts.slices);
    parts.by_beams = Divider((uint32_t)a.beams);
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

template <typename V, int kBeams, bool kStream = false>
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
            if (in_place && parents[j0 + j] == j0 + j) continue;
            char *to = out + (int64_t)(j0 + j) * out_beam;
            if constexpr (kStream) {
                typedef V Anywhere __attribute__((aligned(1)));
                __builtin_nontemporal_store(v[j], reinterpret_cast<Anywhere *>(to));
            } else {
                __builtin_memcpy(to, &v[j], sizeof(V));
            }
        }
    }
}

typedef uint32_t Words4 __attribute__((ext_vector_type(4)));

template <int kBeams, bool kStream>
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
        uint64_t at = (i - run * state.pieces.d) * 16;
        // the end of a run: its last 16 bytes, which have some in common with the piece before.  In place
        // that one may be written already, and the end keeps to its own, in halves of halves.
        if (!in_place && s.run_bytes >= 16) at = min(at, s.run_bytes - 16);
        const char *in = static_cast<const char *>(s.in) + (int64_t)search * s.in_search + (int64_t)run * s.in_run + at;
        char *out = static_cast<char *>(s.out) + (int64_t)search * s.out_search + (int64_t)run * s.out_run + at;
        const uint64_t left = s.run_bytes - at;
        if (left >= 16) {
            move<Words4, kBeams, kStream>(in, out, s.in_beam, s.out_beam, parents, beams, n, in_place);
            continue;
        }
        uint32_t o = 0;
        if (left & 8) move<uint64_t, kBeams>(in, out, s.in_beam, s.out_beam, parents, beams, n, in_place), o += 8;
        if (left & 4) move<uint32_t, kBeams>(in + o, out + o, s.in_beam, s.out_beam, parents, beams, n, in_place), o += 4;
        if (left & 2) move<uint16_t, kBeams>(in + o, out + o, s.in_beam, s.out_beam, parents, beams, n, in_place), o += 2;
        if (left & 1) move<uint8_t, kBeams>(in + o, out + o, s.in_beam, s.out_beam, parents, beams, n, in_place);
    }
}

}  // namespace

uint64_t beam_select_workspace(const spiky_lm_beams_args &a) {
    Parts parts;
    cut(a, parts);
    return a.searches * a.beams * parts.slices * (sizeof(float2) + a.n * 8);
}

hipError_t launch_beam_select(const spiky_lm_beams_args &a, void *workspace, hipStream_t st) {
    Parts parts;
    cut(a, parts);
    const uint64_t rows = a.searches * a.beams;
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
    const dim3 searches((uint32_t)min(a.searches, (uint64_t)kSearchesX), (uint32_t)((a.searches + kSearchesX - 1) / kSearchesX));
    k_beam_join<<<searches, dim3(kJoinThreads), 0, st>>>(a, parts);
    return hipGetLastError();
}

hipError_t launch_reorder(const spiky_lm_state *states, uint64_t count, const void *parents, bool parents_i64,
                          uint64_t searches, uint64_t beams, uint64_t n, hipStream_t st) {
    // Results past twice the last cache do not stay there for their reader.  Stored past it, bf16 states of 4, 8,
    // 16, 32 and 64 beams, 1.6 GB of results, take 433, 445, 486, 462 and 454 us against 468, 467, 495, 478 and
    // 491, and in place, where beams that stay are not moved, 344, 421, 473, 427 and 480 against 367, 446, 485,
    // 446 and 519.  The call by itself gains as much at 0.5 GB (147 for 167); at 175 MB, which a reader finds in
    // the cache, it takes 42 to 47 for 47 to 54, and in place 35 to 52 either way.
    uint64_t bytes = 0;
    for (uint64_t i = 0; i < count; i++) bytes += states[i].runs * states[i].run_bytes * n * searches;
    const bool stream = bytes >= 2 * kLastCache;
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
            const hipError_t e = n <= 4 ? stream ? go(k_reorder<4, true>) : go(k_reorder<4, false>)
                                 : n <= 8 ? stream ? go(k_reorder<8, true>) : go(k_reorder<8, false>)
                                 : n <= 16 ? stream ? go(k_reorder<16, true>) : go(k_reorder<16, false>)
                                 : n <= 32 ? stream ? go(k_reorder<32, true>) : go(k_reorder<32, false>)
                                 : stream ? go(k_reorder<64, true>) : go(k_reorder<64, false>);
            if (e != hipSuccess) return e;
        }
    }
    return hipSuccess;
}

}  // namespace lm
}  // namespace spiky
