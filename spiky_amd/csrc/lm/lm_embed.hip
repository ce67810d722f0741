// lm_embed.hip -- token embeddings and their gradient (gfx950).
#include "lm_tokens.h"

namespace spiky {
namespace lm {
namespace {

constexpr int kThreads = 256;

template <typename A, typename B>
constexpr int piece() {  // columns of a piece: 16 bytes of the narrower type
    return 16 / (sizeof(A) < sizeof(B) ? sizeof(A) : sizeof(B));
}

// ---- lookup ------------------------------------------------------------------
// Reads the distinct rows and writes every one: bound by HBM where it is large.  The pieces of
// all rows are numbered through as in dropout; a thread takes kPieces of them.
template <typename Tok, typename W, typename T, int kPieces>
__global__ __launch_bounds__(kThreads) void k_embed(const Tok *__restrict__ tokens, const W *__restrict__ weight,
                                                    int64_t stride, T *__restrict__ out, uint64_t n, uint64_t vocab,
                                                    uint64_t cols, Divider row_pieces, float scale) {
    constexpr int N = piece<W, T>();
    const uint64_t first = (uint64_t)blockIdx.x * (kThreads * kPieces);
    const uint64_t row0 = first < 0x100000000ull ? row_pieces.divide((uint32_t)first) : first / row_pieces.d;
    const uint32_t piece0 = (uint32_t)(first - row0 * row_pieces.d);
    // first all tokens, then all pieces, then the results: no load waits for another piece's
    uint64_t row[kPieces], token[kPieces];
    Place<N> place[kPieces];
    Raw<W, N> raw[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; i++) {
        const uint64_t at = (uint64_t)piece0 + i * kThreads + threadIdx.x;
        // a long row ends at most once in the workgroup's pieces, a short one's numbers fit 32 bits
        const uint32_t down = row_pieces.d >= kThreads * kPieces ? at >= row_pieces.d
                                                                 : row_pieces.divide((uint32_t)at);
        row[i] = row0 + down;
        place[i].set(cols, (at - (uint64_t)down * row_pieces.d) * N);
        token[i] = (uint64_t)(int64_t)tokens[min(row[i], n - 1)];
    }
#pragma unroll
    for (int i = 0; i < kPieces; i++) {
        const W *from = weight + (int64_t)(token[i] < vocab ? token[i] : 0) * stride + place[i].col;
        if (cols >= N && vocab > 0)
            __builtin_memcpy(raw[i].w, from, sizeof(raw[i].w));
        else
            raw[i].clear(), raw[i].load(from, vocab > 0 ? place[i].n : 0);
    }
#pragma unroll
    for (int i = 0; i < kPieces; i++) {
        if (row[i] >= n) break;
        float v[N];
#pragma unroll
        for (int k = 0; k < N; k++) {
            v[k] = token[i] < vocab ? raw[i][k] * scale : 0.f;
            // the product rounds to 32 bits and then to T, for every T alike
            if (sizeof(T) == 2) asm("" : "+v"(v[k]));
        }
        store(out + row[i] * cols + place[i].col, v, place[i].n);
    }
}

template <typename Tok, typename W, typename T>
hipError_t lookup(const spiky_lm_embed_args &a, void *out, hipStream_t st) {
    constexpr uint64_t N = piece<W, T>();
    const uint64_t row_pieces = (a.cols + N - 1) / N, pieces = a.n * row_pieces;
    const Divider by((uint32_t)row_pieces);
    auto go = [&](auto kernel, uint64_t each) {
        const uint64_t groups = (pieces + kThreads * each - 1) / (kThreads * each);
        if (groups * kThreads > 0xffffffffull) return hipErrorInvalidValue;
        kernel<<<dim3((uint32_t)groups), dim3(kThreads), 0, st>>>(
            static_cast<const Tok *>(a.tokens), static_cast<const W *>(a.weight), a.weight_stride,
            static_cast<T *>(out), a.n, a.vocab, a.cols, by, (float)a.scale);
        return hipGetLastError();
    };
    // a piece a thread where more would leave CUs idle
    return pieces < 8 * kCUs * kThreads ? go(k_embed<Tok, W, T, 1>, 1) : go(k_embed<Tok, W, T, 4>, 4);
}

// ---- gradient ------------------------------------------------------------------
// The tokens' positions, sorted by token and for each token in ascending order, and where each
// token's begin: start [vocab + 1], order [start[vocab]]; and for every chunk of `chunk` sorted positions
// the run of one token that its first position is in.  One launch without any exchange between
// workgroups: a workgroup owns `range` consecutive tokens of the vocabulary, reads all n, lists its
// own for each wave's share of the positions, counts these and the ones below its range, adds up,
// and places its own.  A wave with more of its own than its list holds reads its share again.
// Tokens outside the vocabulary are in no range.
struct Run {
    uint32_t from, to, token, unused;
};

constexpr int kSortWaves = 16, kMostRange = 1024;
constexpr uint32_t kList = 512;                        // of a wave
constexpr uint32_t kListShare = 0xffffffffu / kMostRange;  // positions of a share that a list's words can tell apart

// A token as 32 bits: those outside any vocabulary stay outside.
__device__ __forceinline__ uint32_t narrow(int64_t token) {
    return (uint64_t)token >> 32 ? ~0u : (uint32_t)token;
}
__device__ __forceinline__ uint32_t narrow(int32_t token) { return (uint32_t)token; }

// A workgroup's part: its tokens' positions to `order`, which takes the ones of this range from
// *from_below on.  In the end counts [kSortWaves - 1][o] is where those of token base + o end.
template <typename Tok, typename Start>
__device__ __forceinline__ void sort_range(const Tok *tokens, uint32_t n, uint32_t base, uint32_t size, uint32_t range,
                                           uint32_t *counts, uint32_t (*lists)[kList], uint32_t *order, bool from_below,
                                           Start start) {
    __shared__ uint32_t below_of[kSortWaves], sum_of[kSortWaves];
    const uint32_t wave = threadIdx.x / 64, lane = threadIdx.x & 63;
    const uint64_t lower = ((uint64_t)1 << lane) - 1;
    for (uint32_t i = threadIdx.x; i < kSortWaves * range; i += kSortWaves * 64) counts[i] = 0;
    __syncthreads();
    const uint32_t share = (n / (kSortWaves * 64) + 1) * 64;
    const uint32_t begin = min(wave * share, n), end = min(begin + share, n);
    uint32_t *mine = counts + wave * range, *list = lists[wave], below = 0, listed = 0;
    // More at once make the code longer than they save: a launch waits for its instructions too.  2, 4, 8
    // and 16 take 8.0, 8.4, 9.5 and 10.5 us for 8192 tokens of 256.
    constexpr int kAhead = 2;
    // fn(position of the wave's lane 0, the lane's token)
    auto each = [&](auto fn) {
        if (begin >= end) return;
        Tok id[kAhead], next[kAhead];  // no lane's load hangs on a condition: all are in flight at once
#pragma unroll
        for (int k = 0; k < kAhead; k++) next[k] = tokens[min(begin + k * 64 + lane, end - 1)];
        for (uint32_t at = begin; at < end; at += 64 * kAhead) {
#pragma unroll
            for (int k = 0; k < kAhead; k++) id[k] = next[k];
#pragma unroll
            for (int k = 0; k < kAhead; k++) next[k] = tokens[min(at + (kAhead + k) * 64 + lane, end - 1)];
#pragma unroll
            for (int k = 0; k < kAhead; k++) fn(at + k * 64, at + k * 64 + lane < end ? narrow(id[k]) : ~0u);
        }
    };
    each([&](uint32_t first, uint32_t id) {
        const uint32_t o = id - base;
        below += id < base;  // base <= vocab, so tokens outside are not
        const uint64_t own = __ballot(o < size);
        if (own == 0) return;
        // many lanes with one token, as where a batch is padded with it, count as one: 32768 times one
        // token take 25 us against 43
        uint32_t counted = ~0u;
        if (__popcll(own) >= 16) {
            counted = __builtin_amdgcn_readlane(o, __builtin_ctzll(own));
            const uint64_t same = __ballot(o == counted);
            if (lane == 0) atomicAdd(&mine[counted], (uint32_t)__popcll(same));
        }
        if (o < size) {
            if (o != counted) atomicAdd(&mine[o], 1u);
            const uint32_t at = listed + __popcll(own & lower);
            if (at < kList) list[at] = (first - begin + lane) * kMostRange + o;
        }
        listed += __popcll(own);
    });
    for (int k = 32; k >= 1; k /= 2) below += __shfl_xor(below, k);
    if (lane == 0) below_of[wave] = below;
    __syncthreads();
    uint32_t total = 0;
    if (threadIdx.x < size)
        for (int w = 0; w < kSortWaves; w++) total += counts[w * range + threadIdx.x];
    uint32_t upto = total;
    for (int k = 1; k < 64; k *= 2) {
        const uint32_t x = __shfl_up(upto, k);
        if (lane >= (uint32_t)k) upto += x;
    }
    if (lane == 63) sum_of[wave] = upto;
    __syncthreads();
    uint32_t at = upto - total;
    for (uint32_t w = 0; w < kSortWaves; w++) at += (from_below ? below_of[w] : 0) + (w < wave ? sum_of[w] : 0);
    if (threadIdx.x < size) {
        start(threadIdx.x, at, total);
        for (int w = 0; w < kSortWaves; w++) {
            const uint32_t c = counts[w * range + threadIdx.x];
            counts[w * range + threadIdx.x] = at;
            at += c;
        }
    }
    __syncthreads();
    // Places the lanes' positions whose tokens are o in the range, or none where that is ~0.
    auto place = [&](uint32_t position, uint32_t o) {
        for (uint64_t left = __ballot(o != ~0u); left;) {
            const uint32_t leader = __builtin_ctzll(left);
            const uint32_t token = __builtin_amdgcn_readlane(o, leader);
            const uint64_t same = __ballot(o == token);
            uint32_t to = 0;
            if (lane == leader) to = atomicAdd(&mine[token], (uint32_t)__popcll(same));
            to = __builtin_amdgcn_readlane(to, leader);
            if (o == token) order[to + __popcll(same & lower)] = position;
            left &= ~same;
        }
    };
    if (listed <= kList && share <= kListShare) {
        for (uint32_t i = 0; i < listed; i += 64) {
            const uint32_t word = i + lane < listed ? list[i + lane] : ~0u;
            place(begin + word / kMostRange, word == ~0u ? ~0u : word % kMostRange);
        }
    } else {
        each([&](uint32_t first, uint32_t id) { place(first + lane, id - base < size ? id - base : ~0u); });
    }
}

template <typename Tok>
__global__ __launch_bounds__(kSortWaves * 64) void k_embed_sort(const Tok *__restrict__ tokens, uint32_t n,
                                                                uint32_t vocab, uint32_t range, uint32_t chunk,
                                                                uint32_t *__restrict__ start,
                                                                uint32_t *__restrict__ order, Run *__restrict__ runs) {
    extern __shared__ uint32_t counts[];  // [kSortWaves][range]
    __shared__ uint32_t lists[kSortWaves][kList];
    const uint32_t base = blockIdx.x * range, size = min(range, vocab - base);
    sort_range(tokens, n, base, size, range, counts, lists, order, true, [&](uint32_t o, uint32_t at, uint32_t total) {
        start[base + o] = at;
        if (base + o == vocab - 1) start[vocab] = at + total;
        for (uint32_t c = (at + chunk - 1) / chunk; c * chunk < at + total; c++) runs[c] = {at, at + total, base + o, 0};
    });
}

// Positions of a token that are added up one after the other: tokens with more ("frequent") go in
// chunks of this many sorted positions, whose sums a launch of its own adds up.  A text's most
// frequent token stands at every tenth position or so: as one row's sum it took 1.9 ms of 32768
// tokens' gradient, ten times the rest.  Fewer positions, down to kLeastChunk, where chunks would not fill the chip.
constexpr uint32_t kMostChunk = 32, kLeastChunk = 8;
constexpr uint64_t kManyGroups = 64 * kCUs;

// The sum over positions [from, to) of the n columns at d_out; `from < to`, n > 0.  No load of a whole
// piece hangs on a condition, so as many rows as registers hold are in flight.
template <int N, typename T>
__device__ __forceinline__ void sum_rows(float (&sum)[N], const T *d_out, int64_t stride, const uint32_t *order,
                                         uint32_t from, uint32_t to, int n) {
    constexpr uint32_t kAhead = 32 / (N * sizeof(T) / 4);
#pragma unroll
    for (int k = 0; k < N; k++) sum[k] = 0.f;
    if (n < N) {  // rows narrower than a piece
        for (uint32_t i = from; i < to; i++) {
            float v[N];
            load(v, d_out + (int64_t)order[i] * stride, n);
#pragma unroll
            for (int k = 0; k < N; k++) sum[k] += v[k];
        }
        return;
    }
    uint32_t at[kAhead], i = from;
#pragma unroll
    for (uint32_t j = 0; j < kAhead; j++) at[j] = order[min(from + j, to - 1)];
    Raw<T, N> raw[kAhead];
    for (; i + kAhead <= to; i += kAhead) {
#pragma unroll
        for (uint32_t j = 0; j < kAhead; j++)
            __builtin_memcpy(raw[j].w, d_out + (int64_t)at[j] * stride, sizeof(raw[j].w));
#pragma unroll
        for (uint32_t j = 0; j < kAhead; j++) at[j] = order[min(i + kAhead + j, to - 1)];
#pragma unroll
        for (uint32_t j = 0; j < kAhead; j++)
#pragma unroll
            for (int k = 0; k < N; k++) sum[k] += raw[j][k];
    }
    // the last few, which for most tokens are one or two and all
#pragma unroll
    for (uint32_t j = 0; j < kAhead; j++)
        if (i + j < to) __builtin_memcpy(raw[j].w, d_out + (int64_t)at[j] * stride, sizeof(raw[j].w));
#pragma unroll
    for (uint32_t j = 0; j < kAhead; j++) {
        if (i + j >= to) break;
#pragma unroll
        for (int k = 0; k < N; k++) sum[k] += raw[j][k];
    }
}

// The first `chunk_groups` workgroups of x take chunks of the sorted positions, `lanes` threads, a
// power of two, each: frequent runs are longer than a chunk, so the only ones that a chunk holds a
// part of are the one of its first position and the one of the next chunk's.  Their sums go to partial
// [2 * chunk] and [2 * chunk + 1].  The others take kRows rows a thread of the table's gradient, of
// tokens that are not frequent.
template <typename T, typename W, uint32_t kRows, bool kStream>
__global__ __launch_bounds__(kThreads) void k_embed_sum(const T *__restrict__ d_out, int64_t stride,
                                                        const uint32_t *__restrict__ start,
                                                        const uint32_t *__restrict__ order,
                                                        const Run *__restrict__ runs, W *__restrict__ d_weight,
                                                        float *__restrict__ partial, uint64_t pitch, uint32_t vocab,
                                                        uint64_t cols, uint32_t size, uint32_t chunks,
                                                        uint32_t chunk_groups, uint32_t lanes, float scale) {
    constexpr int N = piece<W, T>();
    Place<N> place;
    place.set(cols, ((uint64_t)blockIdx.y * lanes + (threadIdx.x & (lanes - 1))) * N);
    const uint32_t rows = kThreads / lanes, own = threadIdx.x / lanes;
    float sum[N];
    if (blockIdx.x < chunk_groups) {
        const uint32_t chunk = blockIdx.x * rows + own, begin = chunk * size;
        if (chunk >= chunks || place.n == 0) return;
        const uint32_t n = start[vocab];
        const Run first = runs[chunk], next = runs[min(chunk + 1, chunks - 1)];  // not written past n
        if (begin >= n) return;
        const uint32_t end = min(begin + size, n);
        if (first.to - first.from > size) {
            sum_rows(sum, d_out + place.col, stride, order, begin, min(end, first.to), place.n);
            store(partial + (uint64_t)chunk * 2 * pitch + place.col, sum, place.n);
        }
        if (begin + size < n && next.from > begin && next.from < end && next.to - next.from > size) {
            sum_rows(sum, d_out + place.col, stride, order, next.from, end, place.n);
            store(partial + ((uint64_t)chunk * 2 + 1) * pitch + place.col, sum, place.n);
        }
        return;
    }
    const uint64_t row0 = (uint64_t)(blockIdx.x - chunk_groups) * (rows * kRows) + own;
    uint32_t from[kRows], to[kRows];
#pragma unroll
    for (uint32_t r = 0; r < kRows; r++) {
        const uint64_t row = row0 + r * rows;
        from[r] = row < vocab ? start[row] : 0;
        to[r] = row < vocab ? start[row + 1] : ~0u;
    }
    if (place.n == 0) return;
#pragma unroll
    for (uint32_t r = 0; r < kRows; r++) {
        if (to[r] - from[r] > size) continue;
        if (from[r] < to[r]) {
            sum_rows(sum, d_out + place.col, stride, order, from[r], to[r], place.n);
        } else {
#pragma unroll
            for (int k = 0; k < N; k++) sum[k] = 0.f;
        }
#pragma unroll
        for (int k = 0; k < N; k++) sum[k] *= scale;
        W *to_row = d_weight + (row0 + r * rows) * cols + place.col;
        if constexpr (kStream)
            stream_out(to_row, sum, place.n);
        else
            store(to_row, sum, place.n);
    }
}

// The rows of frequent tokens, from their chunks' sums: workgroup x adds up the runs whose first whole
// chunk is one of `joined` from x * joined on, 64 lanes a group of columns, wave w the sums number w,
// w + 4, ... of a run.
template <typename W>
__global__ __launch_bounds__(kThreads) void k_embed_join(const uint32_t *__restrict__ start,
                                                         const Run *__restrict__ runs, W *__restrict__ d_weight,
                                                         const float *__restrict__ partial, uint64_t pitch, uint32_t vocab,
                                                         uint64_t cols, uint32_t size, uint32_t chunks,
                                                         uint32_t joined, float scale) {
    constexpr int N = 4, kAhead = 8;
    constexpr uint32_t kWaves = kThreads / 64;
    __shared__ float sums[kWaves - 1][N][64];
    const uint32_t n = start[vocab], wave = threadIdx.x / 64, lane = threadIdx.x & 63;
    // a lane a chunk, the same in all waves
    const uint32_t mine = min(blockIdx.x * joined + lane, chunks - 1);
    const Run run = runs[mine];
    const bool begins = lane < joined && blockIdx.x * joined + lane < chunks && mine * size < n &&
                        run.to - run.from > size && run.from + size > mine * size;
    Place<N> place;
    place.set(cols, ((uint64_t)blockIdx.y * 64 + lane) * N);
    for (uint64_t found = __ballot(begins); found; found &= found - 1) {
        const uint32_t l = __builtin_ctzll(found);
        const uint32_t from = __builtin_amdgcn_readlane(run.from, l), to = __builtin_amdgcn_readlane(run.to, l);
        const uint32_t token = __builtin_amdgcn_readlane(run.token, l);
        const uint32_t chunk = from / size, parts = (to - 1) / size - chunk + 1;
        // a run that begins inside a chunk is that one's second
        const uint32_t skew = from > chunk * size ? 1 : 0;
        const float *p = partial + (uint64_t)chunk * 2 * pitch + place.col;
        float sum[N] = {};
        for (uint32_t i = wave; i < parts; i += kWaves * kAhead) {
            Raw<float, N> raw[kAhead];
#pragma unroll
            for (uint32_t j = 0; j < kAhead; j++) {
                const uint32_t k = min(i + j * kWaves, parts - 1);
                __builtin_memcpy(raw[j].w, p + ((uint64_t)k * 2 + (k == 0 ? skew : 0)) * pitch, sizeof(raw[j].w));
            }
#pragma unroll
            for (uint32_t j = 0; j < kAhead; j++)
#pragma unroll
                for (int k = 0; k < N; k++) sum[k] += i + j * kWaves < parts ? raw[j][k] : 0.f;
        }
        __syncthreads();  // the sums of the run before are read
        if (wave > 0)
            for (int k = 0; k < N; k++) sums[wave - 1][k][lane] = sum[k];
        __syncthreads();
        if (wave > 0 || place.n == 0) continue;
        for (uint32_t w = 0; w < kWaves - 1; w++)
            for (int k = 0; k < N; k++) sum[k] += sums[w][k][lane];
        for (int k = 0; k < N; k++) sum[k] *= scale;
        store(d_weight + (uint64_t)token * cols + place.col, sum, place.n);
    }
}

// Both in one launch, for few positions: a workgroup takes `range` tokens and a slab of `lanes` pieces of
// their rows, sorts for itself, and adds up.  Its groups of `lanes` threads take a token each, and all
// of them one that has more than kTogether positions, a share each.  64 positions of 256 columns in a
// table of 256 rows take 5 us, in three launches 14.
constexpr uint32_t kSmall = 8192, kTogether = 16;
constexpr uint64_t kSmallBytes = 2 << 20;

template <typename Tok, typename T, typename W>
__global__ __launch_bounds__(kSortWaves * 64) void k_embed_small(const Tok *__restrict__ tokens,
                                                                 const T *__restrict__ d_out, int64_t stride,
                                                                 W *__restrict__ d_weight, uint32_t n, uint32_t vocab,
                                                                 uint64_t cols, uint32_t range, uint32_t lanes,
                                                                 float scale) {
    constexpr int N = piece<W, T>();
    constexpr uint32_t kAll = kSortWaves * 64;
    extern __shared__ uint32_t counts[];  // [kSortWaves][range], then the order [n]
    __shared__ union {
        uint32_t lists[kSortWaves][kList];
        float partial[N][kAll];
    } shared;
    __shared__ uint32_t together[kSmall / kTogether], n_together;
    static_assert(sizeof(shared) <= 32768, "two workgroups to a CU");
    uint32_t *order = counts + kSortWaves * range;
    const uint32_t base = blockIdx.x * range, size = min(range, vocab - base);
    if (threadIdx.x == 0) n_together = 0;
    // the first barrier lies between this and the calls
    sort_range(tokens, n, base, size, range, counts, shared.lists, order, false, [&](uint32_t o, uint32_t, uint32_t total) {
        if (total > kTogether) together[atomicAdd(&n_together, 1u)] = o;
    });
    __syncthreads();
    const uint32_t *ends = counts + (kSortWaves - 1) * range;
    const uint32_t group = threadIdx.x / lanes, groups = kAll / lanes;
    Place<N> place;
    place.set(cols, ((uint64_t)blockIdx.y * lanes + (threadIdx.x & (lanes - 1))) * N);
    d_out += place.col;
    d_weight += (uint64_t)base * cols + place.col;
    float sum[N];
    for (uint32_t h = 0; h < n_together; h++) {
        const uint32_t o = together[h], from = o ? ends[o - 1] : 0, to = ends[o];
        const uint32_t share = (to - from + groups - 1) / groups, begin = from + group * share;
        if (begin < to && place.n > 0) {
            sum_rows(sum, d_out, stride, order, begin, min(begin + share, to), place.n);
        } else {
#pragma unroll
            for (int k = 0; k < N; k++) sum[k] = 0.f;
        }
#pragma unroll
        for (int k = 0; k < N; k++) shared.partial[k][threadIdx.x] = sum[k];
        __syncthreads();
        for (uint32_t half = kAll / 2; half >= lanes; half /= 2) {
            if (threadIdx.x < half)
#pragma unroll
                for (int k = 0; k < N; k++) shared.partial[k][threadIdx.x] += shared.partial[k][threadIdx.x + half];
            __syncthreads();
        }
        if (group == 0 && place.n > 0) {
#pragma unroll
            for (int k = 0; k < N; k++) sum[k] = shared.partial[k][threadIdx.x] * scale;
            store(d_weight + o * cols, sum, place.n);
        }
        __syncthreads();
    }
    if (place.n == 0) return;
    for (uint32_t o = group; o < size; o += groups) {
        const uint32_t from = o ? ends[o - 1] : 0, to = ends[o];
        if (to - from > kTogether) continue;
        if (from < to) {
            sum_rows(sum, d_out, stride, order, from, to, place.n);
        } else {
#pragma unroll
            for (int k = 0; k < N; k++) sum[k] = 0.f;
        }
#pragma unroll
        for (int k = 0; k < N; k++) sum[k] *= scale;
        store(d_weight + o * cols, sum, place.n);
    }
}

// Few enough: here one workgroup adds up a frequent token's rows, and every slab's workgroups read all
// positions.  Where no cache holds the gradient, one launch and three take 27 and 31 us for 512
// positions of 1024 bf16 columns (1 MB) in a table of 50000 rows, 26 and 32 for 8192 of 64 fp32 (2 MB)
// in one of 152000, 35 and 33 for 2048 of 1024 bf16 (4 MB), 29 and 22 for 8192 of 256 fp32 (8 MB) in
// one of 256.
template <typename W, typename T>
bool is_small(const spiky_lm_embed_args &a, uint32_t &lanes, uint64_t &slabs) {
    constexpr uint64_t N = piece<W, T>();
    const uint64_t pieces = (a.cols + N - 1) / N;
    lanes = 1;
    while (lanes < pieces && lanes < 64) lanes *= 2;
    slabs = (pieces + lanes - 1) / lanes;
    return slabs <= 2 && a.n * slabs <= kSmall && a.n * a.cols * sizeof(T) <= kSmallBytes;
}

// Positions of a chunk, a power of two, and chunks: half a workgroup of pieces of four columns to a CU,
// or chunks of the fewest positions.  8192 positions of 256 columns, one in nine the same token, take
// 22.3 us with 16 positions to a chunk, 24.6 with 8 and 23.4 with 32, which is as good from 1001 columns on.
uint64_t chunk_of(const spiky_lm_embed_args &a) {
    uint64_t chunk = kMostChunk;
    while (chunk > kLeastChunk && a.n / chunk * ((a.cols + 3) / 4) < kCUs / 2 * kThreads) chunk /= 2;
    return chunk;
}
uint64_t chunks_of(const spiky_lm_embed_args &a) { return (a.n + chunk_of(a) - 1) / chunk_of(a); }

// The workspace: runs, starts, order, and the chunks' sums.
uint64_t start_at(const spiky_lm_embed_args &a) { return chunks_of(a) * sizeof(Run); }
uint64_t order_at(const spiky_lm_embed_args &a) { return start_at(a) + (a.vocab + 1) * 4; }
uint64_t partial_at(const spiky_lm_embed_args &a) { return order_at(a) + a.n * 4; }
uint64_t pitch_of(const spiky_lm_embed_args &a) { return max(a.cols, (uint64_t)4); }  // of a chunk's sums: a piece at least

uint32_t range_of(const spiky_lm_embed_args &a) {
    return (uint32_t)min(max((a.vocab + kCUs - 1) / kCUs, (uint64_t)1), (uint64_t)kMostRange);
}

template <typename W, typename T>
hipError_t sums(const spiky_lm_embed_args &a, const void *d_out_, int64_t stride, void *d_weight_, const Run *runs,
                const uint32_t *start, const uint32_t *order, float *partial, hipStream_t st) {
    constexpr uint64_t N = piece<W, T>();
    const T *d_out = static_cast<const T *>(d_out_);
    W *d_weight = static_cast<W *>(d_weight_);
    const uint64_t pieces = (a.cols + N - 1) / N;
    uint32_t lanes = 1;
    while (lanes < pieces && lanes < kThreads) lanes *= 2;
    const uint32_t rows = kThreads / lanes, chunk = (uint32_t)chunk_of(a), chunks = (uint32_t)chunks_of(a);
    const uint32_t groups = a.n > chunk ? (chunks + rows - 1) / rows : 0;  // no token is frequent among fewer
    const uint64_t slabs = (pieces + lanes - 1) / lanes;
    auto go = [&](auto kernel, uint64_t each) {
        const uint64_t all = groups + (a.vocab + rows * each - 1) / (rows * each);
        if (all * kThreads > 0xffffffffull) return hipErrorInvalidValue;
        kernel<<<dim3((uint32_t)all, (uint32_t)slabs), dim3(kThreads), 0, st>>>(
            d_out, stride, start, order, runs, d_weight, partial, pitch_of(a), (uint32_t)a.vocab, a.cols, chunk, chunks,
            groups, lanes, (float)a.scale);
        return hipGetLastError();
    };
    // Several rows to a thread where there are enough: most have no token, and only their zeros to write.
    // 1, 4, 8 and 16 rows take 424, 325, 332 and 373 us of 32768 tokens' 4096 bf16 columns and 152000
    // rows.  A table that the last cache would not hold for its reader is stored past it, where a thread's
    // piece is one store: 16384 tokens' 600 MB of 4096 columns in fp32 take 161 and, stored as usual, 195 us,
    // in bf16 123 and 167; 2.4 GB 466 and 528, 442 and 475.  fp32 rows of 16-bit results are two
    // stores a piece, and go as usual: 185 us for 283, 488 for 1090.  Of smaller tables it hangs on the tokens:
    // 256 MB in fp32 take 111 and 126 us with 16384 of them, 55 and 41 with 256.
    const bool many = a.vocab / rows * slabs >= kManyGroups;
    const hipError_t e = [&] {
        if (!many) return go(k_embed_sum<T, W, 1, false>, 1);
        if constexpr (N * sizeof(W) == 16)
            if (a.vocab * a.cols * sizeof(W) >= kLastCache * 2) return go(k_embed_sum<T, W, 4, true>, 4);
        return go(k_embed_sum<T, W, 4, false>, 4);
    }();
    if (e != hipSuccess || groups == 0) return e;
    // most chunks begin no run: where there are many, a workgroup looks at several
    const uint32_t col_groups = (uint32_t)((a.cols + 255) / 256), joined = (uint64_t)chunks * col_groups > 4 * kCUs ? 8 : 1;
    k_embed_join<W><<<dim3((chunks + joined - 1) / joined, col_groups), dim3(kThreads), 0, st>>>(
        start, runs, d_weight, partial, pitch_of(a), (uint32_t)a.vocab, a.cols, chunk, chunks, joined, (float)a.scale);
    return hipGetLastError();
}

// go(a value of the table's type, a value of out's)
template <typename F>
hipError_t by_types(int weight, int out, F &&go) {
    if (weight == SPIKY_F32)
        return out == SPIKY_F32 ? go(0.f, 0.f) : out == SPIKY_BF16 ? go(0.f, bf16()) : go(0.f, f16());
    if (weight == SPIKY_BF16) return out == SPIKY_F32 ? go(bf16(), 0.f) : go(bf16(), bf16());
    return out == SPIKY_F32 ? go(f16(), 0.f) : go(f16(), f16());
}

}  // namespace

hipError_t launch_embed(const spiky_lm_embed_args &a, void *out, hipStream_t st) {
    return by_types(a.weight_dtype, a.out_dtype, [&](auto w, auto t) {
        return a.tokens_i64 ? lookup<int64_t, decltype(w), decltype(t)>(a, out, st)
                            : lookup<int32_t, decltype(w), decltype(t)>(a, out, st);
    });
}

uint64_t embed_workspace(const spiky_lm_embed_args &a) { return partial_at(a) + chunks_of(a) * 2 * pitch_of(a) * 4; }

template <typename Tok, typename W, typename T>
hipError_t gradient(const spiky_lm_embed_args &a, const void *d_out, int64_t stride, void *d_weight, void *workspace,
                    hipStream_t st) {
    uint32_t lanes;
    uint64_t slabs;
    if (is_small<W, T>(a, lanes, slabs)) {
        const uint32_t vocab = (uint32_t)a.vocab, range = range_of(a), lds = (kSortWaves * range + (uint32_t)a.n) * 4;
        k_embed_small<Tok, T, W><<<dim3((vocab + range - 1) / range, (uint32_t)slabs), dim3(kSortWaves * 64), lds, st>>>(
            static_cast<const Tok *>(a.tokens), static_cast<const T *>(d_out), stride, static_cast<W *>(d_weight),
            (uint32_t)a.n, vocab, a.cols, range, lanes, (float)a.scale);
        return hipGetLastError();
    }
    char *w = static_cast<char *>(workspace);
    Run *runs = reinterpret_cast<Run *>(w);
    uint32_t *start = reinterpret_cast<uint32_t *>(w + start_at(a)), *order = reinterpret_cast<uint32_t *>(w + order_at(a));
    const uint32_t vocab = (uint32_t)a.vocab, range = range_of(a);
    k_embed_sort<Tok><<<dim3((vocab + range - 1) / range), dim3(kSortWaves * 64), kSortWaves * range * 4, st>>>(
        static_cast<const Tok *>(a.tokens), (uint32_t)a.n, vocab, range, (uint32_t)chunk_of(a), start, order, runs);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    return sums<W, T>(a, d_out, stride, d_weight, runs, start, order, reinterpret_cast<float *>(w + partial_at(a)), st);
}

hipError_t launch_embed_backward(const spiky_lm_embed_args &a, const void *d_out, int64_t d_out_stride, void *d_weight,
                                 void *workspace, hipStream_t st) {
    return by_types(a.weight_dtype, a.out_dtype, [&](auto w, auto t) {
        return a.tokens_i64 ? gradient<int64_t, decltype(w), decltype(t)>(a, d_out, d_out_stride, d_weight, workspace, st)
                            : gradient<int32_t, decltype(w), decltype(t)>(a, d_out, d_out_stride, d_weight, workspace, st);
    });
}

}  // namespace lm
}  // namespace spiky
