// lm_logits.hip -- penalties, biases, temperature and masks on logits (gfx950).
#include <type_traits>

#include "lm_kernels.h"

namespace spiky {
namespace lm {
namespace {

// Tokens of a history from which 1024 threads count them: where workgroups are few (128 rows of
// 8991 entries with 31972 tokens take 25 us against 30), and, from twice as many on, where
// chunks of 16384 entries and more, which read it less often, fill the chip (256 rows of 152000:
// 6000 tokens 53 us against 49, 8192 55 both, 16384 60 against 88, 32768 80 against 156).  In
// between the chunks of 256 threads are faster (46 rows of 97950 with 22483: 27 against 36).
constexpr uint64_t kLong = 4096;
constexpr size_t kMostLds = 150000;  // of 160 KiB, beside a list of sparse biases

// The word of an entry in LDS: flags, and in the bits below the times that it is
// among the tokens after the prompt.  Histories short enough leave bits 18 to 29
// for the slot of its sum of sparse biases, if there are no more of these; for
// others the slots have an array.
constexpr uint32_t kSeen = 0x80000000u;    // among the prompt's tokens
constexpr uint32_t kBiased = 0x40000000u;  // among the bias ids
constexpr uint32_t kSlotShift = 18, kSlotMask = 0xfff;

__host__ __device__ __forceinline__ bool slots_in_words(uint64_t history, uint64_t n_bias) {
    return history < 1u << kSlotShift && n_bias <= kSlotMask + 1;
}

// A value that no one writes during the launch, read the same by all lanes: a
// scalar load, which does not queue with the lanes' loads.
template <typename T>
__device__ __forceinline__ T scalar(const T *p) {
    typedef __attribute__((address_space(4))) const T *Constant;
    return *(Constant)(uintptr_t)p;
}

__device__ __forceinline__ uint32_t length_at(const void *p, bool i64, uint32_t row, uint32_t most) {
    if (!p) return most;
    const int64_t n = i64 ? scalar(static_cast<const int64_t *>(p) + row) : scalar(static_cast<const int32_t *>(p) + row);
    return n < 0 ? 0 : n < (int64_t)most ? (uint32_t)n : most;
}

// An element `at` elements past a pointer that is the same for all lanes: one
// 32-bit offset a lane.
template <typename T>
__device__ __forceinline__ T *past(T *p, uint32_t at) {
    using C = std::conditional_t<std::is_const_v<T>, const char, char>;
    return reinterpret_cast<T *>(reinterpret_cast<C *>(p) + at * (uint32_t)sizeof(T));
}

// The tokens a thread holds at a time: numbers at + thread, at + thread + kThreads, ...
template <typename T, uint32_t kThreads>
struct Tokens {
    static constexpr uint32_t kAhead = 64 / sizeof(T);
    T id[kAhead];

    // Those past `end` are -1.
    __device__ __forceinline__ void load(const T *tokens, uint32_t at, uint32_t end) {
        if (at + kAhead * kThreads <= end) {
#pragma unroll
            for (uint32_t k = 0; k < kAhead; k++) id[k] = *past(tokens + at + k * kThreads, threadIdx.x);
            return;
        }
#pragma unroll
        for (uint32_t k = 0; k < kAhead; k++) {
            id[k] = (T)-1;
            if (at + k * kThreads + threadIdx.x < end) id[k] = *past(tokens + at + k * kThreads, threadIdx.x);
        }
    }
    // Adds those before len to the words of the chunk's entries.  A workgroup's
    // kThreads are nearly always all of the prompt or all after it, and whole.
    __device__ __forceinline__ void count(uint32_t at, uint32_t len, uint32_t prompt, uint32_t base, uint32_t size,
                                          uint32_t *words) const {
#pragma unroll
        for (uint32_t k = 0; k < kAhead; k++) {
            const uint32_t i = at + k * kThreads;
            if (i >= len) break;
            // base < 2^31, so a negative token stays past any chunk
            const uint32_t o = (uint32_t)id[k] - base;
            bool there = o < size;
            if (sizeof(T) == 8) there = there && (uint32_t)((uint64_t)id[k] >> 32) == 0;
            if (i >= prompt) {
                if (i + kThreads > len) there = there && i + threadIdx.x < len;
                if (there) atomicAdd(&words[o], 1u);
            } else {
                const bool said = there && i + threadIdx.x >= prompt && i + threadIdx.x < len;
                if (there && i + threadIdx.x < prompt) atomicOr(&words[o], kSeen);
                if (said) atomicAdd(&words[o], 1u);
            }
        }
    }
};

// Bias id number k of the row, or -1, and its value.
__device__ __forceinline__ int64_t bias_id(const spiky_lm_logits_args &a, uint32_t row, uint64_t k) {
    const uint64_t at = (uint64_t)row * a.bias_ids_stride + k;
    if (k >= a.n_bias) return -1;
    return a.bias_ids_i64 ? static_cast<const int64_t *>(a.bias_ids)[at] : static_cast<const int32_t *>(a.bias_ids)[at];
}

__device__ __forceinline__ float bias_value(const spiky_lm_logits_args &a, uint32_t row, uint64_t k) {
    return k < a.n_bias ? a.bias_values[(uint64_t)row * a.bias_values_stride + k] : 0.f;
}

// The sums of the row's sparse biases for the chunk's entries.  The ids go by
// kThreads: those in the chunk are listed in their order, and the first of each
// entry adds up the others, so repeated ids are added in their order whatever the
// threads do.
template <uint32_t kThreads>
struct Sparse {
    alignas(16) uint32_t list_id[kThreads + 16];
    float list_value[kThreads];
    uint32_t wave_count[2][kThreads / 64], taken;

    // Before a barrier: how many of the threads' ids are in the chunk.
    __device__ __forceinline__ uint64_t announce(int64_t id, uint32_t turn, uint32_t base, uint32_t size) {
        const uint64_t all = __ballot((uint64_t)id - base < size);
        if ((threadIdx.x & 63) == 0) wave_count[turn][threadIdx.x / 64] = __popcll(all);
        return all;
    }

    // After it.  Ends with a barrier.
    __device__ __forceinline__ void add(const spiky_lm_logits_args &a, uint32_t row, uint32_t base, uint32_t size,
                                        int64_t id, float value, uint64_t all, uint32_t *words, uint16_t *slots,
                                        float *sums) {
        const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid / 64;
        const bool in_words = slots_in_words(a.history, a.n_bias);
        uint32_t turn = 0;
        for (uint64_t k0 = 0;;) {
            uint32_t at = __popcll(all & ((1ull << lane) - 1)), listed = 0;
#pragma unroll
            for (uint32_t w = 0; w < kThreads / 64; w++) {
                if (w < wave) at += wave_count[turn][w];
                listed += wave_count[turn][w];
            }
            if (listed) {
                if (all >> lane & 1) {
                    list_id[at] = (uint32_t)id - base;
                    list_value[at] = value;
                }
                if (tid < 16) list_id[listed + tid] = ~0u;  // the search goes by 16
                __syncthreads();
                if (tid < listed) {
                    const uint32_t mine = list_id[tid];
                    bool leads = true;
                    float sum = 0.f;
                    for (uint32_t j0 = 0; j0 < listed; j0 += 16) {
                        uint4 ids[4];
#pragma unroll
                        for (int q = 0; q < 4; q++) ids[q] = *reinterpret_cast<const uint4 *>(&list_id[j0 + 4 * q]);
                        uint32_t same = 0;
#pragma unroll
                        for (int q = 0; q < 4; q++)
                            same |= (ids[q].x == mine ? 1u : 0u) << 4 * q | (ids[q].y == mine ? 2u : 0u) << 4 * q |
                                    (ids[q].z == mine ? 4u : 0u) << 4 * q | (ids[q].w == mine ? 8u : 0u) << 4 * q;
                        for (; same; same &= same - 1) {
                            const uint32_t j = j0 + __builtin_ctz(same);
                            leads = leads && j >= tid;
                            sum += list_value[j];
                        }
                    }
                    if (leads) {
                        const uint32_t w = words[mine];
                        if (w & kBiased) {  // by ids before these
                            sums[in_words ? w >> kSlotShift & kSlotMask : slots[mine]] += sum;
                        } else {
                            const uint32_t slot = atomicAdd(&taken, 1u);
                            sums[slot] = sum;
                            if (!in_words) slots[mine] = (uint16_t)slot;
                            // tokens may be counted meanwhile, in other bits
                            atomicOr(&words[mine], kBiased | (in_words ? slot << kSlotShift : 0));
                        }
                    }
                }
            }
            k0 += kThreads;
            if (k0 >= a.n_bias) break;
            turn ^= 1;
            id = bias_id(a, row, k0 + tid), value = bias_value(a, row, k0 + tid);
            all = announce(id, turn, base, size);
            __syncthreads();
        }
        __syncthreads();
    }
};

// A workgroup of kThreads takes a chunk of a row, of kThreads * P * N entries or others.  Counts
// of the row's tokens in the chunk, and which entries have sparse biases, are words in LDS, so
// the logits are read and written once and no count is kept in memory.  Loads are issued in the
// order in which they are waited for: tokens, sparse biases, logits, bias, mask; in chunks of
// another size the last three by the piece, after the counts.
//
// 512 rows of 152000 bf16 logits to fp32, inputs not in the caches: 76 us without more (6.1
// TB/s); 4096 tokens a row add 14, a shared bias 15, a mask 2 and 64 sparse biases 5, all of
// them together 58, where the waves wait for each other's phases and for L2, which reads a
// row's tokens for each of its chunks.  256 threads are faster than 512 and 1024 there (all
// together, in an earlier form: 166, 198, 242), for barriers hold fewer waves; 8 pieces a
// thread no faster than 4 (144, 141).
//
// The bound of 7 waves is measured for 2-byte logits to fp32, which spill nothing under it (127 us
// with everything set, 98 of HBM).  Under it fp32 to fp32 spills 46 registers (225 us, 129 of HBM) and
// a 2-byte result 16 (125 us, 66 of HBM); other bounds have not been measured for these.
template <typename TI, typename TO, int N, int P, uint32_t kThreads>
__global__ __launch_bounds__(kThreads, kThreads == 256 ? 7 : 1) void k_logits(spiky_lm_logits_args a, uint32_t chunk) {
    // words where there are tokens or bias ids; with bias ids as many sums as may be needed, and slots
    extern __shared__ uint4 space[];
    __shared__ Sparse<kThreads> sparse;
    uint32_t *const words = reinterpret_cast<uint32_t *>(space);
    float *const sums = reinterpret_cast<float *>(words + chunk);
    uint16_t *const slots = reinterpret_cast<uint16_t *>(sums + min((uint64_t)chunk, a.n_bias));
    // Workgroups go round the 8 XCDs in their order: the chunks of a row, which read the same
    // tokens, to one of them, as far as rows come in eights (512 rows of 152000 with 4096 tokens,
    // nothing else set: 90 us against 95).  A chunk of all rows before the next one would share
    // the bias, but reads the logits in too many places at once (all set: 143 against 134).
    uint32_t row = blockIdx.y, number = blockIdx.x;
    if (row < (gridDim.y & ~7u)) {
        const uint32_t at = blockIdx.y * gridDim.x + blockIdx.x, step = at / 8;
        row = step / gridDim.x * 8 + at % 8;
        number = step % gridDim.x;
    }
    const uint32_t tid = threadIdx.x, base = number * chunk;
    const uint32_t size = min(chunk, (uint32_t)a.vocab - base);
    const bool marks = a.tokens || a.bias_ids;
    const TI *in = static_cast<const TI *>(a.logits) + (int64_t)row * a.logits_stride + base;
    TO *out = static_cast<TO *>(a.out) + (int64_t)row * a.out_stride + base;
    const uint64_t bias_at = (uint64_t)row * a.bias_stride + base;

    const uint32_t history = (uint32_t)a.history;
    const uint64_t first = (uint64_t)row * a.tokens_stride;
    Tokens<int32_t, kThreads> short_ids;
    Tokens<int64_t, kThreads> long_ids;
    if (a.tokens) {
        if (a.tokens_i64)
            long_ids.load(static_cast<const int64_t *>(a.tokens) + first, 0, history);
        else
            short_ids.load(static_cast<const int32_t *>(a.tokens) + first, 0, history);
    }
    int64_t sparse_id = -1;
    float sparse_value = 0.f;
    if (a.bias_ids) sparse_id = bias_id(a, row, tid), sparse_value = bias_value(a, row, tid);
    const float rho = a.repetition_rows ? scalar(a.repetition_rows + row) : a.repetition;
    const float phi = a.frequency_rows ? scalar(a.frequency_rows + row) : a.frequency;
    const float pi = a.presence_rows ? scalar(a.presence_rows + row) : a.presence;
    const float heat = a.temperature_rows ? scalar(a.temperature_rows + row) : a.temperature;

    struct Piece {
        Raw<TI, N> x;
        Raw<float, N> bias;                // half of the words where it is of a shorter type
        uint32_t allowed[(N + 3) / 4];     // a byte an entry, or the byte that holds the piece's bits
    };
    auto load = [&](Piece &q, uint32_t o, int n) {
        q.x.load_end(past(in, o), n);
        if (a.bias) {
            if (a.bias_dtype == SPIKY_F32) {
                q.bias.load_end(past(static_cast<const float *>(a.bias) + bias_at, o), n);
            } else {
                Raw<bf16, N> half;
                half.load_end(past(static_cast<const bf16 *>(a.bias) + bias_at, o), n);
                __builtin_memcpy(q.bias.w, half.w, sizeof(half.w));
            }
        }
        if (!a.mask) return;
        if (a.mask_bits) {
            // chunks start at multiples of 32 entries, so a piece's bits lie in one byte
            const uint32_t *m = static_cast<const uint32_t *>(a.mask) + (int64_t)row * a.mask_stride;
            q.allowed[0] = *past(reinterpret_cast<const uint8_t *>(m) + base / 8, o / 8);
        } else {
            const uint8_t *m = past(static_cast<const uint8_t *>(a.mask) + (int64_t)row * a.mask_stride + base, o);
            if (n >= N) {
                __builtin_memcpy(q.allowed, m, N);
            } else {
#pragma unroll
                for (int i = 0; i < N; i++) {
                    if (i % 4 == 0) q.allowed[i / 4] = 0;
                    if (i < n) q.allowed[i / 4] |= (uint32_t)m[i] << (8 * (i % 4));
                }
            }
        }
    };
    // Products with reciprocals.  Those of subnormal numbers would pass the largest: a penalty is scaled
    // to a normal one first, and so is what it divides; a temperature divides.
    const float lift = fabsf(rho) < 0x1p-126f ? 0x1p24f : 1.f, less = 1.f / (rho * lift);
    const float cool = heat > 0.f ? 1.f / heat : 1.f;
    const bool divide_heat = heat > 0.f && __builtin_isinf(cool);
    const uint32_t count_mask = slots_in_words(a.history, a.n_bias) ? (1u << kSlotShift) - 1 : kBiased - 1;
    auto finish = [&](const Piece &q, uint32_t o, int n) {
        float x[N];
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = q.x[i];
        if (a.bias) {
            if (a.bias_dtype == SPIKY_F32) {
#pragma unroll
                for (int i = 0; i < N; i++) x[i] += q.bias[i];
            } else {
                Raw<bf16, N> b;
                Raw<f16, N> f;
                __builtin_memcpy(b.w, q.bias.w, sizeof(b.w));
                __builtin_memcpy(f.w, q.bias.w, sizeof(f.w));
#pragma unroll
                for (int i = 0; i < N; i++) x[i] += a.bias_dtype == SPIKY_BF16 ? b[i] : f[i];
            }
        }
        if (marks) {
            uint32_t w[N], any = 0;
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                const uint4 four = space[o / 4 + i / 4];
                w[i] = four.x, w[i + 1] = four.y, w[i + 2] = four.z, w[i + 3] = four.w;
                any |= four.x | four.y | four.z | four.w;
            }
            if (any & kBiased) {
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (w[i] & kBiased)
                        x[i] += sums[slots_in_words(a.history, a.n_bias) ? w[i] >> kSlotShift & kSlotMask : slots[o + i]];
            }
            if (any & (kSeen | count_mask)) {
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const uint32_t times = w[i] & count_mask;
                    const float y = x[i] > 0.f ? x[i] * lift * less : x[i] * rho;
                    x[i] = w[i] & (kSeen | count_mask) ? y : x[i];
                    x[i] = times ? x[i] - (phi * (float)times + pi) : x[i];
                }
            }
        }
        if (divide_heat) {
#pragma unroll
            for (int i = 0; i < N; i++) x[i] /= heat;
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) x[i] *= cool;
        }
        if (a.mask) {
            if (a.mask_bits) {
                const uint32_t bits = q.allowed[0] >> (o % 8);
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const uint32_t keep = (uint32_t)((int32_t)(bits << (31 - i)) >> 31);
                    x[i] = __uint_as_float((__float_as_uint(x[i]) & keep) | (0xff800000u & ~keep));
                }
            } else {
#pragma unroll
                for (int i = 0; i < N; i++)
                    x[i] = q.allowed[i / 4] >> (8 * (i % 4)) & 0xff ? x[i] : -__builtin_inff();
            }
        }
        // 512 rows of 152000, stored so and as usual: 97 and 130 us where the last cache holds the
        // inputs, 128 and 130 where it does not; with a reader of the result behind the call, which
        // then finds less of it there, 218 and 222, 64 rows of 130000 25.3 and 26.8, 4 rows 8.0 and 8.1
        stream_out(past(out, o), x, n);
    };

    const bool whole = size == kThreads * P * N;
    Piece piece[P];
    if (whole)
#pragma unroll
        for (int p = 0; p < P; p++) load(piece[p], (p * kThreads + tid) * N, N);
    uint32_t len = 0, prompt = 0;
    if (a.tokens) {
        len = length_at(a.lengths, a.lengths_i64, row, history);
        if (a.prompt_lengths) prompt = length_at(a.prompt_lengths, a.lengths_i64, row, len);
    }
    if (marks) {
        for (uint32_t i = tid; i < chunk / 4; i += kThreads) space[i] = make_uint4(0, 0, 0, 0);
        uint64_t all = 0;
        if (a.bias_ids) all = sparse.announce(sparse_id, 0, base, size);
        if (tid == 0) sparse.taken = 0;
        __syncthreads();
        if (a.tokens) {
            auto count_all = [&](auto &ids, auto *tokens) {
                uint32_t at = 0;
                while (true) {
                    ids.count(at, len, prompt, base, size, words);
                    at += ids.kAhead * kThreads;
                    if (at >= len) break;
                    ids.load(tokens + first, at, len);
                }
            };
            if (a.tokens_i64)
                count_all(long_ids, static_cast<const int64_t *>(a.tokens));
            else
                count_all(short_ids, static_cast<const int32_t *>(a.tokens));
        }
        if (a.bias_ids)
            sparse.add(a, row, base, size, sparse_id, sparse_value, all, words, slots, sums);
        else
            __syncthreads();
    }
    if (whole) {
#pragma unroll
        for (int p = 0; p < P; p++) finish(piece[p], (p * kThreads + tid) * N, N);
    } else {
#pragma unroll 1
        for (uint32_t o = tid * N; o < size; o += kThreads * N) {
            const int n = size - o < N ? (int)(size - o) : N;
            load(piece[0], o, n);
            finish(piece[0], o, n);
        }
    }
}

template <typename TI, typename TO>
hipError_t launch(const spiky_lm_logits_args &a, hipStream_t st) {
    constexpr int N = sizeof(TO) == 4 ? 4 : 8, kMost = 16 / N;
    // enough workgroups for the chip, but no more than a row's history is worth reading for
    auto workgroups = [&](uint64_t entries) { return (a.vocab + entries - 1) / entries * a.rows; };
    const bool wide = a.tokens && a.history > kLong &&
                      (workgroups(4096) < 2 * kCUs || (a.history >= 2 * kLong && workgroups(16384) >= 2 * kCUs));
    uint64_t chunk = wide ? 32768 : 256 * 16;
    auto lds_of = [&](uint64_t entries) {
        size_t bytes = a.tokens || a.bias_ids ? entries * sizeof(uint32_t) : 0;
        if (a.bias_ids)
            bytes += (a.n_bias < entries ? a.n_bias : entries) * sizeof(float) +
                     (slots_in_words(a.history, a.n_bias) ? 0 : entries * sizeof(uint16_t));
        return bytes;
    };
    while (chunk > (wide ? 1024 : 256) * N && (workgroups(chunk) < 2 * kCUs || lds_of(chunk) > kMostLds)) chunk /= 2;
    const uint64_t chunks = (a.vocab + chunk - 1) / chunk;
    const size_t lds = lds_of(chunk);
    // 65535 rows a launch, in y
    for (uint64_t row0 = 0; row0 < a.rows; row0 += 65535) {
        const uint32_t n = (uint32_t)(a.rows - row0 < 65535 ? a.rows - row0 : 65535);
        spiky_lm_logits_args part = a;
        auto skip = [&](auto *&p, int64_t bytes) {
            using P = std::remove_reference_t<decltype(p)>;
            if (p) p = (P)((uintptr_t)p + (uint64_t)bytes * row0);
        };
        skip(part.logits, a.logits_stride * (int64_t)sizeof(TI));
        skip(part.out, a.out_stride * (int64_t)sizeof(TO));
        skip(part.tokens, a.tokens_stride * (a.tokens_i64 ? 8 : 4));
        skip(part.lengths, a.lengths_i64 ? 8 : 4);
        skip(part.prompt_lengths, a.lengths_i64 ? 8 : 4);
        skip(part.repetition_rows, 4);
        skip(part.presence_rows, 4);
        skip(part.frequency_rows, 4);
        skip(part.temperature_rows, 4);
        skip(part.bias, a.bias_stride * (a.bias_dtype == SPIKY_F32 ? 4 : 2));
        skip(part.bias_ids, a.bias_ids_stride * (a.bias_ids_i64 ? 8 : 4));
        skip(part.bias_values, a.bias_values_stride * 4);
        skip(part.mask, a.mask_stride * (a.mask_bits ? 4 : 1));
        const dim3 grid((uint32_t)chunks, n);
        if (wide)
            k_logits<TI, TO, N, 1, 1024><<<grid, dim3(1024), lds, st>>>(part, (uint32_t)chunk);
        else if (chunk == 256 * 16)
            k_logits<TI, TO, N, kMost, 256><<<grid, dim3(256), lds, st>>>(part, (uint32_t)chunk);
        else if (chunk == 256 * 8)
            k_logits<TI, TO, N, kMost / 2, 256><<<grid, dim3(256), lds, st>>>(part, (uint32_t)chunk);
        else
            k_logits<TI, TO, N, 1, 256><<<grid, dim3(256), lds, st>>>(part, (uint32_t)chunk);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return err;
    }
    return hipSuccess;
}

}  // namespace

hipError_t launch_process_logits(const spiky_lm_logits_args &a, hipStream_t st) {
    if (a.dtype == SPIKY_F32) return launch<float, float>(a, st);
    if (a.dtype == SPIKY_BF16)
        return a.out_dtype == SPIKY_F32 ? launch<bf16, float>(a, st) : launch<bf16, bf16>(a, st);
    return a.out_dtype == SPIKY_F32 ? launch<f16, float>(a, st) : launch<f16, f16>(a, st);
}

}  // namespace lm
}  // namespace spiky
