// lm_logits.hip -- penalties, biases, temperature and masks on logits (gfx950).
#include <type_traits>

#include "lm_kernels.h"

namespace spiky {
namespace lm {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kSeen = 0x80000000u;    // among the prompt's tokens
constexpr uint32_t kBiased = 0x40000000u;  // among the bias ids
constexpr uint32_t kCount = 0x3fffffffu;   // times among the tokens after the prompt
constexpr uint32_t kList = 256;            // bias entries of a chunk held in LDS

__device__ __forceinline__ int64_t id_at(const void *p, bool i64, uint64_t i) {
    return i64 ? static_cast<const int64_t *>(p)[i] : static_cast<const int32_t *>(p)[i];
}

__device__ __forceinline__ uint64_t length_at(const void *p, bool i64, uint32_t row, uint64_t most) {
    if (!p) return most;
    const int64_t n = id_at(p, i64, row);
    return n < 0 ? 0 : (uint64_t)n < most ? (uint64_t)n : most;
}

// One workgroup to a chunk of a row's vocabulary.  The chunk's counts of the
// row's tokens, and which entries have sparse biases, are words in LDS, so the
// logits are read and written once and no count is kept in memory.
template <typename TI, typename TO, int N>
__global__ __launch_bounds__(kThreads) void k_logits(spiky_lm_logits_args a, uint32_t chunk) {
    extern __shared__ uint32_t words[];  // [chunk], where there are tokens or bias ids
    __shared__ uint32_t list_id[kList];
    __shared__ float list_value[kList];
    __shared__ uint32_t listed;
    const uint32_t tid = threadIdx.x, row = blockIdx.y;
    const uint64_t base = (uint64_t)blockIdx.x * chunk;
    const uint32_t size = (uint32_t)min((uint64_t)chunk, a.vocab - base);
    const bool marks = a.tokens || a.bias_ids;
    if (marks) {
        for (uint32_t i = tid; i < size; i += kThreads) words[i] = 0;
        __syncthreads();
        if (a.tokens) {
            const uint64_t len = length_at(a.lengths, a.lengths_i64, row, a.history);
            const uint64_t prompt = a.prompt_lengths ? length_at(a.prompt_lengths, a.lengths_i64, row, len) : 0;
            const uint64_t first = (uint64_t)row * a.tokens_stride;
            for (uint64_t i = tid; i < len; i += kThreads) {
                const uint64_t o = (uint64_t)id_at(a.tokens, a.tokens_i64, first + i) - base;
                if (o >= size) continue;
                if (i < prompt)
                    atomicOr(&words[o], kSeen);
                else
                    atomicAdd(&words[o], 1u);
            }
        }
        // the chunk's sparse biases in their order, by the first wave
        if (a.bias_ids && tid < 64) {
            const uint64_t first = (uint64_t)row * a.bias_ids_stride, firstv = (uint64_t)row * a.bias_values_stride;
            uint32_t count = 0;
            for (uint64_t k0 = 0; k0 < a.n_bias; k0 += 64) {
                const uint64_t k = k0 + tid;
                const uint64_t o = k < a.n_bias ? (uint64_t)id_at(a.bias_ids, a.bias_ids_i64, first + k) - base : size;
                const bool in = o < size;
                const uint64_t all = __ballot(in);
                const uint32_t at = count + __popcll(all & ((1ull << tid) - 1));
                if (in) {
                    atomicOr(&words[o], kBiased);
                    if (at < kList) {
                        list_id[at] = (uint32_t)o;
                        list_value[at] = a.bias_values[firstv + k];
                    }
                }
                count += __popcll(all);
            }
            if (tid == 0) listed = count;
        }
        __syncthreads();
    }
    const float rho = a.repetition_rows ? a.repetition_rows[row] : a.repetition;
    const float phi = a.frequency_rows ? a.frequency_rows[row] : a.frequency;
    const float pi = a.presence_rows ? a.presence_rows[row] : a.presence;
    const float heat = a.temperature_rows ? a.temperature_rows[row] : a.temperature;
    const float less = 1.f / rho, cool = heat > 0.f ? 1.f / heat : 1.f;
    const TI *in = static_cast<const TI *>(a.logits) + (int64_t)row * a.logits_stride + base;
    TO *out = static_cast<TO *>(a.out) + (int64_t)row * a.out_stride + base;
    for (uint32_t o = tid * N; o < size; o += kThreads * N) {
        const int n = size - o < N ? (int)(size - o) : N;
        float x[N], b[N];
        load(x, in + o, n);
        if (a.bias) {
            const uint64_t at = (uint64_t)row * a.bias_stride + base + o;
            if (a.bias_dtype == SPIKY_F32)
                load(b, static_cast<const float *>(a.bias) + at, n);
            else if (a.bias_dtype == SPIKY_BF16)
                load(b, static_cast<const bf16 *>(a.bias) + at, n);
            else
                load(b, static_cast<const f16 *>(a.bias) + at, n);
#pragma unroll
            for (int i = 0; i < N; i++) x[i] += b[i];
        }
        if (marks) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const uint32_t w = i < n ? words[o + i] : 0;
                if (w & kBiased) {
                    float s = 0.f;
                    if (listed <= kList) {
                        for (uint32_t k = 0; k < listed; k++)
                            if (list_id[k] == o + i) s += list_value[k];
                    } else {
                        const uint64_t first = (uint64_t)row * a.bias_ids_stride;
                        for (uint64_t k = 0; k < a.n_bias; k++)
                            if ((uint64_t)id_at(a.bias_ids, a.bias_ids_i64, first + k) == base + o + i)
                                s += a.bias_values[(uint64_t)row * a.bias_values_stride + k];
                    }
                    x[i] += s;
                }
                const uint32_t times = w & kCount;
                if (w & (kSeen | kCount)) x[i] = x[i] > 0.f ? x[i] * less : x[i] * rho;
                if (times) x[i] -= phi * (float)times + pi;
            }
        }
#pragma unroll
        for (int i = 0; i < N; i++) x[i] *= cool;
        if (a.mask) {
            if (a.mask_bits) {
                // the piece's bits lie in one or two words
                const uint32_t *m = static_cast<const uint32_t *>(a.mask) + (int64_t)row * a.mask_stride;
                const uint64_t v = base + o;
                const uint32_t shift = (uint32_t)(v & 31);
                uint64_t bits = m[v / 32];
                if (shift + n > 32) bits |= (uint64_t)m[v / 32 + 1] << 32;
                bits >>= shift;
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (!(bits >> i & 1)) x[i] = -__builtin_inff();
            } else {
                const uint8_t *m = static_cast<const uint8_t *>(a.mask) + (int64_t)row * a.mask_stride + base + o;
                uint8_t allowed[N];
                if (n >= N) {
                    __builtin_memcpy(allowed, m, N);
                } else {
#pragma unroll
                    for (int i = 0; i < N; i++) allowed[i] = i < n ? m[i] : 0;
                }
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (!allowed[i]) x[i] = -__builtin_inff();
            }
        }
        store(out + o, x, n);
    }
}

template <typename TI, typename TO>
hipError_t launch(const spiky_lm_logits_args &a, hipStream_t st) {
    constexpr int N = 8;
    // enough workgroups for the chip, but no more than a row's history is worth reading for
    uint64_t chunk = 8192;
    while (chunk > 2048 && (a.vocab + chunk - 1) / chunk * a.rows < 2 * kCUs) chunk /= 2;
    const uint64_t chunks = (a.vocab + chunk - 1) / chunk;
    if (chunks > 0xffffffffull / kThreads) return hipErrorInvalidValue;
    const size_t lds = a.tokens || a.bias_ids ? chunk * sizeof(uint32_t) : 0;
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
        k_logits<TI, TO, N><<<dim3((uint32_t)chunks, n), dim3(kThreads), lds, st>>>(part, (uint32_t)chunk);
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
