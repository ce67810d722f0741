// lm_dropout.hip -- dropout whose mask is recomputed, never stored (gfx950).
#include "lm_kernels.h"

namespace spiky {
namespace lm {
namespace {

constexpr int kThreads = 256;
constexpr int kPieces = 4;  // 16-byte pieces of a thread

// x / d for x < 2^32 by a product and two shifts (Granlund and Montgomery,
// "Division by invariant integers using multiplication", 1994).
struct Divider {
    uint32_t d, m, s1, s2;
    explicit Divider(uint32_t d_) : d(d_) {
        uint32_t l = 0;
        while (l < 32 && ((uint64_t)1 << l) < d) l++;
        m = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << l) - d)) / d + 1);
        s1 = l < 1 ? l : 1;
        s2 = l < 1 ? 0 : l - 1;
    }
    __device__ __forceinline__ uint32_t divide(uint32_t x) const {
        const uint32_t t = __umulhi(m, x);
        return (t + ((x - t) >> s1)) >> s2;
    }
};

// Reads and writes once: 16384 x 8192 bf16 take 96 us, 5.6 TB/s (a large copy runs
// at 4.9 to 5.4).  The generator's 14 products of 32 x 32 bits for four columns make
// most of 44.6 M vector instructions, 73 us at one in 4 cycles.  A row is cut into pieces of 16 bytes, and the
// pieces of all rows are numbered through; thread t of a workgroup takes pieces
// t, t + 256, ... of the workgroup's kThreads * kPieces.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_dropout(const T *__restrict__ x, int64_t x_stride,
                                                      T *__restrict__ y, uint64_t rows,
                                                      uint64_t cols, Divider row_pieces,
                                                      DropArgs args) {
    constexpr int N = 16 / sizeof(T);
    const Dropper d = dropper(args);
    const uint64_t first = (uint64_t)blockIdx.x * (kThreads * kPieces);
    // workgroup-uniform: the row and the piece in it of the workgroup's first piece
    const uint64_t row0 = first < 0x100000000ull ? row_pieces.divide((uint32_t)first) : first / row_pieces.d;
    const uint32_t piece0 = (uint32_t)(first - row0 * row_pieces.d);
#pragma unroll
    for (int i = 0; i < kPieces; i++) {
        const uint64_t at = (uint64_t)piece0 + i * kThreads + threadIdx.x;
        // a long row ends at most once in the workgroup's pieces, a short one's numbers fit 32 bits
        const uint32_t down = row_pieces.d >= kThreads * kPieces ? at >= row_pieces.d
                                                                 : row_pieces.divide((uint32_t)at);
        const uint64_t row = row0 + down;
        if (row >= rows) break;
        Place<N> place;
        place.set(cols, (at - (uint64_t)down * row_pieces.d) * N);
        float v[N];
        load(v, x + (int64_t)row * x_stride + place.col, place.n);
        drop(v, d, (uint32_t)row, place.col);
        if (sizeof(T) == 2) {
            // the product rounds to 32 bits and then to T, for every T alike: without this the
            // compiler rounds fp16 products once (v_fma_mixlo_f16)
#pragma unroll
            for (int k = 0; k < N; k++) asm("" : "+v"(v[k]));
        }
        store(y + row * cols + place.col, v, place.n);
    }
}

template <typename T>
hipError_t launch(const void *x, int64_t x_stride, void *y, uint64_t rows, uint64_t cols,
                  const DropArgs &drop, hipStream_t st) {
    constexpr uint64_t N = 16 / sizeof(T);
    const uint64_t row_pieces = (cols + N - 1) / N;
    const uint64_t groups = (rows * row_pieces + kThreads * kPieces - 1) / (kThreads * kPieces);
    if (groups * kThreads > 0xffffffffull) return hipErrorInvalidValue;
    k_dropout<T><<<dim3((uint32_t)groups), dim3(kThreads), 0, st>>>(
        static_cast<const T *>(x), x_stride, static_cast<T *>(y), rows, cols,
        Divider((uint32_t)row_pieces), drop);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_dropout(const void *x, int64_t x_stride, void *y, uint64_t rows, uint64_t cols,
                          int dtype, const DropArgs &drop, hipStream_t st) {
    if (dtype == SPIKY_F32) return launch<float>(x, x_stride, y, rows, cols, drop, st);
    if (dtype == SPIKY_BF16) return launch<bf16>(x, x_stride, y, rows, cols, drop, st);
    return launch<f16>(x, x_stride, y, rows, cols, drop, st);
}

}  // namespace lm
}  // namespace spiky
