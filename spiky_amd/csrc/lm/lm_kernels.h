// lm_kernels.h -- what the language-model operators' kernels share (gfx950):
// element types, rows in 16-byte pieces, the dropout generator, row sums.
//
// Internal to libspiky_lut.so; the public C ABI is include/spiky_lm.h.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../../include/spiky_lm.h"

namespace spiky {
namespace lm {

constexpr uint32_t kCUs = 256;
constexpr uint64_t kLastCache = 256u << 20;  // bytes

// ---- elements --------------------------------------------------------------
struct bf16 {
    uint16_t bits;
};
typedef _Float16 f16;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16 x) { return __uint_as_float((uint32_t)x.bits << 16); }
__device__ __forceinline__ float to_f32(f16 x) { return (float)x; }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) {
    return x;
}
// Round to nearest, ties to even (the compiler's conversion, v_cvt_pk_bf16_f32).
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(float x) {
    const __bf16 b = (__bf16)x;
    bf16 r;
    __builtin_memcpy(&r, &b, 2);
    return r;
}
template <>
__device__ __forceinline__ f16 from_f32<f16>(float x) {
    return (f16)x;
}

// The words of N elements as they were loaded, so that a load may be in flight
// while the values of the row before are worked on.  A whole piece is one load of
// its full width at any alignment of the element type (the target's unaligned
// access mode).
template <typename T, int N>
struct Raw {
    static constexpr int kWords = N * sizeof(T) / 4;
    uint32_t w[kWords];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kWords; i++) w[i] = 0;
    }
    // n of them exist, the others are 0.  A short piece goes element by element in
    // a loop, which costs no registers: for rows narrower than a piece.
    __device__ __forceinline__ void load(const T *p, int n) {
        if (n >= N) {
            __builtin_memcpy(w, p, sizeof(w));
            return;
        }
        if (n <= 0) return;
        clear();
#pragma unroll 1
        for (int i = n - 1; i >= 0; i--) {
            uint32_t x = 0;
            __builtin_memcpy(&x, p + i, sizeof(T));
#pragma unroll
            for (int k = kWords - 1; k > 0; k--)
                w[k] = sizeof(T) == 4 ? w[k - 1] : w[k] << 16 | w[k - 1] >> 16;
            w[0] = sizeof(T) == 4 ? x : w[0] << 16 | x;
        }
    }
    // The same with a short piece's loads in flight at once: for the ends of rows.
    __device__ __forceinline__ void load_end(const T *p, int n) {
        if (n >= N) {
            __builtin_memcpy(w, p, sizeof(w));
            return;
        }
        clear();
        if (n <= 0) return;
        T t[N];
#pragma unroll
        for (int i = 0; i < N; i++) t[i] = p[i < n ? i : 0];
#pragma unroll
        for (int i = 0; i < N; i++) {
            uint32_t x = 0;
            __builtin_memcpy(&x, &t[i], sizeof(T));
            x = i < n ? x : 0;
            w[i * sizeof(T) / 4] |= sizeof(T) == 4 ? x : x << (16 * (i % 2));
        }
    }
    __device__ __forceinline__ float operator[](int i) const {
        T t;
        if (sizeof(T) == 4) {
            __builtin_memcpy(&t, &w[i], sizeof(T));
        } else {
            const uint16_t h = (uint16_t)(w[i / 2] >> (16 * (i % 2)));
            __builtin_memcpy(&t, &h, 2);
        }
        return to_f32(t);
    }
};

// N elements from p, of which the first n exist; the others read as 0.
template <typename T, int N>
__device__ __forceinline__ void load(float (&v)[N], const T *p, int n) {
    Raw<T, N> raw;
    raw.clear();
    raw.load(p, n);
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = raw[i];
}

// The first n of N elements, a short piece's in halves of halves.
template <typename T, int N>
__device__ __forceinline__ void store(T *p, const float (&v)[N], int n) {
    T t[N];
#pragma unroll
    for (int i = 0; i < N; i++) t[i] = from_f32<T>(v[i]);
    if (n >= N) {
        __builtin_memcpy(p, t, sizeof(t));
        return;
    }
#pragma unroll
    for (int step = N / 2; step >= 1; step /= 2) {
        if (!(n & step)) continue;
        __builtin_memcpy(p, t, step * sizeof(T));
        p += step;
#pragma unroll
        for (int i = 0; i < step; i++) t[i] = t[i + step];
    }
}

// The same past the caches' ordinary replacement, so that what other workgroups read again stays in L2.
// One store a thread: nothing puts the parts of a line together that several store one after the other.
template <typename T, int N>
__device__ __forceinline__ void stream_out(T *p, const float (&v)[N], int n) {
    static_assert(N * sizeof(T) == 16, "16-byte pieces");
    if (n < N) {
        store(p, v, n);
        return;
    }
    typedef uint32_t Piece __attribute__((ext_vector_type(4), aligned(2)));
    T t[N];
#pragma unroll
    for (int i = 0; i < N; i++) t[i] = from_f32<T>(v[i]);
    Piece q;
    __builtin_memcpy(&q, t, sizeof(q));
    __builtin_nontemporal_store(q, reinterpret_cast<Piece *>(p));
}

// A thread's piece of N columns of every row.  The last piece of a row that N does
// not divide is the row's last N columns, and has the others of them in common
// with the piece before: both work them out alike, and only one counts them in
// sums, so no lane takes another path than its wave's.  Rows of fewer than N
// columns are one short piece.
template <int N>
struct Place {
    uint64_t col;   // its first column
    uint32_t own;   // bit i: column col + i counts as this piece's
    int n;          // columns of it that exist: N, or fewer in narrow rows; 0: no piece

    __device__ __forceinline__ void set(uint64_t cols, uint64_t nominal) {
        constexpr uint32_t kAll = N < 32 ? (1u << N) - 1 : ~0u;
        col = nominal, own = kAll, n = N;
        if (nominal >= cols) {
            col = 0, own = 0, n = 0;
        } else if (cols < N) {
            n = (int)cols;
            own = (1u << n) - 1;
        } else if (nominal + N > cols) {
            col = cols - N;
            own = kAll & kAll << (nominal - col);
        }
    }
};

// x / d for x < 2^32 by a product and two shifts (Granlund and Montgomery,
// "Division by invariant integers using multiplication", 1994).
struct Divider {
    uint32_t d, m, s1, s2;
    Divider() : Divider(1) {}
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

// ---- dropout ---------------------------------------------------------------
// The kept elements of a tensor are a function of (seed, offset, row, column)
// alone: 7 rounds of Philox4x32 (Salmon, Moraes, Dror, Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", 2011) give four 32-bit words for four columns.
// Seven rounds are the fewest the authors find to pass BigCrush; a round is two
// 32 x 32 -> 64 products at a quarter of the VALU rate, and ten of them take
// longer than the copy of a 2-byte element.
struct Dropper {
    uint32_t threshold;  // kept: word >= threshold
    float scale;         // 1 / (1 - p); 0: nothing is kept
    uint32_t k0, k1, o0, o1;
};

struct DropArgs {
    uint32_t threshold;
    float scale;
    uint64_t seed, offset;
    const int64_t *rng;
};

__device__ __forceinline__ Dropper dropper(const DropArgs &a) {
    const uint64_t seed = a.rng ? (uint64_t)a.rng[0] : a.seed;
    const uint64_t offset = a.rng ? (uint64_t)a.rng[1] : a.offset;
    return {a.threshold,    a.scale, (uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)offset,
            (uint32_t)(offset >> 32)};
}

__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
    return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);  // one instruction; the compiler takes two for a ^ b ^ c
}

// Bit i: the group's column i is kept.
__device__ __forceinline__ uint32_t kept4(const Dropper &d, uint32_t row, uint32_t group) {
    uint32_t c0 = group, c1 = row, c2 = d.o0, c3 = d.o1, k0 = d.k0, k1 = d.k1;
#pragma unroll
    for (int i = 0; i < 7; i++) {
        const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = xor3((uint32_t)(p1 >> 32), c1, k0);
        c1 = (uint32_t)p1;
        c2 = xor3((uint32_t)(p0 >> 32), c3, k1);
        c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return (c0 >= d.threshold ? 1 : 0) | (c1 >= d.threshold ? 2 : 0) | (c2 >= d.threshold ? 4 : 0) |
           (c3 >= d.threshold ? 8 : 0);
}

// The same for the N columns from col on.
template <int N>
__device__ __forceinline__ uint32_t kept(const Dropper &d, uint32_t row, uint64_t col) {
    static_assert(N % 4 == 0 && N <= 28, "whole groups");
    const uint32_t group = (uint32_t)(col / 4), within = (uint32_t)col & 3;
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < N; i += 4) bits |= kept4(d, row, group + i / 4) << i;
    if (within) bits = (bits | kept4(d, row, group + N / 4) << N) >> within;
    return d.scale != 0.f ? bits : 0;
}

// x where bit i is set, else 0, whatever x is.
__device__ __forceinline__ float where(uint32_t bits, int i, float x) {
    return __int_as_float(__float_as_int(x) & ((int32_t)(bits << (31 - i)) >> 31));
}

template <int N>
__device__ __forceinline__ void drop(float (&v)[N], const Dropper &d, uint32_t row, uint64_t col) {
    const uint32_t bits = kept<N>(d, row, col);
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = where(bits, i, v[i] * d.scale);
}

// ---- launchers -------------------------------------------------------------
hipError_t launch_dropout(const void *x, int64_t x_stride, void *y, uint64_t rows, uint64_t cols,
                          int dtype, const DropArgs &drop, hipStream_t st);

hipError_t launch_residual_norm(const spiky_lm_residual_args &a, const DropArgs &drop, void *out,
                                void *normed, hipStream_t st);
uint64_t residual_norm_workspace(const spiky_lm_residual_args &a, const spiky_lm_residual_grads &g);
hipError_t launch_residual_norm_backward(const spiky_lm_residual_args &a, const DropArgs &drop,
                                         const spiky_lm_residual_grads &g, hipStream_t st);

hipError_t launch_process_logits(const spiky_lm_logits_args &a, hipStream_t st);

}  // namespace lm
}  // namespace spiky
