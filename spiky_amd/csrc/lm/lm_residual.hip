// lm_residual.hip -- the residual join of a block, forward and backward (gfx950).
//
// Forward, per row:  v = post(a) w1 + b1,  d = dropout(v),
//   z = alpha r + beta g d,  h = pre(z) w2 + b2.
// Backward from dz and dh, with n1 = post(a), n2 = pre(z), r1 and r2 their
// reciprocal deviations, means over the row's columns:
//   t  = dh w2
//   q  = dz + r2 (t - [mean t] - n2 mean(t n2))     dw2 = sum dh n2   db2 = sum dh
//   dr = alpha q      dg = sum beta d q
//   dv = keep / (1 - p) beta g q                    dw1 = sum dv n1   db1 = sum dv
//   dn = dv w1
//   da = r1 (dn - [mean dn] - n1 mean(dn n1))
// ([..] in layer norms only).  z is formed again from r and a, not read back
// from its rounded copy, so n2 is the forward's own.
//
// Both directions are bound by memory where the work is large: 16384 rows of 4096,
// bf16 beside an fp32 residual, take 155-176 us forward (805 MB, 4.6-5.2 TB/s; a large
// copy runs at 4.9 to 5.4) and 268-299 us backward (1.24 GB, 4.1-4.6 TB/s), the less in a
// process that has worked on nothing else, with the vector unit
// busy half of the time, a third of that with the dropout's generator.  A backward
// pass in two passes over the inputs took 808.  Small calls are bound by the host.
#include "lm_kernels.h"

namespace spiky {
namespace lm {
namespace {

// What a call has, as bits of Join::has: tests of them in a row's loop cost no
// registers, those of the pointers two each.
enum : uint32_t {
    kBranch = 1, kDz = 2, kDh = 4, kDrops = 8, kPost = 16, kPostLayer = 32, kPreLayer = 64, kDr = 128, kDa = 256,
    kGate = 512, kRowGate = 1 << 10, kDgate = 1 << 11, kRowDgate = 1 << 12, kW1 = 1 << 13, kB1 = 1 << 14, kW2 = 1 << 15,
    kPart = 1 << 16  // and the four bits above: column sums number 0 to 4
};

// The bits where they are used: the compiler would take each test out of the row's
// loop and keep its result in two registers over it.
__device__ __forceinline__ uint32_t here(uint32_t has) {
    asm("" : "+s"(has));
    return has;
}

// The kernels' view of a call.
template <typename TZ, typename TA>
struct Join {
    const TZ *r;
    const TA *a;
    int64_t r_stride, a_stride;
    const void *w1, *b1, *g, *w2, *b2;
    bool par_f32, gate_f32;
    int post, pre;
    float post_eps, pre_eps, alpha, beta, inv_cols;
    bool drops;
    DropArgs drop;
    uint32_t rows, gate_rows;
    uint32_t row0;  // the launch's first row
    uint64_t cols;
    float4 *stats;
    TZ *out;
    TA *normed;
    // backward
    uint32_t has;
    const TZ *dz;
    const TA *dh;
    int64_t dz_stride, dh_stride;
    TZ *dr;
    TA *da;
    void *dgate;      // full gates: written by element
    float4 *row_sums; // [rows]: mean t, mean t n2, mean dn, mean dn n1
    float *part[5];   // column sums of w1, b1, w2, b2, g: one row a chunk, or null
    uint32_t chunk;                    // rows of a chunk
    uint32_t span, chunks_per_span;    // chunks_per_span > 0: so many chunks to each span rows, none across two spans
};

// N values of a parameter row at column col, n of them in the row.
template <typename T, int N>
__device__ __forceinline__ void param(float (&v)[N], const void *p, bool f32, uint64_t at, int n) {
    if (f32)
        load(v, static_cast<const float *>(p) + at, n);
    else
        load(v, static_cast<const T *>(p) + at, n);
}

template <int CTRL>
__device__ __forceinline__ float add_dpp(float x) {
    return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}

// Sum over groups of L lanes (8, 16, 32 or 64), in every lane: exchanges inside
// quads, eights and sixteens by DPP, then between rows of 16 and halves.
template <int L>
__device__ __forceinline__ float lanes_sum(float x) {
    x = add_dpp<0xB1>(x);   // quad_perm 1 0 3 2
    x = add_dpp<0x4E>(x);   // quad_perm 2 3 0 1
    x = add_dpp<0x141>(x);  // row_half_mirror
    if (L >= 16) x = add_dpp<0x140>(x);  // row_mirror
    if (L >= 32) {
        auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
    if (L >= 64) {
        auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
    return x;
}

__device__ __forceinline__ int piece_size(uint64_t cols, uint64_t col, int n) {
    return col >= cols ? 0 : cols - col < (uint64_t)n ? (int)(cols - col) : n;
}

// v = n1 w1 + b1 and then d = dropout(v), from n1.
template <typename TA, int N, typename J>
__device__ __forceinline__ void affine_drop(float (&v)[N], const J &j, const Dropper &dr, uint32_t row,
                                            uint64_t col, int n) {
    if (j.w1) {
        float w[N];
        param<TA>(w, j.w1, j.par_f32, col, n);
#pragma unroll
        for (int i = 0; i < N; i++) v[i] *= w[i];
    }
    if (j.b1) {
        float b[N];
        param<TA>(b, j.b1, j.par_f32, col, n);
#pragma unroll
        for (int i = 0; i < N; i++) v[i] += b[i];
    }
    if (j.drops) drop(v, dr, row, col);
}

template <typename TA, int N, typename J>
__device__ __forceinline__ void gate_of(float (&g)[N], const J &j, uint32_t gate_row, uint64_t col, int n) {
    if (j.g) {
        param<TA>(g, j.g, j.gate_f32, (uint64_t)gate_row * j.cols + col, n);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) g[i] = 1.f;
    }
}

// Sums of K values over the `waves` waves of a row (TPR > 64) or its TPR lanes,
// in every lane.  The waves' sums go through LDS, two buffers in turn: a buffer
// is written again only after the barrier of the call in between, which its
// readers have passed.  Lane i reads the sums of wave i % 16.
template <int TPR, int K>
__device__ __forceinline__ void row_sums(float (&x)[K], float4 (*lds)[(K + 3) / 4][16], uint32_t &turn,
                                         uint32_t waves) {
#pragma unroll
    for (int k = 0; k < K; k++) x[k] = lanes_sum<(TPR < 64 ? TPR : 64)>(x[k]);
    if constexpr (TPR > 64) {
        constexpr int H = (K + 3) / 4;
        float v[4 * H];
#pragma unroll
        for (int k = 0; k < 4 * H; k++) v[k] = k < K ? x[k < K ? k : 0] : 0.f;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int h = 0; h < H; h++)
                lds[turn][h][threadIdx.x / 64] = make_float4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]);
        __syncthreads();
        const uint32_t wave = threadIdx.x & 15;
#pragma unroll
        for (int h = 0; h < H; h++) {
            const float4 f = wave < waves ? lds[turn][h][wave] : make_float4(0.f, 0.f, 0.f, 0.f);
            v[4 * h] = f.x, v[4 * h + 1] = f.y, v[4 * h + 2] = f.z, v[4 * h + 3] = f.w;
        }
#pragma unroll
        for (int k = 0; k < K; k++) x[k] = lanes_sum<16>(v[k]);
        turn ^= 1;
    }
}

// ---- forward ---------------------------------------------------------------
// A piece of a row.  SHORT: rows may be narrower than a piece.
template <bool SHORT, typename T, int N>
__device__ __forceinline__ void fetch_piece(Raw<T, N> &raw, const T *p, int n) {
    if (SHORT)
        raw.load(p, n);
    else if (n)
        __builtin_memcpy(raw.w, p, sizeof(raw.w));
}

template <bool SHORT, typename T, int N>
__device__ __forceinline__ void store_piece(T *p, const float (&v)[N], int n) {
    if (SHORT)
        store(p, v, n);
    else if (n)
        store(p, v, N);
}

// N values of a parameter or gate row: its words as loaded (half of them where it
// is of a shorter type than float), and their values.
template <typename TA, bool SHORT, int N>
__device__ __forceinline__ void words_of(Raw<float, N> &raw, const void *p, bool f32, uint64_t at, int n) {
    if (sizeof(TA) == 4 || f32) {
        fetch_piece<SHORT>(raw, static_cast<const float *>(p) + at, n);
    } else {
        Raw<TA, N> half;
        __builtin_memcpy(half.w, raw.w, sizeof(half.w));
        fetch_piece<SHORT>(half, static_cast<const TA *>(p) + at, n);
        __builtin_memcpy(raw.w, half.w, sizeof(half.w));
    }
}

template <typename TA, int N>
__device__ __forceinline__ void values_of(float (&v)[N], const Raw<float, N> &raw, bool f32) {
    if (sizeof(TA) == 4 || f32) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = raw[i];
    } else {
        Raw<TA, N> half;
        __builtin_memcpy(half.w, raw.w, sizeof(half.w));
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = half[i];
    }
}

// A row in the registers of TPR threads (TPR > 64: of the workgroup, of up to TPR),
// P pieces of N columns each: every input is read once, the sums of both norms run
// over registers.  The row's loads are issued before the first sum, and with 8
// columns a thread the parameters' too; with 16 these would halve the waves (2597
// rows of 9564: 119 us so, 107 without).  A workgroup has one round of rows and
// leaves: walking many with the parameters in registers and the next row's loads
// ahead needs twice the registers, so half the waves (16384 rows of 8192 bf16: 287
// us against 232).  FULL: with layer norms or biases.
template <typename TZ, typename TA, int N, int P, int TPR, bool FULL>
__global__ __launch_bounds__(TPR <= 64 ? 256 : TPR) void k_join(Join<TZ, TA> j) {
    constexpr int kSlots = TPR <= 64 ? 256 / TPR : 1, Q = N * P <= 8 ? P : 1;
    constexpr bool AHEAD = N * P <= 8;
    __shared__ float4 red[TPR > 64 ? 2 : 1][1][16];
    uint32_t turn = 0;
    const uint32_t threads = TPR <= 64 ? TPR : blockDim.x, waves = blockDim.x / 64;
    const uint32_t lane = TPR <= 64 ? threadIdx.x % TPR : threadIdx.x;
    uint32_t row = j.row0 + blockIdx.x * kSlots + (kSlots > 1 ? threadIdx.x / TPR : 0);
    if (TPR == 64) row = __builtin_amdgcn_readfirstlane(row);
    if (kSlots > 1 && row >= j.rows) return;

    Place<N> at[P];
    Raw<TZ, N> z_raw[P];
    Raw<TA, N> a_raw[P];
    Raw<float, N> g[P], w[Q], b[FULL ? Q : 1];
#pragma unroll
    for (int p = 0; p < P; p++) {
        at[p].set(j.cols, (uint64_t)(p * threads + lane) * N);
        a_raw[p].clear(), z_raw[p].clear(), g[p].clear();
        if (AHEAD || p == 0) {
            w[AHEAD ? p : 0].clear();
            if (FULL) b[FULL && AHEAD ? p : 0].clear();
        }
        if (j.a) fetch_piece<false>(a_raw[p], j.a + (int64_t)row * j.a_stride + at[p].col, at[p].n);
        fetch_piece<false>(z_raw[p], j.r + (int64_t)row * j.r_stride + at[p].col, at[p].n);
    }
    const uint64_t gate_at = j.g ? (uint64_t)(row / j.gate_rows) * j.cols : 0;
    auto parameters = [&](int p, const void *weight, const void *bias) {
        const int q = AHEAD ? p : 0;
        if (weight) words_of<TA, false>(w[q], weight, j.par_f32, at[p].col, at[p].n);
        if constexpr (FULL)
            if (bias) words_of<TA, false>(b[q], bias, j.par_f32, at[p].col, at[p].n);
    };
#pragma unroll
    for (int p = 0; p < P; p++) {
        if (j.g) words_of<TA, false>(g[p], j.g, j.gate_f32, gate_at + at[p].col, at[p].n);
        if (AHEAD) parameters(p, j.w1, j.b1);
    }
    auto affine = [&](float (&x)[N], int p, const void *weight, const void *bias) {
        const int q = AHEAD ? p : 0;
        if (!AHEAD) parameters(p, weight, bias);
        float f[N];
        if (weight) {
            values_of<TA>(f, w[q], j.par_f32);
#pragma unroll
            for (int i = 0; i < N; i++) x[i] *= f[i];
        }
        if constexpr (FULL) {
            if (bias) {
                values_of<TA>(f, b[q], j.par_f32);
#pragma unroll
                for (int i = 0; i < N; i++) x[i] += f[i];
            }
        }
    };
    // Mean (layer) and reciprocal deviation of the row in x.
    auto deviation = [&](const float (&x)[P][N], int kind, float eps, float &mean) {
        float s[1] = {0.f};
        mean = 0.f;
        if (FULL && kind == SPIKY_NORM_LAYER) {
#pragma unroll
            for (int p = 0; p < P; p++)
#pragma unroll
                for (int i = 0; i < N; i++) s[0] += where(at[p].own, i, x[p][i]);
            row_sums<TPR, 1>(s, red, turn, waves);
            mean = s[0] * j.inv_cols;
            s[0] = 0.f;
        }
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int i = 0; i < N; i++) {
                const float d = where(at[p].own, i, x[p][i] - mean);
                s[0] += d * d;
            }
        row_sums<TPR, 1>(s, red, turn, waves);
        return rsqrtf(s[0] * j.inv_cols + eps);
    };

    float z[P][N];
    float4 st = {0.f, 1.f, 0.f, 1.f};
    const uint64_t row_at = (uint64_t)row * j.cols;
    if (j.a) {
        float v[P][N];
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int i = 0; i < N; i++) v[p][i] = a_raw[p][i];
        if (j.post != SPIKY_NORM_NONE) {
            st.y = deviation(v, j.post, j.post_eps, st.x);
#pragma unroll
            for (int p = 0; p < P; p++)
#pragma unroll
                for (int i = 0; i < N; i++) v[p][i] = (v[p][i] - st.x) * st.y;
        }
        const Dropper dr = dropper(j.drop);
#pragma unroll
        for (int p = 0; p < P; p++) {
            float f[N];
            affine(v[p], p, j.w1, j.b1);
            if (j.drops) drop(v[p], dr, row, at[p].col);
#pragma unroll
            for (int i = 0; i < N; i++) f[i] = 1.f;
            if (j.g) values_of<TA>(f, g[p], j.gate_f32);
#pragma unroll
            for (int i = 0; i < N; i++) z[p][i] = j.alpha * z_raw[p][i] + j.beta * (f[i] * v[p][i]);
        }
    } else {
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int i = 0; i < N; i++) z[p][i] = z_raw[p][i];
    }
    if (AHEAD && j.pre != SPIKY_NORM_NONE)
#pragma unroll
        for (int p = 0; p < P; p++) parameters(p, j.w2, j.b2);
    if (j.a)
#pragma unroll
        for (int p = 0; p < P; p++) store_piece<false>(j.out + row_at + at[p].col, z[p], at[p].n);
    if (j.pre != SPIKY_NORM_NONE) {
        st.w = deviation(z, j.pre, j.pre_eps, st.z);
#pragma unroll
        for (int p = 0; p < P; p++) {
#pragma unroll
            for (int i = 0; i < N; i++) z[p][i] = (z[p][i] - st.z) * st.w;
            affine(z[p], p, j.w2, j.b2);
            store_piece<false>(j.normed + row_at + at[p].col, z[p], at[p].n);
        }
    }
    if (j.stats && lane == 0) j.stats[row] = st;
}

// Rows of any width: a workgroup walks its row once for each sum.
template <typename TZ, typename TA, int N, int WG>
__global__ __launch_bounds__(WG) void k_join_any(Join<TZ, TA> j) {
    __shared__ float4 red[2][1][16];
    uint32_t turn = 0;
    const uint32_t row = j.row0 + blockIdx.x;
    const TZ *r = j.r + (int64_t)row * j.r_stride;
    const TA *a = j.a + (int64_t)row * j.a_stride;
    const Dropper dr = dropper(j.drop);
    const uint32_t gate_row = j.g ? row / j.gate_rows : 0;
    float4 st = {0.f, 1.f, 0.f, 1.f};
    auto sum_of = [&](auto &&piece) {
        float s[1] = {0.f};
        for (uint64_t col = (uint64_t)threadIdx.x * N; col < j.cols; col += WG * N)
            s[0] += piece(col, piece_size(j.cols, col, N));
        row_sums<WG, 1>(s, red, turn, WG / 64);
        return s[0];
    };
    auto deviation = [&](int kind, float eps, float &mean, auto &&read) {
        mean = 0.f;
        if (kind == SPIKY_NORM_LAYER)
            mean = j.inv_cols * sum_of([&](uint64_t col, int n) {
                       float x[N], s = 0.f;
                       read(x, col, n);
#pragma unroll
                       for (int i = 0; i < N; i++) s += i < n ? x[i] : 0.f;
                       return s;
                   });
        const float m = mean;
        return rsqrtf(eps + j.inv_cols * sum_of([&](uint64_t col, int n) {
                                float x[N], s = 0.f;
                                read(x, col, n);
#pragma unroll
                                for (int i = 0; i < N; i++) s += i < n ? (x[i] - m) * (x[i] - m) : 0.f;
                                return s;
                            }));
    };
    if (j.a && j.post != SPIKY_NORM_NONE)
        st.y = deviation(j.post, j.post_eps, st.x, [&](float (&x)[N], uint64_t col, int n) { load(x, a + col, n); });
    auto joined = [&](float (&z)[N], uint64_t col, int n) {
        load(z, r + col, n);
        if (!j.a) return;
        float v[N], g[N];
        load(v, a + col, n);
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = (v[i] - st.x) * st.y;
        affine_drop<TA>(v, j, dr, row, col, n);
        gate_of<TA>(g, j, gate_row, col, n);
#pragma unroll
        for (int i = 0; i < N; i++) z[i] = j.alpha * z[i] + j.beta * (g[i] * v[i]);
    };
    if (j.pre != SPIKY_NORM_NONE) st.w = deviation(j.pre, j.pre_eps, st.z, joined);
    for (uint64_t col = (uint64_t)threadIdx.x * N; col < j.cols; col += WG * N) {
        const int n = piece_size(j.cols, col, N);
        float z[N], w[N], b[N];
        joined(z, col, n);
        if (j.a) store(j.out + (uint64_t)row * j.cols + col, z, n);
        if (j.pre == SPIKY_NORM_NONE) continue;
        if (j.w2) param<TA>(w, j.w2, j.par_f32, col, n);
        if (j.b2) param<TA>(b, j.b2, j.par_f32, col, n);
#pragma unroll
        for (int i = 0; i < N; i++) {
            z[i] = (z[i] - st.z) * st.w;
            if (j.w2) z[i] *= w[i];
            if (j.b2) z[i] += b[i];
        }
        store(j.normed + (uint64_t)row * j.cols + col, z, n);
    }
    if (j.stats && threadIdx.x == 0) j.stats[row] = st;
}

// ---- backward --------------------------------------------------------------
// The rows [row, end) of chunk number `chunk`.
template <typename J>
__device__ __forceinline__ void chunk_rows(const J &j, uint32_t chunk, uint32_t &row, uint32_t &end) {
    if (j.chunks_per_span) {
        const uint32_t first = chunk / j.chunks_per_span * j.span;
        const uint64_t from = (uint64_t)(chunk % j.chunks_per_span) * j.chunk;
        row = first + (uint32_t)min(from, (uint64_t)j.span);
        end = first + (uint32_t)min(from + j.chunk, (uint64_t)j.span);
    } else {
        const uint64_t from = (uint64_t)chunk * j.chunk;
        row = (uint32_t)min(from, (uint64_t)j.rows);
        end = (uint32_t)min(from + j.chunk, (uint64_t)j.rows);
    }
}

// The column sums of a backward pass, numbered as Join::part.
enum { kSumW1, kSumB1, kSumW2, kSumB2, kSumG };

// What a thread has of one piece of N columns on the way back: parameters, the
// loads of the next row, and what the row's sums are awaited with.  FULL: with
// layer norms or biases.  LEAN: w2 and b1 are read again for every row.
template <typename TZ, typename TA, int N, bool FULL, bool SHORT, bool LEAN = false>
struct Piece {
    static constexpr int K = FULL ? 8 : 3;
    Place<N> at;
    float w1[N], w2[LEAN ? 1 : N], b1[FULL && !LEAN ? N : 1], g[N];
    Raw<TZ, N> z_raw, dz_raw;
    Raw<TA, N> a_raw, dh_raw;
    Raw<float, N> g_raw;  // half of the words where the gate is of a shorter type
    float n1[N], n2[N], e[N];
    uint32_t keep;  // bit i: column i is not dropped

    template <typename J>
    __device__ __forceinline__ void place(const J &j, uint64_t column) {
        at.set(j.cols, column);
        z_raw.clear(), dz_raw.clear(), a_raw.clear(), dh_raw.clear(), g_raw.clear();
    }
    template <typename J>
    __device__ __forceinline__ void parameter(float (&v)[N], const J &j, const void *p, bool there, float absent) const {
        if (there) {
            Raw<float, N> raw;
            raw.clear();
            words_of<TA, SHORT>(raw, p, j.par_f32, at.col, at.n);
            values_of<TA>(v, raw, j.par_f32);
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) v[i] = absent;
        }
    }
    template <typename J>
    __device__ __forceinline__ void parameters(const J &j) {
        parameter(w1, j, j.w1, j.has & kW1, 1.f);
        if constexpr (!LEAN) parameter(w2, j, j.w2, j.has & kW2, 1.f);
        if constexpr (FULL && !LEAN) parameter(b1, j, j.b1, j.has & kB1, 0.f);
#pragma unroll
        for (int i = 0; i < N; i++)
            if (!(j.has & kGate)) g[i] = 1.f;
    }
    template <typename J>
    __device__ __forceinline__ void load_gate(const J &j, uint32_t gate_row) {
        words_of<TA, SHORT>(g_raw, j.g, j.gate_f32, (uint64_t)gate_row * j.cols + at.col, at.n);
    }
    template <typename J>
    __device__ __forceinline__ void take_gate(const J &j) {
        values_of<TA>(g, g_raw, j.gate_f32);
    }
    template <typename J>
    __device__ __forceinline__ void fetch(const J &j, uint32_t row, bool row_gates) {
        const uint32_t has = here(j.has);
        if (has & kDz) fetch_piece<SHORT>(dz_raw, j.dz + (int64_t)row * j.dz_stride + at.col, at.n);
        if (has & kBranch) fetch_piece<SHORT>(a_raw, j.a + (int64_t)row * j.a_stride + at.col, at.n);
        if (has & kDh) {
            fetch_piece<SHORT>(z_raw, j.r + (int64_t)row * j.r_stride + at.col, at.n);
            fetch_piece<SHORT>(dh_raw, j.dh + (int64_t)row * j.dh_stride + at.col, at.n);
        }
        if (row_gates) load_gate(j, row);
    }
    // v of the forward pass, and then d: a dropped element is 0 whatever it holds.
    __device__ __forceinline__ float dropped(const Dropper &dr, int i, const float (&b)[N]) const {
        float v = n1[i] * w1[i];
        if (FULL) v += b[i];
        return where(keep, i, v * dr.scale);
    }
    // The post norm's bias, and the pre norm's weight, as the row's sums want them.
    template <typename J>
    __device__ __forceinline__ void bias_of(float (&v)[N], const J &j, uint32_t has) const {
        if constexpr (!FULL) return;
        if constexpr (LEAN) {
            parameter(v, j, j.b1, has & kB1, 0.f);
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) v[i] = b1[FULL && !LEAN ? i : 0];
        }
    }
    template <typename J>
    __device__ __forceinline__ void weight_of(float (&v)[N], const J &j, uint32_t has) const {
        if constexpr (LEAN) {
            parameter(v, j, j.w2, has & kW2, 1.f);
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) v[i] = w2[LEAN ? 0 : i];
        }
    }
    // The row's values from its loads, and the piece's share of the row's sums s;
    // add(k, v) adds v to the column sums k.
    template <typename J, typename F>
    __device__ __forceinline__ void consume(const J &j, const Dropper &dr, const float4 &st, uint32_t row,
                                            float (&s)[K], F &&add) {
        const uint32_t has = here(j.has);
        const float r2 = has & kDh ? st.w : 0.f;
        float dw2[N], db2[FULL ? N : 1], b[N], w[N];
        bias_of(b, j, has);
        weight_of(w, j, has);
        const float kept_scale = dr.scale * j.beta;
        keep = has & kDrops ? kept<N>(dr, row, at.col) : ~0u;
        const uint32_t counts = keep & at.own;
#pragma unroll
        for (int i = 0; i < N; i++) {
            n1[i] = (a_raw[i] - st.x) * st.y;
            float z = z_raw[i];
            if (has & kBranch) z = j.alpha * z + j.beta * (g[i] * dropped(dr, i, b));
            n2[i] = has & kDh ? (z - st.z) * r2 : 0.f;
            const float dh = dh_raw[i], t = dh * w[i];
            e[i] = dz_raw[i] + r2 * t;
            dw2[i] = dh * n2[i];
            const float c = where(counts, i, kept_scale * g[i] * w1[i]), own_t = where(at.own, i, t);
            const float ce = where(counts, i, c * e[i]), cn = c * n1[i];
            s[0] += own_t * n2[i];
            s[1] += ce * n1[i];
            s[2] += cn * n2[i];
            if constexpr (FULL) {
                db2[i] = dh;
                s[3] += own_t;
                s[4] += ce;
                s[5] += c;
                s[6] += c * n2[i];
                s[7] += cn;
            }
        }
        if (has & kPart << kSumW2) add(kSumW2, dw2);
        if constexpr (FULL)
            if (has & kPart << kSumB2) add(kSumB2, db2);
    }
    // The row's gradients, from its means (mean t, mean t n2, mean dn, mean dn n1).
    template <typename J, typename F>
    __device__ __forceinline__ void finish(const J &j, const Dropper &dr, const float4 &st, const float4 &m,
                                           uint32_t row, F &&add) {
        const uint32_t has = here(j.has);
        const float kept_scale = dr.scale * j.beta;
        const float r2 = has & kDh ? st.w : 0.f, alpha = has & kBranch ? j.alpha : 1.f;
        const uint64_t to = (uint64_t)row * j.cols + at.col;
        float out[N], da[N], dg[N], dw1[N], db1[N], b[N];
        bias_of(b, j, has);
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float q = e[i] - r2 * (m.x + n2[i] * m.y);
            out[i] = alpha * q;
            dg[i] = j.beta * (dropped(dr, i, b) * q);
            db1[i] = where(keep, i, kept_scale * (g[i] * q));
            dw1[i] = db1[i] * n1[i];
            da[i] = db1[i];
            if (has & kPost) da[i] = st.y * (db1[i] * w1[i] - m.z - n1[i] * m.w);
        }
        if (has & kDr) store_piece<SHORT>(j.dr + to, out, at.n);
        if (has & kDa) store_piece<SHORT>(j.da + to, da, at.n);
        if (has & kRowDgate)
            store_gate(j, row, dg);
        else if (has & (kDgate | kPart << kSumG))
            add(kSumG, dg);
        if (has & kPart << kSumW1) add(kSumW1, dw1);
        if constexpr (FULL)
            if (has & kPart << kSumB1) add(kSumB1, db1);
    }
    template <typename J>
    __device__ __forceinline__ void store_gate(const J &j, uint32_t gate_row, const float (&dg)[N]) const {
        const uint64_t to = (uint64_t)gate_row * j.cols + at.col;
        if (sizeof(TA) == 4 || j.gate_f32)
            store_piece<SHORT>(static_cast<float *>(j.dgate) + to, dg, at.n);
        else
            store_piece<SHORT>(static_cast<TA *>(j.dgate) + to, dg, at.n);
    }
};

// A row's means from its sums.  q is linear in the sums of the pre norm, so those
// of the post norm follow from sums that need none of them, and a row has one
// reduction: with c = keep / (1 - p) beta g w1 and e = dz + r2 t,
//   sum dn n1 = sum c n1 e - r2 (mean t sum c n1 + mean(t n2) sum c n1 n2)
// and alike without n1.
template <bool FULL, typename J, int K>
__device__ __forceinline__ float4 row_means(const J &j, const float4 &st, const float (&s)[K]) {
    const uint32_t has = here(j.has);
    const float r2 = has & kDh ? st.w : 0.f;
    float4 m = {0.f, s[0] * j.inv_cols, 0.f, 0.f};
    if (FULL && has & kPreLayer) m.x = s[FULL ? 3 : 0] * j.inv_cols;
    if (has & kPost) {
        m.w = s[1] - r2 * (m.y * s[2]);
        if constexpr (FULL) {
            m.w -= r2 * (m.x * s[7]);
            if (has & kPostLayer) m.z = (s[4] - r2 * (m.x * s[5] + m.y * s[6])) * j.inv_cols;
        }
        m.w *= j.inv_cols;
    }
    return m;
}

// Rows of 8 to 8192 columns: a workgroup walks the rows of its chunk (a slot of TPR
// lanes its share of them), a thread always with the same columns, so every input
// crosses HBM once.  Parameters stay in registers; column sums are in LDS, each
// thread's its own: a read and a write of LDS a row, a tenth of the time that the
// row takes in HBM, for registers that make 3 waves of 2 to a SIMD (33822 rows of
// 640 fp32 with layer norms 234 -> 161 us).  The next row's loads are issued before
// the reduction, into the registers that this row's left.  Above 4096 columns 512
// threads have 16 columns each.  All of these spill: 14 registers with rms norms beside
// fp32, 22 to 37 with layer norms, 86 and 112 for fp32.  1024 threads of 8, which may use
// 128 registers, spilled more when they were compared (8192 rows of 8192 bf16: 370 us
// against 255), before a call's parts were bits and parameters could be read again.  With
// layer norms w2 and b1 are read again for every row (410 -> 341 us).
template <typename TZ, typename TA, int N, int P, int TPR, bool FULL>
__global__ __launch_bounds__(TPR <= 64 ? 256 : TPR) void k_join_back(Join<TZ, TA> j) {
    constexpr int kThreads = TPR <= 64 ? 256 : TPR, kSlots = TPR <= 64 ? 256 / TPR : 1;
    constexpr int W = N * P, K = FULL ? 8 : 3, kQuads = W / 4;
    __shared__ float4 red[TPR > 64 ? 2 : 1][(K + 3) / 4][16];
    // sums of w1, w2, g and, FULL, b1; five of 8192 columns would not fit, so those of b2 stay in registers
    constexpr int kInLds = FULL ? 4 : 3;
    __shared__ float4 acc[kInLds][kQuads][kThreads];
    const uint32_t threads = TPR <= 64 ? TPR : blockDim.x, waves = blockDim.x / 64;
    const uint32_t lane = TPR <= 64 ? threadIdx.x % TPR : threadIdx.x;
    uint32_t row, end, turn = 0;
    chunk_rows(j, blockIdx.x, row, end);
    if (kSlots > 1) {
        uint32_t share = (end - row + kSlots - 1) / kSlots;
        if (!j.chunks_per_span) share = (share + j.span - 1) / j.span * j.span;  // whole spans
        row += min(end - row, threadIdx.x / TPR * share);
        end = row + min(end - row, share);
    }
    if (TPR == 64) row = __builtin_amdgcn_readfirstlane(row), end = __builtin_amdgcn_readfirstlane(end);
    const Dropper dr = dropper(j.drop);  // of scale 1 where nothing is dropped
    const bool row_gates = j.has & kRowGate;
    uint32_t gate_row = j.has & kGate ? row / j.gate_rows : 0, in_gate = j.has & kGate ? row - gate_row * j.gate_rows : 0;

    auto slot_of = [](int k) { return k == kSumW1 ? 0 : k == kSumW2 ? 1 : k == kSumG ? 2 : 3; };
    float acc_b2[P][N];
    Piece<TZ, TA, N, FULL, false, FULL && (N * P > 8)> x[P];
    float4 st = {0.f, 1.f, 0.f, 1.f};
#pragma unroll
    for (int p = 0; p < P; p++) {
        x[p].place(j, (uint64_t)(p * threads + lane) * N);
        if (row < end) x[p].fetch(j, row, row_gates);
    }
    if (row < end) st = j.stats[row];
#pragma unroll
    for (int k = 0; k < kInLds; k++)
#pragma unroll
        for (int q = 0; q < kQuads; q++) acc[k][q][threadIdx.x] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int p = 0; p < P; p++) {
        x[p].parameters(j);
        if (j.has & kGate && !row_gates && row < end) x[p].load_gate(j, gate_row), x[p].take_gate(j);
#pragma unroll
        for (int i = 0; i < N; i++) acc_b2[p][i] = 0.f;
    }

    for (; row < end; row++) {
        float s[K];
#pragma unroll
        for (int k = 0; k < K; k++) s[k] = 0.f;
        const float4 now = st;
        auto adds_to = [&](int p) {
            return [&acc_b2, slot_of, p](int k, const float (&v)[N]) {
                if (FULL && k == kSumB2) {
#pragma unroll
                    for (int i = 0; i < N; i++) acc_b2[p][i] += v[i];
                    return;
                }
#pragma unroll
                for (int i = 0; i < N; i += 4) {
                    float4 &f = acc[slot_of(k)][(p * N + i) / 4][threadIdx.x];
                    float4 t = f;
                    t.x += v[i], t.y += v[i + 1], t.z += v[i + 2], t.w += v[i + 3];
                    f = t;
                }
            };
        };
#pragma unroll
        for (int p = 0; p < P; p++) {
            if (row_gates) x[p].take_gate(j);
            x[p].consume(j, dr, now, row, s, adds_to(p));
        }
        if (row + 1 < end) {
            st = j.stats[row + 1];
#pragma unroll
            for (int p = 0; p < P; p++) x[p].fetch(j, row + 1, row_gates);
        }
        row_sums<TPR, K>(s, red, turn, waves);
        const float4 m = row_means<FULL>(j, now, s);
#pragma unroll
        for (int p = 0; p < P; p++) x[p].finish(j, dr, now, m, row, adds_to(p));
        if (j.has & kGate && !row_gates && ++in_gate == j.gate_rows) {
            // the rows of a gate end here, and with them its sum, where no other chunk has some of them
#pragma unroll
            for (int p = 0; p < P; p++) {
                if (j.has & kDgate) {
                    float dg[N];
#pragma unroll
                    for (int i = 0; i < N; i += 4) {
                        float4 &f = acc[2][(p * N + i) / 4][threadIdx.x];
                        dg[i] = f.x, dg[i + 1] = f.y, dg[i + 2] = f.z, dg[i + 3] = f.w;
                        f = make_float4(0.f, 0.f, 0.f, 0.f);
                    }
                    x[p].store_gate(j, gate_row, dg);
                }
                if (row + 1 < end) x[p].load_gate(j, gate_row + 1), x[p].take_gate(j);
            }
            in_gate = 0;
            gate_row++;
        }
    }

    auto write_sums = [&](int k, const float4 (*sums)[kThreads]) {
        float *part = j.part[k] + (uint64_t)blockIdx.x * j.cols;
        if constexpr (kSlots == 1) {
#pragma unroll
            for (int p = 0; p < P; p++) {
                float v[N];
#pragma unroll
                for (int i = 0; i < N; i += 4) {
                    const float4 f = sums[(p * N + i) / 4][threadIdx.x];
                    v[i] = f.x, v[i + 1] = f.y, v[i + 2] = f.z, v[i + 3] = f.w;
                }
                store_piece<false>(part + x[p].at.col, v, x[p].at.n);
            }
        } else {
            const uint32_t cols = (uint32_t)j.cols, last = (cols - 1) / N;
            for (uint32_t c = threadIdx.x; c < cols; c += 256) {
                const uint32_t piece = c / N;
                const uint32_t i = piece < last ? c % N : c - (cols - N);
                const uint32_t q = (piece / TPR * N + i) / 4, l = piece % TPR;
                float v = 0.f;
#pragma unroll
                for (int slot = 0; slot < kSlots; slot++)
                    v += reinterpret_cast<const float *>(&sums[q][slot * TPR + l])[i % 4];
                part[c] = v;
            }
        }
    };
    if (kSlots > 1) __syncthreads();
    if (j.has & kPart << kSumW1) write_sums(kSumW1, acc[0]);
    if (j.has & kPart << kSumW2) write_sums(kSumW2, acc[1]);
    if (j.has & kPart << kSumG) write_sums(kSumG, acc[2]);
    if constexpr (FULL) {
        if (j.has & kPart << kSumB1) write_sums(kSumB1, acc[3]);
        if (j.has & kPart << kSumB2) {
            if (kSlots > 1) __syncthreads();
#pragma unroll
            for (int p = 0; p < P; p++)
#pragma unroll
                for (int i = 0; i < N; i += 4)
                    acc[0][(p * N + i) / 4][threadIdx.x] =
                        make_float4(acc_b2[p][i], acc_b2[p][i + 1], acc_b2[p][i + 2], acc_b2[p][i + 3]);
            if (kSlots > 1) __syncthreads();
            write_sums(kSumB2, acc[0]);
        }
    }
}

// Wider rows, and those narrower than a piece, take two passes over the inputs: the
// means of each row, then columns.  1392 rows of 10700 fp16: 32 and 40 us, for 41 of
// HBM in one pass.  A thread's registers do not hold such a row's inputs and sums; a row
// of 2-byte elements in LDS, its column sums in registers, would fit to 16384 columns and
// has not been built.
template <typename TZ, typename TA, int N, int WG, bool FULL>
__global__ __launch_bounds__(WG) void k_join_back_rows(Join<TZ, TA> j) {
    constexpr int K = FULL ? 8 : 3;
    __shared__ float4 red[2][(K + 3) / 4][16];
    const uint32_t row = j.row0 + blockIdx.x;
    const Dropper dr = dropper(j.drop);
    const float4 st = j.stats[row];
    float s[K];
#pragma unroll
    for (int k = 0; k < K; k++) s[k] = 0.f;
    for (uint64_t col = (uint64_t)threadIdx.x * N; col < j.cols; col += WG * N) {
        Piece<TZ, TA, N, FULL, true> x;
        x.place(j, col);
        x.fetch(j, row, false);
        x.parameters(j);
        if (j.has & kGate) x.load_gate(j, row / j.gate_rows), x.take_gate(j);
        x.consume(j, dr, st, row, s, [](int, auto &) {});
    }
    uint32_t turn = 0;
    row_sums<WG, K>(s, red, turn, WG / 64);
    if (threadIdx.x == 0) j.row_sums[row] = row_means<FULL>(j, st, s);
}

// The gradients, and the sums over the rows of a chunk for N columns a thread.
template <typename TZ, typename TA, int N, bool FULL>
__global__ __launch_bounds__(64) void k_join_back_cols(Join<TZ, TA> j) {
    constexpr int K = FULL ? 8 : 3;
    Piece<TZ, TA, N, FULL, true> x;
    x.place(j, ((uint64_t)blockIdx.x * 64 + threadIdx.x) * N);
    if (x.at.n == 0) return;
    uint32_t row, end;
    chunk_rows(j, blockIdx.y, row, end);
    if (row >= end) return;
    const Dropper dr = dropper(j.drop);  // of scale 1 where nothing is dropped
    const bool row_gates = j.has & kRowGate;
    uint32_t gate_row = j.has & kGate ? row / j.gate_rows : 0, in_gate = j.has & kGate ? row - gate_row * j.gate_rows : 0;
    float acc[5][N], s[K];
#pragma unroll
    for (int k = 0; k < 5; k++)
#pragma unroll
        for (int i = 0; i < N; i++) acc[k][i] = 0.f;
    x.fetch(j, row, row_gates);
    float4 st = j.stats[row], m = j.row_sums[row];
    x.parameters(j);
    if (j.has & kGate && !row_gates) x.load_gate(j, gate_row), x.take_gate(j);
    auto add = [&](int k, const float (&v)[N]) {
#pragma unroll
        for (int i = 0; i < N; i++) acc[k][i] += v[i];
    };
    for (; row < end; row++) {
        const float4 now = st, means = m;
#pragma unroll
        for (int k = 0; k < K; k++) s[k] = 0.f;
        if (row_gates) x.take_gate(j);
        x.consume(j, dr, now, row, s, add);
        if (row + 1 < end) {
            st = j.stats[row + 1], m = j.row_sums[row + 1];
            x.fetch(j, row + 1, row_gates);
        }
        x.finish(j, dr, now, means, row, add);
        if (j.has & kGate && !row_gates && ++in_gate == j.gate_rows) {
            if (j.has & kDgate) {
                x.store_gate(j, gate_row, acc[kSumG]);
#pragma unroll
                for (int i = 0; i < N; i++) acc[kSumG][i] = 0.f;
            }
            if (row + 1 < end) x.load_gate(j, gate_row + 1), x.take_gate(j);
            in_gate = 0;
            gate_row++;
        }
    }
#pragma unroll
    for (int k = 0; k < 5; k++)
        if (j.part[k]) store(j.part[k] + (uint64_t)blockIdx.y * j.cols + x.at.col, acc[k], x.at.n);
}

// Column sums of the chunks' rows, in one order: out[g][c] = the sum of the
// `count` rows of part from g * count on.
struct Sums {
    const float *part[5];
    void *out[5];
    bool f32[5];
    uint32_t count[5], groups[5];  // groups: 0 where there is no sum
};

// A workgroup takes 32 columns, its thread (k, c) every 32nd row from k on.
template <typename TA>
__global__ __launch_bounds__(1024) void k_join_sums(Sums s, uint64_t cols) {
    __shared__ float lds[32][33];
    // blockIdx.y counts through the groups of all sums
    uint32_t group = blockIdx.y;
    int k = 0;
    while (group >= s.groups[k]) group -= s.groups[k++];
    const uint32_t c = threadIdx.x & 31, first = threadIdx.x / 32, count = s.count[k];
    const uint64_t col = (uint64_t)blockIdx.x * 32 + c;
    const float *p = s.part[k] + (uint64_t)group * count * cols + col;
    float sum = 0.f;
    if (col < cols)
#pragma unroll 8
        for (uint32_t r = first; r < count; r += 32) sum += p[(uint64_t)r * cols];
    lds[first][c] = sum;
    __syncthreads();
    // row `first` of the transposed sums: its 32 lanes hold one column's
    sum = lanes_sum<32>(lds[c][first]);
    const uint64_t to = (uint64_t)blockIdx.x * 32 + first;
    if (c != 0 || to >= cols) return;
    const uint64_t at = (uint64_t)group * cols + to;
    if (s.f32[k])
        static_cast<float *>(s.out[k])[at] = sum;
    else
        static_cast<TA *>(s.out[k])[at] = from_f32<TA>(sum);
}

// ---- host ------------------------------------------------------------------
template <typename TZ, typename TA>
Join<TZ, TA> view(const spiky_lm_residual_args &a, const DropArgs &drop) {
    Join<TZ, TA> j = {};
    j.r = static_cast<const TZ *>(a.residual);
    j.a = static_cast<const TA *>(a.branch);
    j.r_stride = a.residual_stride;
    j.a_stride = a.branch_stride;
    j.w1 = a.post_weight;
    j.b1 = a.post_bias;
    j.g = a.gate;
    j.w2 = a.pre_weight;
    j.b2 = a.pre_bias;
    j.par_f32 = a.par_f32 != 0;
    j.gate_f32 = a.gate_f32 != 0;
    j.post = a.post_norm;
    j.pre = a.pre_norm;
    j.post_eps = (float)a.post_eps;
    j.pre_eps = (float)a.pre_eps;
    j.alpha = (float)a.residual_scale;
    j.beta = (float)a.branch_scale;
    j.inv_cols = (float)(1.0 / (double)a.cols);
    j.drops = a.branch && a.dropout_p > 0.0;
    j.drop = drop;
    if (!j.drops) j.drop.scale = 1.f;
    j.rows = (uint32_t)a.rows;
    j.gate_rows = a.gate ? (uint32_t)a.gate_rows : (uint32_t)a.rows;
    j.cols = a.cols;
    j.stats = reinterpret_cast<float4 *>(a.stats);
    return j;
}

// A workgroup of `threads` to every `kRows` rows, in launches of fewer than 2^32 threads.
template <typename J, typename F>
hipError_t over_rows(J &j, uint32_t kRows, uint32_t threads, F &&launch) {
    const uint64_t most = (uint64_t)(0xffffffffu / threads) * kRows;
    for (uint64_t row0 = 0; row0 < j.rows; row0 += most) {
        const uint64_t n = j.rows - row0 < most ? j.rows - row0 : most;
        j.row0 = (uint32_t)row0;
        launch(dim3((uint32_t)((n + kRows - 1) / kRows)), dim3(threads));
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return err;
    }
    return hipSuccess;
}

// W columns a thread.  Rows of up to 1024 columns have a wave, which needs no
// barrier: 33822 rows of 640 fp32 take 85 us against 118 in workgroups of 160
// threads, 14400 of 646 fp16 38 against 42.  Narrower ones have as few lanes as hold
// them (262144 rows of 64 bf16 beside fp32 with 8 lanes 38 us forward, 68 backward,
// with 16 54 and 94).
template <typename TZ, typename TA, int W, int TPR, bool FULL>
hipError_t run_rows(Join<TZ, TA> &j, hipStream_t st) {
    constexpr int N = sizeof(TA) == 4 ? 4 : 8;
    const uint32_t threads = TPR <= 64 ? 256 : (uint32_t)((j.cols + W - 1) / W + 63) & ~63u;
    return over_rows(j, TPR <= 64 ? 256 / TPR : 1, threads, [&](dim3 grid, dim3 block) {
        k_join<TZ, TA, N, W / N, TPR, FULL><<<grid, block, 0, st>>>(j);
    });
}

template <typename TZ, typename TA, bool FULL>
hipError_t run_forward(Join<TZ, TA> &j, hipStream_t st) {
    constexpr int N = sizeof(TA) == 4 ? 4 : 8;
    if (j.cols < 8)  // narrower than a piece
        return over_rows(j, 1, 64, [&](dim3 grid, dim3 block) { k_join_any<TZ, TA, N, 64><<<grid, block, 0, st>>>(j); });
    if (j.cols <= 64) return run_rows<TZ, TA, 8, 8, FULL>(j, st);
    if (j.cols <= 128) return run_rows<TZ, TA, 8, 16, FULL>(j, st);
    if (j.cols <= 256) return run_rows<TZ, TA, 8, 32, FULL>(j, st);
    if (j.cols <= 512) return run_rows<TZ, TA, 8, 64, FULL>(j, st);
    if (j.cols <= 1024) return run_rows<TZ, TA, 16, 64, FULL>(j, st);
    if (j.cols <= 2048) return run_rows<TZ, TA, 8, 256, FULL>(j, st);
    if (j.cols <= 4096) return run_rows<TZ, TA, 8, 512, FULL>(j, st);
    if (j.cols <= 8192) return run_rows<TZ, TA, 8, 1024, FULL>(j, st);
    if (j.cols <= 16384) return run_rows<TZ, TA, 16, 1024, FULL>(j, st);
    return over_rows(j, 1, 1024, [&](dim3 grid, dim3 block) { k_join_any<TZ, TA, N, 1024><<<grid, block, 0, st>>>(j); });
}

bool is_full(const spiky_lm_residual_args &a) {
    return a.post_norm == SPIKY_NORM_LAYER || a.pre_norm == SPIKY_NORM_LAYER || a.post_bias || a.pre_bias;
}

template <typename TZ, typename TA>
hipError_t forward(const spiky_lm_residual_args &a, const DropArgs &drop, void *out, void *normed,
                   hipStream_t st) {
    Join<TZ, TA> j = view<TZ, TA>(a, drop);
    j.out = static_cast<TZ *>(out);
    j.normed = static_cast<TA *>(normed);
    return is_full(a) ? run_forward<TZ, TA, true>(j, st) : run_forward<TZ, TA, false>(j, st);
}

// How the rows are cut into chunks, and the workspace's regions.
struct Plan {
    uint32_t tpr;  // lanes of a row in k_join_back, 1024: a workgroup's; 0: the passes for any row
    uint32_t chunk, chunks, span, chunks_per_span;
    bool part[5];
    uint64_t row_sums, parts[5], bytes;
};

// Columns of a thread of k_join_back.
constexpr uint64_t kBackCols = 8;
constexpr uint64_t kLeast = 8;

Plan plan(const spiky_lm_residual_args &a, const spiky_lm_residual_grads &g) {
    Plan p = {};
    const uint64_t threads = (a.cols + kBackCols - 1) / kBackCols;
    p.tpr = threads <= 8 ? 8 : threads <= 16 ? 16 : threads <= 32 ? 32 : threads <= 64 ? 64 : threads <= 1024 ? 1024 : 0;
    if (a.cols < kBackCols) p.tpr = 0;
    const uint64_t span = a.gate && g.d_gate ? a.gate_rows : a.rows;
    const uint64_t slots = p.tpr && p.tpr <= 64 ? 256 / p.tpr : 1;
    const uint64_t waves = p.tpr && p.tpr <= 64 ? 4 : (threads + 63) / 64;
    uint64_t chunk;
    if (p.tpr) {
        // 16 waves to a CU, where each has kLeast rows of its own; at least one workgroup to a CU.  Fewer
        // rows to more workgroups: 1024 rows of 4096 in 512 workgroups 34 us, in 256 27; 8192 rows of 1024
        // with 4 rows to a workgroup 35 and 7.4 for the sums, with 8 35 and 4.5
        const uint64_t most = kCUs * (waves > 8 ? 1 : 16 / waves);
        chunk = (a.rows + most - 1) / most;
        const uint64_t one_each = (a.rows + kCUs - 1) / kCUs, least = kLeast * slots;
        if (chunk < least) chunk = one_each < least ? one_each : least;
        if (chunk < slots) chunk = slots;
    } else {
        chunk = (a.rows + 2 * kCUs - 1) / (2 * kCUs);
        if (chunk < 8) chunk = 8;
    }
    if (span >= chunk) {
        p.chunks_per_span = (uint32_t)((span + chunk - 1) / chunk);
        chunk = (span + p.chunks_per_span - 1) / p.chunks_per_span;
        p.chunks = (uint32_t)(a.rows / span * p.chunks_per_span);
    } else {
        chunk = chunk / span * span;
        p.chunks = (uint32_t)((a.rows + chunk - 1) / chunk);
    }
    p.chunk = (uint32_t)chunk;
    p.span = (uint32_t)span;
    p.part[0] = g.d_post_weight != nullptr;
    p.part[1] = g.d_post_bias != nullptr;
    p.part[2] = g.d_pre_weight != nullptr;
    p.part[3] = g.d_pre_bias != nullptr;
    p.part[4] = g.d_gate != nullptr && p.chunks_per_span > 0;
    p.row_sums = 0;
    uint64_t at = p.tpr ? 0 : (a.rows * sizeof(float4) + 255) & ~255ull;
    for (int k = 0; k < 5; k++) {
        p.parts[k] = at;
        if (p.part[k]) at += ((uint64_t)p.chunks * a.cols * sizeof(float) + 255) & ~255ull;
    }
    p.bytes = at;
    return p;
}

template <typename TZ, typename TA, bool FULL>
hipError_t run_back(Join<TZ, TA> &j, const Plan &p, hipStream_t st) {
    constexpr int N = sizeof(TA) == 4 ? 4 : 8, P = kBackCols / N;
    if (!p.tpr) {
        const hipError_t err = over_rows(j, 1, 512, [&](dim3 grid, dim3 block) {
            k_join_back_rows<TZ, TA, N, 512, FULL><<<grid, block, 0, st>>>(j);
        });
        if (err != hipSuccess) return err;
        const uint64_t tiles = (j.cols + 64 * N - 1) / (64 * N);
        // fewer than 2048 chunks, in y
        k_join_back_cols<TZ, TA, N, FULL><<<dim3((uint32_t)tiles, p.chunks), dim3(64), 0, st>>>(j);
        return hipGetLastError();
    }
    const dim3 grid(p.chunks);
    const uint32_t threads = (uint32_t)((j.cols + kBackCols - 1) / kBackCols + 63) & ~63u;
    if (p.tpr == 8)
        k_join_back<TZ, TA, N, P, 8, FULL><<<grid, dim3(256), 0, st>>>(j);
    else if (p.tpr == 16)
        k_join_back<TZ, TA, N, P, 16, FULL><<<grid, dim3(256), 0, st>>>(j);
    else if (p.tpr == 32)
        k_join_back<TZ, TA, N, P, 32, FULL><<<grid, dim3(256), 0, st>>>(j);
    else if (p.tpr == 64)
        k_join_back<TZ, TA, N, P, 64, FULL><<<grid, dim3(256), 0, st>>>(j);
    else if (threads <= 128)
        k_join_back<TZ, TA, N, P, 128, FULL><<<grid, dim3(threads), 0, st>>>(j);
    else if (threads <= 256)
        k_join_back<TZ, TA, N, P, 256, FULL><<<grid, dim3(threads), 0, st>>>(j);
    else if (threads <= 512)
        k_join_back<TZ, TA, N, P, 512, FULL><<<grid, dim3(threads), 0, st>>>(j);
    else
        k_join_back<TZ, TA, N, 2 * P, 512, FULL><<<grid, dim3((threads / 2 + 63) & ~63u), 0, st>>>(j);
    return hipGetLastError();
}

template <typename TZ, typename TA>
hipError_t backward(const spiky_lm_residual_args &a, const DropArgs &drop, const spiky_lm_residual_grads &g,
                    hipStream_t st) {
    const Plan p = plan(a, g);
    Join<TZ, TA> j = view<TZ, TA>(a, drop);
    char *ws = static_cast<char *>(g.workspace);
    j.dz = static_cast<const TZ *>(g.d_out);
    j.dh = static_cast<const TA *>(g.d_normed);
    j.dz_stride = g.d_out_stride;
    j.dh_stride = g.d_normed_stride;
    j.dr = static_cast<TZ *>(g.d_residual);
    j.da = static_cast<TA *>(g.d_branch);
    j.dgate = p.part[4] ? nullptr : g.d_gate;
    j.row_sums = reinterpret_cast<float4 *>(ws + p.row_sums);
    for (int k = 0; k < 5; k++) j.part[k] = p.part[k] ? reinterpret_cast<float *>(ws + p.parts[k]) : nullptr;
    auto bit = [](bool set, uint32_t b) { return set ? b : 0u; };
    j.has = bit(j.a, kBranch) | bit(j.dz, kDz) | bit(j.dh, kDh) | bit(j.drops, kDrops) | bit(j.post, kPost) |
            bit(j.post == SPIKY_NORM_LAYER, kPostLayer) | bit(j.pre == SPIKY_NORM_LAYER, kPreLayer) | bit(j.dr, kDr) |
            bit(j.da, kDa) | bit(j.g, kGate) | bit(j.g && j.gate_rows == 1, kRowGate) | bit(j.dgate, kDgate) |
            bit(j.dgate && j.gate_rows == 1, kRowDgate) | bit(j.w1, kW1) | bit(j.b1, kB1) | bit(j.w2, kW2);
    for (int k = 0; k < 5; k++) j.has |= bit(j.part[k], kPart << k);
    j.chunk = p.chunk;
    j.span = p.span;
    j.chunks_per_span = p.chunks_per_span;
    hipError_t err = is_full(a) ? run_back<TZ, TA, true>(j, p, st) : run_back<TZ, TA, false>(j, p, st);
    if (err != hipSuccess) return err;
    Sums s = {};
    void *outs[5] = {g.d_post_weight, g.d_post_bias, g.d_pre_weight, g.d_pre_bias, g.d_gate};
    uint32_t groups = 0;
    for (int k = 0; k < 5; k++) {
        s.part[k] = j.part[k];
        s.out[k] = outs[k];
        s.f32[k] = k == 4 ? j.gate_f32 : j.par_f32;
        s.count[k] = k == 4 ? p.chunks_per_span : p.chunks;
        s.groups[k] = !s.part[k] ? 0 : k == 4 && p.chunks_per_span ? p.chunks / p.chunks_per_span : 1;
        groups += s.groups[k];
    }
    if (groups == 0) return hipSuccess;
    k_join_sums<TA><<<dim3((uint32_t)((a.cols + 31) / 32), groups), dim3(1024), 0, st>>>(s, a.cols);
    return hipGetLastError();
}

template <typename F>
hipError_t by_type(const spiky_lm_residual_args &a, F &&f) {
    if (a.act_dtype == SPIKY_F32) return f(float{}, float{});
    if (a.act_dtype == SPIKY_BF16) return a.res_dtype == SPIKY_F32 ? f(float{}, bf16{}) : f(bf16{}, bf16{});
    return a.res_dtype == SPIKY_F32 ? f(float{}, f16{}) : f(f16{}, f16{});
}

}  // namespace

hipError_t launch_residual_norm(const spiky_lm_residual_args &a, const DropArgs &drop, void *out, void *normed,
                                hipStream_t st) {
    return by_type(a, [&](auto z, auto t) {
        return forward<decltype(z), decltype(t)>(a, drop, out, normed, st);
    });
}

uint64_t residual_norm_workspace(const spiky_lm_residual_args &a, const spiky_lm_residual_grads &g) {
    return plan(a, g).bytes;
}

hipError_t launch_residual_norm_backward(const spiky_lm_residual_args &a, const DropArgs &drop,
                                         const spiky_lm_residual_grads &g, hipStream_t st) {
    return by_type(a, [&](auto z, auto t) {
        return backward<decltype(z), decltype(t)>(a, drop, g, st);
    });
}

}  // namespace lm
}  // namespace spiky
