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
#include "lm_kernels.h"

namespace spiky {
namespace lm {
namespace {

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

// Sum over groups of L lanes (16, 32 or 64), in every lane: exchanges inside
// quads, eights and sixteens by DPP, then between rows of 16 and halves.
template <int L>
__device__ __forceinline__ float lanes_sum(float x) {
    x = add_dpp<0xB1>(x);   // quad_perm 1 0 3 2
    x = add_dpp<0x4E>(x);   // quad_perm 2 3 0 1
    x = add_dpp<0x141>(x);  // row_half_mirror
    x = add_dpp<0x140>(x);  // row_mirror
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

// Sums of K values over the TPR threads of a row.  Rows of more than a wave go
// through LDS, two buffers in turn: a buffer is written again only after the
// barrier of the call in between, which its readers have passed.
template <int TPR, int K>
struct RowSum {
    static constexpr int kWaves = TPR / 64;
    float (*lds)[K][16];
    int turn = 0;
    __device__ __forceinline__ void operator()(float (&x)[K]) {
#pragma unroll
        for (int k = 0; k < K; k++) x[k] = lanes_sum<(TPR < 64 ? TPR : 64)>(x[k]);
        if constexpr (TPR > 64) {
            if ((threadIdx.x & 63) == 0)
#pragma unroll
                for (int k = 0; k < K; k++) lds[turn][k][threadIdx.x / 64] = x[k];
            __syncthreads();
#pragma unroll
            for (int k = 0; k < K; k++) {
                float s = 0.f;
#pragma unroll
                for (int w = 0; w < kWaves; w++) s += lds[turn][k][w];
                x[k] = s;
            }
            turn ^= 1;
        }
    }
};

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

// ---- forward ---------------------------------------------------------------
// A row in the registers of TPR threads, P pieces of N columns each: every
// input is read once, the sums of both norms run over registers.
template <typename TZ, typename TA, int N, int P, int TPR>
__global__ __launch_bounds__(TPR < 256 && TPR <= 64 ? 256 : TPR) void k_join(Join<TZ, TA> j) {
    constexpr int kRows = TPR <= 64 ? 256 / TPR : 1;
    __shared__ float red[TPR > 64 ? 2 : 1][1][16];
    RowSum<TPR, 1> row_sum{red};
    const uint32_t lane = threadIdx.x % TPR;
    const uint32_t row = j.row0 + blockIdx.x * kRows + threadIdx.x / TPR;
    if (TPR <= 64 && row >= j.rows) return;
    float z[P][N], v[P][N];
    int n[P];
    const TZ *r = j.r + (int64_t)row * j.r_stride;
    const TA *a = j.a + (int64_t)row * j.a_stride;
#pragma unroll
    for (int p = 0; p < P; p++) {
        const uint64_t col = (uint64_t)(p * TPR + lane) * N;
        n[p] = piece_size(j.cols, col, N);
        load(z[p], r + col, n[p]);
        if (j.a) load(v[p], a + col, n[p]);
    }
    // mean (layer) and reciprocal deviation of the row held in x
    auto deviation = [&](float (&x)[P][N], int kind, float eps, float &mean) {
        float s[1] = {0.f};
        mean = 0.f;
        if (kind == SPIKY_NORM_LAYER) {
#pragma unroll
            for (int p = 0; p < P; p++)
#pragma unroll
                for (int i = 0; i < N; i++) s[0] += x[p][i];
            row_sum(s);
            mean = s[0] * j.inv_cols;
            s[0] = 0.f;
        }
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int i = 0; i < N; i++) {
                const float d = i < n[p] ? x[p][i] - mean : 0.f;
                s[0] += d * d;
            }
        row_sum(s);
        return rsqrtf(s[0] * j.inv_cols + eps);
    };
    float4 st = {0.f, 1.f, 0.f, 1.f};
    if (j.a) {
        if (j.post != SPIKY_NORM_NONE) {
            st.y = deviation(v, j.post, j.post_eps, st.x);
#pragma unroll
            for (int p = 0; p < P; p++)
#pragma unroll
                for (int i = 0; i < N; i++) v[p][i] = (v[p][i] - st.x) * st.y;
        }
        const Dropper dr = dropper(j.drop);
        const uint32_t gate_row = j.g ? row / j.gate_rows : 0;
#pragma unroll
        for (int p = 0; p < P; p++) {
            const uint64_t col = (uint64_t)(p * TPR + lane) * N;
            float g[N];
            affine_drop<TA>(v[p], j, dr, row, col, n[p]);
            gate_of<TA>(g, j, gate_row, col, n[p]);
#pragma unroll
            for (int i = 0; i < N; i++) z[p][i] = j.alpha * z[p][i] + j.beta * (g[i] * v[p][i]);
            store(j.out + (uint64_t)row * j.cols + col, z[p], n[p]);
        }
    }
    if (j.pre != SPIKY_NORM_NONE) {
        // columns past the row's end hold what affine_drop made of zeros
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int i = 0; i < N; i++)
                if (i >= n[p]) z[p][i] = 0.f;
        st.w = deviation(z, j.pre, j.pre_eps, st.z);
#pragma unroll
        for (int p = 0; p < P; p++) {
            const uint64_t col = (uint64_t)(p * TPR + lane) * N;
            float w[N], b[N];
            if (j.w2) param<TA>(w, j.w2, j.par_f32, col, n[p]);
            if (j.b2) param<TA>(b, j.b2, j.par_f32, col, n[p]);
#pragma unroll
            for (int i = 0; i < N; i++) {
                z[p][i] = (z[p][i] - st.z) * st.w;
                if (j.w2) z[p][i] *= w[i];
                if (j.b2) z[p][i] += b[i];
            }
            store(j.normed + (uint64_t)row * j.cols + col, z[p], n[p]);
        }
    }
    if (j.stats && lane == 0) j.stats[row] = st;
}

// Rows of any width: a workgroup walks its row once for each sum.
template <typename TZ, typename TA, int N>
__global__ __launch_bounds__(1024) void k_join_wide(Join<TZ, TA> j) {
    __shared__ float red[2][1][16];
    RowSum<1024, 1> row_sum{red};
    const uint32_t row = j.row0 + blockIdx.x;
    const TZ *r = j.r + (int64_t)row * j.r_stride;
    const TA *a = j.a + (int64_t)row * j.a_stride;
    const Dropper dr = dropper(j.drop);
    const uint32_t gate_row = j.g ? row / j.gate_rows : 0;
    float4 st = {0.f, 1.f, 0.f, 1.f};
    auto sum_of = [&](auto &&piece) {
        float s[1] = {0.f};
        for (uint64_t col = (uint64_t)threadIdx.x * N; col < j.cols; col += 1024 * N)
            s[0] += piece(col, piece_size(j.cols, col, N));
        row_sum(s);
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
    for (uint64_t col = (uint64_t)threadIdx.x * N; col < j.cols; col += 1024 * N) {
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

// Rows of up to 1024 * N * P columns: a workgroup walks the rows of its chunk (a
// slot of TPR lanes its share of them), a thread always with the same columns,
// so parameters and column sums stay in registers and every input crosses HBM
// once.  q is linear in the sums of the pre norm, so those of the post norm
// follow from sums that need none of them, and a row has one reduction: with
// c = keep / (1 - p) beta g w1 and e = dz + r2 t,
//   sum dn n1 = sum c n1 e - r2 (mean t sum c n1 + mean(t n2) sum c n1 n2)
// and alike without n1.  The next row's loads are issued before the reduction,
// into the registers that this row's left.  FULL: with layer norms or biases.
template <typename TZ, typename TA, int N, int P, int TPR, bool FULL>
__global__ __launch_bounds__(TPR <= 64 ? 256 : TPR) void k_join_back(Join<TZ, TA> j) {
    constexpr int kSlots = TPR <= 64 ? 256 / TPR : 1, W = N * P, K = FULL ? 8 : 3;
    __shared__ float4 red[TPR > 64 ? 2 : 1][(K + 3) / 4][16];
    __shared__ float joint[kSlots > 1 ? kSlots : 1][kSlots > 1 ? TPR * W : 1];
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
    const Dropper dr = dropper(j.drop);
    const bool row_gates = j.g && j.gate_rows == 1;
    uint32_t gate_row = j.g ? row / j.gate_rows : 0, in_gate = j.g ? row - gate_row * j.gate_rows : 0;

    uint64_t col[P];
    int n[P];
    float w1[P][N], w2[P][N], b1[FULL ? P : 1][N], g[P][N];
    float acc_w1[P][N], acc_w2[P][N], acc_g[P][N], acc_b1[FULL ? P : 1][N], acc_b2[FULL ? P : 1][N];
    Raw<TZ, N> z_raw[P], dz_raw[P];
    Raw<TA, N> a_raw[P], dh_raw[P];
    Raw<float, N> g_raw[P];  // half of the words where the gate is of a shorter type
    float4 st = {0.f, 1.f, 0.f, 1.f};

    auto gate_words = [&](int p, uint32_t at_row) {
        const uint64_t at = (uint64_t)at_row * j.cols + col[p];
        if (sizeof(TA) == 4 || j.gate_f32) {
            g_raw[p].load(static_cast<const float *>(j.g) + at, n[p]);
        } else {
            Raw<TA, N> half;
            half.load(static_cast<const TA *>(j.g) + at, n[p]);
            __builtin_memcpy(g_raw[p].w, half.w, sizeof(half.w));
        }
    };
    auto gate_values = [&](int p) {
        if (sizeof(TA) == 4 || j.gate_f32) {
#pragma unroll
            for (int i = 0; i < N; i++) g[p][i] = g_raw[p][i];
        } else {
            Raw<TA, N> half;
            __builtin_memcpy(half.w, g_raw[p].w, sizeof(half.w));
#pragma unroll
            for (int i = 0; i < N; i++) g[p][i] = half[i];
        }
    };
    auto fetch = [&](uint32_t r) {
        st = j.stats[r];
#pragma unroll
        for (int p = 0; p < P; p++) {
            if (j.dz) dz_raw[p].load(j.dz + (int64_t)r * j.dz_stride + col[p], n[p]);
            if (j.a) a_raw[p].load(j.a + (int64_t)r * j.a_stride + col[p], n[p]);
            if (j.dh) {
                z_raw[p].load(j.r + (int64_t)r * j.r_stride + col[p], n[p]);
                dh_raw[p].load(j.dh + (int64_t)r * j.dh_stride + col[p], n[p]);
            }
            if (row_gates) gate_words(p, r);
        }
    };
#pragma unroll
    for (int p = 0; p < P; p++) {
        col[p] = (uint64_t)(p * threads + lane) * N;
        n[p] = piece_size(j.cols, col[p], N);
        z_raw[p].clear(), dz_raw[p].clear(), a_raw[p].clear(), dh_raw[p].clear(), g_raw[p].clear();
    }
    if (row < end) fetch(row);
#pragma unroll
    for (int p = 0; p < P; p++) {
        // columns past the row's end have weights of 0, so they add nothing to any sum
        if (j.w1) param<TA>(w1[p], j.w1, j.par_f32, col[p], n[p]);
        if (j.w2) param<TA>(w2[p], j.w2, j.par_f32, col[p], n[p]);
        if (FULL && j.b1) param<TA>(b1[p], j.b1, j.par_f32, col[p], n[p]);
        if (j.g && !row_gates && row < end) gate_words(p, gate_row), gate_values(p);
#pragma unroll
        for (int i = 0; i < N; i++) {
            if (!j.w1) w1[p][i] = i < n[p] ? 1.f : 0.f;
            if (!j.w2) w2[p][i] = 1.f;
            if (FULL && !j.b1) b1[FULL ? p : 0][i] = 0.f;
            if (!j.g) g[p][i] = 1.f;
            acc_w1[p][i] = acc_w2[p][i] = acc_g[p][i] = 0.f;
            if (FULL) acc_b1[FULL ? p : 0][i] = acc_b2[FULL ? p : 0][i] = 0.f;
        }
    }
    const float alpha = j.a ? j.alpha : 1.f;

    for (; row < end; row++) {
        float n1[P][N], n2[P][N], e[P][N], keep[P][N];
        float s[K];
#pragma unroll
        for (int k = 0; k < K; k++) s[k] = 0.f;
        const float r1 = st.y, r2 = j.dh ? st.w : 0.f;
#pragma unroll
        for (int p = 0; p < P; p++) {
            if (row_gates) gate_values(p);
#pragma unroll
            for (int i = 0; i < N; i++) {
                keep[p][i] = 1.f;
                n1[p][i] = (a_raw[p][i] - st.x) * st.y;
            }
            if (j.drops) drop(keep[p], dr, row, col[p]);
#pragma unroll
            for (int i = 0; i < N; i++) {
                float v = n1[p][i] * w1[p][i];
                if (FULL) v += b1[FULL ? p : 0][i];
                const bool kept = keep[p][i] != 0.f;
                v = kept ? v * keep[p][i] : 0.f;  // a dropped element is 0 whatever it holds
                float z = z_raw[p][i];
                if (j.a) z = alpha * z + j.beta * (g[p][i] * v);
                n2[p][i] = j.dh ? (z - st.z) * r2 : 0.f;
                const float dh = dh_raw[p][i], t = dh * w2[p][i];
                e[p][i] = dz_raw[p][i] + r2 * t;
                acc_w2[p][i] += dh * n2[p][i];
                const float c = keep[p][i] * (j.beta * g[p][i]) * w1[p][i];
                const float ce = kept ? c * e[p][i] : 0.f, cn = c * n1[p][i];
                s[0] += t * n2[p][i];
                s[1] += ce * n1[p][i];
                s[2] += cn * n2[p][i];
                if constexpr (FULL) {
                    acc_b2[p][i] += dh;
                    s[3] += t;
                    s[4] += ce;
                    s[5] += c;
                    s[6] += c * n2[p][i];
                    s[7] += cn;
                }
            }
        }
        if (row + 1 < end) fetch(row + 1);
        row_sums<TPR, K>(s, red, turn, waves);
        // means over the row
        float mean_t = 0.f, mean_tn, mean_dn = 0.f, mean_dnn = 0.f;
        mean_tn = s[0] * j.inv_cols;
        if (FULL && j.pre == SPIKY_NORM_LAYER) mean_t = s[FULL ? 3 : 0] * j.inv_cols;
        if (j.post != SPIKY_NORM_NONE) {
            mean_dnn = s[1] - r2 * (mean_tn * s[2]);
            if constexpr (FULL) {
                mean_dnn -= r2 * (mean_t * s[7]);
                if (j.post == SPIKY_NORM_LAYER)
                    mean_dn = (s[4] - r2 * (mean_t * s[5] + mean_tn * s[6])) * j.inv_cols;
            }
            mean_dnn *= j.inv_cols;
        }
        const bool gate_ends = j.dgate && in_gate + 1 == j.gate_rows;
#pragma unroll
        for (int p = 0; p < P; p++) {
            const uint64_t at = (uint64_t)row * j.cols + col[p];
            float out[N], da[N];
#pragma unroll
            for (int i = 0; i < N; i++) {
                const float q = e[p][i] - r2 * (mean_t + n2[p][i] * mean_tn);
                out[i] = alpha * q;
                const bool kept = keep[p][i] != 0.f;
                float v = n1[p][i] * w1[p][i];
                if (FULL) v += b1[FULL ? p : 0][i];
                v = kept ? v * keep[p][i] : 0.f;
                acc_g[p][i] += j.beta * (v * q);
                const float dv = kept ? j.beta * (g[p][i] * q) * keep[p][i] : 0.f;
                acc_w1[p][i] += dv * n1[p][i];
                if (FULL) acc_b1[FULL ? p : 0][i] += dv;
                da[i] = dv;
                if (j.post != SPIKY_NORM_NONE) da[i] = r1 * (dv * w1[p][i] - mean_dn - n1[p][i] * mean_dnn);
            }
            if (j.dr) store(j.dr + at, out, n[p]);
            if (j.da) store(j.da + at, da, n[p]);
            if (gate_ends) {
                const uint64_t to = (uint64_t)gate_row * j.cols + col[p];
                if (sizeof(TA) == 4 || j.gate_f32)
                    store(static_cast<float *>(j.dgate) + to, acc_g[p], n[p]);
                else
                    store(static_cast<TA *>(j.dgate) + to, acc_g[p], n[p]);
#pragma unroll
                for (int i = 0; i < N; i++) acc_g[p][i] = 0.f;
            }
        }
        if (j.g && ++in_gate == j.gate_rows) {
            in_gate = 0;
            gate_row++;
            if (!row_gates && row + 1 < end)
#pragma unroll
                for (int p = 0; p < P; p++) gate_words(p, gate_row), gate_values(p);
        }
    }

    auto column_sums = [&](float *part, float (&acc)[P][N]) {
        if (!part) return;
        part += (uint64_t)blockIdx.x * j.cols;
        if constexpr (kSlots == 1) {
#pragma unroll
            for (int p = 0; p < P; p++) store(part + col[p], acc[p], n[p]);
        } else {
            __syncthreads();
#pragma unroll
            for (int p = 0; p < P; p++)
#pragma unroll
                for (int i = 0; i < N; i++) joint[threadIdx.x / TPR][(p * TPR + lane) * N + i] = acc[p][i];
            __syncthreads();
            for (uint32_t c = threadIdx.x; c < TPR * W && c < j.cols; c += 256) {
                float sum = 0.f;
#pragma unroll
                for (int k = 0; k < kSlots; k++) sum += joint[k][c];
                part[c] = sum;
            }
        }
    };
    column_sums(j.part[0], acc_w1);
    column_sums(j.part[2], acc_w2);
    column_sums(j.part[4], acc_g);
    if constexpr (FULL) {
        column_sums(j.part[1], acc_b1);
        column_sums(j.part[3], acc_b2);
    }
}

// Wider rows take two passes over the inputs: the sums over each row, then
// columns.
//
// What a piece of N columns of one row holds on the way back.
template <typename TZ, typename TA, int N>
struct Piece {
    float dz[N], dh[N], n2[N], t[N];  // t = dh w2
    float n1[N], d[N], g[N], keep[N];

    // Everything that does not depend on sums over the row.
    template <typename J>
    __device__ __forceinline__ void read(const J &j, const Dropper &dr, const float4 &st, uint32_t row,
                                         uint32_t gate_row, uint64_t col, int n) {
        if (j.dz)
            load(dz, j.dz + (int64_t)row * j.dz_stride + col, n);
        else
#pragma unroll
            for (int i = 0; i < N; i++) dz[i] = 0.f;
        if (j.a) {
            load(n1, j.a + (int64_t)row * j.a_stride + col, n);
#pragma unroll
            for (int i = 0; i < N; i++) {
                n1[i] = (n1[i] - st.x) * st.y;
                d[i] = n1[i];
                keep[i] = 1.f;
            }
            if (j.w1) {
                float w[N];
                param<TA>(w, j.w1, j.par_f32, col, n);
#pragma unroll
                for (int i = 0; i < N; i++) d[i] *= w[i];
            }
            if (j.b1) {
                float b[N];
                param<TA>(b, j.b1, j.par_f32, col, n);
#pragma unroll
                for (int i = 0; i < N; i++) d[i] += b[i];
            }
            if (j.drops) {
                drop(keep, dr, row, col);
                // a dropped element is 0 whatever it holds
#pragma unroll
                for (int i = 0; i < N; i++) d[i] = keep[i] != 0.f ? d[i] * keep[i] : 0.f;
            }
            gate_of<TA>(g, j, gate_row, col, n);
        }
        if (j.dh) {
            float z[N], w[N];
            load(dh, j.dh + (int64_t)row * j.dh_stride + col, n);
            load(z, j.r + (int64_t)row * j.r_stride + col, n);
            if (j.a)
#pragma unroll
                for (int i = 0; i < N; i++) z[i] = j.alpha * z[i] + j.beta * (g[i] * d[i]);
            if (j.w2) param<TA>(w, j.w2, j.par_f32, col, n);
#pragma unroll
            for (int i = 0; i < N; i++) {
                n2[i] = i < n ? (z[i] - st.z) * st.w : 0.f;
                t[i] = j.w2 ? dh[i] * w[i] : dh[i];
            }
        }
    }

    // q in place of dz.
    template <typename J>
    __device__ __forceinline__ void through_pre(const J &j, const float4 &st, float mean_t, float mean_tn) {
        if (!j.dh) return;
#pragma unroll
        for (int i = 0; i < N; i++) dz[i] += st.w * (t[i] - mean_t - n2[i] * mean_tn);
    }

    // dv, from q.
    template <typename J>
    __device__ __forceinline__ void through_gate(const J &j, float (&dv)[N]) const {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float x = j.beta * (g[i] * dz[i]);
            dv[i] = !j.drops ? x : keep[i] != 0.f ? x * keep[i] : 0.f;
        }
    }
};

// The sums over each row, and dr.
template <typename TZ, typename TA, int N, int WG>
__global__ __launch_bounds__(WG) void k_join_back_rows(Join<TZ, TA> j) {
    __shared__ float red[2][2][16];
    RowSum<WG, 2> row_sum{red};
    const uint32_t row = j.row0 + blockIdx.x;
    const Dropper dr = dropper(j.drop);
    const uint32_t gate_row = j.g ? row / j.gate_rows : 0;
    const float4 st = j.stats[row];
    float4 sums = {0.f, 0.f, 0.f, 0.f};
    Piece<TZ, TA, N> x;
    if (j.dh) {
        float s[2] = {0.f, 0.f};
        for (uint64_t col = (uint64_t)threadIdx.x * N; col < j.cols; col += WG * N) {
            x.read(j, dr, st, row, gate_row, col, piece_size(j.cols, col, N));
#pragma unroll
            for (int i = 0; i < N; i++) {
                s[0] += x.t[i];
                s[1] += x.t[i] * x.n2[i];
            }
        }
        row_sum(s);
        sums.x = j.pre == SPIKY_NORM_LAYER ? s[0] * j.inv_cols : 0.f;
        sums.y = s[1] * j.inv_cols;
    }
    float s[2] = {0.f, 0.f};
    for (uint64_t col = (uint64_t)threadIdx.x * N; col < j.cols; col += WG * N) {
        const int n = piece_size(j.cols, col, N);
        x.read(j, dr, st, row, gate_row, col, n);
        x.through_pre(j, st, sums.x, sums.y);
        if (j.dr) {
            float d[N];
            const float alpha = j.a ? j.alpha : 1.f;
#pragma unroll
            for (int i = 0; i < N; i++) d[i] = alpha * x.dz[i];
            store(j.dr + (uint64_t)row * j.cols + col, d, n);
        }
        if (j.a && j.post != SPIKY_NORM_NONE) {
            float dv[N], w[N];
            x.through_gate(j, dv);
            if (j.w1) param<TA>(w, j.w1, j.par_f32, col, n);
#pragma unroll
            for (int i = 0; i < N; i++) {
                const float dn = i < n ? (j.w1 ? dv[i] * w[i] : dv[i]) : 0.f;
                s[0] += dn;
                s[1] += dn * x.n1[i];
            }
        }
    }
    if (j.a && j.post != SPIKY_NORM_NONE) {
        row_sum(s);
        sums.z = j.post == SPIKY_NORM_LAYER ? s[0] * j.inv_cols : 0.f;
        sums.w = s[1] * j.inv_cols;
    }
    if (threadIdx.x == 0) j.row_sums[row] = sums;
}

// da, and the sums over the rows of a chunk for N columns a thread.
template <typename TZ, typename TA, int N>
__global__ __launch_bounds__(64) void k_join_back_cols(Join<TZ, TA> j) {
    const uint64_t col = ((uint64_t)blockIdx.x * 64 + threadIdx.x) * N;
    const int n = piece_size(j.cols, col, N);
    if (n == 0) return;
    uint32_t row, end;
    chunk_rows(j, blockIdx.y, row, end);
    const Dropper dr = dropper(j.drop);
    float acc[5][N];
#pragma unroll
    for (int k = 0; k < 5; k++)
#pragma unroll
        for (int i = 0; i < N; i++) acc[k][i] = 0.f;
    Piece<TZ, TA, N> x;
    for (; row < end; row++) {
        const uint32_t gate_row = j.g ? row / j.gate_rows : 0;
        const float4 st = j.stats[row], sums = j.row_sums[row];
        x.read(j, dr, st, row, gate_row, col, n);
        if (j.dh) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                acc[2][i] += x.dh[i] * x.n2[i];
                acc[3][i] += x.dh[i];
            }
        }
        if (!j.a) continue;
        x.through_pre(j, st, sums.x, sums.y);
        float dv[N];
        x.through_gate(j, dv);
        if (j.dgate || j.part[4]) {
            float dg[N];
#pragma unroll
            for (int i = 0; i < N; i++) {
                dg[i] = j.beta * (x.d[i] * x.dz[i]);
                acc[4][i] += dg[i];
            }
            // the rows of a gate end here: its sum is whole, or the gate has one row for each
            if (j.dgate && (row + 1) % j.gate_rows == 0) {
                const uint64_t at = (uint64_t)gate_row * j.cols + col;
                if (j.gate_f32)
                    store(static_cast<float *>(j.dgate) + at, acc[4], n);
                else
                    store(static_cast<TA *>(j.dgate) + at, acc[4], n);
#pragma unroll
                for (int i = 0; i < N; i++) acc[4][i] = 0.f;
            }
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
            acc[0][i] += dv[i] * x.n1[i];
            acc[1][i] += dv[i];
        }
        if (j.da) {
            if (j.post != SPIKY_NORM_NONE) {
                float w[N];
                if (j.w1) param<TA>(w, j.w1, j.par_f32, col, n);
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const float dn = j.w1 ? dv[i] * w[i] : dv[i];
                    dv[i] = st.y * (dn - sums.z - x.n1[i] * sums.w);
                }
            }
            store(j.da + (uint64_t)row * j.cols + col, dv, n);
        }
    }
#pragma unroll
    for (int k = 0; k < 5; k++)
        if (j.part[k]) store(j.part[k] + (uint64_t)blockIdx.y * j.cols + col, acc[k], n);
}

// Column sums of the chunks' rows, in one order: out[g][c] = the sum of the
// `count` rows of part from g * count on.
struct Sums {
    const float *part[5];
    void *out[5];
    bool f32[5];
    uint32_t count[5], groups[5];
};

// A workgroup takes 32 columns, its thread (k, c) every 32nd row from k on.
template <typename TA>
__global__ __launch_bounds__(1024) void k_join_sums(Sums s, uint64_t cols) {
    __shared__ float lds[32][33];
    const int k = blockIdx.z;
    if (!s.part[k] || blockIdx.y >= s.groups[k]) return;
    const uint32_t c = threadIdx.x & 31, first = threadIdx.x / 32, count = s.count[k];
    const uint64_t col = (uint64_t)blockIdx.x * 32 + c;
    const float *p = s.part[k] + (uint64_t)blockIdx.y * count * cols + col;
    float sum = 0.f;
    if (col < cols)
#pragma unroll 8
        for (uint32_t r = first; r < count; r += 32) sum += p[(uint64_t)r * cols];
    lds[first][c] = sum;
    __syncthreads();
    // row `first` of the transposed sums: its 32 lanes hold one column's
    sum = lds[c][first];
    sum = lanes_sum<32>(sum);
    const uint64_t to = (uint64_t)blockIdx.x * 32 + first;
    if (c != 0 || to >= cols) return;
    const uint64_t at = (uint64_t)blockIdx.y * cols + to;
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

template <typename TZ, typename TA, int N, int P, int TPR>
hipError_t run_rows(Join<TZ, TA> &j, hipStream_t st) {
    return over_rows(j, TPR <= 64 ? 256 / TPR : 1, TPR <= 64 ? 256 : TPR, [&](dim3 grid, dim3 block) {
        k_join<TZ, TA, N, P, TPR><<<grid, block, 0, st>>>(j);
    });
}

template <typename TZ, typename TA>
hipError_t forward(const spiky_lm_residual_args &a, const DropArgs &drop, void *out, void *normed,
                   hipStream_t st) {
    constexpr int N = sizeof(TA) == 4 ? 4 : 8;
    Join<TZ, TA> j = view<TZ, TA>(a, drop);
    j.out = static_cast<TZ *>(out);
    j.normed = static_cast<TA *>(normed);
    const uint64_t pieces = (a.cols + N - 1) / N;
    if (pieces <= 16) return run_rows<TZ, TA, N, 1, 16>(j, st);
    if (pieces <= 32) return run_rows<TZ, TA, N, 1, 32>(j, st);
    if (pieces <= 64) return run_rows<TZ, TA, N, 1, 64>(j, st);
    if (pieces <= 128) return run_rows<TZ, TA, N, 1, 128>(j, st);
    if (pieces <= 256) return run_rows<TZ, TA, N, 1, 256>(j, st);
    if (pieces <= 512) return run_rows<TZ, TA, N, 1, 512>(j, st);
    if (pieces <= 1024) return run_rows<TZ, TA, N, 1, 1024>(j, st);
    if (pieces <= 2048) return run_rows<TZ, TA, N, 2, 1024>(j, st);
    return over_rows(j, 1, 1024, [&](dim3 grid, dim3 block) { k_join_wide<TZ, TA, N><<<grid, block, 0, st>>>(j); });
}

// How the rows are cut into chunks, and the workspace's regions.
struct Plan {
    uint32_t tpr;  // lanes of a row in k_join_back, 1024 for all rows of more than 64; 0: the passes for wider rows
    uint32_t chunk, chunks, span, chunks_per_span;
    bool part[5];
    uint64_t row_sums, parts[5], bytes;
};

// Columns of a thread of k_join_back.
constexpr uint64_t kBackCols = 8;

Plan plan(const spiky_lm_residual_args &a, const spiky_lm_residual_grads &g) {
    Plan p = {};
    const uint64_t threads = (a.cols + kBackCols - 1) / kBackCols;
    p.tpr = threads <= 16 ? 16 : threads <= 32 ? 32 : threads <= 64 ? 64 : threads <= 1024 ? 1024 : 0;
    const uint64_t span = a.gate && g.d_gate ? a.gate_rows : a.rows;
    // two workgroups to a CU; one, where that leaves each fewer than two rounds of rows
    const uint64_t slots = p.tpr && p.tpr <= 64 ? 256 / p.tpr : 1;
    const uint64_t most = a.rows >= 4 * kCUs * slots ? 2 * kCUs : kCUs;
    uint64_t chunk = (a.rows + most - 1) / most;
    if (chunk < slots) chunk = slots;
    if (!p.tpr && chunk < 8) chunk = 8;
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
void run_back(const Join<TZ, TA> &j, const Plan &p, hipStream_t st) {
    constexpr int N = sizeof(TA) == 4 ? 4 : 8, P = kBackCols / N;
    const dim3 grid(p.chunks);
    const uint32_t threads = (uint32_t)((j.cols + kBackCols - 1) / kBackCols + 63) & ~63u;
    if (p.tpr == 16)
        k_join_back<TZ, TA, N, P, 16, FULL><<<grid, dim3(256), 0, st>>>(j);
    else if (p.tpr == 32)
        k_join_back<TZ, TA, N, P, 32, FULL><<<grid, dim3(256), 0, st>>>(j);
    else if (p.tpr == 64)
        k_join_back<TZ, TA, N, P, 64, FULL><<<grid, dim3(256), 0, st>>>(j);
    else if (threads <= 256)
        k_join_back<TZ, TA, N, P, 256, FULL><<<grid, dim3(threads), 0, st>>>(j);
    else if (threads <= 512)
        k_join_back<TZ, TA, N, P, 512, FULL><<<grid, dim3(threads), 0, st>>>(j);
    else
        k_join_back<TZ, TA, N, P, 1024, FULL><<<grid, dim3(threads), 0, st>>>(j);
}

template <typename TZ, typename TA>
hipError_t backward(const spiky_lm_residual_args &a, const DropArgs &drop, const spiky_lm_residual_grads &g,
                    hipStream_t st) {
    constexpr int N = sizeof(TA) == 4 ? 4 : 8;
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
    j.chunk = p.chunk;
    j.span = p.span;
    j.chunks_per_span = p.chunks_per_span;
    hipError_t err;
    if (p.tpr) {
        if (a.post_norm == SPIKY_NORM_LAYER || a.pre_norm == SPIKY_NORM_LAYER || a.post_bias || a.pre_bias)
            run_back<TZ, TA, true>(j, p, st);
        else
            run_back<TZ, TA, false>(j, p, st);
    } else {
        err = over_rows(j, 1, 256, [&](dim3 grid, dim3 block) {
            k_join_back_rows<TZ, TA, N, 256><<<grid, block, 0, st>>>(j);
        });
        if (err != hipSuccess) return err;
        const uint64_t tiles = (a.cols + 64 * N - 1) / (64 * N);
        // fewer than 2048 chunks, in y
        k_join_back_cols<TZ, TA, N><<<dim3((uint32_t)tiles, p.chunks), dim3(64), 0, st>>>(j);
    }
    err = hipGetLastError();
    if (err != hipSuccess) return err;
    Sums s = {};
    void *outs[5] = {g.d_post_weight, g.d_post_bias, g.d_pre_weight, g.d_pre_bias, g.d_gate};
    uint32_t groups = 0;
    for (int k = 0; k < 5; k++) {
        s.part[k] = j.part[k];
        s.out[k] = outs[k];
        s.f32[k] = k == 4 ? j.gate_f32 : j.par_f32;
        s.count[k] = k == 4 ? p.chunks_per_span : p.chunks;
        s.groups[k] = k == 4 && p.chunks_per_span ? p.chunks / p.chunks_per_span : 1;
        if (s.part[k] && s.groups[k] > groups) groups = s.groups[k];
    }
    if (groups == 0) return hipSuccess;
    k_join_sums<TA><<<dim3((uint32_t)((a.cols + 31) / 32), groups, 5), dim3(1024), 0, st>>>(s, a.cols);
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
