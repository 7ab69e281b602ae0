// Layer norm over the last dimension, forward and backward (gat_layer_norm,
// gat_layer_norm_backward).
//
//   m = mean(x)   v = mean((x - m)^2)   r = 1 / sqrt(v + eps)   z = (x - m) r
//   y = z w + b
//   h = g w       dx = r (h - mean(h) - z mean(h z))
//   dw = sum over rows of g z            db = sum over rows of g
//
// Bound: memory.  The forward has to read x and write y, the backward to read x
// and g and write dx, so each is one pass: a row is held in registers (as it is
// stored, 16 bytes a vector) between the sums and the output, and the variance is
// the mean of the squared deviations, not a difference of two large sums.
//
// A row belongs to LPR lanes (8 to 64 lanes of a wave, or a whole workgroup of 256
// for rows over 128 vectors) with NV vectors each; the groups walk the rows with
// a stride that is a multiple of 8 rows, so a group's rows all start at the same
// offset from a 16-byte boundary and a lane keeps the same columns: w, b and the
// sums of dw and db stay in registers over the group's rows, also where the row
// length is odd.  The vectors at a row's two ends then hold elements of its neighbours:
// they are loaded whole all the same and those elements set to zero, save in the tensor's
// first and last row, where the vector would reach out of the tensor (10,007 x 1,433 bf16
// forward: 33 -> 24 us against element by element).
//
// dw and db: per-lane float32 sums over the group's rows, added up over the
// workgroup's groups in LDS, one partial row per workgroup; k_norm_columns adds
// those up in a fixed order.  No atomics: the result depends on the shape alone.
//
// Measured: 32,768 x 2,048 bf16 forward 46.5 us (5.8 TB/s), a training step 140 us (537 MB,
// 3.8 TB/s); 400,000 x 64 bf16 forward 17.8 us (5.8 TB/s); 10,007 x 1,433 fp16 forward 21 us
// (2.7 TB/s: one workgroup a row, a row's two exchanges are not covered).  Above 8,192 columns
// the backward's 8 or 16 vectors a lane do not fit its registers (600 to 700 bytes of scratch a
// lane): 4,096 x 16,384 bf16, a training step, 340 us (537 MB, 1.6 TB/s).

#include "gat_seq.h"

namespace {

constexpr int kNormBlock = 256;

struct NormArgs {
    const void* x;
    const void* g;  // backward: the incoming gradient
    void* out;      // forward: y, backward: dx
    const void* w;  // may be null (1)
    const void* b;  // may be null (0)
    float* stats;   // [rows, 2] mean, r; forward: may be null
    float* part;    // backward: [workgroups, 2, cols], may be null
    long long ld_x, ld_g, ld_out;
    int rows, cols;
    float eps;
    int inner_x, inner_g;  // rows 1 .. inner - 1 have a vector's width of the tensor on both sides
    int whole_g, whole_out;  // the tensor's rows have x's offset from a 16-byte boundary
};

// Sums of two values over the LPR lanes that share a row, given to all of them.
// `red`: LDS for LPR = 256, a slot of its own per call of the row loop's parity.
template <int LPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float (*red)[2]) {
    constexpr int W = LPR < kWave ? LPR : kWave;
    a = lanes_sum<W>(a);
    b = lanes_sum<W>(b);
    if constexpr (LPR > kWave) {
        const int wave = threadIdx.x / kWave;
        if (threadIdx.x % kWave == 0) {
            red[wave][0] = a;
            red[wave][1] = b;
        }
        __syncthreads();
        a = b = 0.f;
#pragma unroll
        for (int k = 0; k < LPR / kWave; ++k) {
            a += red[k][0];
            b += red[k][1];
        }
    }
}

// A lane's columns of w or b.  Where the row does not start on a 16-byte boundary they lie
// across the vectors of w: then the workgroup's copy in LDS (LPR <= 64) is read element by
// element instead of memory.
template <typename T, int LPR, int NV>
__device__ __forceinline__ void load_params(typename Vec16<T>::type* out, const void* from, float none,
                                            int phase, int cols, T* lds) {
    constexpr int N = Vec16<T>::N;
    const int lane = threadIdx.x % LPR;
    const T* w = static_cast<const T*>(from);
    if (w == nullptr) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int c = (i * LPR + lane) * N - phase + e;
                out[i][e] = c >= 0 && c < cols ? (T)none : (T)0.f;
            }
        return;
    }
    if constexpr (LPR <= kWave) {
        __syncthreads();
        for (int c = threadIdx.x; c < cols; c += kNormBlock) lds[c] = w[c];
        __syncthreads();
        w = lds;
    }
    const bool whole = LPR > kWave && phase == 0 && phase_of(w) == 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) out[i] = load_vec<T>(w, (i * LPR + lane) * N - phase, cols, whole);
}

// Columns [col0, col0 + N) of a row as one aligned vector where `inner` says that what lies
// around the row's ends is the tensor's too; elements outside the row are zeros.
template <typename T>
__device__ __forceinline__ typename Vec16<T>::type load_cols(const T* row, int col0, int cols,
                                                             bool whole, bool inner) {
    constexpr int N = Vec16<T>::N;
    if (!inner) return load_vec<T>(row, col0, cols, whole);
    typename Vec16<T>::type v{};
    if (col0 < cols && col0 + N > 0) {
        v = *reinterpret_cast<const typename Vec16<T>::type*>(row + col0);
        if (col0 < 0 || col0 + N > cols) {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (col0 + e < 0 || col0 + e >= cols) v[e] = (T)0.f;
        }
    }
    return v;
}

// One vector a lane: six waves a SIMD (32,768 x 2,048 bf16: 48 -> 46.5 us against the five
// that the compiler takes by itself; eight spill, 60 us).
template <typename T, int LPR, int NV>
__global__ __launch_bounds__(kNormBlock, (NV == 1 ? 6 : 1)) void k_norm_fwd(NormArgs p) {
    constexpr int N = Vec16<T>::N;
    constexpr int RPB = kNormBlock / LPR;
    typedef typename Vec16<T>::type V;
    __shared__ float red[4][4][2];
    __shared__ T wl[LPR <= kWave ? LPR * NV * N : 1];
    const int lane = threadIdx.x % LPR;
    const int group = blockIdx.x * RPB + threadIdx.x / LPR;
    const int groups = gridDim.x * RPB;
    const T* x = static_cast<const T*>(p.x);
    const int phase = phase_of(x + (long long)group * p.ld_x);
    constexpr bool AHEAD = NV <= 4;  // the next row's loads fly meanwhile, registers permitting
    V v[NV], next[NV], w[NV], b[NV];
    auto load_row = [&](V* to, long long row) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            to[i] = load_cols<T>(x + row * p.ld_x, (i * LPR + lane) * N - phase, p.cols, true,
                                 row > 0 && row < p.inner_x);
    };
    if (AHEAD && group < p.rows) load_row(next, group);
    load_params<T, LPR, NV>(w, p.w, 1.f, phase, p.cols, wl);
    load_params<T, LPR, NV>(b, p.b, 0.f, phase, p.cols, wl);
    const float inv = 1.f / (float)p.cols;
    int turn = 0;
    // groups of one workgroup leave together where they meet at barriers (LPR = 256)
    for (long long row = group; row < p.rows; row += groups, turn ^= 2) {
        float s = 0.f, unused = 0.f;
        if (!AHEAD) load_row(next, row);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            v[i] = next[i];
#pragma unroll
            for (int e = 0; e < N; ++e) s += (float)v[i][e];
        }
        if (AHEAD && row + groups < p.rows) load_row(next, row + groups);
        row_sum2<LPR>(s, unused, red[turn]);
        // Divided, not times 1 / cols: the product's rounding, which the compiler may also leave
        // out of v - mean, would give rows of one value deviations from their mean, which
        // 1 / sqrt(eps) enlarges (3 columns of 1000: z = 9e-3 for 0).
        const float mean = s / (float)p.cols;
        float q = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int c = (i * LPR + lane) * N - phase + e;
                const float d = (float)v[i][e] - mean;
                q += c >= 0 && c < p.cols ? d * d : 0.f;
            }
        row_sum2<LPR>(q, unused, red[turn + 1]);
        const float r = 1.f / sqrtf(q * inv + p.eps);
        if (p.stats != nullptr && lane == 0) {
            p.stats[2 * row] = mean;
            p.stats[2 * row + 1] = r;
        }
        T* yr = static_cast<T*>(p.out) + row * p.ld_out;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            V y;
#pragma unroll
            for (int e = 0; e < N; ++e)
                y[e] = (T)(((float)v[i][e] - mean) * r * (float)w[i][e] + (float)b[i][e]);
            store_vec<T>(yr, (i * LPR + lane) * N - phase, p.cols, p.whole_out, y);
        }
    }
}

template <typename T, int LPR, int NV>
__global__ __launch_bounds__(kNormBlock) void k_norm_bwd(NormArgs p) {
    constexpr int N = Vec16<T>::N;
    constexpr int RPB = kNormBlock / LPR;
    typedef typename Vec16<T>::type V;
    constexpr int COLS = LPR * NV * N;
    __shared__ float red[4][4][2];
    __shared__ __align__(16) float cs[RPB > 1 ? 2 * COLS : 1];
    const int lane = threadIdx.x % LPR;
    const int group = blockIdx.x * RPB + threadIdx.x / LPR;
    const int groups = gridDim.x * RPB;
    const T* x = static_cast<const T*>(p.x);
    const int phase = phase_of(x + (long long)group * p.ld_x);
    constexpr bool AHEAD = NV <= 2;
    V v[NV], g[NV], vn[NV], gn[NV], w[NV];
    float mean = 0.f, r = 0.f;
    auto load_row = [&](long long row) {
        const T* gr = static_cast<const T*>(p.g) + row * p.ld_g;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c0 = (i * LPR + lane) * N - phase;
            vn[i] = load_cols<T>(x + row * p.ld_x, c0, p.cols, true, row > 0 && row < p.inner_x);
            gn[i] = load_cols<T>(gr, c0, p.cols, p.whole_g, row > 0 && row < p.inner_g);
        }
        mean = p.stats[2 * row];
        r = p.stats[2 * row + 1];
    };
    if (AHEAD && group < p.rows) load_row(group);
    load_params<T, LPR, NV>(w, p.w, 1.f, phase, p.cols, reinterpret_cast<T*>(cs));
    float dw[NV][N] = {}, db[NV][N] = {};
    const float inv = 1.f / (float)p.cols;
    int turn = 0;
    for (long long row = group; row < p.rows; row += groups, turn ^= 1) {
        if (!AHEAD) load_row(row);
        const float m = mean, rs = r;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            v[i] = vn[i];
            g[i] = gn[i];
        }
        if (AHEAD && row + groups < p.rows) load_row(row + groups);
        float sh = 0.f, shz = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < N; ++e) {
                // outside the row g and w are 0, so nothing is added there; d is finite where z
                // of a large mean is not, whose product with 0 would reach the whole row
                const float d = (float)v[i][e] - m;
                const float h = (float)g[i][e] * (float)w[i][e];
                sh += h;
                shz += h * d;
                dw[i][e] += (float)g[i][e] * (d * rs);
                db[i][e] += (float)g[i][e];
            }
        row_sum2<LPR>(sh, shz, red[turn]);
        sh *= inv;
        shz *= rs * inv;
        if (p.out != nullptr) {
            T* dr = static_cast<T*>(p.out) + row * p.ld_out;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                V d;
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const float z = ((float)v[i][e] - m) * rs;
                    d[e] = (T)(rs * ((float)g[i][e] * (float)w[i][e] - sh - z * shz));
                }
                store_vec<T>(dr, (i * LPR + lane) * N - phase, p.cols, p.whole_out, d);
            }
        }
    }
    if (p.part == nullptr) return;
    float* part = p.part + (size_t)blockIdx.x * 2 * p.cols;
    if constexpr (RPB == 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int c = (i * LPR + lane) * N - phase + e;
                if (c < 0 || c >= p.cols) continue;
                part[c] = dw[i][e];
                part[p.cols + c] = db[i][e];
            }
    } else {
        __syncthreads();  // cs held w
        // The groups' columns may be shifted against each other (odd row lengths), so
        // they take turns: group j adds its sums to those of the groups before it.
        for (int j = 0; j < RPB; ++j) {
            if (threadIdx.x / LPR == j) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const int c = (i * LPR + lane) * N - phase + e;
                        if (c < 0 || c >= p.cols) continue;
                        cs[c] = (j == 0 ? 0.f : cs[c]) + dw[i][e];
                        cs[COLS + c] = (j == 0 ? 0.f : cs[COLS + c]) + db[i][e];
                    }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < p.cols; c += kNormBlock) {
            part[c] = cs[c];
            part[p.cols + c] = cs[COLS + c];
        }
    }
}

// out[c] = sum over the partial rows, for the 2 * cols sums (dw, then db); 32 columns
// by 32 strided partial chains a workgroup, joined in LDS in a fixed order.
constexpr int kColsTile = 32;

template <typename T>
__global__ __launch_bounds__(1024) void k_norm_columns(const float* part, int parts, int cols,
                                                       T* dw, T* db) {
    __shared__ float s[32][kColsTile + 1];
    const int c = blockIdx.x * kColsTile + threadIdx.x % kColsTile;
    const int k = threadIdx.x / kColsTile;
    float a = 0.f;
    if (c < 2 * cols) {
#pragma unroll 8
        for (int j = k; j < parts; j += 32) a += part[(size_t)j * 2 * cols + c];
    }
    s[k][threadIdx.x % kColsTile] = a;
    __syncthreads();
    if (k != 0 || c >= 2 * cols) return;
    a = 0.f;
#pragma unroll
    for (int j = 0; j < 32; ++j) a += s[j][threadIdx.x];
    if (c < cols) {
        if (dw != nullptr) dw[c] = (T)a;
    } else if (db != nullptr) {
        db[c - cols] = (T)a;
    }
}

// The lanes and vectors of a row: the fewest lanes that hold it with one vector each,
// then more vectors, then a whole workgroup.  `vecs`: 16-byte vectors that a row of
// any phase may span.
struct NormShape {
    int lpr, nv;
};

inline NormShape norm_shape(int cols, int dtype, bool aligned) {
    const int n = 16 / (int)dtype_size(dtype);
    const int vecs = (cols + (aligned ? 0 : n - 1) + n - 1) / n;
    if (vecs <= 8) return {8, 1};
    if (vecs <= 16) return {16, 1};
    if (vecs <= 32) return {32, 1};
    if (vecs <= 64) return {64, 1};
    if (vecs <= 128) return {64, 2};
    if (vecs <= 256) return {256, 1};
    if (vecs <= 512) return {256, 2};
    if (vecs <= 1024) return {256, 4};
    if (vecs <= 2048) return {256, 8};
    if (vecs <= 4096 && n == 4) return {256, 16};  // registers as for 8 vectors of 8
    return {0, 0};
}

// Workgroups of a launch over `rows` rows: a multiple of 8 row groups in all.
inline int norm_grid(int rows, int lpr, int most) {
    const int rpb = kNormBlock / lpr;
    const int step = rpb >= 8 ? 1 : 8 / rpb;
    long long g = ((long long)rows + rpb - 1) / rpb;
    if (g > most) g = most;
    return (int)((g + step - 1) / step * step);
}

// Workgroups that are resident at once on all 256 CUs, which is what a launch gets at most:
// every group then walks rows to the end, none waits for a second turn (20,000 x 3,001 fp16
// forward: 97 us with 2,048, 81 us so).
template <auto KERNEL>
int resident() {
    static const int n = [] {
        int per_cu = 0;
        const hipError_t e =
            hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, KERNEL, kNormBlock, 0);
        return 256 * (e == hipSuccess && per_cu > 0 ? per_cu : 4);
    }();
    return n;
}

// The backward's workgroups each leave a partial row of 2 * cols sums: at most this many.
constexpr int kNormBwdGrid = 1024;

// `parts`: the backward's workgroups
template <typename T, bool BWD>
hipError_t norm_launch(const NormShape& sh, const NormArgs& a, int* parts, hipStream_t s) {
#define GAT_NORM_CASE(L, V)                                                              \
    if (sh.lpr == L && sh.nv == V) {                                                     \
        if constexpr (BWD) {                                                             \
            *parts = norm_grid(a.rows, L, std::min(resident<k_norm_bwd<T, L, V>>(),      \
                                                   kNormBwdGrid));                       \
            k_norm_bwd<T, L, V><<<*parts, kNormBlock, 0, s>>>(a);                        \
        } else {                                                                         \
            const int grid = norm_grid(a.rows, L, resident<k_norm_fwd<T, L, V>>());      \
            k_norm_fwd<T, L, V><<<grid, kNormBlock, 0, s>>>(a);                          \
        }                                                                                \
        return hipGetLastError();                                                        \
    }
    GAT_NORM_CASE(8, 1)
    GAT_NORM_CASE(16, 1)
    GAT_NORM_CASE(32, 1)
    GAT_NORM_CASE(64, 1)
    GAT_NORM_CASE(64, 2)
    GAT_NORM_CASE(256, 1)
    GAT_NORM_CASE(256, 2)
    GAT_NORM_CASE(256, 4)
    GAT_NORM_CASE(256, 8)
    if constexpr (sizeof(T) == 4) {
        GAT_NORM_CASE(256, 16)
    }
#undef GAT_NORM_CASE
    return hipErrorInvalidValue;
}

template <bool BWD>
hipError_t norm_by_type(const NormShape& sh, const NormArgs& a, int dtype, int* parts, hipStream_t s) {
    if (dtype == GAT_F32) return norm_launch<float, BWD>(sh, a, parts, s);
    if (dtype == GAT_BF16) return norm_launch<bf16, BWD>(sh, a, parts, s);
    return norm_launch<f16, BWD>(sh, a, parts, s);
}

// The tensor's rows lie as x's against the 16-byte boundaries.
inline int lies_as(const void* x, long long ld_x, const void* t, long long ld, int dtype) {
    const uintptr_t z = dtype_size(dtype);
    return ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(t)) & 15) == 0 &&
           ((uintptr_t)(ld_x - ld) * z & 15) == 0;
}

// Rows [1, n) of a tensor have at least a vector's width of it before and behind them.
inline int inner_rows(int rows, long long ld, int whole, int dtype) {
    return whole && ld >= 16 / (int)dtype_size(dtype) ? rows - 1 : 0;
}

inline bool norm_aligned(const void* x, long long ld, int dtype) {
    return (reinterpret_cast<uintptr_t>(x) & 15) == 0 && ((uintptr_t)ld * dtype_size(dtype) & 15) == 0;
}

}  // namespace

extern "C" {

int gat_layer_norm(const void* x, long long ld_x, int rows, int cols, const void* w,
                   const void* b, float eps, void* y, long long ld_y, float* stats, int dtype,
                   void* stream) {
    if (rows < 0 || cols <= 0 || !known_dtype(dtype) || !(eps >= 0.f)) return GAT_EINVAL;
    const NormShape sh = norm_shape(cols, dtype, norm_aligned(x, ld_x, dtype));
    if (sh.lpr == 0) return GAT_EUNSUPPORTED;
    if (rows == 0) return GAT_OK;
    if (x == nullptr || y == nullptr || ld_x < 0 || ld_y < cols || !element_aligned(x, dtype) ||
        !element_aligned(y, dtype))
        return GAT_EINVAL;
    NormArgs a{};
    a.x = x;
    a.out = y;
    a.w = w;
    a.b = b;
    a.stats = stats;
    a.ld_x = ld_x;
    a.ld_out = ld_y;
    a.rows = rows;
    a.cols = cols;
    a.eps = eps;
    a.inner_x = inner_rows(rows, ld_x, 1, dtype);
    a.whole_out = lies_as(x, ld_x, y, ld_y, dtype);
    return status_of(norm_by_type<false>(sh, a, dtype, nullptr, static_cast<hipStream_t>(stream)));
}

int gat_layer_norm_backward_workspace_size(int rows, int cols, int dtype, size_t* bytes) {
    if (rows < 0 || cols <= 0 || !known_dtype(dtype) || bytes == nullptr) return GAT_EINVAL;
    size_t most = 0;  // x's alignment is not known here: the larger of the two
    for (int aligned = 0; aligned < 2; ++aligned) {
        const NormShape sh = norm_shape(cols, dtype, aligned != 0);
        if (sh.lpr == 0) {
            if (aligned) return GAT_EUNSUPPORTED;
            continue;
        }
        most = std::max(most, (size_t)norm_grid(rows, sh.lpr, kNormBwdGrid));
    }
    *bytes = most * 2 * (size_t)cols * sizeof(float);
    return GAT_OK;
}

int gat_layer_norm_backward(const void* g, long long ld_g, const void* x, long long ld_x, int rows,
                            int cols, const void* w, const float* stats, void* dx,
                            long long ld_dx, void* dw, void* db, void* workspace,
                            size_t workspace_bytes, int dtype, void* stream) {
    if (rows < 0 || cols <= 0 || !known_dtype(dtype)) return GAT_EINVAL;
    const NormShape sh = norm_shape(cols, dtype, norm_aligned(x, ld_x, dtype));
    if (sh.lpr == 0) return GAT_EUNSUPPORTED;
    const bool sums = dw != nullptr || db != nullptr;
    int parts = rows > 0 ? norm_grid(rows, sh.lpr, kNormBwdGrid) : 0;
    if (sums && workspace_bytes < (size_t)parts * 2 * cols * sizeof(float)) return GAT_EWORKSPACE;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (rows > 0) {
        if (g == nullptr || x == nullptr || stats == nullptr || ld_x < 0 || ld_g < 0 ||
            (dx != nullptr && (ld_dx < cols || !element_aligned(dx, dtype))) ||
            (sums && workspace == nullptr) || !element_aligned(x, dtype) ||
            !element_aligned(g, dtype))
            return GAT_EINVAL;
        NormArgs a{};
        a.x = x;
        a.g = g;
        a.out = dx;
        a.w = w;
        a.stats = const_cast<float*>(stats);
        a.part = sums ? static_cast<float*>(workspace) : nullptr;
        a.ld_x = ld_x;
        a.ld_g = ld_g;
        a.ld_out = ld_dx;
        a.rows = rows;
        a.cols = cols;
        a.inner_x = inner_rows(rows, ld_x, 1, dtype);
        a.whole_g = lies_as(x, ld_x, g, ld_g, dtype);
        a.inner_g = inner_rows(rows, ld_g, a.whole_g, dtype);
        a.whole_out = dx != nullptr && lies_as(x, ld_x, dx, ld_dx, dtype);
        const hipError_t e = norm_by_type<true>(sh, a, dtype, &parts, s);
        if (e != hipSuccess) return status_of(e);
    }
    if (!sums) return GAT_OK;
    const int grid = (2 * cols + kColsTile - 1) / kColsTile;
    const float* part = static_cast<const float*>(workspace);
    if (dtype == GAT_F32)
        k_norm_columns<float><<<grid, 1024, 0, s>>>(part, parts, cols, static_cast<float*>(dw),
                                                    static_cast<float*>(db));
    else if (dtype == GAT_BF16)
        k_norm_columns<bf16><<<grid, 1024, 0, s>>>(part, parts, cols, static_cast<bf16*>(dw),
                                                   static_cast<bf16*>(db));
    else
        k_norm_columns<f16><<<grid, 1024, 0, s>>>(part, parts, cols, static_cast<f16*>(dw),
                                                  static_cast<f16*>(db));
    return status_of(hipGetLastError());
}

}  // extern "C"
