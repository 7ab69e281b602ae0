// Embedding lookup with a scale, and the gradient of its table (gat_embedding,
// gat_embedding_grad).
//
//   y[t] = scale * w[ids[t]]          dw[v] = scale * sum over t with ids[t] = v of g[t]
//
// Bound: memory.  The lookup reads a row and writes a row per token; the gradient has
// to read g once and write the whole table once.
//
// Gradient: the tokens are sorted by id (stable, so each id's tokens stay in order) and
// each table row is then one sum over its tokens' rows of g, written once, zeros
// included: no atomics and no separate clearing pass, and the result does not depend on
// timing.  An id with many tokens would keep one row's lanes busy long after the rest: the
// sorted order is cut into pieces, the pieces of an id with more tokens than a piece are
// summed by workgroups of their own, and the partial sums are joined in order.
// Sums are float32 and rounded once, after the scale.
//
// Few tokens (few_tokens): one launch instead of the sort's four and more.  A workgroup owns
// kOwnRows table rows, picks their tokens out of all ids in order, and sums as above.
//
// Sort: least significant digit first, 8 bits a pass, over (id, token) pairs; an id that
// takes no gradient (out of range, or the padding id) sorts behind the table as id
// `vocab`.  A pass is two launches: digit counts per workgroup, then every workgroup
// adds up the counts before its own and writes its pairs in order.  The workgroups are
// limited to 256 so that this sum stays short.
//
// Measured, 65,536 tokens of 1,024 bf16 over 50,021 rows: lookup 44 us, sort 20 us (two passes),
// sums 67 us, joins 6 us (474 MB in 136 us, 3.5 TB/s).

#include "gat_seq.h"

namespace {

constexpr int kSortBlock = 1024;
constexpr int kSortWaves = kSortBlock / kWave;
constexpr int kSortMinItems = 1024;
constexpr int kSortMaxBlocks = 256;
constexpr int kMinPiece = 16, kMaxPieces = 2048;
constexpr int kFewTokens = 1024, kOwnRows = 64, kOwnHot = 32;
constexpr long long kMaxTokens = 1ll << 30;
constexpr int kEmbedBlock = 256;

struct Ids {
    const void* ids;
    int is64;
    long long padding;  // an id without a gradient, or -1
    int vocab;
};

__device__ __forceinline__ long long id_at(const Ids& s, long long t) {
    return s.is64 ? static_cast<const long long*>(s.ids)[t]
                  : (long long)static_cast<const int*>(s.ids)[t];
}

__device__ __forceinline__ unsigned key_at(const Ids& s, long long t) {
    const long long id = id_at(s, t);
    return id >= 0 && id < s.vocab && id != s.padding ? (unsigned)id : (unsigned)s.vocab;
}

// ---------------------------------------------------------------------------
// Lookup: LPR lanes per token, 16 bytes a lane and step.
// ---------------------------------------------------------------------------
template <typename T, int LPR>
__global__ __launch_bounds__(kEmbedBlock) void k_embed(Ids s, long long tokens, const T* w,
                                                       long long ld_w, int cols, float scale,
                                                       T* out, long long ld_out, int whole) {
    constexpr int N = Vec16<T>::N;
    constexpr int TPB = kEmbedBlock / LPR;
    const int lane = threadIdx.x % LPR;
    for (long long t = (long long)blockIdx.x * TPB + threadIdx.x / LPR; t < tokens;
         t += (long long)gridDim.x * TPB) {
        const long long id = id_at(s, t);
        const bool in = id >= 0 && id < s.vocab;
        const T* row = w + (in ? id : 0) * ld_w;
        const float f = in ? scale : NAN;  // an id outside the table shows
        T* to = out + t * ld_out;
        for (int c = lane * N; c < cols; c += LPR * N) {
            typename Vec16<T>::type v = load_vec<T>(row, c, in ? cols : 0, whole), y;
#pragma unroll
            for (int e = 0; e < N; ++e) y[e] = (T)((float)v[e] * f);
            store_vec<T>(to, c, cols, whole, y);
        }
    }
}

// ---------------------------------------------------------------------------
// Sort
// ---------------------------------------------------------------------------
template <bool FIRST>
__global__ __launch_bounds__(kSortBlock) void k_sort_count(Ids s, const unsigned* keys, int n,
                                                           int per, int shift, unsigned* counts) {
    __shared__ unsigned h[256];
    if (threadIdx.x < 256) h[threadIdx.x] = 0;
    __syncthreads();
    const int a = blockIdx.x * per, e = a + per < n ? a + per : n;
    for (int i = a + threadIdx.x; i < e; i += kSortBlock) {
        const unsigned k = FIRST ? key_at(s, i) : keys[i];
        atomicAdd(&h[(k >> shift) & 255], 1u);
    }
    __syncthreads();
    if (threadIdx.x < 256) counts[blockIdx.x * 256 + threadIdx.x] = h[threadIdx.x];
}

template <bool FIRST>
__global__ __launch_bounds__(kSortBlock) void k_sort_place(Ids s, const unsigned* keys,
                                                           const unsigned* toks, int n, int per,
                                                           int shift, const unsigned* counts,
                                                           unsigned* keys_out, unsigned* toks_out) {
    __shared__ unsigned base[256], wave_count[kSortWaves][256], sums[2][4][256];
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    {
        // of digit d: its count in the workgroups before this one and in all, by four
        // threads a digit
        const int d = tid % 256, quarter = tid / 256;
        unsigned before = 0, total = 0;
#pragma unroll 8
        for (int b = quarter; b < (int)gridDim.x; b += 4) {
            const unsigned c = counts[b * 256 + d];
            before += b < (int)blockIdx.x ? c : 0;
            total += c;
        }
        sums[0][quarter][d] = before;
        sums[1][quarter][d] = total;
    }
    __syncthreads();
    if (wave == 0) {  // where each digit begins: lane l adds up digits 4 l .. 4 l + 3
        unsigned t[4], all = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int d = 4 * lane + k;
            t[k] = all;
            all += sums[1][0][d] + sums[1][1][d] + sums[1][2][d] + sums[1][3][d];
        }
        unsigned upto = all;
#pragma unroll
        for (int off = 1; off < kWave; off <<= 1) {
            const unsigned v = __shfl_up(upto, off);
            if (lane >= off) upto += v;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int d = 4 * lane + k;
            base[d] = upto - all + t[k] + sums[0][0][d] + sums[0][1][d] + sums[0][2][d] + sums[0][3][d];
        }
    }
    const int a = blockIdx.x * per, e = a + per < n ? a + per : n;
    for (int i0 = a; i0 < e; i0 += kSortBlock) {
#pragma unroll
        for (int k = 0; k < 4; ++k) wave_count[wave][4 * lane + k] = 0;
        __syncthreads();
        const int i = i0 + tid;
        const bool in = i < e;
        const unsigned key = in ? (FIRST ? key_at(s, i) : keys[i]) : 0;
        const unsigned digit = (key >> shift) & 255;
        // the lanes of this wave with the same digit
        unsigned long long same = __ballot(in);
#pragma unroll
        for (int b = 0; b < 8; ++b) {
            const unsigned long long m = __ballot((digit >> b) & 1);
            same &= (digit >> b) & 1 ? m : ~m;
        }
        const unsigned rank = __popcll(same & ((1ull << lane) - 1));
        if (in && rank == 0) wave_count[wave][digit] = __popcll(same);
        __syncthreads();
        if (in) {
            unsigned at = base[digit] + rank;
            for (int k = 0; k < wave; ++k) at += wave_count[k][digit];
            keys_out[at] = key;
            toks_out[at] = FIRST ? (unsigned)i : toks[i];
        }
        __syncthreads();
        if (tid < 256) {
            unsigned c = 0;
#pragma unroll
            for (int k = 0; k < kSortWaves; ++k) c += wave_count[k][tid];
            base[tid] += c;
        }
        __syncthreads();
    }
}

// first[v] = position of the first sorted token with id >= v, for v in [0, vocab].
// A lane writes the ids between its token's and the one before; a wide gap is shared
// by the wave.
__global__ __launch_bounds__(256) void k_sort_firsts(const unsigned* keys, int n, int vocab,
                                                     int* first) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    const int lane = threadIdx.x % kWave;
    int lo = 0, hi = -1;  // first[lo .. hi] = i
    if (i <= n) {
        lo = i > 0 ? (int)keys[i - 1] + 1 : 0;
        hi = i < n ? (int)keys[i] : vocab;
    }
    const bool wide = hi - lo >= 16;
    if (!wide)
        for (int v = lo; v <= hi; ++v) first[v] = i;
    for (unsigned long long m = __ballot(wide); m != 0; m &= m - 1) {
        const int l = __ffsll((long long)m) - 1;
        const int a = __shfl(lo, l), b = __shfl(hi, l), at = __shfl(i, l);
        for (int v = a + lane; v <= b; v += kWave) first[v] = at;
    }
}

// ---------------------------------------------------------------------------
// Sums
// ---------------------------------------------------------------------------

// acc += the rows of g of sorted tokens [a, e), `step` apart, columns [c, c + N)
template <typename T, int U = 8>
__device__ __forceinline__ void add_rows(float (&acc)[Vec16<T>::N], const T* g, long long ld_g,
                                         const unsigned* toks, int a, int e, int step, int c,
                                         int cols, bool whole) {
    constexpr int N = Vec16<T>::N;
    for (int i = a; i < e; i += U * step) {  // U rows in flight, also where fewer are left
        typename Vec16<T>::type v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            v[u] = typename Vec16<T>::type{};
            if (i + u * step < e)
                v[u] = load_vec<T>(g + (long long)toks[i + u * step] * ld_g, c, cols, whole);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < N; ++k) acc[k] += (float)v[u][k];
    }
}

// acc of the workgroup's groups added up in order into group 0's
template <int N, int LPR>
__device__ __forceinline__ void join_groups(float (&acc)[N], float* lds) {
    constexpr int G = kEmbedBlock / LPR;
    const int lane = threadIdx.x % LPR, grp = threadIdx.x / LPR;
    if constexpr (G > 1) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k) lds[(grp * N + k) * LPR + lane] = acc[k];
        __syncthreads();
        if (grp == 0)
            for (int j = 1; j < G; ++j)
#pragma unroll
                for (int k = 0; k < N; ++k) acc[k] += lds[(j * N + k) * LPR + lane];
    }
}

// Table rows of ids with more tokens than a piece: piece j's workgroup takes the one whose
// tokens begin in it, if there is one.
template <typename T, int LPR>
__global__ __launch_bounds__(kEmbedBlock) void k_embed_join(const unsigned* keys, const int* first,
                                                            int n, int vocab, int piece, int cols,
                                                            const float* part, float scale, T* dw,
                                                            long long ld_dw, int whole) {
    constexpr int N = Vec16<T>::N;
    __shared__ float lds[kEmbedBlock * N];
    const int j = blockIdx.x;
    const int a = j * piece, e = a + piece < n ? a + piece : n;
    const unsigned id = keys[e - 1];
    if (id >= (unsigned)vocab) return;
    const int f = first[id], l = first[id + 1];
    if (l - f <= piece || f < a) return;
    const int lane = threadIdx.x % LPR, grp = threadIdx.x / LPR;
    const int c = (blockIdx.y * LPR + lane) * N;
    const int last = (l - 1) / piece;
    float acc[N] = {};
    if (c < cols) {
#pragma unroll 8
        for (int p = j + grp; p <= last; p += kEmbedBlock / LPR) {
            const float* row = part + (size_t)(2 * p + (p == j && f != a ? 1 : 0)) * cols;
#pragma unroll
            for (int k = 0; k < N; ++k) acc[k] += c + k < cols ? row[c + k] : 0.f;
        }
    }
    join_groups<N, LPR>(acc, lds);
    if (grp == 0 && c < cols) {
        typename Vec16<T>::type y;
#pragma unroll
        for (int k = 0; k < N; ++k) y[k] = (T)(acc[k] * scale);
        store_vec<T>(dw + (long long)id * ld_dw, c, cols, whole, y);
    }
}

// Piece j's partial sums, part[2 j + slot]: slot 0 the id that the piece begins with,
// slot 1 the one that it ends with, where that id has more tokens than a piece.
template <typename T, int LPR>
__device__ __forceinline__ void sum_piece(const unsigned* keys, const unsigned* toks, const int* first,
                                          int n, int vocab, int piece, const T* g, long long ld_g,
                                          int cols, int whole, float* part, int at, int slab,
                                          float* lds) {
    constexpr int N = Vec16<T>::N;
    const int j = at >> 1, slot = at & 1;
    const int a = j * piece, e = a + piece < n ? a + piece : n;
    const unsigned head = keys[a], id = slot == 0 ? head : keys[e - 1];
    if (id >= (unsigned)vocab || (slot == 1 && id == head)) return;
    const int f = first[id], l = first[id + 1];
    if (l - f <= piece) return;
    const int from = f > a ? f : a, to = l < e ? l : e;
    const int lane = threadIdx.x % LPR, grp = threadIdx.x / LPR;
    const int c = (slab * LPR + lane) * N;
    float acc[N] = {};
    if (c < cols)
        add_rows<T>(acc, g, ld_g, toks, from + grp, to, kEmbedBlock / LPR, c, cols, whole);
    join_groups<N, LPR>(acc, lds);
    if (grp == 0) {
        float* p = part + (size_t)at * cols;
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (c + k < cols) p[c + k] = acc[k];
    }
}

// All other table rows, those of ids without a token too: R rows a group, whose tokens lie
// together in the sorted order, so that U rows of g are in flight across the table rows'
// borders (most ids have few tokens).
template <typename T, int LPR, int R>
__device__ __forceinline__ void sum_rows(const unsigned* toks, const int* first, int vocab, int piece,
                                         const T* g, long long ld_g, int whole_g, int cols, float scale,
                                         T* dw, long long ld_dw, int whole, int block) {
    constexpr int N = Vec16<T>::N, U = 8;
    typedef typename Vec16<T>::type V;
    const int lane = threadIdx.x % LPR;
    const int slabs = (cols + LPR * N - 1) / (LPR * N);
    const int v0 = (block / slabs * (kEmbedBlock / LPR) + threadIdx.x / LPR) * R;
    const int c = (block % slabs * LPR + lane) * N;
    if (v0 >= vocab) return;  // lanes behind the last column stay: they hand out tokens
    const int rows = vocab - v0 < R ? vocab - v0 : R;
    int at[R + 1];
#pragma unroll
    for (int r = 0; r <= R; ++r) at[r] = first[v0 + (r < rows ? r : rows)];
    for (int r = 0; r < rows;) {
        // rows r .. e - 1 with at most a piece each; row e has more, or is not ours
        int e = r, end = at[0], cur_end = 0;
#pragma unroll
        for (int k = 0; k < R; ++k)
            if (k == e && k < rows && at[k + 1] - at[k] <= piece) e = k + 1;
        int p = 0;
#pragma unroll
        for (int k = 0; k < R; ++k) {
            p = k == r ? at[k] : p;
            cur_end = k == r ? at[k + 1] : cur_end;
            end = k + 1 == e ? at[k + 1] : end;
        }
        if (e == r) {
            ++r;
            continue;
        }
        float acc[N] = {};
        auto finish = [&]() {  // row r is whole
            V y;
#pragma unroll
            for (int k = 0; k < N; ++k) {
                y[k] = (T)(acc[k] * scale);
                acc[k] = 0.f;
            }
            store_vec<T>(dw + (long long)(v0 + r) * ld_dw, c, cols, whole, y);
            ++r;
#pragma unroll
            for (int k = 0; k < R; ++k) cur_end = k == r ? at[k + 1] : cur_end;
        };
        for (; p < end; p += U) {
            V x[U];
            const unsigned mine = toks[p + lane % U < end ? p + lane % U : end - 1];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const unsigned tok = __shfl(mine, u, LPR);
                if (p + u < end) x[u] = load_vec<T>(g + (long long)tok * ld_g, c, cols, whole_g);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (p + u >= end) break;
                while (p + u >= cur_end) finish();
#pragma unroll
                for (int k = 0; k < N; ++k) acc[k] += (float)x[u][k];
            }
        }
        while (r < e) finish();
    }
}

// Both in one launch, `blocks` workgroups of pieces last (first: 144.5 us for 65,536 tokens,
// 50,021 x 1024 bf16, forward and gradient; last: 140.1 us, as two launches take).
template <typename T, int LPR, int R>
__global__ __launch_bounds__(kEmbedBlock) void k_embed_sums(
    const unsigned* keys, const unsigned* toks, const int* first, int n, int vocab, int piece, int blocks,
    const T* g, long long ld_g, int whole_g, int cols, float scale, float* part, T* dw, long long ld_dw,
    int whole) {
    __shared__ float lds[kEmbedBlock * Vec16<T>::N];
    const int slabs = (cols + LPR * Vec16<T>::N - 1) / (LPR * Vec16<T>::N);
    const int rest = (int)gridDim.x - blocks, at = (int)blockIdx.x - rest;
    if (at >= 0)
        sum_piece<T, LPR>(keys, toks, first, n, vocab, piece, g, ld_g, cols, whole_g, part, at / slabs,
                          at % slabs, lds);
    else
        sum_rows<T, LPR, R>(toks, first, vocab, piece, g, ld_g, whole_g, cols, scale, dw, ld_dw, whole,
                            blockIdx.x);
}

// Few tokens: table rows [kOwnRows * blockIdx.x, ...).  Rows with up to kOwnHot tokens are one
// group's, walking the workgroup's list; for the others the groups share the tokens.
template <typename T, int LPR>
__global__ __launch_bounds__(kEmbedBlock) void k_embed_own(Ids s, int n, const T* g, long long ld_g,
                                                           int whole_g, int cols, float scale, T* dw,
                                                           long long ld_dw, int whole) {
    constexpr int N = Vec16<T>::N, U = 8, G = kEmbedBlock / LPR, WAVES = kEmbedBlock / kWave;
    typedef typename Vec16<T>::type V;
    __shared__ unsigned list[kFewTokens];  // row << 16 | token, ascending tokens
    __shared__ int found[kOwnRows], wave_found[WAVES];
    __shared__ float lds[kEmbedBlock * N];
    const int tid = threadIdx.x, lane = tid % LPR, grp = tid / LPR;
    const int v0 = blockIdx.x * kOwnRows;
    const int rows = s.vocab - v0 < kOwnRows ? s.vocab - v0 : kOwnRows;
    const int c = (blockIdx.y * LPR + lane) * N;
    if (tid < kOwnRows) found[tid] = 0;
    __syncthreads();  // no tokens: nothing below waits before found is read
    int total = 0;
    for (int t0 = 0; t0 < n; t0 += kEmbedBlock) {
        const int t = t0 + tid;
        const int r = t < n ? (int)key_at(s, t) - v0 : -1;
        const bool ours = r >= 0 && r < rows;
        const unsigned long long m = __ballot(ours);
        if (tid % kWave == 0) wave_found[tid / kWave] = __popcll(m);
        __syncthreads();
        int at = total + __popcll(m & ((1ull << (tid % kWave)) - 1));
#pragma unroll
        for (int k = 0; k < WAVES; ++k) {
            if (k < tid / kWave) at += wave_found[k];
            total += wave_found[k];
        }
        if (ours) {
            list[at] = (unsigned)r << 16 | (unsigned)t;
            atomicAdd(&found[r], 1);
        }
        __syncthreads();
    }
    // acc += the rows of g whose list entries belong to row r, every `step`th from `skip` on
    const unsigned long long mine =
        LPR == kWave ? ~0ull : ((1ull << (LPR & 63)) - 1) << (tid % kWave / LPR * LPR);
    auto sum = [&](float(&acc)[N], int r, int skip, int step) {
        for (int i0 = 0; i0 < total; i0 += LPR) {
            const unsigned entry = i0 + lane < total ? list[i0 + lane] : ~0u;
            unsigned long long m = __ballot((int)(entry >> 16) == r) & mine;
            while (m != 0) {
                V x[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    for (; m != 0 && skip > 0; --skip) m &= m - 1;
                    const int from = m != 0 ? __ffsll((long long)m) - 1 : 0;
                    const unsigned tok = __shfl(entry, from) & 0xFFFF;
                    x[u] = V{};
                    if (m != 0) {
                        x[u] = load_vec<T>(g + (long long)tok * ld_g, c, cols, whole_g);
                        m &= m - 1;
                        skip = step - 1;
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int k = 0; k < N; ++k) acc[k] += (float)x[u][k];
            }
        }
    };
    auto store = [&](const float(&acc)[N], int r) {
        V y;
#pragma unroll
        for (int k = 0; k < N; ++k) y[k] = (T)(acc[k] * scale);
        store_vec<T>(dw + (long long)(v0 + r) * ld_dw, c, cols, whole, y);
    };
    for (int r = grp; r < rows; r += G) {
        if (found[r] > kOwnHot) continue;
        float acc[N] = {};
        if (found[r] > 0) sum(acc, r, 0, 1);
        store(acc, r);
    }
    for (int r = 0; r < rows; ++r) {
        if (found[r] <= kOwnHot) continue;
        float acc[N] = {};
        sum(acc, r, grp, G);
        join_groups<N, LPR>(acc, lds);
        if (grp == 0) store(acc, r);
    }
}

// One launch beats the sort where launches are the time: every workgroup looks at all ids, and
// one that is all tokens' is summed by one workgroup, so the tokens are few; table rows are
// limited so that the looking stays below writing the rows.
inline bool few_tokens(long long tokens, int vocab) {
    return tokens <= kFewTokens && vocab <= 1 << 20;
}

// lanes per row: the power of two in [8, 64] that covers it, if one does
inline int embed_lanes(int cols, int dtype) {
    const int n = 16 / (int)dtype_size(dtype);
    const int vecs = (cols + n - 1) / n;
    return vecs <= 8 ? 8 : vecs <= 16 ? 16 : vecs <= 32 ? 32 : 64;
}

// A launch has at most 65535 slabs of 64 vectors for a row; columns beyond them would also
// wrap the lookup's int steps.
inline bool cols_fit(int cols, int dtype) {
    return cols > 0 && cols <= 65535 * kWave * (16 / (int)dtype_size(dtype));
}

inline bool rows_whole(const void* p, long long ld, int dtype) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ((uintptr_t)ld * dtype_size(dtype) & 15) == 0;
}

// Tokens of a piece: few, so that no group adds up many rows in a line, but at most
// kMaxPieces pieces in all, whose partial sums an id of all tokens joins in a line (sums and
// joins of 60,157 tokens over 512 x 64 float32, a third of them one id: 34 us with 4096, 21
// with 2048, 22 with 1024; 65,536 over 50,021 x 1,024 bf16: 81, 73 and 72).
inline int piece_of(int n) {
    int p = kMinPiece;
    while ((long long)p * kMaxPieces < n) p *= 2;
    return p;
}

struct SortPlan {
    int per, blocks, passes;
};
inline SortPlan sort_plan(int n, int vocab) {
    SortPlan s;
    s.per = (n + kSortMaxBlocks - 1) / kSortMaxBlocks;
    if (s.per < kSortMinItems) s.per = kSortMinItems;
    s.blocks = (n + s.per - 1) / s.per;
    int bits = 0;
    while (bits < 32 && ((unsigned)vocab >> bits) != 0) ++bits;
    s.passes = (bits + 7) / 8;
    return s;
}

// Workspace: two sets of (key, token) arrays, the digit counts, first[], the pieces'
// partial sums.
struct GradLayout {
    size_t keys[2], toks[2], counts, first, part, bytes;
};
inline GradLayout grad_layout(int n, int vocab, int cols) {
    GradLayout l;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += align_up(bytes);
        return here;
    };
    for (int k = 0; k < 2; ++k) {
        l.keys[k] = take((size_t)n * 4);
        l.toks[k] = take((size_t)n * 4);
    }
    l.counts = take((size_t)kSortMaxBlocks * 256 * 4);
    l.first = take(((size_t)vocab + 1) * 4);
    const int piece = piece_of(n);
    l.part = take(((size_t)n + piece - 1) / piece * 2 * cols * 4);
    l.bytes = at;
    return l;
}

template <typename T, int LPR>
int embed_grad_sums(const unsigned* keys, const unsigned* toks, const int* first, int n, int vocab,
                    const T* g, long long ld_g, int cols, float scale, float* part, T* dw,
                    long long ld_dw, int dtype, hipStream_t s) {
    constexpr int N = Vec16<T>::N;
    const int whole_g = rows_whole(g, ld_g, dtype), whole = rows_whole(dw, ld_dw, dtype);
    const int slabs = (cols + LPR * N - 1) / (LPR * N);
    const int piece = piece_of(n);
    const int pieces = n > piece ? (n + piece - 1) / piece : 0;  // one id has no more than a piece else
    constexpr int RPB = kEmbedBlock / LPR;
    // several table rows a group where there are enough of them for all CUs
    auto sums = [&](auto r) {
        constexpr int R = decltype(r)::value;
        const int groups = (vocab + R - 1) / R, blocks = 2 * pieces * slabs;
        k_embed_sums<T, LPR, R>
            <<<(unsigned)(blocks + (groups + RPB - 1) / RPB * slabs), kEmbedBlock, 0, s>>>(
                keys, toks, first, n, vocab, piece, blocks, g, ld_g, whole_g, cols, scale, part, dw, ld_dw,
                whole);
    };
    if ((long long)vocab * slabs >= 4ll * 256 * 8 * RPB)
        sums(std::integral_constant<int, 4>());
    else
        sums(std::integral_constant<int, 1>());
    if (pieces > 0)
        k_embed_join<T, LPR><<<dim3(pieces, slabs), kEmbedBlock, 0, s>>>(
            keys, first, n, vocab, piece, cols, part, scale, dw, ld_dw, whole);
    return status_of(hipGetLastError());
}

template <typename T>
int embed_grad_by_lanes(int lanes, const unsigned* keys, const unsigned* toks, const int* first,
                        int n, int vocab, const void* g, long long ld_g, int cols, float scale,
                        float* part, void* dw, long long ld_dw, int dtype, hipStream_t s) {
    const T* gt = static_cast<const T*>(g);
    T* dt = static_cast<T*>(dw);
    auto call = [&](auto l) {
        return embed_grad_sums<T, decltype(l)::value>(keys, toks, first, n, vocab, gt, ld_g, cols,
                                                      scale, part, dt, ld_dw, dtype, s);
    };
    if (lanes == 8) return call(std::integral_constant<int, 8>());
    if (lanes == 16) return call(std::integral_constant<int, 16>());
    if (lanes == 32) return call(std::integral_constant<int, 32>());
    return call(std::integral_constant<int, 64>());
}

template <typename T>
int embed_by_lanes(int lanes, const Ids& ids, long long tokens, const void* w, long long ld_w,
                   int cols, float scale, void* out, long long ld_out, int dtype, hipStream_t s) {
    const int whole = rows_whole(w, ld_w, dtype) && rows_whole(out, ld_out, dtype);
    auto call = [&](auto l) {
        constexpr int L = decltype(l)::value;
        const int grid = grid_for(tokens, kEmbedBlock / L, 256 * 32);
        k_embed<T, L><<<grid, kEmbedBlock, 0, s>>>(ids, tokens, static_cast<const T*>(w), ld_w,
                                                   cols, scale, static_cast<T*>(out), ld_out, whole);
        return status_of(hipGetLastError());
    };
    if (lanes == 8) return call(std::integral_constant<int, 8>());
    if (lanes == 16) return call(std::integral_constant<int, 16>());
    if (lanes == 32) return call(std::integral_constant<int, 32>());
    return call(std::integral_constant<int, 64>());
}

template <typename T>
int embed_own_by_lanes(int lanes, const Ids& ids, int n, const void* g, long long ld_g, int cols,
                       float scale, void* dw, long long ld_dw, int dtype, hipStream_t s) {
    const int whole_g = rows_whole(g, ld_g, dtype), whole = rows_whole(dw, ld_dw, dtype);
    auto call = [&](auto l) {
        constexpr int L = decltype(l)::value;
        const int slabs = (cols + L * Vec16<T>::N - 1) / (L * Vec16<T>::N);
        k_embed_own<T, L><<<dim3((ids.vocab + kOwnRows - 1) / kOwnRows, slabs), kEmbedBlock, 0, s>>>(
            ids, n, static_cast<const T*>(g), ld_g, whole_g, cols, scale, static_cast<T*>(dw), ld_dw, whole);
        return status_of(hipGetLastError());
    };
    if (lanes == 8) return call(std::integral_constant<int, 8>());
    if (lanes == 16) return call(std::integral_constant<int, 16>());
    if (lanes == 32) return call(std::integral_constant<int, 32>());
    return call(std::integral_constant<int, 64>());
}

inline bool ids_fit(const void* ids, int ids64, long long tokens) {
    return tokens == 0 ||
           (ids != nullptr && (reinterpret_cast<uintptr_t>(ids) & (ids64 ? 7 : 3)) == 0);
}

}  // namespace

extern "C" {

int gat_embedding(const void* ids, int ids64, long long tokens, const void* w, long long ld_w,
                  int vocab, int cols, float scale, void* out, long long ld_out, int dtype,
                  void* stream) {
    if (tokens < 0 || tokens > kMaxTokens || vocab <= 0 || !known_dtype(dtype) || !cols_fit(cols, dtype) ||
        ld_w < cols || ld_out < cols || !ids_fit(ids, ids64, tokens))
        return GAT_EINVAL;
    if (tokens == 0) return GAT_OK;
    if (w == nullptr || out == nullptr || !element_aligned(w, dtype) || !element_aligned(out, dtype))
        return GAT_EINVAL;
    const Ids s{ids, ids64, -1, vocab};
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int lanes = embed_lanes(cols, dtype);
    if (dtype == GAT_F32)
        return embed_by_lanes<float>(lanes, s, tokens, w, ld_w, cols, scale, out, ld_out, dtype, st);
    if (dtype == GAT_BF16)
        return embed_by_lanes<bf16>(lanes, s, tokens, w, ld_w, cols, scale, out, ld_out, dtype, st);
    return embed_by_lanes<f16>(lanes, s, tokens, w, ld_w, cols, scale, out, ld_out, dtype, st);
}

int gat_embedding_grad_workspace_size(long long tokens, int vocab, int cols, size_t* bytes) {
    if (tokens < 0 || tokens > kMaxTokens || vocab <= 0 || vocab > kMaxTokens || cols <= 0 || bytes == nullptr)
        return GAT_EINVAL;
    *bytes = few_tokens(tokens, vocab) ? 0 : grad_layout((int)tokens, vocab, cols).bytes;
    return GAT_OK;
}

int gat_embedding_grad(const void* ids, int ids64, long long tokens, const void* g, long long ld_g,
                       int vocab, int cols, float scale, long long padding, void* dw,
                       long long ld_dw, void* workspace, size_t workspace_bytes, int dtype,
                       void* stream) {
    if (tokens < 0 || tokens > kMaxTokens || vocab <= 0 || vocab > kMaxTokens || !known_dtype(dtype) ||
        !cols_fit(cols, dtype) || ld_g < 0 || ld_dw < cols || dw == nullptr || !element_aligned(dw, dtype) ||
        !ids_fit(ids, ids64, tokens) ||
        (tokens > 0 && (g == nullptr || !element_aligned(g, dtype))))
        return GAT_EINVAL;
    const int n = (int)tokens;
    const Ids s{ids, ids64, padding, vocab};
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int lanes = embed_lanes(cols, dtype);
    if (few_tokens(n, vocab)) {
        if (dtype == GAT_F32)
            return embed_own_by_lanes<float>(lanes, s, n, g, ld_g, cols, scale, dw, ld_dw, dtype, st);
        if (dtype == GAT_BF16)
            return embed_own_by_lanes<bf16>(lanes, s, n, g, ld_g, cols, scale, dw, ld_dw, dtype, st);
        return embed_own_by_lanes<f16>(lanes, s, n, g, ld_g, cols, scale, dw, ld_dw, dtype, st);
    }
    const GradLayout l = grad_layout(n, vocab, cols);
    if (workspace == nullptr || workspace_bytes < l.bytes) return GAT_EWORKSPACE;
    if ((reinterpret_cast<uintptr_t>(workspace) & 15) != 0) return GAT_EINVAL;
    char* ws = static_cast<char*>(workspace);
    unsigned* keys[2] = {reinterpret_cast<unsigned*>(ws + l.keys[0]),
                         reinterpret_cast<unsigned*>(ws + l.keys[1])};
    unsigned* toks[2] = {reinterpret_cast<unsigned*>(ws + l.toks[0]),
                         reinterpret_cast<unsigned*>(ws + l.toks[1])};
    unsigned* counts = reinterpret_cast<unsigned*>(ws + l.counts);
    int* first = reinterpret_cast<int*>(ws + l.first);
    float* part = reinterpret_cast<float*>(ws + l.part);
    int cur = 0;
    if (n > 0) {
        const SortPlan p = sort_plan(n, vocab);
        for (int k = 0; k < p.passes; ++k) {
            const int shift = 8 * k;
            if (k == 0) {
                k_sort_count<true><<<p.blocks, kSortBlock, 0, st>>>(s, nullptr, n, p.per, shift, counts);
                k_sort_place<true><<<p.blocks, kSortBlock, 0, st>>>(s, nullptr, nullptr, n, p.per, shift,
                                                                    counts, keys[0], toks[0]);
            } else {
                k_sort_count<false><<<p.blocks, kSortBlock, 0, st>>>(s, keys[cur], n, p.per, shift,
                                                                     counts);
                k_sort_place<false><<<p.blocks, kSortBlock, 0, st>>>(s, keys[cur], toks[cur], n, p.per,
                                                                     shift, counts, keys[cur ^ 1],
                                                                     toks[cur ^ 1]);
                cur ^= 1;
            }
        }
    }
    k_sort_firsts<<<n / 256 + 1, 256, 0, st>>>(keys[cur], n, vocab, first);
    if (dtype == GAT_F32)
        return embed_grad_by_lanes<float>(lanes, keys[cur], toks[cur], first, n, vocab, g, ld_g, cols,
                                          scale, part, dw, ld_dw, dtype, st);
    if (dtype == GAT_BF16)
        return embed_grad_by_lanes<bf16>(lanes, keys[cur], toks[cur], first, n, vocab, g, ld_g, cols,
                                         scale, part, dw, ld_dw, dtype, st);
    return embed_grad_by_lanes<f16>(lanes, keys[cur], toks[cur], first, n, vocab, g, ld_g, cols, scale,
                                    part, dw, ld_dw, dtype, st);
}

}  // extern "C"
