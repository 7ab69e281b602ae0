// Attention over packed sequences, forward and backward (gat_packed_attention,
// gat_packed_attention_backward).
//
// Sequence b has the queries ptr[b] .. ptr[b+1] of q and the keys kv_ptr[b] ..
// kv_ptr[b+1] of k and v.  Per query head h, with key head h / G (G query heads share
// a key head):
//   P = softmax(scale q k^T over the visible keys)        y = P v
//   dP = g v^T     dS = P (dP - sum_d g y)
//   dq = scale dS k    dk = scale sum_heads dS^T q    dv = sum_heads P^T g
// Causal: key j is visible to query i iff j <= i + (keys - queries).  A query that
// sees no key gives y = 0, lse = -inf and no gradient.
//
// One tile shape carries all three kernels.  A wave owns 32 COLUMNS (queries in the
// forward and the dq kernel, keys in the dk/dv kernel; 16 for narrow float32 heads), one per
// lane and half wave, and streams ROWS of the other side through LDS, 32 at a time:
//   scores[row][col]  = rows . columns        A: rows from LDS, B: columns in registers
//   acc[d][col]      += X^T[d][row] W[row][col]     W: the scores after the softmax
// A 32x32 matrix product leaves lane (col, half) with rows 8 i + 4 half + 0..3, and that
// is the order in which it takes W back as its B operand: the scores never leave the
// registers, and the softmax sums of a column are one lane's own plus one exchange
// between the halves.  X^T comes out of LDS by the transposing 64-bit read.
//
// The query heads that share a key head are rows of one packed axis (row = query * G +
// head in group): a tile holds whole groups, keys are read once for the group, and dk
// and dv sum over the heads inside the kernel.
//
// Tiles are found without a launch that counts them: the sequence boundaries bnd are
// monotone, so slot(s) = bnd[s] / tile + s leaves every sequence at least the slots it
// needs.  The rows before the first and behind the last sequence form sequences without
// keys, so their outputs and gradients are zeros.
//
// Bound: matrix products where sequences are long, the keys' and values' bytes where queries
// are few, softmax arithmetic and latency where heads are narrow and sequences short.
// Measured, by box: prompts of 300 to 6,000 tokens, 16 heads of 128 over 4, bf16, causal:
// 546-584 us (967-905 TFLOP/s; the softmax arithmetic of its 10^9 scores takes as long as the
// products); 8 sequences of 2,048 with the backward: 1,047-1,084 us; one query for each of 48
// sequences of up to 8,192, 32 heads of 128 over 8: 165 us (4.6 TB/s); 512 graphs of 85 to 150
// nodes, 8 heads of 8, float32, with the backward: 277 us.

#include "gat_seq.h"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

struct Rows {  // a [tokens, heads, dim] tensor; strides in elements
    const void* p;
    long long row, head;
};

struct AttnArgs {
    Rows q, k, v, g, o;  // o: the forward's output
    void* low;           // bf16: what o's rounding left, as o lies; may be null
    Rows dq, dk, dv;
    float* lse;    // [queries, heads]
    float* delta;  // [queries, heads] sum_d g y
    const void *ptr, *kv_ptr;
    float* part;  // partial results of a split axis
    int ptr64, count;
    int nq, nk;  // rows of q and of k
    int kv_heads, group, dim;
    unsigned div_mul, div_shift;  // row / group
    float scale;
    int causal, splits;
    int by_xcd;  // place_of
};

// The scores are formed as |scale| (+-columns) . rows, so that their maximum is that of the
// products; a scale of 0 as 1 times zero columns (0 times a hidden row's -inf is no score).
__device__ __forceinline__ float score_scale(float scale) { return scale == 0.f ? 1.f : fabsf(scale); }

__device__ __forceinline__ int div_group(const AttnArgs& a, int r) {
    return a.group == 1 ? r : (int)(__umulhi((unsigned)r, a.div_mul) >> a.div_shift);
}

// bnd[0] = 0, bnd[1 .. count + 1] = ptr, bnd[count + 2] = n: sequences 1 .. count are
// the caller's, 0 and count + 1 the rows outside them.  Values are held to [0, n].
__device__ __forceinline__ int bound_at(const void* ptr, int ptr64, int count, int n, int s) {
    if (s <= 0) return 0;
    if (s >= count + 2) return n;
    const long long v = ptr64 ? static_cast<const long long*>(ptr)[s - 1]
                              : (long long)static_cast<const int*>(ptr)[s - 1];
    return (int)(v < 0 ? 0 : v > n ? n : v);
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

struct Tile {
    int first, len;              // the sequence's rows on the tile's axis
    int other_first, other_len;  // and on the other; none outside the caller's sequences
    int index;                   // tile within the sequence
};

// The sequence and the tile of a slot; 64 boundaries a step, then the four that count at once.
__device__ __forceinline__ Tile tile_of(const void* ptr, const void* other, int ptr64, int count, int n,
                                        int other_n, int group, int size, int slot) {
    const int lane = threadIdx.x % kWave;
    int lo = 0, hi = count + 2;
    while (hi - lo > 1) {
        const int step = (hi - lo + kWave - 1) / kWave;
        const int at = lo + lane * step;
        bool ok = false;
        if (at < hi)
            ok = (long long)bound_at(ptr, ptr64, count, n, at) * group / size + at <= slot;
        const int got = __popcll(__ballot(ok));
        lo += (got > 0 ? got - 1 : 0) * step;
        if (lo + step < hi) hi = lo + step;
    }
    const bool ours = lo >= 1 && lo <= count;
    const int a = bound_at(ptr, ptr64, count, n, lo), b = bound_at(ptr, ptr64, count, n, lo + 1);
    const int c = ours ? bound_at(other, ptr64, count, other_n, lo) : 0;
    const int d = ours ? bound_at(other, ptr64, count, other_n, lo + 1) : 0;
    Tile t;
    t.first = uniform(a);
    t.len = uniform(b > a ? b - a : 0);
    t.other_first = uniform(c);
    t.other_len = uniform(d > c ? d - c : 0);
    t.index = uniform(slot - (int)((long long)a * group / size + lo));
    return t;
}

// Workgroups go round the 8 XCDs, each with an L2 of its own.  Where the key heads divide
// evenly among the XCDs, an XCD gets workgroups of one head (or of heads of its own), so that
// the rows they stream are read into one L2 or few, not into all (causal prompts of 300 to
// 6000 tokens, 4 key heads of 128: 602 us plainly, 571 us so; a packed training batch, heads
// of 64: 305 us and 268 us).  Narrow heads, whose rows are a part of a line: 8 heads of 8 over 512
// graphs, training, 281 us plainly and 279 us so in float32, 224 us either way in bf16; 8 heads
// of 32 in bf16 lose, 290 us plainly and 297 us so.  Single waves stream rows that no other
// workgroup reads: 164.3 us plainly, 165.6 us so, for one query each of 48 sequences.
struct Place {
    int slot, kh;
};
__device__ __forceinline__ Place place_of(const AttnArgs& a) {
    if (a.by_xcd) {  // gridDim.x is a multiple of 8
        const unsigned id = blockIdx.y * gridDim.x + blockIdx.x, xcd = id % 8, at = id / 8;
        if (a.kv_heads >= 8) return {(int)(at % gridDim.x), (int)(xcd + at / gridDim.x * 8)};
        return {(int)(at * (8 / a.kv_heads) + xcd / a.kv_heads), (int)(xcd % a.kv_heads)};
    }
    return {(int)blockIdx.x, (int)blockIdx.y};
}

inline long long slots_of(long long n, int group, int size, int count) {
    return n * group / size + count + 2;
}

// ---------------------------------------------------------------------------
// Matrix products.  K of a step: two 16-byte vectors, one per half wave.
// ---------------------------------------------------------------------------
__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(f32x4 a, f32x4 b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
}

// W: columns of a wave.  32 with 32x32 products; 16 with 16x16 ones for narrow float32 heads,
// where 32-wide tiles of the head dimension would be mostly empty.  The lanes that share a
// column are its PARTS.  A step covers ROWS rows with 16 scores a lane, register i of part p
// holding row row_of(i, p); an accumulator's register e holds dimension row_of(e, p) of its
// tile.
template <typename T, int DP>
struct Shape {
    static constexpr int N = Vec16<T>::N;
    static constexpr int W = sizeof(T) == 4 && DP <= 16 ? 16 : 32;
    static constexpr int PARTS = kWave / W, ROWS = 16 * PARTS;
    static constexpr int STEPS = W == 16 ? 1 : DP / (2 * N);  // products of a score tile
    static constexpr int DT = W == 16 ? 1 : (DP + 31) / 32;   // tiles of the head dimension
    static constexpr int CPR = DP / N;                        // 16-byte vectors of a row
    static constexpr int AR = W == 16 ? 4 : 16;               // registers of an accumulator
    static constexpr int FN = W == 16 ? DP / 4 : N;           // a lane's dimensions of a step
    typedef float Acc __attribute__((ext_vector_type(AR)));
    typedef T Frag __attribute__((ext_vector_type(FN)));
    static __device__ __forceinline__ int row_of(int i, int part) {
        return 4 * PARTS * (i / 4) + 4 * part + i % 4;
    }
    // A tile of `rows` in LDS, rows without gaps (as the loads to LDS write them).  Vector c
    // of row r lies at place c ^ turn(r), so that what LDS serves in one cycle, 256 bytes,
    // meets all 64 banks: one vector of 16 rows (the scores' reads), four of 4 rows (bf16's
    // transposing reads; counted in bf16: no conflict.  float32 reads X one element a lane:
    // heads of 8 conflict in 42 to 48% of the LDS cycles).  With 8-row turns, two rows a bank:
    // 2.6 more cycles a read.  The last tile of the head dimension may read past DP, into what
    // follows.
    static constexpr int slab(int rows) { return rows * DP; }
    static constexpr int kSlack = 32;
    static __device__ __forceinline__ int turn(int r) {
        if constexpr (CPR % 16 == 0) return (r & 3) << 2 | (r >> 2 & 3);
        if constexpr (CPR % 8 == 0) return (r >> 1 & 1) << 2 | (r >> 2 & 3);
        if constexpr (CPR % 4 == 0) return r >> 2 & 3;
        return r >> 3 & 1;
    }
};

// Asks the compiler to spread the LDS reads of a whole tile between its matrix products, not
// to gather them just before their use (bf16: prompts 602 -> 588 us, packed training 306 ->
// 297 us; float32's 64-cycle products cover them as they are).
template <typename T, bool MASK>
__device__ __forceinline__ void schedule() {
    if constexpr (sizeof(T) == 2 && !MASK) __builtin_amdgcn_iglp_opt(0);
}

enum AttnPass { kFwd, kDq, kDkv };

// What the registers are held to: two waves a SIMD to have one's softmax under the other's
// matrix products, as many as fit where the tiles are narrow and waiting is most of the time
// (graphs of 85 to 150 nodes, 8 heads of 8, float32, one training step: 300 us with what the
// compiler takes, 278 us with these).  bf16 heads over 64: dq too (8 sequences of 2048, 16 heads
// of 128 over 4, causal, one training step: 1215 us with one wave, 1087 us with two); dk and
// dv, whose two accumulators are 128 registers there, spill under two (1645 us).  Heads of 64
// spill 116-132 bytes a lane in dk and dv under two, heads of 128 28 (bf16) and 80 (float32) in
// the forward.
// Single-wave workgroups have row tiles of their own in LDS: those of narrow float32 heads are
// resident three or four times a SIMD, not six, and float32 heads over 32 once; the compiler
// says so of each.
template <typename T, int DP>
constexpr int waves_per_simd(AttnPass pass) {
    if (Shape<T, DP>::W == 16) return pass == kDkv ? 4 : 6;
    return pass == kFwd || DP <= 64 || (pass == kDq && sizeof(T) == 2) ? 2 : 1;
}

// scores[row][col] of ROWS rows in LDS against the wave's columns
template <typename T, int DP>
__device__ __forceinline__ f32x16 scores(const T* rows, const typename Shape<T, DP>::Frag* cols) {
    typedef Shape<T, DP> S;
    const int lane = threadIdx.x % kWave, row = lane % S::W, part = lane / S::W;
    f32x16 c = {};
    if constexpr (S::W == 32) {
        const T* at = rows + row * DP;
        const int place = part ^ S::turn(row);
#pragma unroll
        for (int s = 0; s < S::STEPS; ++s)
            c = mma(*reinterpret_cast<const typename Vec16<T>::type*>(at + ((2 * s) ^ place) * S::N),
                    cols[s], c);
    } else {
        const T* at = rows + row * DP + ((part * S::FN / S::N) ^ S::turn(row)) * S::N + part * S::FN % S::N;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const auto x = *reinterpret_cast<const typename S::Frag*>(at + 16 * u * DP);
            f32x4 t = {};
#pragma unroll
            for (int e = 0; e < S::FN; ++e)
                t = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], cols[0][e], t, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; ++e) c[4 * u + e] = t[e];
        }
    }
    return c;
}

// four rows of one column of a row-major tile in LDS
__device__ __forceinline__ bf16x4 read_transposed(const bf16* p) {
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    return __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                          (lds_s16x4*)(__attribute__((address_space(3))) void*)p));
}

// acc[d][col] += sum over ROWS rows of X[row][d] w[row][col].  bf16: w is rounded to bf16; FINE
// adds the product with what that leaves.
template <int DP, bool FINE = false>
__device__ __forceinline__ void add_products(f32x16* acc, const bf16* rows, const f32x16& w) {
    typedef Shape<bf16, DP> S;
    const int lane = threadIdx.x % kWave;
    const int row = 4 * (lane / 32) + lane % 16 / 4;
    const bf16* at = rows + row * DP + lane % 2 * 4;
    const int vec = lane % 32 / 16 * 2 + lane % 4 / 2;
    const int place_lo = vec ^ S::turn(row), place_hi = vec ^ S::turn(row + 8);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        bf16x8 b, left;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            b[e] = (bf16)w[8 * s + e];
            if constexpr (FINE) left[e] = (bf16)(w[8 * s + e] - (float)b[e]);
        }
#pragma unroll
        for (int t = 0; t < S::DT; ++t) {
            const bf16x4 lo = read_transposed(at + 16 * s * DP + ((4 * t) ^ place_lo) * 8);
            const bf16x4 hi = read_transposed(at + (16 * s + 8) * DP + ((4 * t) ^ place_hi) * 8);
            const bf16x8 x = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            acc[t] = mma(x, b, acc[t]);
            if constexpr (FINE) acc[t] = mma(x, left, acc[t]);
        }
    }
}
template <int DP, bool FINE = false>
__device__ __forceinline__ void add_products(typename Shape<float, DP>::Acc* acc, const float* rows,
                                             const f32x16& w) {
    typedef Shape<float, DP> S;
    const int lane = threadIdx.x % kWave, part = lane / S::W, d = lane % S::W;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int row = S::row_of(i, part);
        const float* x = rows + row * DP + d % 4;
        const int place = d / 4 ^ S::turn(row);
#pragma unroll
        for (int t = 0; t < S::DT; ++t) {
            const float v = x[((8 * t) ^ place) * 4];
            if constexpr (S::W == 32)
                acc[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, w[i], acc[t], 0, 0, 0);
            else
                acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, w[i], acc[t], 0, 0, 0);
        }
    }
}

// over the lanes that share a column
template <int W>
__device__ __forceinline__ float parts_sum(float v) {
    if (W == 16) v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}
template <int W>
__device__ __forceinline__ float parts_max(float v) {
    if (W == 16) v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}

// A column's dimensions out of memory: step s of lane (col, part) holds FN of them from
// (2 s + part) FN on; zeros where `in` is false and beyond `dim`.
template <typename T, int DP>
__device__ __forceinline__ void load_columns(typename Shape<T, DP>::Frag* cols, const T* row, int dim,
                                             bool in, bool negate) {
    typedef Shape<T, DP> S;
    const int part = threadIdx.x % kWave / S::W;
#pragma unroll
    for (int s = 0; s < S::STEPS; ++s) {
        typename S::Frag v = {};
        const int d = (2 * s + part) * S::FN;
        if (in && d < dim) v = *reinterpret_cast<const typename S::Frag*>(row + d);
        cols[s] = negate ? -v : v;
    }
}

// ---------------------------------------------------------------------------
// Causal tiles that some column of the workgroup does not see in whole: a hidden row has
// W = 0, but 0 times an infinity or NaN in its X would still reach the column.  Such a
// tile is looked over when it has arrived (`bad` takes its number); when it holds one, its
// non-finite values are cleared in LDS once the scores are formed, and after the matrix
// product their share is added for the rows that are seen.  All other rows get the same
// bits as from a finite tile.
// ---------------------------------------------------------------------------
__device__ __forceinline__ bool non_finite(float v) {
    return (__float_as_uint(v) & 0x7F800000u) == 0x7F800000u;
}

// Whether a tile holds an infinity or NaN: *bad = tag.  CLEAR: puts zeros in their place.
template <typename T, int DP, int NW, int BN, bool CLEAR>
__device__ __forceinline__ void look_over(T* lds, int* bad, int tag) {
    typedef Shape<T, DP> S;
    typedef typename Vec16<T>::type V;
    bool any = false;
#pragma unroll 1
    for (int at = threadIdx.x; at < BN * S::CPR; at += NW * kWave) {
        V x = reinterpret_cast<V*>(lds)[at];
#pragma unroll
        for (int e = 0; e < S::N; ++e)
            if (non_finite((float)x[e])) {
                any = true;
                x[e] = (T)0.f;
            }
        if (CLEAR && any) reinterpret_cast<V*>(lds)[at] = x;
    }
    if (!CLEAR && any) *bad = tag;
}

// bit i of `seen`: the column sees row r0 + row_of(i, part)
template <typename T, int DP, typename F>
__device__ __forceinline__ void add_non_finite(typename Shape<T, DP>::Acc* acc, f32x16 w, unsigned seen,
                                               int r0, int end, int dim, F addr) {
    typedef Shape<T, DP> S;
    const int lane = threadIdx.x % kWave, part = lane / S::W;
#pragma unroll 1
    for (int i = 0; i < 16; ++i) {
        const float here = w[0];
        w = __builtin_shufflevector(w, w, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15, 0);
#pragma unroll 1
        for (int k = 0; k < S::PARTS; ++k) {
            const float f = __shfl(here, lane % S::W + S::W * k);
            const unsigned sees = __shfl(seen, lane % S::W + S::W * k);
            const int row = r0 + S::row_of(i, k);
            if (row >= end || !((sees >> i) & 1)) continue;
            const T* x = addr(row);
#pragma unroll
            for (int t = 0; t < S::DT; ++t)
#pragma unroll
                for (int e = 0; e < S::AR; ++e) {
                    const int d = 32 * t + S::row_of(e, part);
                    const float v = d < dim ? (float)x[d] : 0.f;
                    if (non_finite(v)) acc[t][e] += f * v;
                    // one value at a time: all of them in flight would take the registers
                    // that the ordinary tiles need
                    asm volatile("" ::: "memory");
                }
        }
    }
}

// Row tiles go from memory straight into LDS (buffer loads with the lds bit: 64 lanes leave
// 64 consecutive vectors), two tiles deep: a tile is loaded while the one before it is
// worked on, without a register in between.  The buffer's size ends with the last row, so
// rows behind it and dimensions behind `dim` arrive as zeros.
typedef int i32x4 __attribute__((ext_vector_type(4)));

// (m0 is on the clobber list so that no value of the compiler's own stays in it across the
// statement; the compiler warns that it would not save m0, which nothing here asks of it)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_to_lds(i32x4 buffer, unsigned offset, unsigned lds) {
    // m0 holds the LDS address; the nops cover scalar operands that a vector instruction wrote
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds),
                 "v"(offset), "s"(buffer)
                 : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

__device__ __forceinline__ i32x4 make_buffer(const void* p, unsigned bytes) {
    const unsigned long long a = reinterpret_cast<unsigned long long>(p);
    i32x4 b;
    b[0] = uniform((int)(unsigned)a);
    b[1] = uniform((int)(unsigned)(a >> 32) & 0xFFFF);
    b[2] = uniform((int)bytes);
    b[3] = 0x00020000;
    return b;
}

__device__ __forceinline__ unsigned lds_address(const void* p) {
    return (unsigned)(unsigned long long)(__attribute__((address_space(3))) const void*)p;
}

template <typename T, int DP, int NW, int BN>
struct Loader {
    typedef Shape<T, DP> S;
    static constexpr int LOADS = (BN * S::CPR + kWave - 1) / kWave;  // of a wave each
    static constexpr int CNT = (LOADS + NW - 1) / NW;
    // A wave's loads lie STEP rows apart; where that is a multiple of 16 they differ by one
    // value for all lanes.
    static constexpr int STEP = NW * kWave % S::CPR == 0 ? NW * kWave / S::CPR : 0;
    static constexpr bool EVEN = CNT == 1 || (STEP > 0 && STEP % 16 == 0);
    unsigned offset[EVEN ? 1 : CNT];  // of this lane's vectors within a tile

    __device__ __forceinline__ void init(long long row_elements, int dim) {
#pragma unroll
        for (int j = 0; j < (EVEN ? 1 : CNT); ++j) {
            const int at = (threadIdx.x / kWave + NW * j) * kWave + threadIdx.x % kWave;
            const int r = at / S::CPR, c = at % S::CPR ^ S::turn(r);
            offset[j] = c * S::N < dim ? (unsigned)(r * (int)row_elements + c * S::N) * (unsigned)sizeof(T)
                                       : 0x80000000u;
        }
    }
    // rows [0, rows) from `base` on, into `lds`
    __device__ __forceinline__ void load(const T* base, int row_elements, int rows, int dim,
                                         T* lds) const {
        const int n = rows < BN ? rows : BN;
        const i32x4 b = make_buffer(base, (unsigned)((n - 1) * row_elements + dim) * (unsigned)sizeof(T));
        const unsigned to = lds_address(lds);
#pragma unroll
        for (int j = 0; j < CNT; ++j) {
            const int k = uniform(threadIdx.x / kWave) + NW * j;
            if (LOADS % NW != 0 && k >= LOADS) break;
            // added to the lane's offset, not as the scalar one: that is no part of what the
            // buffer's size is compared with
            const unsigned more = EVEN ? (unsigned)(j * STEP * row_elements) * (unsigned)sizeof(T) : 0u;
            load_to_lds(b, offset[EVEN ? 0 : j] + more, uniform((int)(to + k * kWave * 16)));
        }
    }
    // The same for rows of the packed (query, head of the group) axis: rows [r0, end), row r
    // being head r % group of query r / group.
    __device__ __forceinline__ void load_packed(const AttnArgs& a, const T* base, const Rows& x, int r0,
                                                int end, T* lds) const {
        const int i0 = uniform(div_group(a, r0));
        const i32x4 b = make_buffer(base + (long long)i0 * x.row, 0x7FFFFFFFu);
        const unsigned to = lds_address(lds);
#pragma unroll
        for (int j = 0; j < CNT; ++j) {
            const int k = uniform(threadIdx.x / kWave) + NW * j;
            if (LOADS % NW != 0 && k >= LOADS) break;
            const int at = k * kWave + threadIdx.x % kWave;
            const int r = r0 + at / S::CPR, i = div_group(a, r);
            const unsigned o = (unsigned)((i - i0) * (int)x.row + (r - i * a.group) * (int)x.head) *
                                   (unsigned)sizeof(T) + offset[EVEN ? 0 : j];
            load_to_lds(b, r < end ? o : 0x80000000u, uniform((int)(to + k * kWave * 16)));
        }
    }
};

// acc[d][col] of one column as a row of U: T, or float32 for partial sums
template <typename T, int DP, typename U>
__device__ __forceinline__ void store_column(U* row, const typename Shape<T, DP>::Acc* acc, float f,
                                             int dim) {
    typedef Shape<T, DP> S;
    const int part = threadIdx.x % kWave / S::W;
    typedef U V4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int t = 0; t < S::DT; ++t)
#pragma unroll
        for (int i = 0; i < S::AR / 4; ++i) {
            const int d = 32 * t + S::row_of(4 * i, part);
            if (d >= dim) continue;
            V4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = (U)(acc[t][4 * i + e] * f);
            *reinterpret_cast<V4*>(row + d) = y;
        }
}

// Scores whose reference m is further than this from 0 (in log2) are subtracted before they
// are scaled: the difference of near floats is exact, while m c is rounded, by 2^-14 here and
// by more than exp2 holds beyond 2^31 (prompts 543 -> 546 us, single tokens 165 -> 166.5 us).
constexpr float kFar = 1024.f;
// The backward has the float32 lse alone, whose rounding is a factor of P: 2^(2^-13) for an lse
// of 1024.  Where it could be 2^(1/2), a row without a gradient is left out (P = 0) and any
// other makes its gradients NaN, not numbers without a digit.
constexpr float kFarthest = 4194304.f;
__device__ __forceinline__ bool beyond_lse(float lse2) {
    return fabsf(lse2) > kFarthest && fabsf(lse2) < INFINITY;
}

constexpr float kRescale = 8.f;  // log2 of how far p may pass 1 before the sums are rescaled

// ---------------------------------------------------------------------------
// Forward: columns = queries, rows = keys.  One pass with a running reference m: p =
// exp(s - m), sums of p and p v; m follows the maximum only when that has grown by over
// 2^8, so most tiles skip the rescaling of the accumulators (p stays far inside float32
// and keeps its relative precision in bf16).  p is rounded to v's type for the second
// product (single waves: in two halves), the sum l uses the unrounded p.
// ---------------------------------------------------------------------------
template <typename T, int DP, int NW, int R>
__global__ __launch_bounds__(NW * kWave, (waves_per_simd<T, DP>(kFwd))) void k_attn_fwd(AttnArgs a) {
    typedef Shape<T, DP> S;
    typedef typename S::Frag Frag;
    typedef typename S::Acc Acc;
    constexpr int W = S::W, ROWS = S::ROWS, BM = W * NW, BN = ROWS * R, SLAB = S::slab(BN);
    __shared__ __align__(16) T lds[4 * SLAB + S::kSlack];  // keys and values, two tiles of each
    __shared__ int bad;
    if (threadIdx.x == 0) bad = 0;
    const Place where = place_of(a);
    // later tiles of a causal sequence take longer: they go first
    const Tile t = tile_of(a.ptr, a.kv_ptr, a.ptr64, a.count, a.nq, a.nk, a.group, BM,
                           gridDim.x - 1 - where.slot);
    const int rows = t.len * a.group;
    if (t.index < 0 || (long long)t.index * BM >= rows) return;
    const int kh = where.kh;
    const int k0 = t.other_first, nk = t.other_len;
    const int lane = threadIdx.x % kWave, part = lane / W;
    const int r0 = t.index * BM + threadIdx.x / kWave * W;
    const int r = r0 + lane % W;
    // the keys that a row sees: [0, limit)
    auto limit = [&](int row) {
        if (!a.causal) return nk;
        const int l = div_group(a, row) + nk - t.len + 1;
        return l < 0 ? 0 : l > nk ? nk : l;
    };
    const bool mine = r < rows;
    const int rc = mine ? r : rows - 1;
    const int qi = div_group(a, rc), gi = rc - qi * a.group;
    const int head = kh * a.group + gi;
    const int lim = limit(rc);
    const int lim_last = uniform(r0 < rows ? limit(r0 + W - 1 < rows ? r0 + W - 1 : rows - 1) : 0);
    const int last = t.index * BM + BM - 1;
    const int lim_block = uniform(limit(last < rows ? last : rows - 1));
    const int lim_whole = uniform(limit(t.index * BM));  // keys that all rows see
    int from = 0, to = lim_block;
    if (a.splits > 1) {
        const int per = ((lim_block + a.splits - 1) / a.splits + BN - 1) / BN * BN;
        from = blockIdx.z * per;
        to = from + per < lim_block ? from + per : lim_block;
    }

    Frag qc[S::STEPS];
    load_columns<T, DP>(qc,
                        static_cast<const T*>(a.q.p) + (long long)(t.first + qi) * a.q.row +
                            (long long)head * a.q.head,
                        a.dim, mine && a.scale != 0.f, a.scale < 0.f);
    const T* kb = static_cast<const T*>(a.k.p) + (long long)k0 * a.k.row + (long long)kh * a.k.head;
    const T* vb = static_cast<const T*>(a.v.p) + (long long)k0 * a.v.row + (long long)kh * a.v.head;
    auto v_at = [&](int row) { return vb + (long long)row * a.v.row; };
    const float c = score_scale(a.scale) * kLog2e;

    Loader<T, DP, NW, BN> kl, vl;
    kl.init(a.k.row, a.dim);
    vl.init(a.v.row, a.dim);
    auto load_tile = [&](int n0, T* to_lds) {
        kl.load(kb + (long long)n0 * a.k.row, (int)a.k.row, nk - n0, a.dim, to_lds);
        vl.load(vb + (long long)n0 * a.v.row, (int)a.v.row, nk - n0, a.dim, to_lds + SLAB);
    };
    Acc acc[S::DT] = {};
    float m = -INFINITY, l = 0.f;
    // One tile.  MASK: some column may not see all of its rows; mend: and a hidden one may
    // hold an infinity or NaN.
    auto tile = [&](int n0, const T* lk, const T* lv, auto masks, bool mend) {
        constexpr bool MASK = decltype(masks)::value;
        schedule<T, MASK>();
        f32x16 s[R];
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < R; ++j) {
            s[j] = scores<T, DP>(lk + S::slab(ROWS * j), qc);
            if (MASK) {  // row_of(i, part) = row_of(i, 0) + 4 part: constants on one side
                const int left = lim - n0 - 4 * part;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (ROWS * j + S::row_of(i, 0) >= left) s[j][i] = -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[j][i]);
        }
        mx = parts_max<W>(mx);
        if (__any((mx - m) * c > kRescale)) {  // -inf - -inf: false
            const float to_m = fmaxf(m, mx);
            const float f = m == -INFINITY ? 0.f : exp2f((m - to_m) * c);
            m = to_m;
            l *= f;
#pragma unroll
            for (int d = 0; d < S::DT; ++d) acc[d] *= f;
        }
        float mc = m == -INFINITY ? 0.f : m * c;
        if (__any(fabsf(mc) > kFar && m < INFINITY)) {
            const float ref = m == -INFINITY ? 0.f : m;
            mc = 0.f;
#pragma unroll
            for (int j = 0; j < R; ++j) s[j] -= ref;
        }
#pragma unroll
        for (int j = 0; j < R; ++j) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[j][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][i], c, -mc));
                l += s[j][i];
            }
            // Single waves wait for memory, not for products: what rounding p leaves goes in too
            // (one query each of 48 sequences: y off by 1.64e-3 of its norm, its own rounding,
            // for 2.2e-3; 164 us for 162).  Elsewhere p is rounded once, which leaves y off by
            // 2.1e-3, because the second product would cost more than its rounding is worth:
            // prompts 735 us for 544, 12 sequences with heads of 64, training, 260 us for 246,
            // graphs with 8 heads of 32 73 us for 66 (forward), with 8 heads of 8 228 us for 220.
            add_products<DP, NW == 1>(acc, lv + S::slab(ROWS * j), s[j]);
            if (MASK && mend) {
                unsigned seen = 0;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    seen |= (n0 + ROWS * j + S::row_of(i, part) < lim ? 1u : 0u) << i;
                add_non_finite<T, DP>(acc, s[j], seen, n0 + ROWS * j, nk, a.dim, v_at);
            }
        }
    };
    const int whole = lim_whole < to ? lim_whole : to;  // tiles up to here need no mask
    int n0 = from, turn = 0;
    auto arrive = [&]() {  // tile n0 is in LDS, the next one on its way
        wait_loads();
        __syncthreads();
        if (n0 + BN < to) load_tile(n0 + BN, lds + 2 * SLAB * (turn ^ 1));
        return lds + 2 * SLAB * turn;
    };
    if (from < to) load_tile(from, lds);
    for (; n0 + BN <= whole; n0 += BN, turn ^= 1) {
        const T* at = arrive();
        tile(n0, at, at + SLAB, std::false_type(), false);
    }
    for (; n0 < to; n0 += BN, turn ^= 1) {
        T* at = arrive();
        bool mend = false;
        if (a.causal) {
            look_over<T, DP, NW, BN, false>(at + SLAB, &bad, n0 + 1);
            __syncthreads();
            mend = bad == n0 + 1;
        }
        if (mend) {
            look_over<T, DP, NW, BN, true>(at + SLAB, nullptr, 0);
            __syncthreads();
        }
        if (n0 < lim_last) tile(n0, at, at + SLAB, std::true_type(), mend);
    }
    l = parts_sum<W>(l);
    if (!mine) return;
    const long long qh = (long long)(t.first + qi) * a.kv_heads * a.group + head;
    if (a.splits > 1) {
        const long long at = (long long)blockIdx.z * a.nq * a.kv_heads * a.group + qh;
        store_column<T, DP>(a.part + at * a.dim, acc, 1.f, a.dim);
        float* ml = a.part + (long long)a.splits * a.nq * a.kv_heads * a.group * a.dim;
        if (part == 0) {
            ml[2 * at] = m;
            ml[2 * at + 1] = lim == 0 && blockIdx.z == 0 ? 1.f : l;  // no key: 0 / 1, not 0 / 0
        }
        return;
    }
    T* out = static_cast<T*>(const_cast<void*>(a.o.p)) + (long long)(t.first + qi) * a.o.row +
             (long long)head * a.o.head;
    if (lim == 0) {  // sees no key
#pragma unroll
        for (int d = 0; d < S::DT; ++d) acc[d] = Acc{};
        l = 1.f;
    }
    store_column<T, DP>(out, acc, 1.f / l, a.dim);
    if constexpr (sizeof(T) == 2) {
        if (a.low != nullptr) {
            const float f = 1.f / l;
#pragma unroll
            for (int d = 0; d < S::DT; ++d)
#pragma unroll
                for (int i = 0; i < S::AR; ++i) {
                    const float y = acc[d][i] * f;
                    acc[d][i] = y - (float)(T)y;
                }
            store_column<T, DP>(static_cast<T*>(a.low) + qh * a.dim, acc, 1.f, a.dim);
        }
    }
    if (a.lse != nullptr && part == 0)
        a.lse[qh] = lim == 0 ? -INFINITY : m * score_scale(a.scale) + logf(l);
}

// Joins the forward's splits: y = sum_s f_s acc_s / sum_s f_s l_s, f_s = exp(m_s - max m).
template <typename T>
__global__ __launch_bounds__(256) void k_attn_join(AttnArgs a) {
    const int quads = a.dim / 4;
    const long long n = (long long)a.nq * a.kv_heads * a.group;
    const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
    if (at >= n * quads) return;
    const long long qh = at / quads;
    const int d = (int)(at % quads) * 4;
    const float* ml = a.part + a.splits * n * a.dim;
    float m = -INFINITY;
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) m = fmaxf(m, ml[2 * (s * n + qh)]);
    const float c = score_scale(a.scale) * kLog2e;
    float l = 0.f;
    f32x4 acc = {};
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) {
        const long long i = s * n + qh;
        const float f = m == -INFINITY ? 1.f : exp2f((ml[2 * i] - m) * c);
        l += f * ml[2 * i + 1];
        acc = fma4(f, *reinterpret_cast<const f32x4*>(a.part + i * a.dim + d), acc);
    }
    const long long tok = qh / (a.kv_heads * a.group), head = qh % (a.kv_heads * a.group);
    T* out = static_cast<T*>(const_cast<void*>(a.o.p)) + tok * a.o.row + head * a.o.head + d;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float y = acc[e] / l;
        out[e] = (T)y;
        if (sizeof(T) == 2 && a.low != nullptr) static_cast<T*>(a.low)[qh * a.dim + d + e] = (T)(y - (float)(T)y);
    }
    if (a.lse != nullptr && d == 0)
        a.lse[qh] = m == -INFINITY ? -INFINITY : m * score_scale(a.scale) + logf(l);
}

// out[i] = scale * sum over the splits, of one tensor's partial sums
template <typename T>
__global__ __launch_bounds__(256) void k_attn_sum(const float* part, int splits, long long step,
                                                  long long n, float scale, T* out) {
    const long long at = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (at >= n) return;
    f32x4 s = {};
#pragma unroll 4
    for (int k = 0; k < splits; ++k) s += *reinterpret_cast<const f32x4*>(part + k * step + at);
#pragma unroll
    for (int e = 0; e < 4; ++e) out[at + e] = (T)(s[e] * scale);
}

// ---------------------------------------------------------------------------
// dq: columns = queries, rows = keys.  P comes back from the scores and lse; dS is
// rounded to k's type for the product with k.  sum_d g y is formed here, in float32, and
// left for the dk/dv kernel.
// ---------------------------------------------------------------------------
template <typename T, int DP, int NW, int R>
__global__ __launch_bounds__(NW * kWave, (waves_per_simd<T, DP>(kDq))) void k_attn_dq(AttnArgs a) {
    typedef Shape<T, DP> S;
    typedef typename S::Frag Frag;
    typedef typename S::Acc Acc;
    constexpr int W = S::W, ROWS = S::ROWS, BM = W * NW, BN = ROWS * R, SLAB = S::slab(BN);
    __shared__ __align__(16) T lds[4 * SLAB + S::kSlack];
    __shared__ int bad;
    if (threadIdx.x == 0) bad = 0;
    const Place where = place_of(a);
    // later tiles of a causal sequence take longer: they go first
    const Tile t = tile_of(a.ptr, a.kv_ptr, a.ptr64, a.count, a.nq, a.nk, a.group, BM,
                           gridDim.x - 1 - where.slot);
    const int rows = t.len * a.group;
    if (t.index < 0 || (long long)t.index * BM >= rows) return;
    const int kh = where.kh;
    const int k0 = t.other_first, nk = t.other_len;
    const int lane = threadIdx.x % kWave, part = lane / W;
    const int r0 = t.index * BM + threadIdx.x / kWave * W;
    const int r = r0 + lane % W;
    // the keys that a row sees: [0, limit)
    auto limit = [&](int row) {
        if (!a.causal) return nk;
        const int l = div_group(a, row) + nk - t.len + 1;
        return l < 0 ? 0 : l > nk ? nk : l;
    };
    const bool mine = r < rows;
    const int rc = mine ? r : rows - 1;
    const int qi = div_group(a, rc), gi = rc - qi * a.group;
    const int head = kh * a.group + gi;
    const int lim = limit(rc);
    const int lim_last = uniform(r0 < rows ? limit(r0 + W - 1 < rows ? r0 + W - 1 : rows - 1) : 0);
    const int last = t.index * BM + BM - 1;
    const int lim_block = uniform(limit(last < rows ? last : rows - 1));
    const int lim_whole = uniform(limit(t.index * BM));  // keys that all rows see
    int from = 0, to = lim_block;
    if (a.splits > 1) {
        const int per = ((lim_block + a.splits - 1) / a.splits + BN - 1) / BN * BN;
        from = blockIdx.z * per;
        to = from + per < lim_block ? from + per : lim_block;
    }

    Frag qc[S::STEPS], gc[S::STEPS];
    const long long tok = t.first + qi;
    const long long qh = tok * a.kv_heads * a.group + head;
    load_columns<T, DP>(qc, static_cast<const T*>(a.q.p) + tok * a.q.row + (long long)head * a.q.head,
                        a.dim, mine && a.scale != 0.f, a.scale < 0.f);
    load_columns<T, DP>(gc, static_cast<const T*>(a.g.p) + tok * a.g.row + (long long)head * a.g.head,
                        a.dim, mine, false);
    // From y and, in bf16, what its rounding left: the rounding alone would be the larger part
    // of dq's error where few keys are seen (measured at 64 to 1000 keys: 3.0e-3 to 2.5e-3 of
    // dq's norm against 2.3e-3 to 2.45e-3)
    float delta = 0.f;
    auto add_delta = [&](const T* from_row) {
        Frag oc[S::STEPS];
        load_columns<T, DP>(oc, from_row, a.dim, mine, false);
#pragma unroll
        for (int s = 0; s < S::STEPS; ++s)
#pragma unroll
            for (int e = 0; e < S::FN; ++e) delta = fmaf((float)gc[s][e], (float)oc[s][e], delta);
    };
    if (sizeof(T) == 2 && a.low != nullptr) add_delta(static_cast<const T*>(a.low) + qh * a.dim);
    add_delta(static_cast<const T*>(a.o.p) + tok * a.o.row + (long long)head * a.o.head);
    delta = parts_sum<W>(delta);
    float lse2 = mine ? a.lse[qh] * kLog2e : 0.f, some = 0.f;
#pragma unroll
    for (int s = 0; s < S::STEPS; ++s)
#pragma unroll
        for (int e = 0; e < S::FN; ++e) some = fmaxf(some, fabsf((float)gc[s][e]));
    some = parts_max<W>(some);
    if (beyond_lse(lse2)) {
        lse2 = INFINITY;
        if (some > 0.f) delta = NAN;
    }
    if (mine && part == 0 && blockIdx.z == 0) a.delta[qh] = delta;
    const T* kb = static_cast<const T*>(a.k.p) + (long long)k0 * a.k.row + (long long)kh * a.k.head;
    const T* vb = static_cast<const T*>(a.v.p) + (long long)k0 * a.v.row + (long long)kh * a.v.head;
    auto k_at = [&](int row) { return kb + (long long)row * a.k.row; };
    const float c = score_scale(a.scale) * kLog2e;

    Loader<T, DP, NW, BN> kl, vl;
    kl.init(a.k.row, a.dim);
    vl.init(a.v.row, a.dim);
    auto load_tile = [&](int n0, T* to_lds) {
        kl.load(kb + (long long)n0 * a.k.row, (int)a.k.row, nk - n0, a.dim, to_lds);
        vl.load(vb + (long long)n0 * a.v.row, (int)a.v.row, nk - n0, a.dim, to_lds + SLAB);
    };
    Acc acc[S::DT] = {};
    auto tile = [&](int n0, T* lk, const T* lv, auto masks, bool mend) {
        constexpr bool MASK = decltype(masks)::value;
        schedule<T, MASK>();
        f32x16 s[R], dp[R];
        const int left = lim - n0 - 4 * part;
#pragma unroll
        for (int j = 0; j < R; ++j) {
            s[j] = scores<T, DP>(lk + S::slab(ROWS * j), qc);
            dp[j] = scores<T, DP>(lv + S::slab(ROWS * j), gc);
        }
#pragma unroll
        for (int j = 0; j < R; ++j) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][i], c, -lse2));
                s[j][i] = p * (dp[j][i] - delta);
                if (MASK && ROWS * j + S::row_of(i, 0) >= left) s[j][i] = 0.f;
            }
        }
        if (MASK && mend) {  // the scores need the keys as they are, the product needs them cleared
            __syncthreads();
            look_over<T, DP, NW, BN, true>(lk, nullptr, 0);
            __syncthreads();
        }
#pragma unroll
        for (int j = 0; j < R; ++j) {
            // Narrow heads are bound by latency, not by products: what rounding dS leaves goes
            // in too (512 graphs of 85 to 150 nodes, 8 heads of 8, training: dq off by 1.8e-3
            // of its norm, of which 1.7e-3 its own rounding, for 2.6e-3; 220 us for 215).
            // Wider ones round it once, dq off by 2.4e-3 (1.7e-3 with both halves; 12 sequences,
            // heads of 64: 259 us for 246, heads of 128: 1126 us for 1074).
            add_products<DP, DP <= 32>(acc, lk + S::slab(ROWS * j), s[j]);
            if (MASK && mend) {
                unsigned seen = 0;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    seen |= (n0 + ROWS * j + S::row_of(i, part) < lim ? 1u : 0u) << i;
                add_non_finite<T, DP>(acc, s[j], seen, n0 + ROWS * j, nk, a.dim, k_at);
            }
        }
    };
    const int whole = lim_whole < to ? lim_whole : to;
    int n0 = from, turn = 0;
    auto arrive = [&]() {
        wait_loads();
        __syncthreads();
        if (n0 + BN < to) load_tile(n0 + BN, lds + 2 * SLAB * (turn ^ 1));
        return lds + 2 * SLAB * turn;
    };
    if (from < to) load_tile(from, lds);
    for (; n0 + BN <= whole; n0 += BN, turn ^= 1) {
        T* at = arrive();
        tile(n0, at, at + SLAB, std::false_type(), false);
    }
    for (; n0 < to; n0 += BN, turn ^= 1) {
        T* at = arrive();
        bool mend = false;
        if (a.causal) {
            look_over<T, DP, NW, BN, false>(at, &bad, n0 + 1);
            __syncthreads();
            mend = bad == n0 + 1;
        }
        if (n0 < lim_last || mend) tile(n0, at, at + SLAB, std::true_type(), mend);
    }
    if (!mine) return;
    if (a.splits > 1) {
        const long long at = (long long)blockIdx.z * a.nq * a.kv_heads * a.group + qh;
        store_column<T, DP>(a.part + at * a.dim, acc, 1.f, a.dim);
        return;
    }
    store_column<T, DP>(static_cast<T*>(const_cast<void*>(a.dq.p)) + tok * a.dq.row +
                            (long long)head * a.dq.head,
                        acc, a.scale, a.dim);
}

// ---------------------------------------------------------------------------
// dk, dv: columns = keys, rows = (query, head of the group).
// ---------------------------------------------------------------------------
template <typename T, int DP, int NW, int R>
__global__ __launch_bounds__(NW * kWave, (waves_per_simd<T, DP>(kDkv))) void k_attn_dkv(AttnArgs a) {
    typedef Shape<T, DP> S;
    typedef typename S::Frag Frag;
    typedef typename S::Acc Acc;
    constexpr int W = S::W, ROWS = S::ROWS, BM = W * NW, BN = ROWS * R, SLAB = S::slab(BN);
    __shared__ __align__(16) T lds[4 * SLAB + S::kSlack];  // q and g, two tiles of each
    __shared__ __align__(16) float sums[2 * 2 * BN];               // lse and delta of their rows
    __shared__ int bad;
    if (threadIdx.x == 0) bad = 0;
    const Place where = place_of(a);
    const Tile t = tile_of(a.kv_ptr, a.ptr, a.ptr64, a.count, a.nk, a.nq, 1, BM, where.slot);
    if (t.index < 0 || (long long)t.index * BM >= t.len) return;
    const int kh = where.kh;
    const int q0 = t.other_first, nq = t.other_len;
    const int rows = nq * a.group;
    const int lane = threadIdx.x % kWave, part = lane / W;
    const int c0 = t.index * BM + threadIdx.x / kWave * W;
    const int key = c0 + lane % W;
    const bool mine = key < t.len;
    const int kc = mine ? key : t.len - 1;
    // the rows that see a key: [start, rows)
    auto start = [&](int k) {
        if (!a.causal) return 0;
        const int i = k - (t.len - nq);
        return i < 0 ? 0 : i >= nq ? rows : i * a.group;
    };
    const int beg = start(kc);
    const int beg_first = uniform(c0 < t.len ? start(c0) : rows);  // the wave's smallest
    // the first row from which on all of the workgroup's keys are seen
    const int beg_whole = start(t.index * BM + BM - 1 < t.len ? t.index * BM + BM - 1 : t.len - 1);
    int from = start(t.index * BM) / BN * BN, to = rows;
    if (a.splits > 1) {
        const int per = ((rows - from + a.splits - 1) / a.splits + BN - 1) / BN * BN;
        from += blockIdx.z * per;
        to = from + per < rows ? from + per : rows;
    }

    Frag kcol[S::STEPS], vcol[S::STEPS];
    const long long tok = t.first + kc;
    load_columns<T, DP>(kcol, static_cast<const T*>(a.k.p) + tok * a.k.row + (long long)kh * a.k.head,
                        a.dim, mine && a.scale != 0.f, a.scale < 0.f);
    load_columns<T, DP>(vcol, static_cast<const T*>(a.v.p) + tok * a.v.row + (long long)kh * a.v.head,
                        a.dim, mine, false);
    // Rows behind the last arrive as zeros and have p = exp(0 - inf) = 0, but zero times a key's
    // infinity is NaN: the last tile of a wave with such a key is masked.
    float zero = 0.f;
#pragma unroll
    for (int i = 0; i < S::STEPS; ++i)
#pragma unroll
        for (int e = 0; e < S::FN; ++e) zero = fmaf((float)kcol[i][e], 0.f, fmaf((float)vcol[i][e], 0.f, zero));
    const bool odd = __any(zero != 0.f);
    const T* qb = static_cast<const T*>(a.q.p) + (long long)q0 * a.q.row +
                  (long long)kh * a.group * a.q.head;
    const T* gb = static_cast<const T*>(a.g.p) + (long long)q0 * a.g.row +
                  (long long)kh * a.group * a.g.head;
    auto q_at = [&](int row) {
        const int i = div_group(a, row);
        return qb + (long long)i * a.q.row + (long long)(row - i * a.group) * a.q.head;
    };
    auto g_at = [&](int row) {
        const int i = div_group(a, row);
        return gb + (long long)i * a.g.row + (long long)(row - i * a.group) * a.g.head;
    };
    // lse and delta of a row tile
    constexpr int NT = NW * kWave, PER = (BN + NT - 1) / NT;
    float rl[PER], rd[PER];
    auto load_sums = [&](int n0) {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int row = n0 + j * NT + threadIdx.x;
            const bool in = j * NT + threadIdx.x < BN && row < rows;
            const int i = in ? div_group(a, row) : 0;
            const long long qh =
                in ? ((long long)(q0 + i) * a.kv_heads + kh) * a.group + (row - i * a.group) : 0;
            rl[j] = in ? a.lse[qh] : INFINITY;  // exp(s - inf) = 0 behind the last row
            rd[j] = in ? a.delta[qh] : 0.f;
        }
    };
    const float c = score_scale(a.scale) * kLog2e;

    Loader<T, DP, NW, BN> ld;
    ld.init(0, a.dim);
    auto load_tile = [&](int n0, T* to_lds) {
        ld.load_packed(a, qb, a.q, n0, rows, to_lds);
        ld.load_packed(a, gb, a.g, n0, rows, to_lds + SLAB);
    };
    Acc dk[S::DT] = {}, dv[S::DT] = {};
    auto tile = [&](int n0, T* lq, T* lg, const float* ll, auto masks, bool mend) {
        constexpr bool MASK = decltype(masks)::value;
        schedule<T, MASK>();
        f32x16 p[R], ds[R];
        const int hidden = beg - n0 - 4 * part, behind = rows - n0 - 4 * part;
#pragma unroll
        for (int j = 0; j < R; ++j) {
            p[j] = scores<T, DP>(lq + S::slab(ROWS * j), kcol);
            ds[j] = scores<T, DP>(lg + S::slab(ROWS * j), vcol);
        }
#pragma unroll
        for (int j = 0; j < R; ++j)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const f32x4 l4 = *reinterpret_cast<const f32x4*>(ll + ROWS * j + S::row_of(4 * b, part));
                const f32x4 d4 = *reinterpret_cast<const f32x4*>(ll + BN + ROWS * j + S::row_of(4 * b, part));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = 4 * b + e;
                    p[j][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[j][i], c, -l4[e]));
                    ds[j][i] = p[j][i] * (ds[j][i] - d4[e]);
                    const int r = ROWS * j + S::row_of(i, 0);
                    if (MASK && (r < hidden || r >= behind)) p[j][i] = ds[j][i] = 0.f;
                }
            }
        if (MASK && mend) {
            __syncthreads();
            look_over<T, DP, NW, BN, true>(lq, nullptr, 0);
            look_over<T, DP, NW, BN, true>(lg, nullptr, 0);
            __syncthreads();
        }
#pragma unroll
        for (int j = 0; j < R; ++j) {
            // P and dS are rounded to g's and q's type here: dk off by 2.4e-3 of its norm and dv by
            // 2.3e-3, their own rounding 1.7e-3 of it.  Both halves would leave just that, for
            // 283 us instead of 246 (12 sequences, heads of 64, training), 1156 instead of 1074
            // (heads of 128) and 237 instead of 220 (graphs, 8 heads of 8): two more products
            // a tile, not one as in dq.
            add_products<DP>(dv, lg + S::slab(ROWS * j), p[j]);
            add_products<DP>(dk, lq + S::slab(ROWS * j), ds[j]);
            if (MASK && mend) {
                const int n = n0 + ROWS * j;
                unsigned seen = 0;
#pragma unroll
                for (int i = 0; i < 16; ++i) seen |= (n + S::row_of(i, part) >= beg ? 1u : 0u) << i;
                add_non_finite<T, DP>(dv, p[j], seen, n, rows, a.dim, g_at);
                add_non_finite<T, DP>(dk, ds[j], seen, n, rows, a.dim, q_at);
            }
        }
    };
    int n0 = from, turn = 0;
    auto arrive = [&]() {
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (j * NT + threadIdx.x < BN) {
                const float l = rl[j] * kLog2e;
                sums[turn * 2 * BN + j * NT + threadIdx.x] =
                    beyond_lse(l) ? rd[j] == 0.f ? INFINITY : NAN : l;
                sums[(turn * 2 + 1) * BN + j * NT + threadIdx.x] = rd[j];
            }
        wait_loads();
        __syncthreads();
        if (n0 + BN < to) {
            load_sums(n0 + BN);
            load_tile(n0 + BN, lds + 2 * SLAB * (turn ^ 1));
        }
        return lds + 2 * SLAB * turn;
    };
    if (from < to) {
        load_sums(from);
        load_tile(from, lds);
    }
    for (; n0 < to && n0 < beg_whole; n0 += BN, turn ^= 1) {  // causal: the first tiles
        T* at = arrive();
        look_over<T, DP, NW, BN, false>(at, &bad, n0 + 1);
        look_over<T, DP, NW, BN, false>(at + SLAB, &bad, n0 + 1);
        __syncthreads();
        const bool mend = bad == n0 + 1;
        if (n0 + BN > beg_first || mend)
            tile(n0, at, at + SLAB, sums + turn * 2 * BN, std::true_type(), mend);
    }
    const int whole = odd ? to - BN + 1 : to;
    for (; n0 < whole; n0 += BN, turn ^= 1) {
        T* at = arrive();
        tile(n0, at, at + SLAB, sums + turn * 2 * BN, std::false_type(), false);
    }
    if (n0 < to) {
        T* at = arrive();
        tile(n0, at, at + SLAB, sums + turn * 2 * BN, std::true_type(), false);
    }
    if (!mine) return;
    if (a.splits > 1) {
        const long long n = (long long)a.nk * a.kv_heads;
        const long long at = (long long)blockIdx.z * n + tok * a.kv_heads + kh;
        store_column<T, DP>(a.part + at * a.dim, dk, 1.f, a.dim);
        store_column<T, DP>(a.part + (a.splits * n + at) * a.dim, dv, 1.f, a.dim);
        return;
    }
    store_column<T, DP>(static_cast<T*>(const_cast<void*>(a.dk.p)) + tok * a.dk.row +
                            (long long)kh * a.dk.head, dk, a.scale, a.dim);
    store_column<T, DP>(static_cast<T*>(const_cast<void*>(a.dv.p)) + tok * a.dv.row +
                            (long long)kh * a.dv.head, dv, 1.f, a.dim);
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

// A launch's waves per workgroup and its splits of the streamed axis, from the average
// lengths (the lengths themselves are on the device).  One sequence far longer than the rest of a
// large batch is therefore streamed by as few waves as the others: of a thousand single queries,
// 999 over ten keys and one over 100,000, the long one is one wave's.
struct Plan {
    int waves, splits;
};

// The columns of a wave (Shape::W) for these heads.
inline int wave_columns(int dim, int dtype) { return dtype == GAT_F32 && dim <= 16 ? 16 : 32; }

// cols: rows of the axis whose tiles the grid walks; streamed: the other's; w: wave_columns;
// want_waves: a SIMD's, below which the streamed axis is split.
inline Plan plan_of(long long cols, long long streamed, int count, int kv_heads, int w,
                    int want_waves) {
    const int n = count > 0 ? count : 1;
    auto tiles = [&](int waves) {
        return std::max<long long>(n, (cols + w * waves - 1) / (w * waves)) * kv_heads;
    };
    Plan p;
    // A workgroup shares its row tiles between its waves; short sequences fill one or two,
    // and fewer than 4 workgroups a CU leave CUs idle behind the longest.
    p.waves = cols <= (long long)w * n ? 1 : cols <= 2ll * w * n || tiles(4) < 4 * 256 ? 2 : 4;
    // Split into 256 rows or more each.
    const long long waves = tiles(p.waves) * p.waves;
    const long long want = (want_waves * 4ll * 256 + waves - 1) / waves;
    p.splits = (int)std::max<long long>(1, std::min<long long>({want, streamed / n / 256, 128}));
    return p;
}

struct AttnSizes {
    Plan fwd, dq, dkv;
    size_t fwd_bytes, delta_bytes, dq_bytes, dkv_bytes;
};

inline AttnSizes attn_sizes(long long nq, long long nk, int count, int heads, int kv_heads, int dim,
                            int dtype) {
    AttnSizes s;
    const int group = heads / kv_heads;
    const int w = wave_columns(dim, dtype);
    // dk and dv stream `group` rows for each query, so that the first keys of a long causal
    // sequence outlast the rest: more splits (a packed training batch: 3 waves 262 us, 6 255 us,
    // 9 268 us)
    s.fwd = plan_of(nq * group, nk, count, kv_heads, w, 3);
    s.dq = s.fwd;
    s.dkv = plan_of(nk, nq * group, count, kv_heads, w, 6);
    const size_t q = (size_t)nq * heads, k = (size_t)nk * kv_heads;
    s.fwd_bytes = s.fwd.splits > 1 ? s.fwd.splits * q * (dim + 2) * sizeof(float) : 0;
    s.delta_bytes = align_up(q * sizeof(float));
    s.dq_bytes = s.dq.splits > 1 ? s.dq.splits * q * dim * sizeof(float) : 0;
    s.dkv_bytes = s.dkv.splits > 1 ? 2 * s.dkv.splits * k * dim * sizeof(float) : 0;
    return s;
}

// What the kernels need of a call's sizes and layouts.
inline int attn_check(int nq, int nk, int count, int heads, int kv_heads, int dim, int dtype) {
    if (nq < 0 || nk < 0 || count < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 ||
        dim <= 0 || (dtype != GAT_F32 && dtype != GAT_BF16))
        return GAT_EINVAL;
    if (dim > GAT_PACKED_MAX_DIM || dim % (16 / (int)dtype_size(dtype)) != 0 ||
        (long long)nq * (heads / kv_heads) > 0x3FFFFFFF || nk > 0x3FFFFFFF || count > 0x3FFFFFFF ||
        kv_heads > 65535)
        return GAT_EUNSUPPORTED;
    return GAT_OK;
}

// group: the heads that a tile's offsets span (q and its like), 0 where each has its own base
inline bool vec_rows(const Rows& r, int dim, int group, int dtype) {
    const int n = 16 / (int)dtype_size(dtype);
    return (reinterpret_cast<uintptr_t>(r.p) & 15) == 0 && r.row % n == 0 && r.head % n == 0 &&
           r.row >= dim && r.row <= (1 << 22) && r.head >= 0 &&
           r.head * group <= (1 << 28);  // offsets within a tile fit 31 bits of bytes
}

inline void set_group(AttnArgs& a, int group) {
    a.group = group;
    int s = 0;  // row / group = umulhi(row, mul) >> shift for rows below 2^31
    while ((1 << (s + 1)) < group) ++s;
    a.div_shift = s;
    a.div_mul = group == 1 ? 0 : (unsigned)(((1ull << (32 + s)) + group - 1) / group);
}

template <typename T, int DP, AttnPass PASS>
int attn_launch(const AttnArgs& a, const Plan& p, hipStream_t s) {
    const bool keys = PASS == kDkv;
    const long long need = slots_of(keys ? a.nk : a.nq, keys ? 1 : a.group, Shape<T, DP>::W * p.waves, a.count);
    const long long slots = a.by_xcd ? (need + 7) / 8 * 8 : need;
    if (slots * 64 * p.waves > 0xFFFFFFFFll) return GAT_EUNSUPPORTED;  // lanes of one launch
    const dim3 grid((unsigned)slots, a.kv_heads, p.splits);
    // row tiles a step: two where the registers allow it (their chains interleave)
    constexpr int R = sizeof(T) == 4 ? 1 : PASS == kFwd || DP <= 64 ? 2 : 1;
    auto call = [&](auto waves) {
        constexpr int NW = decltype(waves)::value;
        if constexpr (PASS == kFwd) k_attn_fwd<T, DP, NW, NW == 4 ? R : 1><<<grid, 64 * NW, 0, s>>>(a);
        if constexpr (PASS == kDq) k_attn_dq<T, DP, NW, R><<<grid, 64 * NW, 0, s>>>(a);
        if constexpr (PASS == kDkv) k_attn_dkv<T, DP, NW, R><<<grid, 64 * NW, 0, s>>>(a);
    };
    if (p.waves == 1)
        call(std::integral_constant<int, 1>());
    else if (p.waves == 2)
        call(std::integral_constant<int, 2>());
    else
        call(std::integral_constant<int, 4>());
    return status_of(hipGetLastError());
}

template <typename T, AttnPass PASS>
int attn_by_dim(const AttnArgs& a, const Plan& p, hipStream_t s) {
    if constexpr (sizeof(T) == 4) {
        if (a.dim <= 8) return attn_launch<T, 8, PASS>(a, p, s);
    }
    if (a.dim <= 16) return attn_launch<T, 16, PASS>(a, p, s);
    if (a.dim <= 32) return attn_launch<T, 32, PASS>(a, p, s);
    if (a.dim <= 64) return attn_launch<T, 64, PASS>(a, p, s);
    if (a.dim <= 96) return attn_launch<T, 96, PASS>(a, p, s);
    return attn_launch<T, 128, PASS>(a, p, s);
}

template <AttnPass PASS>
int attn_pass(AttnArgs& a, const Plan& p, int dtype, hipStream_t s) {
    a.splits = p.splits;
    a.by_xcd = p.waves > 1 && (a.kv_heads % 8 == 0 || 8 % a.kv_heads == 0);
    return dtype == GAT_F32 ? attn_by_dim<float, PASS>(a, p, s) : attn_by_dim<bf16, PASS>(a, p, s);
}

template <typename T>
int attn_sum(const float* part, int splits, long long n, float scale, const Rows& out,
             hipStream_t s) {
    if (n == 0) return GAT_OK;
    k_attn_sum<T><<<(unsigned)((n / 4 + 255) / 256), 256, 0, s>>>(
        part, splits, n, n, scale, static_cast<T*>(const_cast<void*>(out.p)));
    return status_of(hipGetLastError());
}

}  // namespace

extern "C" {

int gat_packed_attention_workspace_size(int nq, int nk, int count, int heads, int kv_heads, int dim,
                                        int dtype, size_t* bytes) {
    const int rc = attn_check(nq, nk, count, heads, kv_heads, dim, dtype);
    if (rc != GAT_OK) return rc;
    if (bytes == nullptr) return GAT_EINVAL;
    *bytes = attn_sizes(nq, nk, count, heads, kv_heads, dim, dtype).fwd_bytes;
    return GAT_OK;
}

int gat_packed_attention(const void* q, long long q_row, long long q_head, const void* k,
                         long long k_row, long long k_head, const void* v, long long v_row,
                         long long v_head, const void* ptr, const void* kv_ptr, int ptr64, int count,
                         int nq, int nk, int heads, int kv_heads, int dim, float scale, int causal,
                         void* out, void* low, float* lse, void* workspace, size_t workspace_bytes,
                         int dtype, void* stream) {
    const int rc = attn_check(nq, nk, count, heads, kv_heads, dim, dtype);
    if (rc != GAT_OK) return rc;
    if (nq == 0) return GAT_OK;
    AttnArgs a{};
    a.q = {q, q_row, q_head};
    a.k = {k, k_row, k_head};
    a.v = {v, v_row, v_head};
    a.o = {out, (long long)heads * dim, dim};
    if (q == nullptr || out == nullptr || ptr == nullptr || kv_ptr == nullptr ||
        (nk > 0 && (k == nullptr || v == nullptr)))
        return GAT_EINVAL;
    for (const Rows* r : {&a.q, &a.o})
        if (!vec_rows(*r, dim, heads / kv_heads, dtype)) return GAT_EUNSUPPORTED;
    for (const Rows* r : {&a.k, &a.v})
        if (!vec_rows(*r, dim, 0, dtype)) return GAT_EUNSUPPORTED;
    const AttnSizes sz = attn_sizes(nq, nk, count, heads, kv_heads, dim, dtype);
    if (sz.fwd_bytes > 0 && (workspace == nullptr || workspace_bytes < sz.fwd_bytes))
        return GAT_EWORKSPACE;
    if (((reinterpret_cast<uintptr_t>(workspace) | reinterpret_cast<uintptr_t>(low)) & 15) != 0)
        return GAT_EINVAL;
    a.ptr = ptr;
    a.kv_ptr = kv_ptr;
    a.ptr64 = ptr64;
    a.count = count;
    a.nq = nq;
    a.nk = nk;
    a.kv_heads = kv_heads;
    set_group(a, heads / kv_heads);
    a.dim = dim;
    a.scale = scale;
    a.causal = causal;
    a.lse = lse;
    a.low = dtype == GAT_F32 ? nullptr : low;
    a.part = static_cast<float*>(workspace);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int st = attn_pass<kFwd>(a, sz.fwd, dtype, s);
    if (st != GAT_OK || sz.fwd.splits == 1) return st;
    const long long work = (long long)nq * heads * (dim / 4);
    const unsigned grid = (unsigned)((work + 255) / 256);
    if (dtype == GAT_F32)
        k_attn_join<float><<<grid, 256, 0, s>>>(a);
    else
        k_attn_join<bf16><<<grid, 256, 0, s>>>(a);
    return status_of(hipGetLastError());
}

int gat_packed_attention_backward_workspace_size(int nq, int nk, int count, int heads, int kv_heads,
                                                 int dim, int dtype, size_t* bytes) {
    const int rc = attn_check(nq, nk, count, heads, kv_heads, dim, dtype);
    if (rc != GAT_OK) return rc;
    if (bytes == nullptr) return GAT_EINVAL;
    const AttnSizes s = attn_sizes(nq, nk, count, heads, kv_heads, dim, dtype);
    *bytes = s.delta_bytes + std::max(s.dq_bytes, s.dkv_bytes);  // dq is done before dk and dv begin
    return GAT_OK;
}

int gat_packed_attention_backward(const void* g, long long g_row, long long g_head, const void* q,
                                  long long q_row, long long q_head, const void* k, long long k_row,
                                  long long k_head, const void* v, long long v_row, long long v_head,
                                  const void* out, const void* low, const float* lse, const void* ptr,
                                  const void* kv_ptr, int ptr64, int count, int nq, int nk, int heads,
                                  int kv_heads, int dim, float scale, int causal, void* dq, void* dk,
                                  void* dv, void* workspace, size_t workspace_bytes, int dtype,
                                  void* stream) {
    const int rc = attn_check(nq, nk, count, heads, kv_heads, dim, dtype);
    if (rc != GAT_OK) return rc;
    AttnArgs a{};
    a.g = {g, g_row, g_head};
    a.q = {q, q_row, q_head};
    a.k = {k, k_row, k_head};
    a.v = {v, v_row, v_head};
    a.o = {out, (long long)heads * dim, dim};
    a.dq = {dq, (long long)heads * dim, dim};
    a.dk = {dk, (long long)kv_heads * dim, dim};
    a.dv = {dv, (long long)kv_heads * dim, dim};
    if (ptr == nullptr || kv_ptr == nullptr ||
        (nq > 0 && (q == nullptr || g == nullptr || out == nullptr || lse == nullptr || dq == nullptr)) ||
        (nk > 0 && (k == nullptr || v == nullptr || dk == nullptr || dv == nullptr)))
        return GAT_EINVAL;
    for (const Rows* r : {&a.g, &a.q, &a.o, &a.dq})
        if (!vec_rows(*r, dim, heads / kv_heads, dtype)) return GAT_EUNSUPPORTED;
    for (const Rows* r : {&a.k, &a.v, &a.dk, &a.dv})
        if (!vec_rows(*r, dim, 0, dtype)) return GAT_EUNSUPPORTED;
    const AttnSizes sz = attn_sizes(nq, nk, count, heads, kv_heads, dim, dtype);
    if (workspace_bytes < sz.delta_bytes + std::max(sz.dq_bytes, sz.dkv_bytes) ||
        (workspace == nullptr && workspace_bytes > 0))
        return GAT_EWORKSPACE;
    if (((reinterpret_cast<uintptr_t>(workspace) | reinterpret_cast<uintptr_t>(low)) & 15) != 0)
        return GAT_EINVAL;
    a.ptr = ptr;
    a.kv_ptr = kv_ptr;
    a.ptr64 = ptr64;
    a.count = count;
    a.nq = nq;
    a.nk = nk;
    a.kv_heads = kv_heads;
    set_group(a, heads / kv_heads);
    a.dim = dim;
    a.scale = scale;
    a.causal = causal;
    a.lse = const_cast<float*>(lse);
    a.low = dtype == GAT_F32 ? nullptr : const_cast<void*>(low);
    a.delta = static_cast<float*>(workspace);
    a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + sz.delta_bytes);
    hipStream_t s = static_cast<hipStream_t>(stream);
    int st = GAT_OK;
    if (nq > 0) {
        st = attn_pass<kDq>(a, sz.dq, dtype, s);
        if (st == GAT_OK && sz.dq.splits > 1) {
            const long long n = (long long)nq * heads * dim;
            st = dtype == GAT_F32 ? attn_sum<float>(a.part, sz.dq.splits, n, scale, a.dq, s)
                                  : attn_sum<bf16>(a.part, sz.dq.splits, n, scale, a.dq, s);
        }
    }
    if (st != GAT_OK || nk == 0) return st;
    st = attn_pass<kDkv>(a, sz.dkv, dtype, s);
    if (st != GAT_OK || sz.dkv.splits == 1) return st;
    const long long n = (long long)nk * kv_heads * dim;
    const float* pv = a.part + sz.dkv.splits * n;
    st = dtype == GAT_F32 ? attn_sum<float>(a.part, sz.dkv.splits, n, scale, a.dk, s)
                          : attn_sum<bf16>(a.part, sz.dkv.splits, n, scale, a.dk, s);
    if (st != GAT_OK) return st;
    return dtype == GAT_F32 ? attn_sum<float>(pv, sz.dkv.splits, n, 1.f, a.dv, s)
                            : attn_sum<bf16>(pv, sz.dkv.splits, n, 1.f, a.dv, s);
}

}  // extern "C"
