// Feature transforms: affine maps per group of rows, and a shared projection with low-rank adapters (transform.hip: entry
// points and dispatch; transform_rows.hip: products with one result row per feature row; transform_grad.hip: products that
// sum over rows).  Internal.
#pragma once
#include <type_traits>

#include "common.h"

namespace lnasr {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef double f64x2 __attribute__((ext_vector_type(2)));
typedef double f64x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// One 16 x 16 block of a product by the matrix cores.  Every type moves in pieces of 16 bytes: lane l of the wave holds, for
// row (l & 15) of its operand, the E consecutive k of piece (l >> 4) of a 64-byte run.  Which k an instruction contracts is
// free as long as both operands agree, so the piece feeds E / 8 (16 bit), 4 (f32) or 2 (f64) instructions as it lies.
// D[m, n]: lane l holds column n = l & 15 and the four rows m = row(r, l >> 4).
template <typename T>
struct Mat;
template <>
struct Mat<double> {
    using Acc = f64x4;
    using Sum = double;
    static constexpr int E = 2;
    static constexpr int PARTS = 2;
    static __device__ __forceinline__ Acc part(u32x4 a, u32x4 b, Acc c, int j) {
        const f64x2 x = __builtin_bit_cast(f64x2, a), y = __builtin_bit_cast(f64x2, b);
        return __builtin_amdgcn_mfma_f64_16x16x4f64(x[j], y[j], c, 0, 0, 0);
    }
    static __device__ __forceinline__ int row(int r, int kk) { return 4 * r + kk; }
};
template <>
struct Mat<float> {
    using Acc = f32x4;
    using Sum = float;
    static constexpr int E = 4;
    static constexpr int PARTS = 4;
    static __device__ __forceinline__ Acc part(u32x4 a, u32x4 b, Acc c, int j) {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
        return __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
    }
    static __device__ __forceinline__ int row(int r, int kk) { return 4 * kk + r; }
};
template <>
struct Mat<_Float16> {
    using Acc = f32x4;
    using Sum = float;
    static constexpr int E = 8;
    static constexpr int PARTS = 1;
    static __device__ __forceinline__ Acc part(u32x4 a, u32x4 b, Acc c, int) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ int row(int r, int kk) { return 4 * kk + r; }
};
template <>
struct Mat<__bf16> {
    using Acc = f32x4;
    using Sum = float;
    static constexpr int E = 8;
    static constexpr int PARTS = 1;
    static __device__ __forceinline__ Acc part(u32x4 a, u32x4 b, Acc c, int) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ int row(int r, int kk) { return 4 * kk + r; }
};

// The type a projection's narrow middle is held in: never under 32 bits.  (Rounded to 16 bits it took a whole rounding more than the
// results' own, and in f16 a middle past 65504 was lost.)
template <typename T>
using Mid = std::conditional_t<sizeof(T) == 2, float, T>;

template <typename T>
__device__ __forceinline__ typename Mat<T>::Acc mma(u32x4 a, u32x4 b, typename Mat<T>::Acc c) {
#pragma unroll
    for (int j = 0; j < Mat<T>::PARTS; ++j) c = Mat<T>::part(a, b, c, j);
    return c;
}
// acc[i][j] += a[i] b[j]: the instructions of one piece in turns over all of acc, so that none waits for the one before
template <typename T, int I, int J>
__device__ __forceinline__ void mma_all(const u32x4 (&a)[I], const u32x4 (&b)[J], typename Mat<T>::Acc (&acc)[I][J]) {
#pragma unroll
    for (int p = 0; p < Mat<T>::PARTS; ++p)
#pragma unroll
        for (int i = 0; i < I; ++i)
#pragma unroll
            for (int j = 0; j < J; ++j) acc[i][j] = Mat<T>::part(a[i], b[j], acc[i][j], p);
}

// Segments of rows.  offsets may come from device memory that the host has not looked at: every value is brought into
// [0, rows] before it is used, so that an offset out of order gives meaningless numbers but no access out of range.
struct Segments {
    const int64_t* off;      // [S + 1]
    const int32_t* slots;    // [S] or null: segment s belongs to group s
    int S, G;
    int64_t rows;
};
__device__ __forceinline__ int64_t seg_off(const Segments& sg, int s) {
    const int64_t o = sg.off[s];
    return o < 0 ? 0 : o > sg.rows ? sg.rows : o;
}
// group of segment s, or -1
__device__ __forceinline__ int seg_slot(const Segments& sg, int s) {
    const int k = sg.slots ? sg.slots[s] : s;
    return (unsigned)k < (unsigned)sg.G ? k : -1;
}
// The last i in [0, n) with first(i) <= t, -1 if there is none; first must not fall.  The 64 lanes of a wave probe 64 candidates
// at a time: two rounds for 4096 segments.
template <typename F>
__device__ __forceinline__ int wave_search(int n, int64_t t, F first) {
    const int lane = threadIdx.x & 63;
    int lo = 0;
    while (true) {
        const int step = (n + 63) / 64;
        const int64_t at = (int64_t)lane * step;
        const bool below = at < n && first(lo + (int)at) <= t;
        const int cnt = __popcll(__ballot(below));
        if (cnt == 0) return -1;
        const int skip = (cnt - 1) * step;
        lo += skip;
        n = min(step, n - skip);
        if (step == 1) return __builtin_amdgcn_readfirstlane(lo);
    }
}
// The spans of 2^ts rows of a ragged batch, without a table: give segment s the numbers floor(off[s] / 2^ts) + s and on.  They
// never collide (a segment of n rows needs ceil(n / 2^ts) numbers and has at least floor(n / 2^ts) + 1), so floor(rows / 2^ts)
// + S numbers cover every batch; some of them are empty spans.  Returns the segment of span t and its rows r0 .. r1 - 1
// (wave-uniform), -1 if the span is empty.
__device__ __forceinline__ int find_span(const int64_t* off, int S, int64_t rows, int64_t t, int ts, int64_t* r0, int64_t* r1) {
    auto clamped = [&](int s) {
        const int64_t o = off[s];
        return o < 0 ? (int64_t)0 : o > rows ? rows : o;
    };
    const int s = wave_search(S, t, [&](int i) { return (clamped(i) >> ts) + i; });
    if (s < 0) return -1;
    const int64_t o = clamped(s), e = clamped(s + 1);
    *r0 = o + ((t - ((o >> ts) + s)) << ts);
    *r1 = *r0 + (1ll << ts) < e ? *r0 + (1ll << ts) : e;
    return *r0 < *r1 ? s : -1;
}

// 16 bytes of E consecutive elements from element c of a line that ends before `end`; what lies past the end is 0.  The
// address need not be aligned (odd widths: rows of 39 or 351 values).
template <typename T>
__device__ __forceinline__ u32x4 load_piece(const T* line, long c, long end) {
    constexpr int E = Mat<T>::E;
    u32x4 v;
    if (c + E <= end) {
        __builtin_memcpy(&v, line + c, 16);
        return v;
    }
    // (16 bits: adapters of rank 32 beside 16,384 x 1024 x 2048 80 -> 75 us; two or four elements are looked at as soon)
    if (sizeof(T) == 2 && c >= end) return u32x4{0, 0, 0, 0};
    T e[E];
#pragma unroll
    for (int j = 0; j < E; ++j) e[j] = c + j < end ? line[c + j] : (T)0;
    __builtin_memcpy(&v, e, 16);
    return v;
}

// the same as values of type U, which may be wider than those of the line
template <typename U, typename T>
__device__ __forceinline__ u32x4 load_as(const T* line, long c, long end) {
    if constexpr (std::is_same<U, T>::value) {
        return load_piece(line, c, end);
    } else {
        constexpr int E = Mat<U>::E;
        T t[E];
        if (c + E <= end) {
            __builtin_memcpy(t, line + c, sizeof(t));
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j) t[j] = c + j < end ? line[c + j] : (T)0;
        }
        U e[E];
#pragma unroll
        for (int j = 0; j < E; ++j) e[j] = (U)t[j];
        u32x4 v;
        __builtin_memcpy(&v, e, 16);
        return v;
    }
}

// LDS of one wave is its own: order its writes and reads for the compiler (the hardware keeps the order of a wave's LDS accesses)
__device__ __forceinline__ void wave_lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// HIP takes fewer than 2^32 threads along x: beyond 2^31 a launch has rows of blocks, a few of them past the last (their spans are
// empty).  block_id: a block's number, of block_count().
inline dim3 transform_grid(int64_t blocks, int threads) {
    const int64_t most = (1ll << 31) / threads, y = (blocks + most - 1) / most;
    return dim3((unsigned)(y > 1 ? (blocks + y - 1) / y : blocks), (unsigned)(y > 1 ? y : 1));
}
__device__ __forceinline__ unsigned block_count() { return gridDim.x * gridDim.y; }
__device__ __forceinline__ unsigned block_id() { return blockIdx.y * gridDim.x + blockIdx.x; }

// Consecutive block numbers go to the eight dies (XCDs) in turn, each with an L2 of its own: give every die a run of
// neighbouring tiles, so that the tiles that share a matrix or a span of rows share an L2.
__device__ __forceinline__ unsigned die_order(unsigned id, unsigned total) {
    const unsigned per = total / 8, rest = total % 8, die = id % 8, at = id / 8;
    return die * per + min(die, rest) + at;
}

// Tile number -> (m, n): eight tiles of n beside each other before the next of m, so that the tiles a die works on at a time share
// rows and columns about evenly
__device__ __forceinline__ void tile_order(unsigned id, unsigned tiles_m, unsigned tiles_n, unsigned* m, unsigned* n) {
    const unsigned group = id / (8 * tiles_m), wide = min(8u, tiles_n - 8 * group), at = id - group * 8 * tiles_m;
    *m = at / wide;
    *n = 8 * group + at % wide;
}
// 16 bytes a lane from base + offset to LDS at `to` (wave-uniform) + 16 * lane; zeros where offset >= 2^31
__device__ __forceinline__ void bring_piece(const char* base, unsigned offset, char* to) {
    const __amdgpu_buffer_rsrc_t d = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 0x80000000u, 0x00027000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(d, (__attribute__((address_space(3))) void*)to, 16, offset, 0, 0, 0);
}

// A tile of C columns whose k is strided, in LDS as lines of k: the run of 16 columns (sizeof(T) pieces) at place p of line k
// is run p ^ spread(k), so that the lines one fragment read touches (they differ in (lane & 15) >> 2 and lane >> 4 for 16 bit,
// in lane >> 4 alone for the others) lie in other banks.  U: the type the values are multiplied in, T or a wider one.
template <typename T, int C, typename U = T>
__device__ __forceinline__ int spread(int k) {
    constexpr int RUNS = C / 16;
    if ((RUNS & (RUNS - 1)) != 0) return 0;
    if (sizeof(U) != sizeof(T)) return k >> 2 & (RUNS < 4 ? RUNS - 1 : 3);
    if (sizeof(T) == 2) return ((k & 3) | (k >> 1 & 4)) & (RUNS < 8 ? RUNS - 1 : 7);
    if (sizeof(T) == 4) return k >> 2 & (RUNS < 4 ? RUNS - 1 : 3);
    return k >> 1 & (RUNS < 2 ? RUNS - 1 : 1);
}
// the wave's fragment of columns c .. c + 15 (c a multiple of 16) as values of type U, half h of their 128 bytes of k
template <typename T, int C, typename U = T>
__device__ __forceinline__ u32x4 strided_fragment(const char* tile, int h, int c) {
    constexpr int SZ = (int)sizeof(T), E = Mat<U>::E;
    const int lane = threadIdx.x & 63, l15 = lane & 15, kk = lane >> 4;
    u32x4 f;
    if constexpr (SZ == 2 && sizeof(U) == 2) {
        // each 16 lanes read 4 lines of 16 columns, 8 bytes a lane; the lane gets the 4 k of its column
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4 lds16x4;
        const int k = 32 * h + 8 * kk + (l15 >> 2);
        const int at = k * (C * 2) + (((c / 16) ^ spread<T, C>(k)) << 5) + (l15 & 3) * 8;
        const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds16x4*)(tile + at)));
        // (spread(k + 4) == spread(k))
        const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds16x4*)(tile + (at + 4 * (C * 2)))));
        f = u32x4{lo[0], lo[1], hi[0], hi[1]};
    } else {
        U e[E];
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const int k = (4 * h + kk) * E + j;
            e[j] = (U) * (const T*)(tile + k * (C * SZ) + (((c / 16) ^ spread<T, C, U>(k)) * 16 + l15) * SZ);
        }
        __builtin_memcpy(&f, e, 16);
    }
    return f;
}

// y[r, :] = scale_k * (x[r, :] W_k') + bias_k  for the rows of the segments; W_k' = W_k^T (kn false, W_k [n, k]) or W_k (kn
// true, W_k [k, n]).  w_stride 0: one W for all rows, tiles of rows then run across segments; with `low` each row also gets
// p[r, :] L_k' of its segment's group (none where the group is negative).  p, and y where `mid` says so, are of type Mid.
struct RowsArgs {
    Segments sg;
    const void *x, *w, *bias, *p, *low;
    const double* scale;
    void* y;
    int64_t ldx, ldy, ldp;
    int64_t w_stride, bias_stride, low_stride;
    int K, N, R;
    bool kn, mid;
};
int transform_rows(lnasr_ctx* ctx, int dtype, const RowsArgs& a, const char* name);

// out[k, i, j] = sum over the rows r of group k of a[r, i] b[r, j];  cols[k, i] = sum of a[r, i] (or null).  Every group is
// written, zeros where it has no rows.  a is of type Mid with mid_a, b with mid_b (one of them at most, and then no cols).
struct SumArgs {
    Segments sg;
    const int64_t* group_off;   // group g: places group_off[g * group_step] .. group_off[(g + 1) * group_step] of the sorted rows
    int64_t group_step;         // 1; S: all segments as one group
    const int* ord;             // [S] the segments in the order of their groups, or null: the rows as they lie
    const int64_t* place;       // [S + 1] (with ord) places of the sorted segments' rows
    const int64_t* rowmap;      // (with ord, if the segments are short or the rows far apart) the row at each place
    const void *a, *b;
    void *out, *cols;
    int64_t lda, ldb;
    int groups, I, J;
    bool mid_a, mid_b;
};
// Where the sums of a group of several spans lie: place sum_place of span k = 0, 1, .. of a group that begins at row go, of
// sum_places.  With few groups the spans' numbers; else 2 floor(go / 2^ts) + k, whatever the number of groups: a group of L > 2^ts
// rows has ceil(L / 2^ts) <= floor(L / 2^ts) + 1 <= 2 floor(L / 2^ts) spans, and the next one begins floor(L / 2^ts) or more further
// on.  (Groups of one span write no sums: 128 groups of 4096 x 4096, one of them split, took 8.6 GB.)
__host__ __device__ inline bool sum_numbered(int64_t rows, int groups, int ts) { return groups <= rows >> ts; }
inline int64_t sum_places(const SumArgs& a, int ts) { return (a.sg.rows >> ts) + (sum_numbered(a.sg.rows, a.groups, ts) ? a.groups : a.sg.rows >> ts); }
__device__ __forceinline__ int64_t sum_place(const SumArgs& a, int group, int64_t go, int64_t k, int ts) {
    return (go >> ts) + k + (sum_numbered(a.sg.rows, a.groups, ts) ? group : go >> ts);
}
// Span t of 2^ts places of the sorted rows: its group, first place and rows, and where its sums go; false: nothing to do.  (A group
// without rows has one span without rows, to be written as zeros.)
__device__ __forceinline__ bool sum_span(const SumArgs& a, int64_t t, int ts, int* group, int64_t* q0, int* n, bool* whole, int64_t* place) {
    auto clamped = [&](int g) {
        const int64_t o = a.sg.S ? a.group_off[g * a.group_step] : 0;
        return o < 0 ? (int64_t)0 : o > a.sg.rows ? a.sg.rows : o;
    };
    const int g = wave_search(a.groups, t, [&](int i) { return (clamped(i) >> ts) + i; });
    if (g < 0) return false;
    const int64_t go = clamped(g), ge = max(go, clamped(g + 1)), span = t - ((go >> ts) + g);
    *group = g;
    *q0 = go + (span << ts);
    if (span > 0 && *q0 >= ge) return false;
    *n = (int)min(ge - *q0, (int64_t)1 << ts);
    *whole = go + (1ll << ts) >= ge;
    *place = sum_place(a, g, go, span, ts);
    return true;
}
// The rows that lie together from place q of the sorted rows on, at most up to place end: calls each(first row, rows) run by run
template <typename F>
__device__ __forceinline__ void each_run(const SumArgs& a, int64_t q, int64_t end, F each) {
    int i = a.place ? max(0, wave_search(a.sg.S, q, [&](int j) { return a.place[j]; })) : 0;
    while (q < end) {                                     // (one call of `each`: it is a kernel's whole loop)
        int64_t row = q, to = end;
        if (a.place) {
            while (i < a.sg.S && a.place[i + 1] <= q) ++i;
            if (i >= a.sg.S) return;
            to = min(a.place[i + 1], end);
            row = seg_off(a.sg, a.ord[i]) + (q - a.place[i]);
        }
        each(row, (int)(to - q));
        q = to;
    }
}

int transform_sum(lnasr_ctx* ctx, int dtype, const SumArgs& a, const char* name);
// transform_narrow.hip: the same for contiguous rows of a few dozen values of `size` bytes
bool rows_narrow_ok(const RowsArgs& a, int size);
int transform_rows_narrow(lnasr_ctx* ctx, int dtype, const RowsArgs& a, const char* name);
bool sum_narrow_ok(const SumArgs& a);
int transform_sum_narrow(lnasr_ctx* ctx, int dtype, const SumArgs& a, const char* name);
// out and cols from the sums of the spans of 2^ts rows
int transform_join(lnasr_ctx* ctx, const SumArgs& a, int dtype, int ts, const void* parts, const void* col_parts);
// Row strides at which the rows of one step (128 bytes of k) pass the 31 bits of the LDS-DMA's offsets
inline bool transform_far(int64_t ld) { return ld * 128 >= (1ll << 31); }
// Sorts the segments by group (stable): group_off, ord, place, rowmap of a.  Without slots the rows are sorted as they lie.
// ld: the largest row stride of what will be summed.
int transform_sort(lnasr_ctx* ctx, int64_t ld, SumArgs* a);

// Workspace `i` of the feature transforms with room for `bytes`
int transform_ws(lnasr_ctx* ctx, int i, size_t bytes, void** out);
enum { kTrX, kTrOff, kTrSlots, kTrW, kTrBias, kTrA, kTrB, kTrScale, kTrDy, kTrOut0, kTrOut1, kTrOut2, kTrOut3, kTrOut4, kTrLow, kTrDlow,
       kTrSort, kTrPart, kTrCount };

inline size_t transform_size(int dtype) { return dtype == LNASR_F64 ? 8 : dtype == LNASR_F32 ? 4 : 2; }
inline size_t transform_mid_size(int dtype) { return dtype == LNASR_F64 ? 8 : 4; }

}  // namespace lnasr
