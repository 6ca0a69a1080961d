// Feature transforms, products that sum over the rows of a group (transform.h: SumArgs): the gradients of matrices.
#include <algorithm>

#include "transform.h"

namespace lnasr {

// ------------------------------------------------------------------------------------------
// Segments sorted by group, one block: a stable radix sort (eight bits of the group a pass; equal digits of a wave are found
// by ballots), then the running sum of their lengths.  Segments without a group go last and are left out.  Order matters: the
// rows of a group are summed in the order of the batch, so a gradient is the same bits every time.
// ------------------------------------------------------------------------------------------
constexpr int kSortNT = 1024;
__global__ __launch_bounds__(kSortNT) void sort_segments(Segments sg, int passes, int* ord0, int* ord1, int64_t* place,
                                                         int64_t* group_off) {
    __shared__ int base[256], cnt[kSortNT / 64][256];
    __shared__ int64_t part[kSortNT], carry;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    auto key = [&](int s) {
        const int k = seg_slot(sg, s);
        return k < 0 ? sg.G : k;
    };
    for (int i = tid; i < sg.S; i += kSortNT) ord0[i] = i;
    __syncthreads();
    int *in = ord0, *out = ord1;
    for (int p = 0; p < passes; ++p) {
        for (int i = tid; i < 256; i += kSortNT) base[i] = 0;
        __syncthreads();
        for (int i = tid; i < sg.S; i += kSortNT) atomicAdd(&base[key(in[i]) >> (8 * p) & 255], 1);
        __syncthreads();
        if (tid == 0)
            for (int d = 0, sum = 0; d < 256; ++d) {
                const int c = base[d];
                base[d] = sum;
                sum += c;
            }
        for (int c0 = 0; c0 < sg.S; c0 += kSortNT) {
            for (int i = tid; i < kSortNT / 64 * 256; i += kSortNT) cnt[i >> 8][i & 255] = 0;
            __syncthreads();
            const bool live = c0 + tid < sg.S;
            const int s = live ? in[c0 + tid] : 0, d = live ? key(s) >> (8 * p) & 255 : 0;
            uint64_t same = __ballot(live);
#pragma unroll
            for (int bit = 0; bit < 8; ++bit) {
                const uint64_t set = __ballot(d >> bit & 1);
                same &= d >> bit & 1 ? set : ~set;
            }
            const int rank = __popcll(same & ((1ull << lane) - 1));
            if (live && rank == 0) cnt[wave][d] = __popcll(same);
            __syncthreads();
            if (tid < 256) {
                int sum = base[tid];
                for (int w = 0; w < kSortNT / 64; ++w) {
                    const int c = cnt[w][tid];
                    cnt[w][tid] = sum;
                    sum += c;
                }
                base[tid] = sum;
            }
            __syncthreads();
            if (live) out[cnt[wave][d] + rank] = s;
            __syncthreads();
        }
        int* x = in;
        in = out;
        out = x;
    }
    // running sum of the lengths, and where each group begins
    if (tid == 0) carry = 0;
    __syncthreads();
    for (int c0 = 0; c0 < sg.S; c0 += kSortNT) {
        const int i = c0 + tid;
        const bool live = i < sg.S;
        const int s = live ? in[i] : 0, k = live ? key(s) : sg.G;
        int64_t len = live && k < sg.G ? seg_off(sg, s + 1) - seg_off(sg, s) : 0;
        if (len < 0) len = 0;
        part[tid] = len;
        __syncthreads();
        for (int d = 1; d < kSortNT; d *= 2) {
            const int64_t v = tid >= d ? part[tid - d] : 0;
            __syncthreads();
            part[tid] += v;
            __syncthreads();
        }
        const int64_t at = min(carry + part[tid] - len, sg.rows);
        if (live) {
            place[i] = at;
            if (in != ord0) ord0[i] = s;
            const int before = i ? key(in[i - 1]) : -1;
            for (int g = before + 1; g <= k; ++g) group_off[g] = at;
        }
        __syncthreads();
        if (tid == kSortNT - 1) carry += part[tid];
        __syncthreads();
    }
    const int64_t total = min(carry, sg.rows);
    if (tid == 0) place[sg.S] = total;
    const int last = key(in[sg.S - 1]);
    for (int g = last + 1 + tid; g <= sg.G; g += kSortNT) group_off[g] = total;
}

// the row at each place of the sorted order
__global__ __launch_bounds__(256) void map_rows(Segments sg, const int* ord, const int64_t* place, int64_t* rowmap) {
    const int64_t q0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 64, total = place[sg.S];
    if (q0 >= total) return;
    int i = wave_search(sg.S, q0, [&](int j) { return place[j]; });
    if (i < 0) return;
    const int64_t q = q0 + (threadIdx.x & 63);
    if (q >= total) return;
    while (i + 1 < sg.S && place[i + 1] <= q) ++i;
    const int64_t row = seg_off(sg, ord[i]) + q - place[i];
    rowmap[q] = row < sg.rows ? row : sg.rows - 1;
}

int transform_sort(lnasr_ctx* ctx, const Segments& sg, const int64_t** group_off, const int64_t** rowmap) {
    if (!sg.slots) {
        *group_off = sg.off;
        *rowmap = nullptr;
        return 0;
    }
    void* p;
    LN_TRY(transform_ws(ctx, kTrSort, ((size_t)sg.rows + sg.S + 1 + sg.G + 1) * 8 + (size_t)sg.S * 8, &p));
    int64_t* map = (int64_t*)p;
    int64_t* place = map + sg.rows;
    int64_t* goff = place + sg.S + 1;
    int* ord0 = (int*)(goff + sg.G + 1);
    int passes = 1;
    while (passes < 4 && (sg.G >> (8 * passes)) > 0) ++passes;
    LN_LAUNCH(ctx, "sort_segments", sort_segments, dim3(1), dim3(kSortNT), 0, sg, passes, ord0, ord0 + sg.S, place, goff);
    LN_LAUNCH(ctx, "map_rows", map_rows, dim3((unsigned)((sg.rows + 255) / 256)), dim3(256), 0, sg, ord0, place, map);
    *group_off = goff;
    *rowmap = map;
    return 0;
}

// ------------------------------------------------------------------------------------------
// Tiles of TI x TJ results of one group, WI x WJ waves, summed over a span of the group's rows.  The rows are the k of the product,
// strided for both operands: they lie in LDS as lines (strided_fragment).  FROM: 0 through registers; where both operands are made
// of whole aligned 16-byte pieces by LDS-DMA, 1 from rows that lie together (a running base, fixed offsets), 2 from the rows
// that rowmap names.  A group with one span is written at once, the others leave sums of 32
// bits or more per span, which join_parts adds in the order of the spans.
// ------------------------------------------------------------------------------------------
__device__ const u32x4 kZeroPiece = {0, 0, 0, 0};

__device__ __forceinline__ void bring_from(const char* from, char* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

template <typename T, int TI, int TJ, int WI, int WJ, int FROM>
__global__ __launch_bounds__(64 * WI * WJ, 2) void sum_tile(SumArgs a, unsigned tiles_i, unsigned tiles_j, int ts, typename Mat<T>::Sum* parts,
                                                            typename Mat<T>::Sum* col_parts) {
    using M = Mat<T>;
    using Acc = typename M::Acc;
    constexpr int SZ = (int)sizeof(T), E = M::E, KB = 128 / SZ, NT = 64 * WI * WJ, IR = TI / WI / 16, JR = TJ / WJ / 16;
    constexpr int AL = TI * SZ / 16, BL = TJ * SZ / 16;                               // pieces of a line
    constexpr int AP = TI * 8 / NT, BP = TJ * 8 / NT;
    static_assert(TI * 8 % NT == 0 && TJ * 8 % NT == 0, "whole waves of pieces");
    __shared__ __attribute__((aligned(1024))) char lds[2 * (TI + TJ) * 128];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l15 = lane & 15, kk = lane >> 4;
    const int wi = wave / WJ * (TI / WI), wj = wave % WJ * (TJ / WJ);
    const unsigned tiles = tiles_i * tiles_j, id = die_order(blockIdx.x, gridDim.x);
    const int i0 = (int)(id % tiles / tiles_j) * TI, j0 = (int)(id % tiles_j) * TJ;
    const int64_t t = id / tiles;
    // (a span without rows still has its group: a group without rows is written as zeros)
    auto clamped = [&](int g) {
        const int64_t o = a.sg.S ? a.group_off[g * a.group_step] : 0;
        return o < 0 ? (int64_t)0 : o > a.sg.rows ? a.sg.rows : o;
    };
    const int g = wave_search(a.groups, t, [&](int i) { return (clamped(i) >> ts) + i; });
    if (g < 0) return;
    const int64_t go = clamped(g), ge = max(go, clamped(g + 1)), span = t - ((go >> ts) + g), q0 = go + (span << ts);
    if (span > 0 && q0 >= ge) return;
    const int n = (int)min(ge - q0, (int64_t)1 << ts);                                // rows of the span
    const bool whole = go + (1ll << ts) >= ge;

    Acc acc[IR][JR], col[IR];
#pragma unroll
    for (int i = 0; i < IR; ++i) {
        col[i] = Acc{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < JR; ++j) acc[i][j] = Acc{0, 0, 0, 0};
    }
    const bool want_col = a.cols && j0 == 0 && wj == 0;
    u32x4 ones;
    {
        T e[E];
#pragma unroll
        for (int j = 0; j < E; ++j) e[j] = (T)1;
        __builtin_memcpy(&ones, e, 16);
    }
    auto row_of = [&](int k) { return a.rowmap ? a.rowmap[q0 + k] : q0 + k; };
    auto multiply = [&](int buf) {
        const char* as = lds + buf * (TI + TJ) * 128;
        const char* bs = as + TI * 128;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            u32x4 af[IR], bf[JR];
#pragma unroll
            for (int i = 0; i < IR; ++i) af[i] = strided_fragment<T, TI>(as, h, wi + 16 * i);
#pragma unroll
            for (int j = 0; j < JR; ++j) bf[j] = strided_fragment<T, TJ>(bs, h, wj + 16 * j);
#pragma unroll
            for (int i = 0; i < IR; ++i)
#pragma unroll
                for (int j = 0; j < JR; ++j) acc[i][j] = M::mma(af[i], bf[j], acc[i][j]);
            if (want_col)
#pragma unroll
                for (int i = 0; i < IR; ++i) col[i] = M::mma(af[i], ones, col[i]);
        }
    };
    if constexpr (FROM == 1) {
        constexpr unsigned OUT = 0xffffffffu;
        unsigned ao[AP], bo[BP];
#pragma unroll
        for (int i = 0; i < AP; ++i) {
            const int q = tid + NT * i, k = q / AL, c = (q % AL ^ spread<T, TI>(k) * SZ) * E;
            ao[i] = i0 + c < a.I ? (unsigned)k * (unsigned)(a.lda * SZ) + c * SZ : OUT;
        }
#pragma unroll
        for (int i = 0; i < BP; ++i) {
            const int q = tid + NT * i, k = q / BL, c = (q % BL ^ spread<T, TJ>(k) * SZ) * E;
            bo[i] = j0 + c < a.J ? (unsigned)k * (unsigned)(a.ldb * SZ) + c * SZ : OUT;
        }
        const char* ab = (const char*)((const T*)a.a + q0 * a.lda + i0);
        const char* bb = (const char*)((const T*)a.b + q0 * a.ldb + j0);
        auto bring = [&](int buf, int left) {
            char* as = lds + buf * (TI + TJ) * 128;
            const bool tail = left < KB;
#pragma unroll
            for (int i = 0; i < AP; ++i) bring_piece(ab, tail && (tid + NT * i) / AL >= left ? OUT : ao[i], as + (wave * 64 + NT * i) * 16);
#pragma unroll
            for (int i = 0; i < BP; ++i)
                bring_piece(bb, tail && (tid + NT * i) / BL >= left ? OUT : bo[i], as + TI * 128 + (wave * 64 + NT * i) * 16);
            ab += KB * a.lda * SZ;
            bb += KB * a.ldb * SZ;
        };
        if (n > 0) bring(0, n);
        __syncthreads();
        int buf = 0;
        for (int left = n; left > 0; left -= KB, buf ^= 1) {
            if (left > KB) bring(buf ^ 1, left - KB);
            multiply(buf);
            __syncthreads();
        }
    } else if constexpr (FROM == 2) {
        // columns past the end and rows past the span come from a piece of zeros
        auto bring = [&](int buf, int k0) {
            char* as = lds + buf * (TI + TJ) * 128;
#pragma unroll
            for (int i = 0; i < AP; ++i) {
                const int q = tid + NT * i, k = q / AL, c = i0 + (q % AL ^ spread<T, TI>(k) * SZ) * E;
                const bool live = k0 + k < n && c < a.I;
                bring_from(live ? (const char*)((const T*)a.a + row_of(k0 + k) * a.lda + c) : (const char*)&kZeroPiece, as + (wave * 64 + NT * i) * 16);
            }
#pragma unroll
            for (int i = 0; i < BP; ++i) {
                const int q = tid + NT * i, k = q / BL, c = j0 + (q % BL ^ spread<T, TJ>(k) * SZ) * E;
                const bool live = k0 + k < n && c < a.J;
                bring_from(live ? (const char*)((const T*)a.b + row_of(k0 + k) * a.ldb + c) : (const char*)&kZeroPiece,
                           as + TI * 128 + (wave * 64 + NT * i) * 16);
            }
        };
        if (n > 0) bring(0, 0);
        __syncthreads();
        int buf = 0;
        for (int k0 = 0; k0 < n; k0 += KB, buf ^= 1) {
            if (k0 + KB < n) bring(buf ^ 1, k0 + KB);
            multiply(buf);
            __syncthreads();
        }
    } else {
        u32x4 ar[AP], br[BP];
        auto load = [&](int k0) {
#pragma unroll
            for (int i = 0; i < AP; ++i) {
                const int q = tid + NT * i, k = q / AL, c = i0 + (q % AL ^ spread<T, TI>(k) * SZ) * E;
                ar[i] = k0 + k < n ? load_piece((const T*)a.a + row_of(k0 + k) * a.lda, c, a.I) : u32x4{0, 0, 0, 0};
            }
#pragma unroll
            for (int i = 0; i < BP; ++i) {
                const int q = tid + NT * i, k = q / BL, c = j0 + (q % BL ^ spread<T, TJ>(k) * SZ) * E;
                br[i] = k0 + k < n ? load_piece((const T*)a.b + row_of(k0 + k) * a.ldb, c, a.J) : u32x4{0, 0, 0, 0};
            }
        };
        auto store = [&](int buf) {
            char* as = lds + buf * (TI + TJ) * 128;
#pragma unroll
            for (int i = 0; i < AP; ++i) *(u32x4*)(as + (tid + NT * i) * 16) = ar[i];
#pragma unroll
            for (int i = 0; i < BP; ++i) *(u32x4*)(as + TI * 128 + (tid + NT * i) * 16) = br[i];
        };
        if (n > 0) {
            load(0);
            store(0);
        }
        __syncthreads();
        int buf = 0;
        for (int k0 = 0; k0 < n; k0 += KB, buf ^= 1) {
            const bool more = k0 + KB < n;
            if (more) load(k0 + KB);
            multiply(buf);
            if (more) store(buf ^ 1);
            __syncthreads();
        }
    }
#pragma unroll
    for (int i = 0; i < IR; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int ii = i0 + wi + 16 * i + M::row(r, kk);
            if (ii >= a.I) continue;
#pragma unroll
            for (int j = 0; j < JR; ++j) {
                const int jj = j0 + wj + 16 * j + l15;
                if (jj >= a.J) continue;
                if (whole) ((T*)a.out)[((int64_t)g * a.I + ii) * a.J + jj] = (T)acc[i][j][r];
                else parts[(t * a.I + ii) * a.J + jj] = acc[i][j][r];
            }
            if (want_col && l15 == 0) {
                if (whole) ((T*)a.cols)[(int64_t)g * a.I + ii] = (T)col[i][r];
                else col_parts[t * a.I + ii] = col[i][r];
            }
        }
}

template <typename T>
__global__ __launch_bounds__(256) void join_parts(SumArgs a, int ts, const typename Mat<T>::Sum* parts, const typename Mat<T>::Sum* col_parts,
                                                  unsigned per) {
    using Sum = typename Mat<T>::Sum;
    auto clamped = [&](int g) {
        const int64_t o = a.sg.S ? a.group_off[g * a.group_step] : 0;
        return o < 0 ? (int64_t)0 : o > a.sg.rows ? a.sg.rows : o;
    };
    const int g = (int)(blockIdx.x / per);
    const int64_t go = clamped(g), ge = clamped(g + 1), n = (ge - go + (1ll << ts) - 1) >> ts;
    if (n <= 1) return;
    const int64_t t = (go >> ts) + g, size = (int64_t)a.I * a.J;
    for (int64_t e = (int64_t)(blockIdx.x % per) * 256 + threadIdx.x; e < size + a.I; e += (int64_t)per * 256) {
        if (e < size) {
            Sum v = 0;
#pragma unroll 8
            for (int64_t k = 0; k < n; ++k) v += parts[(t + k) * size + e];
            ((T*)a.out)[g * size + e] = (T)v;
        } else if (a.cols) {
            Sum v = 0;
            for (int64_t k = 0; k < n; ++k) v += col_parts[(t + k) * a.I + e - size];
            ((T*)a.cols)[g * a.I + e - size] = (T)v;
        }
    }
}

template <typename T>
static int join_t(lnasr_ctx* ctx, const SumArgs& a, int ts, const void* parts, const void* col_parts) {
    using Sum = typename Mat<T>::Sum;
    const int64_t size = (int64_t)a.I * a.J + a.I, per = std::min<int64_t>((size + 255) / 256, std::max<int64_t>(1, 8192 / a.groups));
    LN_LAUNCH(ctx, "join_parts", (join_parts<T>), dim3((unsigned)(per * a.groups)), dim3(256), 0, a, ts, (const Sum*)parts,
              (const Sum*)col_parts, (unsigned)per);
    return 0;
}

int transform_join(lnasr_ctx* ctx, const SumArgs& a, int dtype, int ts, const void* parts, const void* col_parts) {
    switch (dtype) {
        case LNASR_F64: return join_t<double>(ctx, a, ts, parts, col_parts);
        case LNASR_F32: return join_t<float>(ctx, a, ts, parts, col_parts);
        case LNASR_F16: return join_t<_Float16>(ctx, a, ts, parts, col_parts);
        default: return join_t<__bf16>(ctx, a, ts, parts, col_parts);
    }
}

template <typename T, int TI, int TJ, int WI, int WJ>
static int launch_sum(lnasr_ctx* ctx, const SumArgs& a, const char* name) {
    using Sum = typename Mat<T>::Sum;
    const int64_t ti = (a.I + TI - 1) / TI, tj = (a.J + TJ - 1) / TJ, size = (int64_t)a.I * a.J + a.I, e = 16 / sizeof(T);
    const bool dma = ((uintptr_t)a.a | (uintptr_t)a.b) % 16 == 0 && a.I % e == 0 && a.J % e == 0 && a.lda % e == 0 && a.ldb % e == 0;
    // A span's sums are written and read once more (8 or 16 bytes each) beside its 2 x 2^ts products of each: long spans, but
    // no fewer blocks than the CUs hold at a time (one of 256 x 256, two of 128 x 128, four of 64 x 64).  Where the groups give that many by themselves, only one far over the mean is cut.
    const int64_t want = (TI >= 256 ? 2 : TI >= 128 ? 4 : 8) * ctx->prop.multiProcessorCount;
    int ts = 8;
    while (ts < 40 && (a.sg.rows >> ts) * ti * tj > want) ++ts;
    if (a.groups * ti * tj >= want) ++ts;
    while (ts < 40 && (a.sg.rows >> ts) * size * (int64_t)sizeof(Sum) > (256ll << 20)) ++ts;
    const int64_t spans = (a.sg.rows >> ts) + a.groups;
    LN_REQUIRE(spans * ti * tj < (1ll << 31), "%lld rows in %d groups of %d x %d sums are too many for one call", (long long)a.sg.rows,
               a.groups, a.I, a.J);
    void* parts = nullptr;
    const bool split = a.sg.rows > (1ll << ts);
    if (split) LN_TRY(transform_ws(ctx, kTrPart, (size_t)spans * size * sizeof(Sum), &parts));
    Sum* cp = (Sum*)parts + spans * a.I * a.J;
    const dim3 grid((unsigned)(spans * ti * tj)), block(64 * WI * WJ);
    if (dma && !a.rowmap && std::max(a.lda, a.ldb) * 64 * (int64_t)sizeof(T) < (1ll << 31))
        LN_LAUNCH(ctx, name, (sum_tile<T, TI, TJ, WI, WJ, 1>), grid, block, 0, a, (unsigned)ti, (unsigned)tj, ts, (Sum*)parts, cp);
    else if (dma) LN_LAUNCH(ctx, name, (sum_tile<T, TI, TJ, WI, WJ, 2>), grid, block, 0, a, (unsigned)ti, (unsigned)tj, ts, (Sum*)parts, cp);
    else LN_LAUNCH(ctx, name, (sum_tile<T, TI, TJ, WI, WJ, 0>), grid, block, 0, a, (unsigned)ti, (unsigned)tj, ts, (Sum*)parts, cp);
    if (split) return join_t<T>(ctx, a, ts, (const Sum*)parts, (const Sum*)cp);
    return 0;
}

template <typename T>
static int sum_t(lnasr_ctx* ctx, const SumArgs& a, const char* name) {
    if constexpr (sizeof(T) == 2) {
        if ((int64_t)(a.I / 256) * (a.J / 256) * a.groups >= 128) return launch_sum<T, 256, 256, 2, 4>(ctx, a, name);
        if (a.I > 64 && a.J > 64) return launch_sum<T, 128, 128, 2, 2>(ctx, a, name);
        return launch_sum<T, 64, 64, 2, 2>(ctx, a, name);
    } else if constexpr (sizeof(T) == 4) {
        if (a.I > 64 && a.J > 64) return launch_sum<T, 128, 128, 2, 2>(ctx, a, name);
        return launch_sum<T, 64, 64, 2, 2>(ctx, a, name);
    } else {
        return launch_sum<T, 64, 64, 2, 2>(ctx, a, name);
    }
}

int transform_sum(lnasr_ctx* ctx, int dtype, const SumArgs& a, const char* name) {
    if (a.groups == 0) return 0;
    if (sum_narrow_ok(a)) return transform_sum_narrow(ctx, dtype, a, name);
    switch (dtype) {
        case LNASR_F64: return sum_t<double>(ctx, a, name);
        case LNASR_F32: return sum_t<float>(ctx, a, name);
        case LNASR_F16: return sum_t<_Float16>(ctx, a, name);
        default: return sum_t<__bf16>(ctx, a, name);
    }
}

}  // namespace lnasr
