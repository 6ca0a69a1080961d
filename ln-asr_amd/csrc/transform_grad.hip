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
// Tiles of TI x TJ results of one group, four waves (2 x 2), summed over a span of the group's rows.  Both operands are
// strided in k (their rows are the rows summed over) and lie in LDS as they come.  A group with one span is written at once,
// the others leave sums of 32 bits or more per span, which join_parts adds in the order of the spans.
// ------------------------------------------------------------------------------------------
template <typename T, int TI, int TJ>
__global__ __launch_bounds__(256) void sum_tile(SumArgs a, unsigned tiles_i, unsigned tiles_j, int ts, typename Mat<T>::Sum* parts,
                                                typename Mat<T>::Sum* col_parts) {
    using M = Mat<T>;
    constexpr int E = M::E, KB = 128 / (int)sizeof(T), IR = TI / 32, JR = TJ / 32;
    constexpr int PAD = sizeof(T) == 4 ? 4 : 8, IP = TI + PAD, JP = TJ + PAD;
    constexpr int AP = TI * 8 / 256, BP = TJ * 8 / 256;
    __shared__ __attribute__((aligned(16))) T as[2][KB * IP], bs[2][KB * JP];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l15 = lane & 15, kk = lane >> 4;
    const int wi = (wave >> 1) * (TI / 2), wj = (wave & 1) * (TJ / 2);
    const unsigned tiles = tiles_i * tiles_j;
    const int i0 = (int)(blockIdx.x % tiles / tiles_j) * TI, j0 = (int)(blockIdx.x % tiles_j) * TJ;
    const int64_t t = blockIdx.x / tiles;
    // (a span without rows still has its group: a group without rows is written as zeros)
    int64_t q0 = 0, q1 = 0;
    auto clamped = [&](int g) {
        const int64_t o = a.sg.S ? a.group_off[g * a.group_step] : 0;
        return o < 0 ? (int64_t)0 : o > a.sg.rows ? a.sg.rows : o;
    };
    const int g = wave_search(a.groups, t, [&](int i) { return (clamped(i) >> ts) + i; });
    if (g < 0) return;
    const int64_t go = clamped(g), ge = max(go, clamped(g + 1)), span = t - ((go >> ts) + g);
    q0 = go + (span << ts);
    q1 = min(ge, q0 + (1ll << ts));
    if (span > 0 && q0 >= q1) return;
    const bool whole = go + (1ll << ts) >= ge;

    typename M::Acc acc[IR][JR], col[IR];
#pragma unroll
    for (int i = 0; i < IR; ++i) {
        col[i] = typename M::Acc{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < JR; ++j) acc[i][j] = typename M::Acc{0, 0, 0, 0};
    }
    const bool want_col = a.cols && j0 == 0 && wj == 0;
    u32x4 ones;
    {
        T e[E];
#pragma unroll
        for (int j = 0; j < E; ++j) e[j] = (T)1;
        __builtin_memcpy(&ones, e, 16);
    }
    u32x4 ar[AP], br[BP];
    auto row_of = [&](int64_t q) { return a.rowmap ? a.rowmap[q] : q; };
    auto load = [&](int64_t q) {
#pragma unroll
        for (int i = 0; i < AP; ++i) {
            const int pc = tid + 256 * i, k = pc / (TI / E), c = pc % (TI / E) * E;
            ar[i] = q + k < q1 ? load_piece((const T*)a.a + row_of(q + k) * a.lda, i0 + c, a.I) : u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < BP; ++i) {
            const int pc = tid + 256 * i, k = pc / (TJ / E), c = pc % (TJ / E) * E;
            br[i] = q + k < q1 ? load_piece((const T*)a.b + row_of(q + k) * a.ldb, j0 + c, a.J) : u32x4{0, 0, 0, 0};
        }
    };
    auto store = [&](int buf) {
#pragma unroll
        for (int i = 0; i < AP; ++i) {
            const int pc = tid + 256 * i, k = pc / (TI / E), c = pc % (TI / E) * E;
            *(u32x4*)&as[buf][k * IP + c] = ar[i];
        }
#pragma unroll
        for (int i = 0; i < BP; ++i) {
            const int pc = tid + 256 * i, k = pc / (TJ / E), c = pc % (TJ / E) * E;
            *(u32x4*)&bs[buf][k * JP + c] = br[i];
        }
    };
    auto frag = [&](const T* base, int pitch, int h, int c) {
        const T* p = base + (4 * h + kk) * E * pitch + c;
        T e[E];
        u32x4 v;
#pragma unroll
        for (int j = 0; j < E; ++j) e[j] = p[j * pitch];
        __builtin_memcpy(&v, e, 16);
        return v;
    };
    if (q0 < q1) {
        load(q0);
        store(0);
    }
    __syncthreads();
    int buf = 0;
    for (int64_t q = q0; q < q1; q += KB, buf ^= 1) {
        const bool more = q + KB < q1;
        if (more) load(q + KB);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            u32x4 af[IR], bf[JR];
#pragma unroll
            for (int i = 0; i < IR; ++i) af[i] = frag(as[buf], IP, h, wi + 16 * i + l15);
#pragma unroll
            for (int j = 0; j < JR; ++j) bf[j] = frag(bs[buf], JP, h, wj + 16 * j + l15);
#pragma unroll
            for (int i = 0; i < IR; ++i) {
#pragma unroll
                for (int j = 0; j < JR; ++j) acc[i][j] = M::mma(af[i], bf[j], acc[i][j]);
                if (want_col) col[i] = M::mma(af[i], ones, col[i]);
            }
        }
        if (more) store(buf ^ 1);
        __syncthreads();
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
            for (int64_t k = 0; k < n; ++k) v += parts[(t + k) * size + e];
            ((T*)a.out)[g * size + e] = (T)v;
        } else if (a.cols) {
            Sum v = 0;
            for (int64_t k = 0; k < n; ++k) v += col_parts[(t + k) * a.I + e - size];
            ((T*)a.cols)[g * a.I + e - size] = (T)v;
        }
    }
}

template <typename T, int TI, int TJ>
static int launch_sum(lnasr_ctx* ctx, const SumArgs& a, const char* name) {
    using Sum = typename Mat<T>::Sum;
    const int64_t ti = (a.I + TI - 1) / TI, tj = (a.J + TJ - 1) / TJ, size = (int64_t)a.I * a.J + a.I;
    // spans: as many as it takes to give every CU some eight blocks, none under 256 rows, and no more sums than 256 MB
    // beside one for each group
    int ts = 8;
    while (ts < 40 && ((a.sg.rows >> ts) * ti * tj > 8 * ctx->prop.multiProcessorCount || (a.sg.rows >> ts) * size * (int64_t)sizeof(Sum) > (256ll << 20))) ++ts;
    const int64_t spans = (a.sg.rows >> ts) + a.groups, per = std::min<int64_t>((size + 255) / 256, std::max<int64_t>(1, 8192 / a.groups));
    LN_REQUIRE(spans * ti * tj < (1ll << 31), "%lld rows in %d groups of %d x %d sums are too many for one call", (long long)a.sg.rows,
               a.groups, a.I, a.J);
    void* parts = nullptr;
    const bool split = a.sg.rows > (1ll << ts);
    if (split) LN_TRY(transform_ws(ctx, kTrPart, (size_t)spans * size * sizeof(Sum), &parts));
    Sum* cp = (Sum*)parts + spans * a.I * a.J;
    LN_LAUNCH(ctx, name, (sum_tile<T, TI, TJ>), dim3((unsigned)(spans * ti * tj)), dim3(256), 0, a, (unsigned)ti, (unsigned)tj, ts, (Sum*)parts, cp);
    if (split)
        LN_LAUNCH(ctx, "join_parts", (join_parts<T>), dim3((unsigned)(per * a.groups)), dim3(256), 0, a, ts, (const Sum*)parts, (const Sum*)cp,
                  (unsigned)per);
    return 0;
}

int transform_sum(lnasr_ctx* ctx, int dtype, const SumArgs& a, const char* name) {
    if (a.groups == 0) return 0;
    switch (dtype) {
        case LNASR_F64: return launch_sum<double, 64, 64>(ctx, a, name);
        case LNASR_F32: return launch_sum<float, 64, 64>(ctx, a, name);
        case LNASR_F16: return launch_sum<_Float16, 64, 64>(ctx, a, name);
        default: return launch_sum<__bf16, 64, 64>(ctx, a, name);
    }
}

}  // namespace lnasr
