// Feature transforms, products that sum over the rows of a group (transform.h: SumArgs): the gradients of matrices.
#include <algorithm>

#include "transform.h"

namespace lnasr {

// ------------------------------------------------------------------------------------------
// Segments sorted by group, one block: a stable radix sort (eight bits of the group a pass; equal digits of a wave are found
// by ballots), then the running sum of their lengths.  Segments without a group go last and are left out.  Order matters: the
// rows of a group are summed in the order of the batch, so a gradient is the same bits every time.  Bound by latency:
// 6 us for 300 segments; with everything in LDS it was no faster.
// ------------------------------------------------------------------------------------------
constexpr int kSortNT = 1024;
__global__ __launch_bounds__(kSortNT) void sort_segments(Segments sg, int passes, int* ord0, int* ord1, int64_t* place,
                                                         int64_t* group_off) {
    __shared__ int base[256], cnt[kSortNT / 64][256];
    __shared__ int64_t part[kSortNT / 64], carry;
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
        if (wave == 0) {                                  // running sum, four digits a lane
            int c[4], sum = 0;
            for (int e = 0; e < 4; ++e) c[e] = base[4 * lane + e];
            const int mine = c[0] + c[1] + c[2] + c[3];
            sum = mine;
            for (int d = 1; d < 64; d *= 2) {
                const int v = __shfl_up(sum, d);
                sum += lane >= d ? v : 0;
            }
            sum -= mine;
            for (int e = 0; e < 4; ++e) {
                base[4 * lane + e] = sum;
                sum += c[e];
            }
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
        // running sum of a wave by shuffles, of the waves by the last lanes' sums
        int64_t sum = len;
        for (int d = 1; d < 64; d *= 2) {
            const int64_t v = __shfl_up(sum, d);
            sum += lane >= d ? v : 0;
        }
        if (lane == 63) part[wave] = sum;
        __syncthreads();
        for (int w = 0; w < wave; ++w) sum += part[w];
        const int64_t at = min(carry + sum - len, sg.rows);
        if (live) {
            place[i] = at;
            if (in != ord0) ord0[i] = s;
            const int before = i ? key(in[i - 1]) : -1;
            for (int g = before + 1; g <= k; ++g) group_off[g] = at;
        }
        __syncthreads();
        if (tid == kSortNT - 1) carry = min(carry + sum, sg.rows);
        __syncthreads();
    }
    const int64_t total = carry;
    if (tid == 0) place[sg.S] = total;
    const int last = key(in[sg.S - 1]);
    for (int g = last + 1 + tid; g <= sg.G; g += kSortNT) group_off[g] = total;
}

// the row at each place of the sorted order
__global__ __launch_bounds__(256) void map_rows(Segments sg, const int* ord, const int64_t* place, int64_t* rowmap) {
    const int64_t q0 = ((int64_t)block_id() * 4 + (threadIdx.x >> 6)) * 64, total = place[sg.S];
    if (q0 >= total) return;
    int i = wave_search(sg.S, q0, [&](int j) { return place[j]; });
    if (i < 0) return;
    const int64_t q = q0 + (threadIdx.x & 63);
    if (q >= total) return;
    while (i + 1 < sg.S && place[i + 1] <= q) ++i;
    const int64_t row = seg_off(sg, ord[i]) + q - place[i];
    rowmap[q] = row < sg.rows ? row : sg.rows - 1;
}

// Segments long enough for their rows to be taken run by run.  us, run by run / row by row, segments of 32, 64 and 128 rows: bf16
// 32,768 x 2048 x 1024 660 / 584, 426 / 636, 345 / 679; 16,384 x 512 x 512 105 / 98, 82 / 96, 69 / 92; f32 20,011 x 512 x 429 236 /
// 210, 188 / 210, 150 / 208; f64 20,011 x 128 x 351 92 / 104, 80 / 94, 72 / 107.
static bool rows_together(const Segments& sg) { return sg.rows / sg.S >= 64; }

int transform_sort(lnasr_ctx* ctx, int64_t ld, SumArgs* a) {
    const Segments& sg = a->sg;
    a->rowmap = a->place = nullptr;
    a->ord = nullptr;
    if (!sg.slots) {
        a->group_off = sg.off;
        return 0;
    }
    void* p;
    LN_TRY(transform_ws(ctx, kTrSort, ((size_t)sg.rows + sg.S + 1 + sg.G + 1) * 8 + (size_t)sg.S * 8, &p));
    int64_t* map = (int64_t*)p;
    int64_t* place = map + sg.rows;
    int64_t* goff = place + sg.S + 1;
    int* ord0 = (int*)(goff + sg.G + 1);
    a->group_off = goff;
    const bool mapped = sg.rows > 0 && (!rows_together(sg) || transform_far(ld));
    if (mapped) a->rowmap = map;
    a->place = place;
    a->ord = ord0;
    int passes = 1;
    while (passes < 4 && (sg.G >> (8 * passes)) > 0) ++passes;
    LN_LAUNCH(ctx, "sort_segments", sort_segments, dim3(1), dim3(kSortNT), 0, sg, passes, ord0, ord0 + sg.S, place, goff);
    if (mapped) LN_LAUNCH(ctx, "map_rows", map_rows, transform_grid((sg.rows + 255) / 256, 256), dim3(256), 0, sg, ord0, place, map);
    return 0;
}

// Of up to 64 spans the t-th longest: blocks start in the order of their numbers, and the longest ones are to start first
__device__ __forceinline__ int64_t longest_span(const SumArgs& a, int spans, int64_t t, int ts) {
    const int lane = threadIdx.x & 63;
    int64_t n = -1;                           // rows of span `lane`, -1: none such
    for (int g = 0; g < a.groups; ++g) {
        auto at = [&](int i) {
            const int64_t o = a.sg.S ? a.group_off[i * a.group_step] : 0;
            return o < 0 ? (int64_t)0 : o > a.sg.rows ? a.sg.rows : o;
        };
        const int64_t go = at(g), ge = at(g + 1), q = go + ((lane - ((go >> ts) + g)) << ts);
        if (lane >= (go >> ts) + g) n = q < ge ? min(ge - q, (int64_t)1 << ts) : 0;
    }
    int rank = 0;
    for (int j = 0; j < spans; ++j) {
        const int64_t other = __shfl(n, j);
        rank += other > n || (other == n && j < lane) ? 1 : 0;
    }
    const uint64_t mine = __ballot(lane < spans && rank == (int)t);
    return mine ? __builtin_ctzll(mine) : t;
}
// ------------------------------------------------------------------------------------------
// Tiles of TI x TJ results of one group, WI x WJ waves, summed over a span of the group's rows.  The rows are the k of the product,
// strided for both operands: they lie in LDS as lines (strided_fragment).  TOGETHER: rows that lie together (a segment's) come by
// LDS-DMA step by step, the last and uneven one through registers; otherwise -- segments of a few rows -- all of them through
// registers, row by row as rowmap says, loaded a step ahead.  A group with one span is written at once, the others leave sums of 32
// bits or more per span, which join_parts adds in the order of the spans.
// A: the type of a, B: of b; where they differ (the gradients of adapters) both are multiplied in the wider one, C.
// f32 20,011 rows x 512 x 429: 98 us, 90 TFLOP/s of the 153 of a large library product (CUs busy 72 % of the time: 1120 blocks on
// 1280 places).  bf16 16,384 rows x 16 x 1024, the 16 in f32: 14.8 us, 35 MB (all of it in bf16: 11.6).
// ------------------------------------------------------------------------------------------
template <typename A, typename B>
using Wider = std::conditional_t<(sizeof(A) >= sizeof(B)), A, B>;
// bytes of a step of a and b in LDS
template <typename A, typename B, int TI, int TJ>
constexpr int sum_step() {
    return 128 / (int)sizeof(Wider<A, B>) * (TI * (int)sizeof(A) + TJ * (int)sizeof(B));
}
template <typename T, typename A, typename B, int TI, int TJ, int WI, int WJ, bool TOGETHER>
__global__ __launch_bounds__(64 * WI * WJ, 2) void sum_tile(SumArgs a, unsigned tiles_i, unsigned tiles_j, int ts, typename Mat<T>::Sum* parts,
                                                            typename Mat<T>::Sum* col_parts) {
    using C = Wider<A, B>;
    using M = Mat<C>;
    using Acc = typename M::Acc;
    constexpr int SA = (int)sizeof(A), SB = (int)sizeof(B), EA = 16 / SA, EB = 16 / SB, KB = 128 / (int)sizeof(C), NT = 64 * WI * WJ;
    constexpr int IR = TI / WI / 16, JR = TJ / WJ / 16, STEP = sum_step<A, B, TI, TJ>(), BAT = TI * SA * KB;
    constexpr int AL = TI * SA / 16, BL = TJ * SB / 16;                               // pieces of a line
    constexpr int AN = KB * AL, BN = KB * BL, AP = (AN + NT - 1) / NT, BP = (BN + NT - 1) / NT;
    static_assert(AN % 64 == 0 && BN % 64 == 0, "whole waves of pieces");
    __shared__ __attribute__((aligned(1024))) char lds[2 * STEP];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l15 = lane & 15, kk = lane >> 4;
    const int wi = wave / WJ * (TI / WI), wj = wave % WJ * (TJ / WJ);
    const unsigned tiles = tiles_i * tiles_j, id = die_order(block_id(), block_count());
    const int i0 = (int)(id % tiles / tiles_j) * TI, j0 = (int)(id % tiles_j) * TJ;
    const int64_t t = id / tiles;
    auto brings_a = [&](int i) { return AN % NT == 0 || wave * 64 + NT * i < AN; };
    auto brings_b = [&](int i) { return BN % NT == 0 || wave * 64 + NT * i < BN; };
    int g, n;
    int64_t q0, at;
    bool whole;
    if (!sum_span(a, t, ts, &g, &q0, &n, &whole, &at)) return;

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
        C e[M::E];
#pragma unroll
        for (int j = 0; j < M::E; ++j) e[j] = (C)1;
        __builtin_memcpy(&ones, e, 16);
    }
    auto multiply = [&](int buf) {
        const char* as = lds + buf * STEP;
        const char* bs = as + BAT;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            u32x4 af[IR], bf[JR];
#pragma unroll
            for (int i = 0; i < IR; ++i) af[i] = strided_fragment<A, TI, C>(as, h, wi + 16 * i);
#pragma unroll
            for (int j = 0; j < JR; ++j) bf[j] = strided_fragment<B, TJ, C>(bs, h, wj + 16 * j);
            mma_all<C>(af, bf, acc);
            if (want_col)
#pragma unroll
                for (int i = 0; i < IR; ++i) col[i] = mma<C>(af[i], ones, col[i]);
        }
    };
    // a step through registers: row(k) of its k-th place, for k < left; zeros for the others and past the last column
    u32x4 ar[AP], br[BP];
    auto load = [&](int left, auto row) {
#pragma unroll
        for (int i = 0; i < AP; ++i) {
            const int q = tid + NT * i, k = q / AL, c = i0 + (q % AL ^ spread<A, TI, C>(k) * SA) * EA;
            if (brings_a(i)) ar[i] = k < left ? load_piece((const A*)a.a + row(k) * a.lda, c, a.I) : u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < BP; ++i) {
            const int q = tid + NT * i, k = q / BL, c = j0 + (q % BL ^ spread<B, TJ, C>(k) * SB) * EB;
            if (brings_b(i)) br[i] = k < left ? load_piece((const B*)a.b + row(k) * a.ldb, c, a.J) : u32x4{0, 0, 0, 0};
        }
    };
    auto store = [&](int buf) {
        char* as = lds + buf * STEP;
#pragma unroll
        for (int i = 0; i < AP; ++i)
            if (brings_a(i)) *(u32x4*)(as + (tid + NT * i) * 16) = ar[i];
#pragma unroll
        for (int i = 0; i < BP; ++i)
            if (brings_b(i)) *(u32x4*)(as + BAT + (tid + NT * i) * 16) = br[i];
    };
    if constexpr (TOGETHER) {
        // offsets of this lane's pieces from the step's first; out of range (nothing is read, LDS gets zeros) past the last column.
        // A piece that runs past the last column takes what lies behind it, which no result sees; of a run's last row that may be
        // the array's end, so then the last step goes through registers even if it is a whole one.
        unsigned ao[AP], bo[BP];
#pragma unroll
        for (int i = 0; i < AP; ++i) {
            const int q = tid + NT * i, k = q / AL, c = (q % AL ^ spread<A, TI, C>(k) * SA) * EA;
            ao[i] = i0 + c < a.I ? (unsigned)k * (unsigned)(a.lda * SA) + c * SA : 0xffffffffu;
        }
#pragma unroll
        for (int i = 0; i < BP; ++i) {
            const int q = tid + NT * i, k = q / BL, c = (q % BL ^ spread<B, TJ, C>(k) * SB) * EB;
            bo[i] = j0 + c < a.J ? (unsigned)k * (unsigned)(a.ldb * SB) + c * SB : 0xffffffffu;
        }
        const int uneven = a.I % EA || a.J % EB ? 1 : 0;
        each_run(a, q0, q0 + n, [&](int64_t row0, int rows) {
            const int full = (rows - uneven) / KB;
            const char* ab = (const char*)((const A*)a.a + row0 * a.lda + i0);
            const char* bb = (const char*)((const B*)a.b + row0 * a.ldb + j0);
            auto bring = [&](int buf) {
                char* as = lds + buf * STEP;
#pragma unroll
                for (int i = 0; i < AP; ++i)
                    if (brings_a(i)) bring_piece(ab, ao[i], as + (wave * 64 + NT * i) * 16);
#pragma unroll
                for (int i = 0; i < BP; ++i)
                    if (brings_b(i)) bring_piece(bb, bo[i], as + BAT + (wave * 64 + NT * i) * 16);
                ab += KB * a.lda * SA;
                bb += KB * a.ldb * SB;
            };
            if (full > 0) bring(0);
            const int rest = rows - full * KB;
            if (rest > 0) load(rest, [&](int k) { return row0 + full * KB + k; });
            __syncthreads();
            for (int i = 0; i < full; ++i) {
                if (i + 1 < full) bring((i + 1) & 1);
                multiply(i & 1);
                __syncthreads();
            }
            if (rest > 0) {
                store(0);
                __syncthreads();
                multiply(0);
                __syncthreads();
            }
        });
    } else {
        auto fetch = [&](int k0) { load(n - k0, [&](int k) { return a.rowmap ? a.rowmap[q0 + k0 + k] : q0 + k0 + k; }); };
        if (n > 0) {
            fetch(0);
            store(0);
        }
        __syncthreads();
        int buf = 0;
        for (int k0 = 0; k0 < n; k0 += KB, buf ^= 1) {
            const bool more = k0 + KB < n;
            if (more) fetch(k0 + KB);
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
                else parts[(at * a.I + ii) * a.J + jj] = acc[i][j][r];
            }
            if (want_col && l15 == 0) {
                if (whole) ((T*)a.cols)[(int64_t)g * a.I + ii] = (T)col[i][r];
                else col_parts[at * a.I + ii] = col[i][r];
            }
        }
}

// ------------------------------------------------------------------------------------------
// The same for 16-bit types and wide matrices whose segments are long: 256 x 256 results, eight waves of 128 x 64, steps of 64 rows
// between two pairs of LDS buffers.  While half a step multiplies, the fragments of the next half are read; in the middle of a step
// its own buffers fall free and the step after next is asked for.
// Both operands are strided: which rows the lanes of a fragment hold is free as long as both do alike, so lanes 16 kk .. take rows
// 4 kk .. 4 kk + 3 and 16 more.  Lines of 512 bytes, two to a kilobyte that a wave brings, each kilobyte 64 bytes further on and the
// odd line's runs of 16 columns swapped in pairs: the eight lines that one read touches lie in other banks, and the reads need two
// addresses instead of eight (registers).
// bf16 32,768 rows x 2048 x 1024 in 16 ragged groups: 173 us, 790 TFLOP/s; most of the rest is the longest groups' blocks, one to two
// turns of the CUs (cutting them finer costs as much in sums written and read).
// ------------------------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(512, 2) void sum_deep(SumArgs a, unsigned tiles_i, unsigned tiles_j, int ts, float* parts) {
    using M = Mat<T>;
    using Acc = typename M::Acc;
    constexpr int E = 8, KB = 64, NT = 512, IR = 8, JR = 4, TI = 256, TJ = 256, CHUNK = 1024 + 64, UNIT = 32 * CHUNK;
    static_assert(sizeof(T) == 2, "16-bit types");
    // (four variables, not one array: the compiler then knows that reading one does not wait for what is brought into another)
    __shared__ __attribute__((aligned(64))) char a0[UNIT], b0[UNIT], a1[UNIT], b1[UNIT];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l15 = lane & 15, kk = lane >> 4;
    const int wi = wave / 4 * 128, wj = wave % 4 * 64;
    // (not in die_order: neighbouring blocks are tiles of one span, spread over the dies so that all of them start with the longest)
    const unsigned tiles = tiles_i * tiles_j, id = block_id();
    const int i0 = (int)(id % tiles / tiles_j) * TI, j0 = (int)(id % tiles_j) * TJ;
    const unsigned spans = block_count() / tiles;
    const int64_t t = spans <= 64 ? longest_span(a, spans, id / tiles, ts) : id / tiles;
    int g, n;
    int64_t q0, at;
    bool whole;
    if (!sum_span(a, t, ts, &g, &q0, &n, &whole, &at)) return;

    Acc acc[IR][JR];
#pragma unroll
    for (int i = 0; i < IR; ++i)
#pragma unroll
        for (int j = 0; j < JR; ++j) acc[i][j] = Acc{0, 0, 0, 0};
    struct Frags {
        u32x4 a[IR], b[JR];
    };
    // line k of a unit: chunk k / 2; run r of 16 columns of an odd line lies at r ^ 1
    auto fragment = [&](const char* unit, int h, int c) {
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4 lds16x4;
        const int j = l15 >> 2;                           // lines 32 h + 4 kk + j and 16 further
        const int at = (2 * kk + (j >> 1)) * CHUNK + (j & 1) * 512 + (((c / 16) ^ (j & 1)) << 5) + (l15 & 3) * 8 + 16 * h * CHUNK;
        const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds16x4*)(unit + at)));
        const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds16x4*)(unit + (at + 8 * CHUNK))));
        return u32x4{lo[0], lo[1], hi[0], hi[1]};
    };
    auto read = [&](const char* as, const char* bs, int h, Frags& f) {
#pragma unroll
        for (int j = 0; j < JR; ++j) f.b[j] = fragment(bs, h, wj + 16 * j);
#pragma unroll
        for (int i = 0; i < IR; ++i) f.a[i] = fragment(as, h, wi + 16 * i);
    };
    auto multiply = [&](const Frags& f) {
#pragma unroll
        for (int i = 0; i < IR; ++i)
#pragma unroll
            for (int j = 0; j < JR; ++j) acc[i][j] = mma<T>(f.a[i], f.b[j], acc[i][j]);
    };
    unsigned ao[4], bo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int q = tid + NT * i, k = q / 32, c = (q % 32 ^ (k & 1) * 2) * E;      // the piece at this place
        ao[i] = i0 + c < a.I ? (unsigned)k * (unsigned)(a.lda * 2) + c * 2 : 0xffffffffu;
        bo[i] = j0 + c < a.J ? (unsigned)k * (unsigned)(a.ldb * 2) + c * 2 : 0xffffffffu;
    }
    const int uneven = a.I % E || a.J % E ? 1 : 0;        // as in sum_tile
    each_run(a, q0, q0 + n, [&](int64_t row0, int rows) {
        const int full = (rows - uneven) / KB;
        const char* ab = (const char*)((const T*)a.a + row0 * a.lda + i0);
        const char* bb = (const char*)((const T*)a.b + row0 * a.ldb + j0);
        auto bring = [&](char* as, char* bs) {
#pragma unroll
            for (int i = 0; i < 4; ++i) bring_piece(ab, ao[i], as + (wave + 8 * i) * CHUNK);
#pragma unroll
            for (int i = 0; i < 4; ++i) bring_piece(bb, bo[i], bs + (wave + 8 * i) * CHUNK);
            ab += KB * a.lda * 2;
            bb += KB * a.ldb * 2;
        };
        constexpr int VM0 = 0x0f70;                       // s_waitcnt vmcnt(0), the other counters free
        Frags f0, f1;
        if (full > 0) {
            bring(a0, b0);
            if (full > 1) bring(a1, b1);
            __builtin_amdgcn_s_waitcnt(VM0);
            __builtin_amdgcn_s_barrier();
            read(a0, b0, 0, f0);
            auto interleave = [&]() {                     // a read behind every product, then the other products
#pragma unroll
                for (int j = 0; j < 24; ++j) {
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            };
            // One step from as, bs; the next one in an, bn.  At the barrier the next step has arrived for every wave, and every wave
            // has read all of this one.
            auto run = [&](char* as, char* bs, const char* an, const char* bn) {
                read(as, bs, 1, f1);
                multiply(f0);
                interleave();
                __builtin_amdgcn_s_waitcnt(VM0 & 0xf0ff);
                __builtin_amdgcn_s_barrier();
                __builtin_amdgcn_sched_barrier(0);
                bring(as, bs);
                read(an, bn, 0, f0);
                multiply(f1);
                __builtin_amdgcn_sched_group_barrier(0x020, 8, 0);
                interleave();
            };
            auto turn = [&](int s, char* as, char* bs, const char* an, const char* bn) {
                read(as, bs, 1, f1);
                multiply(f0);
                __builtin_amdgcn_s_waitcnt(VM0 & 0xf0ff);
                __builtin_amdgcn_s_barrier();
                if (s + 2 < full) bring(as, bs);
                if (s + 1 < full) read(an, bn, 0, f0);
                multiply(f1);
            };
            int s = 0;
            for (; s + 4 <= full; s += 2) {
                run(a0, b0, a1, b1);
                run(a1, b1, a0, b0);
            }
            for (; s < full; s += 2) {
                turn(s, a0, b0, a1, b1);
                if (s + 1 < full) turn(s + 1, a1, b1, a0, b0);
            }
            __syncthreads();
        }
        const int rest = rows - full * KB;
        if (rest > 0) {                                   // a last, uneven step through registers
            const int64_t r = row0 + full * KB;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int q = tid + NT * i, k = q / 32, c = (q % 32 ^ (k & 1) * 2) * E, at = (wave + 8 * i) * CHUNK + lane * 16;
                *(u32x4*)(a0 + at) = k < rest ? load_piece((const T*)a.a + (r + k) * a.lda, i0 + c, a.I) : u32x4{0, 0, 0, 0};
                *(u32x4*)(b0 + at) = k < rest ? load_piece((const T*)a.b + (r + k) * a.ldb, j0 + c, a.J) : u32x4{0, 0, 0, 0};
            }
            __syncthreads();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                read(a0, b0, h, f0);
                multiply(f0);
            }
            __syncthreads();
        }
    });
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
                else parts[(at * a.I + ii) * a.J + jj] = acc[i][j][r];
            }
        }
}

// Column sums of a beside sum_deep: cols[k, i] = sum of a[r, i], a span and 512 columns a block, eight of them a thread; the rows of the
// span go to the four waves in turn, which meet in LDS.  bf16 32,768 x 2048: 25 us, 5.3 TB/s.  (Summed beside the products instead, by
// matrix instructions or from LDS, it has no registers left.)
template <typename T>
__global__ __launch_bounds__(256) void sum_cols(SumArgs a, unsigned tiles, int ts, float* col_parts) {
    __shared__ float part[3][64][8];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = (int)(block_id() % tiles) * 512 + lane * 8;
    const int64_t t = block_id() / tiles;
    int g, n;
    int64_t q0, at;
    bool whole;
    if (!sum_span(a, t, ts, &g, &q0, &n, &whole, &at)) return;
    float sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    each_run(a, q0, q0 + n, [&](int64_t row0, int rows) {
#pragma unroll 8
        for (int k = wave; k < rows; k += 4) {
            const u32x4 v = load_piece((const T*)a.a + (row0 + k) * a.lda, c, a.I);
            T e[8];
            __builtin_memcpy(e, &v, 16);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[j] += (float)e[j];
        }
    });
    if (wave)
#pragma unroll
        for (int j = 0; j < 8; ++j) part[wave - 1][lane][j] = sum[j];
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float v = sum[j] + part[0][lane][j] + part[1][lane][j] + part[2][lane][j];
        if (c + j >= a.I) continue;
        if (whole) ((T*)a.cols)[(int64_t)g * a.I + c + j] = (T)v;
        else col_parts[at * a.I + c + j] = v;
    }
}

// out and cols of the groups that have more than one span.  fp64 64 groups of 39 x 39 in 350 spans: 5 us.
template <typename T>
__global__ __launch_bounds__(256) void join_parts(SumArgs a, int ts, const typename Mat<T>::Sum* parts, const typename Mat<T>::Sum* col_parts,
                                                  unsigned per) {
    using Sum = typename Mat<T>::Sum;
    auto clamped = [&](int g) {
        const int64_t o = a.sg.S ? a.group_off[g * a.group_step] : 0;
        return o < 0 ? (int64_t)0 : o > a.sg.rows ? a.sg.rows : o;
    };
    const int g = (int)(block_id() / per);
    if (g >= a.groups) return;
    const int64_t go = clamped(g), ge = clamped(g + 1), n = (ge - go + (1ll << ts) - 1) >> ts;
    if (n <= 1) return;
    const int64_t at = sum_place(a, g, go, 0, ts), size = (int64_t)a.I * a.J;
    // n values `step` apart, in their order, eight on their way at a time
    auto total = [&](const Sum* from, int64_t step) {
        Sum v = 0;
        for (int64_t k = 0; k < n; k += 8) {
            Sum u[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = from[min(k + i, n - 1) * step];
#pragma unroll
            for (int i = 0; i < 8; ++i) v += k + i < n ? u[i] : (Sum)0;
        }
        return (T)v;
    };
    for (int64_t e = (int64_t)(block_id() % per) * 256 + threadIdx.x; e < size + a.I; e += (int64_t)per * 256) {
        if (e < size) ((T*)a.out)[g * size + e] = total(parts + at * size + e, size);
        else if (a.cols) ((T*)a.cols)[g * a.I + e - size] = total(col_parts + at * a.I + e - size, a.I);
    }
}

template <typename T>
static int join_t(lnasr_ctx* ctx, const SumArgs& a, int ts, const void* parts, const void* col_parts) {
    using Sum = typename Mat<T>::Sum;
    const int64_t size = (int64_t)a.I * a.J + a.I, per = std::min<int64_t>((size + 255) / 256, std::max<int64_t>(1, 8192 / a.groups));
    LN_LAUNCH(ctx, "join_parts", (join_parts<T>), transform_grid(per * a.groups, 256), dim3(256), 0, a, ts, (const Sum*)parts,
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

// Length of a span, as a power of two: a span's sums are written and read once more (8 or 16 bytes each) beside its 2 x 2^ts products
// of each, so long ones, but no fewer blocks than the CUs hold at a time (`want`).  Where the groups give that many by themselves,
// only one far over the mean is cut.  Never more than 512 MB of sums (sum_places).
static int span_length(const SumArgs& a, int64_t tiles, int64_t want, size_t sum_size) {
    const int64_t size = (int64_t)a.I * a.J + a.I;
    int ts = 8;
    while (ts < 40 && (a.sg.rows >> ts) * tiles > want) ++ts;
    if (a.groups * tiles >= want) ++ts;
    while (ts < 40 && (a.sg.rows >> ts) * size * (int64_t)sum_size > (256ll << 20)) ++ts;
    return ts;
}

template <typename T, int TI, int TJ, int WI, int WJ, typename A = T, typename B = T>
static int launch_sum(lnasr_ctx* ctx, const SumArgs& a, const char* name) {
    using Sum = typename Mat<T>::Sum;
    constexpr int HOLDS = std::min(8, (160 << 10) / (2 * sum_step<A, B, TI, TJ>()));
    const int64_t ti = (a.I + TI - 1) / TI, tj = (a.J + TJ - 1) / TJ, size = (int64_t)a.I * a.J + a.I;
    const int ts = span_length(a, ti * tj, (int64_t)HOLDS * ctx->prop.multiProcessorCount, sizeof(Sum));
    const int64_t spans = (a.sg.rows >> ts) + a.groups;
    LN_REQUIRE(spans * ti * tj < (1ll << 31), "%lld rows in %d groups of %d x %d sums are too many for one call", (long long)a.sg.rows,
               a.groups, a.I, a.J);
    void* parts = nullptr;
    const bool split = a.sg.rows > (1ll << ts);
    const int64_t places = sum_places(a, ts);
    if (split) LN_TRY(transform_ws(ctx, kTrPart, (size_t)places * size * sizeof(Sum), &parts));
    Sum* cp = (Sum*)parts + places * a.I * a.J;
    const dim3 grid = transform_grid(spans * ti * tj, 64 * WI * WJ), block(64 * WI * WJ);
    // (through registers the rows are rowmap's, or lie as they are summed: transform_sort knows the strides)
    const bool together = !a.rowmap && !transform_far(std::max(a.lda, a.ldb));
    LN_REQUIRE(together || a.rowmap || !a.place, "%s: sorted rows without their map", name);
    if (together) LN_LAUNCH(ctx, name, (sum_tile<T, A, B, TI, TJ, WI, WJ, true>), grid, block, 0, a, (unsigned)ti, (unsigned)tj, ts, (Sum*)parts, cp);
    else LN_LAUNCH(ctx, name, (sum_tile<T, A, B, TI, TJ, WI, WJ, false>), grid, block, 0, a, (unsigned)ti, (unsigned)tj, ts, (Sum*)parts, cp);
    return split ? join_t<T>(ctx, a, ts, parts, cp) : 0;
}

template <typename T>
static int launch_sum_deep(lnasr_ctx* ctx, SumArgs a, const char* name) {
    const int64_t ti = (a.I + 255) / 256, tj = (a.J + 255) / 256;
    void* const cols = a.cols;
    for (int pass = 0; pass < (cols ? 2 : 1); ++pass) {
        // the product, then the column sums: with spans of their own, one after the other in the same workspace
        if (pass) a.J = 0;
        a.cols = pass ? cols : nullptr;
        const int64_t tiles = pass ? (a.I + 511) / 512 : ti * tj, size = (int64_t)a.I * a.J + a.I;
        const int ts = span_length(a, tiles, (pass ? 4 : 1) * ctx->prop.multiProcessorCount, 4);
        const int64_t spans = (a.sg.rows >> ts) + a.groups;
        LN_REQUIRE(spans * tiles < (1ll << 31), "%lld rows in %d groups of %d x %d sums are too many for one call", (long long)a.sg.rows,
                   a.groups, a.I, a.J);
        void* parts = nullptr;
        const bool split = a.sg.rows > (1ll << ts);
        const int64_t places = sum_places(a, ts);
        if (split) LN_TRY(transform_ws(ctx, kTrPart, (size_t)places * size * 4, &parts));
        float* cp = (float*)parts + places * a.I * a.J;
        if (pass) LN_LAUNCH(ctx, "sum_cols", (sum_cols<T>), transform_grid(spans * tiles, 256), dim3(256), 0, a, (unsigned)tiles, ts, cp);
        else LN_LAUNCH(ctx, name, (sum_deep<T>), transform_grid(spans * tiles, 512), dim3(512), 0, a, (unsigned)ti, (unsigned)tj, ts, (float*)parts);
        if (split) LN_TRY(join_t<T>(ctx, a, ts, parts, cp));
    }
    return 0;
}

template <typename T>
static int sum_t(lnasr_ctx* ctx, const SumArgs& a, const char* name) {
    if constexpr (!std::is_same<T, Mid<T>>::value) {
        // (32-bit instructions: tiles of 128 x 128 have nothing to save)
        if (a.mid_a) {
            if (a.I <= 16) return launch_sum<T, 16, 128, 1, 4, Mid<T>, T>(ctx, a, name);
            if (a.I <= 32) return launch_sum<T, 32, 128, 1, 4, Mid<T>, T>(ctx, a, name);
            return launch_sum<T, 64, 64, 2, 2, Mid<T>, T>(ctx, a, name);
        }
        if (a.mid_b) {
            if (a.J <= 16) return launch_sum<T, 128, 16, 4, 1, T, Mid<T>>(ctx, a, name);
            if (a.J <= 32) return launch_sum<T, 128, 32, 4, 1, T, Mid<T>>(ctx, a, name);
            return launch_sum<T, 64, 64, 2, 2, T, Mid<T>>(ctx, a, name);
        }
    }
    // few results on one side: us, 64 x 64 / as narrow as they are: bf16 16,384 x 16 x 1024 26 / 23, f32 20,011 x 16 x 429 33 / 25,
    // x 32 33 / 30, f64 20,011 x 16 x 351 42 / 28, x 32 44 / 37
    if (a.I <= 16) return launch_sum<T, 16, 128, 1, 4>(ctx, a, name);
    if (a.J <= 16) return launch_sum<T, 128, 16, 4, 1>(ctx, a, name);
    if (a.I <= 32) return launch_sum<T, 32, 128, 1, 4>(ctx, a, name);
    if (a.J <= 32) return launch_sum<T, 128, 32, 4, 1>(ctx, a, name);
    if constexpr (sizeof(T) == 2) {
        // 256 x 256 for enough of them with 2048 rows each, from segments long enough for its steps of 64 (us, 64 x 64 / 128 x 128 /
        // 256 x 256; 32,768 x 2048 x 1024 in 1 group 359 / 268 / 146, in 16 323 / 272 / 164, in 64 528 / 418 / 309; 8192 x 1024 x 1024
        // in 16 66 / 61 / 70; 32,768 x 512 x 512 in 1 56 / 57 / 50, in 64 65 / 53 / 78; sorted segments of 128, 256 and 512 rows - / 341
        // / 364, - / 312 / 293, - / 253 / 207).
        if ((int64_t)(a.I / 256) * (a.J / 256) * (a.sg.rows >> 11) >= 128 && (!a.place || a.sg.rows / a.sg.S >= 256) &&
            !transform_far(std::max(a.lda, a.ldb)))
            return launch_sum_deep<T>(ctx, a, name);
        if (a.I > 64 && a.J > 64) return launch_sum<T, 128, 128, 2, 2>(ctx, a, name);
    }
    return launch_sum<T, 64, 64, 2, 2>(ctx, a, name);
}

int transform_sum(lnasr_ctx* ctx, int dtype, const SumArgs& a, const char* name) {
    if (a.groups == 0) return 0;
    if (sum_narrow_ok(a) && !((a.mid_a || a.mid_b) && transform_size(dtype) == 2)) return transform_sum_narrow(ctx, dtype, a, name);
    switch (dtype) {
        case LNASR_F64: return sum_t<double>(ctx, a, name);
        case LNASR_F32: return sum_t<float>(ctx, a, name);
        case LNASR_F16: return sum_t<_Float16>(ctx, a, name);
        default: return sum_t<__bf16>(ctx, a, name);
    }
}

}  // namespace lnasr
