// Feature transforms, products with one result row per feature row (transform.h: RowsArgs).
#include "transform.h"

namespace lnasr {

// Consecutive block numbers go to the eight dies (XCDs) in turn, each with an L2 of its own: give every die a run of
// neighbouring tiles, so that the tiles that share a matrix or a span of rows share an L2.
__device__ __forceinline__ unsigned die_order(unsigned id, unsigned total) {
    const unsigned per = total / 8, rest = total % 8, die = id % 8, at = id / 8;
    return die * per + min(die, rest) + at;
}

// ------------------------------------------------------------------------------------------
// Tiles of TM rows x TN results, four waves.  Both operands pass through LDS in steps of 128 bytes of k: an operand whose k
// is contiguous as rows of eight 16-byte pieces (piece p of row r at p ^ (r & 7): the sixteen rows that a fragment read
// touches then spread over all banks), one whose k is strided (kn) as it lies, padded.  The next step's pieces travel
// through registers while the current one multiplies.
// ------------------------------------------------------------------------------------------
template <typename T, int TM, int TN, int WN, bool KN>
__global__ __launch_bounds__(256) void rows_tile(RowsArgs a, unsigned tiles_n, bool spans, int ts) {
    using M = Mat<T>;
    constexpr int E = M::E, KB = 128 / (int)sizeof(T), WM = 4 / WN, MR = TM / WM / 16, NR = TN / WN / 16;
    constexpr int PAD = sizeof(T) == 4 ? 4 : 8, PITCH = TN + PAD;                 // elements, the strided operand's line
    constexpr int XB = TM * 128, WB = KN ? KB * PITCH * (int)sizeof(T) : TN * 128;
    constexpr int XP = TM * 8 / 256, WP = (TN * 8 + 255) / 256;
    static_assert(TM * 8 % 256 == 0, "whole pieces per thread");
    __shared__ __attribute__((aligned(16))) char lds[2 * (XB + WB)];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l15 = lane & 15, kk = lane >> 4;
    const int wm = wave / WN * (TM / WM), wn = wave % WN * (TN / WN);
    const unsigned id = die_order(blockIdx.x, gridDim.x);
    const int n0 = (int)(id % tiles_n) * TN;
    const int64_t t = id / tiles_n;

    int64_t r0, r1;
    int slot = 0, s = 0;
    if (spans) {
        s = find_span(a.sg.off, a.sg.S, a.sg.rows, t, ts, &r0, &r1);
        if (s < 0) return;
        slot = seg_slot(a.sg, s);
        if (slot < 0) return;
    } else {
        r0 = seg_off(a.sg, 0) + t * TM;
        r1 = seg_off(a.sg, a.sg.S);
        if (r1 > r0 + TM) r1 = r0 + TM;
        if (r0 >= r1) return;
    }
    const int nrow = (int)(r1 - r0);                                                 // 1 .. TM

    typename M::Acc acc[NR][MR];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int m = 0; m < MR; ++m) acc[n][m] = typename M::Acc{0, 0, 0, 0};

    // acc += X W' over k < klen; with `sel` only in the columns (rows of x) for which pred says so
    auto product = [&](const T* x, int64_t ldx, const T* w, int64_t ldw, int klen, auto sel, const bool* pred) {
        constexpr bool SEL = decltype(sel)::value;
        u32x4 xr[XP], wr[WP];
        auto load = [&](int k0) {
#pragma unroll
            for (int i = 0; i < XP; ++i) {
                const int pc = tid + 256 * i, row = pc >> 3;
                xr[i] = load_piece(x + (int64_t)min(row, nrow - 1) * ldx, k0 + (pc & 7) * E, klen);
            }
#pragma unroll
            for (int i = 0; i < WP; ++i) {
                const int pc = tid + 256 * i;
                if (TN * 8 % 256 && pc >= TN * 8) break;
                if (KN) {
                    const int k = pc / (TN / E), c = pc % (TN / E) * E;
                    wr[i] = k0 + k < klen ? load_piece(w + (int64_t)(k0 + k) * ldw, n0 + c, a.N) : u32x4{0, 0, 0, 0};
                } else {
                    const int row = pc >> 3;
                    wr[i] = load_piece(w + (int64_t)min(n0 + row, a.N - 1) * ldw, k0 + (pc & 7) * E, klen);
                }
            }
        };
        auto store = [&](int buf) {
            char* xs = lds + buf * (XB + WB);
            char* ws = xs + XB;
#pragma unroll
            for (int i = 0; i < XP; ++i) {
                const int pc = tid + 256 * i, row = pc >> 3;
                *(u32x4*)(xs + row * 128 + (((pc & 7) ^ (row & 7)) << 4)) = xr[i];
            }
#pragma unroll
            for (int i = 0; i < WP; ++i) {
                const int pc = tid + 256 * i;
                if (TN * 8 % 256 && pc >= TN * 8) break;
                if (KN) {
                    const int k = pc / (TN / E), c = pc % (TN / E) * E;
                    *(u32x4*)(ws + (k * PITCH + c) * (int)sizeof(T)) = wr[i];
                } else {
                    const int row = pc >> 3;
                    *(u32x4*)(ws + row * 128 + (((pc & 7) ^ (row & 7)) << 4)) = wr[i];
                }
            }
        };
        load(0);
        store(0);
        __syncthreads();
        int buf = 0;
        for (int k0 = 0; k0 < klen; k0 += KB, buf ^= 1) {
            const bool more = k0 + KB < klen;
            if (more) load(k0 + KB);
            const char* xs = lds + buf * (XB + WB);
            const char* ws = xs + XB;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                u32x4 xf[MR], wf[NR];
#pragma unroll
                for (int m = 0; m < MR; ++m) {
                    const int row = wm + 16 * m + l15;
                    xf[m] = *(const u32x4*)(xs + row * 128 + (((4 * h + kk) ^ (row & 7)) << 4));
                }
#pragma unroll
                for (int n = 0; n < NR; ++n) {
                    const int c = wn + 16 * n + l15;
                    if (KN) {
                        const T* col = (const T*)ws + (4 * h + kk) * E * PITCH + c;
                        T e[E];
#pragma unroll
                        for (int j = 0; j < E; ++j) e[j] = col[j * PITCH];
                        __builtin_memcpy(&wf[n], e, 16);
                    } else {
                        wf[n] = *(const u32x4*)(ws + c * 128 + (((4 * h + kk) ^ (c & 7)) << 4));
                    }
                }
#pragma unroll
                for (int n = 0; n < NR; ++n)
#pragma unroll
                    for (int m = 0; m < MR; ++m) {
                        const typename M::Acc d = M::mma(wf[n], xf[m], acc[n][m]);
                        if (SEL) {
                            // chosen, not masked by a product with zero: another row's adapter may hold a NaN
#pragma unroll
                            for (int r = 0; r < 4; ++r) acc[n][m][r] = pred[m] ? d[r] : acc[n][m][r];
                        } else {
                            acc[n][m] = d;
                        }
                    }
            }
            if (more) store(buf ^ 1);
            __syncthreads();
        }
    };

    const T* x = (const T*)a.x + r0 * a.ldx;
    product(x, a.ldx, (const T*)a.w + slot * a.w_stride, a.kn ? a.N : a.K, a.K, std::false_type{}, nullptr);

    if (a.low) {
        const T* p = (const T*)a.p + r0 * a.ldp;
        for (s = spans ? s : max(0, wave_search(a.sg.S, r0, [&](int i) { return seg_off(a.sg, i); })); s < a.sg.S; ++s) {
            const int64_t lo = seg_off(a.sg, s), hi = seg_off(a.sg, s + 1);
            if (lo >= r1) break;
            const int k = seg_slot(a.sg, s);
            if (hi <= r0 || lo >= hi || k < 0) continue;
            const T* low = (const T*)a.low + k * a.low_stride;
            if (lo <= r0 && hi >= r1) {
                product(p, a.ldp, low, a.kn ? a.N : a.R, a.R, std::false_type{}, nullptr);
                break;
            }
            bool pred[MR];
#pragma unroll
            for (int m = 0; m < MR; ++m) {
                const int64_t r = r0 + wm + 16 * m + l15;
                pred[m] = r >= lo && r < hi;
            }
            product(p, a.ldp, low, a.kn ? a.N : a.R, a.R, std::true_type{}, pred);
        }
    }

    const typename M::Sum scale = a.scale ? (typename M::Sum)a.scale[slot] : (typename M::Sum)1;
    const T* bias = a.bias ? (const T*)a.bias + slot * a.bias_stride : nullptr;
#pragma unroll
    for (int m = 0; m < MR; ++m) {
        const int row = wm + 16 * m + l15;
        if (row >= nrow) continue;
        T* y = (T*)a.y + (r0 + row) * a.ldy;
#pragma unroll
        for (int n = 0; n < NR; ++n) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int c = n0 + wn + 16 * n + M::row(r, kk);
                if (c >= a.N) continue;
                typename M::Sum v = acc[n][m][r] * scale;
                if (bias) v += (typename M::Sum)bias[c];
                y[c] = (T)v;                                                         // the one rounding of the result
            }
        }
    }
}

template <typename T, int TM, int TN, int WN>
static int launch_tile(lnasr_ctx* ctx, const RowsArgs& a, const char* name) {
    const bool spans = a.w_stride != 0 || a.scale != nullptr || a.bias_stride != 0;
    const int ts = TM == 128 ? 7 : TM == 64 ? 6 : 5;
    static_assert(TM == 128 || TM == 64 || TM == 32, "tile heights");
    const int64_t tiles_n = (a.N + TN - 1) / TN, tiles_m = spans ? a.sg.rows / TM + a.sg.S : (a.sg.rows + TM - 1) / TM;
    LN_REQUIRE(tiles_n * tiles_m < (1ll << 31), "%lld rows x %d results are too many for one call", (long long)a.sg.rows, a.N);
    if (a.kn)
        LN_LAUNCH(ctx, name, (rows_tile<T, TM, TN, WN, true>), dim3((unsigned)(tiles_n * tiles_m)), dim3(256), 0, a, (unsigned)tiles_n, spans, ts);
    else
        LN_LAUNCH(ctx, name, (rows_tile<T, TM, TN, WN, false>), dim3((unsigned)(tiles_n * tiles_m)), dim3(256), 0, a, (unsigned)tiles_n, spans, ts);
    return 0;
}

template <typename T>
static int rows_t(lnasr_ctx* ctx, const RowsArgs& a, const char* name) {
    return launch_tile<T, 64, 64, 2>(ctx, a, name);
}

int transform_rows(lnasr_ctx* ctx, int dtype, const RowsArgs& a, const char* name) {
    if (a.sg.rows == 0 || a.sg.S == 0 || a.N == 0) return 0;
    switch (dtype) {
        case LNASR_F64: return rows_t<double>(ctx, a, name);
        case LNASR_F32: return rows_t<float>(ctx, a, name);
        case LNASR_F16: return rows_t<_Float16>(ctx, a, name);
        default: return rows_t<__bf16>(ctx, a, name);
    }
}

}  // namespace lnasr
