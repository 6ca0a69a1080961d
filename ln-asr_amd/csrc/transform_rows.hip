// Feature transforms, products with one result row per feature row (transform.h: RowsArgs).
#include <algorithm>

#include "transform.h"

namespace lnasr {

// ------------------------------------------------------------------------------------------
// Tiles of TM rows x TN results, WM x WN waves.  Both operands pass through LDS in steps of 128 bytes of k, double buffered, as
// 16-byte pieces in the order of the threads that bring them (LDS-DMA, buffer_load ... lds, needs just that).  Which piece a
// thread brings is chosen so that the reads of a fragment spread over the banks:
//   k contiguous (x, and w [n, k]): rows of 8 pieces; place p of row r holds piece p ^ (r & 7)
//   k strided (w [k, n]): lines of k; a fragment's 16 columns are sizeof(T) pieces, and the run of 16 columns at place p of line k
//     is run p ^ spread(k).  16 bit: ds_read_b64_tr_b16 turns 4 k x 16 columns on the way to the registers.
// DMA: every operand is aligned to 16 bytes and as wide as whole pieces; otherwise the pieces travel through registers, loaded a
// step ahead.  The low-rank product is short and always takes the registers.
// LOW: 0 none; 1 tiles are spans of one segment, whose adapter joins in; 2 tiles of rows that lie together, the adapters of
// every segment they meet join in one after the other (short segments: a span of a few rows would waste its tile).
// ------------------------------------------------------------------------------------------
template <typename T, int TM, int TN, int WM, int WN, bool KN, bool DMA, int LOW>
__global__ __launch_bounds__(64 * WM * WN, 2) void rows_tile(RowsArgs a, unsigned tiles_n, int ts) {
    using M = Mat<T>;
    using Acc = typename M::Acc;
    constexpr int SZ = (int)sizeof(T), E = M::E, KB = 128 / SZ, NT = 64 * WM * WN, MR = TM / WM / 16, NR = TN / WN / 16;
    constexpr int XB = TM * 128, WB = TN * 128, XI = TM * 8 / NT, WI = (TN * 8 + NT - 1) / NT;
    constexpr int LINE = TN * SZ / 16;                                                // pieces of a line of w [k, n]
    static_assert(TM * 8 % NT == 0 && (TN * 8 % NT == 0 || (NT % (TN * 8) == 0)), "whole waves of pieces");
    __shared__ __attribute__((aligned(1024))) char lds[2 * (XB + WB)];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l15 = lane & 15, kk = lane >> 4;
    const int wm = wave / WN * (TM / WM), wn = wave % WN * (TN / WN);
    const bool brings_w = TN * 8 % NT == 0 || tid < TN * 8;                           // uniform over a wave
    const unsigned id = die_order(blockIdx.x, gridDim.x);
    const int n0 = (int)(id % tiles_n) * TN;
    const int64_t t = id / tiles_n;

    int64_t r0, r1;
    int slot = 0, s = 0;
    if (LOW != 2) {
        s = find_span(a.sg.off, a.sg.S, a.sg.rows, t, ts, &r0, &r1);
        if (s < 0) return;
        slot = seg_slot(a.sg, s);
        if (slot < 0 && LOW == 0) return;
    } else {
        r0 = seg_off(a.sg, 0) + t * TM;
        r1 = seg_off(a.sg, a.sg.S);
        if (r1 > r0 + TM) r1 = r0 + TM;
        if (r0 >= r1) return;
    }
    const int nrow = (int)(r1 - r0);                                                 // 1 .. TM

    Acc acc[NR][MR];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int m = 0; m < MR; ++m) acc[n][m] = Acc{0, 0, 0, 0};

    // acc += X W' over the 128 bytes of k in buffer buf; with SEL only in the columns (rows of x) for which pred says so
    auto multiply = [&](int buf, auto sel, const bool* pred) {
        constexpr bool SEL = decltype(sel)::value;
        const char* xs = lds + buf * (XB + WB);
        const char* ws = xs + XB;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            u32x4 xf[MR], wf[NR];
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                const int c = wn + 16 * n;
                if constexpr (!KN) {
                    wf[n] = *(const u32x4*)(ws + (c + l15) * 128 + (((4 * h + kk) ^ (l15 & 7)) << 4));
                } else {
                    wf[n] = strided_fragment<T, TN>(ws, h, c);
                }
            }
#pragma unroll
            for (int m = 0; m < MR; ++m) xf[m] = *(const u32x4*)(xs + (wm + 16 * m + l15) * 128 + (((4 * h + kk) ^ (l15 & 7)) << 4));
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int m = 0; m < MR; ++m) {
                    const Acc d = M::mma(wf[n], xf[m], acc[n][m]);
                    if (SEL) {
                        // chosen, not masked by a product with zero: another row's adapter may hold a NaN
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[n][m][r] = pred[m] ? d[r] : acc[n][m][r];
                    } else {
                        acc[n][m] = d;
                    }
                }
        }
    };

    // through registers
    u32x4 xr[XI], wr[WI];
    auto load = [&](const T* x, int64_t ldx, const T* w, int64_t ldw, int k0, int klen) {
#pragma unroll
        for (int i = 0; i < XI; ++i) {
            const int q = tid + NT * i, row = q >> 3;
            xr[i] = load_piece(x + (int64_t)min(row, nrow - 1) * ldx, k0 + ((q ^ row) & 7) * E, klen);
        }
        if (brings_w)
#pragma unroll
            for (int i = 0; i < WI; ++i) {
                const int q = tid + NT * i;
                if (KN) {
                    const int k = q / LINE, c = (q % LINE ^ spread<T, TN>(k) * SZ) * E;
                    wr[i] = k0 + k < klen ? load_piece(w + (int64_t)(k0 + k) * ldw, n0 + c, a.N) : u32x4{0, 0, 0, 0};
                } else {
                    const int row = q >> 3;
                    wr[i] = load_piece(w + (int64_t)min(n0 + row, a.N - 1) * ldw, k0 + ((q ^ row) & 7) * E, klen);
                }
            }
    };
    auto store = [&](int buf) {
        char* xs = lds + buf * (XB + WB);
#pragma unroll
        for (int i = 0; i < XI; ++i) *(u32x4*)(xs + (tid + NT * i) * 16) = xr[i];
        if (brings_w)
#pragma unroll
            for (int i = 0; i < WI; ++i) *(u32x4*)(xs + XB + (tid + NT * i) * 16) = wr[i];
    };

    const T* x = (const T*)a.x + r0 * a.ldx;
    const T* w = (const T*)a.w + (LOW ? 0 : slot * a.w_stride);
    const int64_t ldw = KN ? a.N : a.K;
    if constexpr (DMA) {
        // offsets of this lane's pieces from the tile's first; out of range (the hardware then writes zeros) where k or n ends
        constexpr unsigned OUT = 0xffffffffu;
        unsigned xo[XI], wo[WI];
        const int xk = ((tid ^ tid >> 3) & 7) * E;                                    // k of the lane's pieces in a step
#pragma unroll
        for (int i = 0; i < XI; ++i) xo[i] = (unsigned)min((tid + NT * i) >> 3, nrow - 1) * (unsigned)(a.ldx * SZ) + xk * SZ;
#pragma unroll
        for (int i = 0; i < WI; ++i) {
            const int q = tid + NT * i;
            if (KN) {
                const int k = q / LINE, c = (q % LINE ^ spread<T, TN>(k) * SZ) * E;
                wo[i] = n0 + c < a.N ? (unsigned)k * (unsigned)(ldw * SZ) + c * SZ : OUT;
            } else {
                wo[i] = (unsigned)min(q >> 3, a.N - 1 - n0) * (unsigned)(ldw * SZ) + xk * SZ;
            }
        }
        const char* xb = (const char*)x;
        const char* wb = (const char*)(KN ? w + n0 : w + (int64_t)n0 * ldw);
        auto bring = [&](int buf, int left) {
            char* xs = lds + buf * (XB + WB);
            const bool tail = left < KB;
#pragma unroll
            for (int i = 0; i < XI; ++i)
                bring_piece(xb, tail && xk >= left ? OUT : xo[i], xs + (wave * 64 + NT * i) * 16);
            if (brings_w)
#pragma unroll
                for (int i = 0; i < WI; ++i)
                    bring_piece(wb, tail && (KN ? (tid + NT * i) / LINE : xk) >= left ? OUT : wo[i], xs + XB + (wave * 64 + NT * i) * 16);
            xb += KB * SZ;
            wb += KN ? KB * ldw * SZ : KB * SZ;
        };
        bring(0, a.K);
        __syncthreads();
        int buf = 0;
        for (int left = a.K; left > 0; left -= KB, buf ^= 1) {
            if (left > KB) bring(buf ^ 1, left - KB);
            multiply(buf, std::false_type{}, nullptr);
            __syncthreads();
        }
    } else {
        load(x, a.ldx, w, ldw, 0, a.K);
        store(0);
        __syncthreads();
        int buf = 0;
        for (int k0 = 0; k0 < a.K; k0 += KB, buf ^= 1) {
            const bool more = k0 + KB < a.K;
            if (more) load(x, a.ldx, w, ldw, k0 + KB, a.K);
            multiply(buf, std::false_type{}, nullptr);
            if (more) store(buf ^ 1);
            __syncthreads();
        }
    }

    auto adapter = [&](int k, auto sel, const bool* pred) {
        const T* p = (const T*)a.p + r0 * a.ldp;
        const T* low = (const T*)a.low + k * a.low_stride;
        for (int k0 = 0; k0 < a.R; k0 += KB) {
            load(p, a.ldp, low, KN ? a.N : a.R, k0, a.R);
            store(0);
            __syncthreads();
            multiply(0, sel, pred);
            __syncthreads();
        }
    };
    if (LOW == 1 && slot >= 0) adapter(slot, std::false_type{}, nullptr);
    if (LOW == 2) {
        for (s = max(0, wave_search(a.sg.S, r0, [&](int i) { return seg_off(a.sg, i); })); s < a.sg.S; ++s) {
            const int64_t lo = seg_off(a.sg, s), hi = seg_off(a.sg, s + 1);
            if (lo >= r1) break;
            const int k = seg_slot(a.sg, s);
            if (hi <= r0 || lo >= hi || k < 0) continue;
            bool pred[MR];
#pragma unroll
            for (int m = 0; m < MR; ++m) {
                const int64_t r = r0 + wm + 16 * m + l15;
                pred[m] = r >= lo && r < hi;
            }
            adapter(k, std::true_type{}, pred);
        }
    }

    const typename M::Sum scale = LOW == 0 && a.scale ? (typename M::Sum)a.scale[slot] : (typename M::Sum)1;
    const T* bias = a.bias ? (const T*)a.bias + (LOW ? 0 : slot * a.bias_stride) : nullptr;
    // four results of a row lie together, but for fp64 (whose instruction spreads them over the rows of its tile)
    constexpr bool RUN = SZ != 8;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
        const int c0 = n0 + wn + 16 * n + (RUN ? 4 * kk : kk);
        typename M::Sum bv[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) bv[r] = bias && c0 + (RUN ? r : 4 * r) < a.N ? (typename M::Sum)bias[c0 + (RUN ? r : 4 * r)] : (typename M::Sum)0;
#pragma unroll
        for (int m = 0; m < MR; ++m) {
            const int row = wm + 16 * m + l15;
            if (row >= nrow) continue;
            T* y = (T*)a.y + (r0 + row) * a.ldy + c0;
            T v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = (T)(acc[n][m][r] * scale + bv[r]);     // the one rounding of the result
            if (RUN && c0 + 4 <= a.N) {
                __builtin_memcpy(y, v, 4 * SZ);
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (c0 + (RUN ? r : 4 * r) < a.N) y[RUN ? r : 4 * r] = v[r];
            }
        }
    }
}

template <typename T, int TM, int TN, int WM, int WN, bool KN, int LOW>
static int launch_tile(lnasr_ctx* ctx, const RowsArgs& a, const char* name) {
    constexpr int ts = TM == 256 ? 8 : TM == 128 ? 7 : 6;
    static_assert(TM == 1 << ts, "tile heights");
    const int64_t tiles_n = (a.N + TN - 1) / TN, tiles_m = LOW != 2 ? a.sg.rows / TM + a.sg.S : (a.sg.rows + TM - 1) / TM;
    LN_REQUIRE(tiles_n * tiles_m < (1ll << 31), "%lld rows x %d results are too many for one call", (long long)a.sg.rows, a.N);
    // 16-byte pieces throughout, and a tile's offsets within 31 bits
    const int64_t e = 16 / sizeof(T), ldw = KN ? a.N : a.K;
    const bool dma = ((uintptr_t)a.x | (uintptr_t)a.w) % 16 == 0 && a.K % e == 0 && (!KN || a.N % e == 0) && a.ldx % e == 0 &&
                     a.ldx * TM * (int64_t)sizeof(T) < (1ll << 31) && ldw * std::max(TN, 64) * (int64_t)sizeof(T) < (1ll << 31);
    const dim3 grid((unsigned)(tiles_n * tiles_m)), block(64 * WM * WN);
    if (dma) LN_LAUNCH(ctx, name, (rows_tile<T, TM, TN, WM, WN, KN, true, LOW>), grid, block, 0, a, (unsigned)tiles_n, ts);
    else LN_LAUNCH(ctx, name, (rows_tile<T, TM, TN, WM, WN, KN, false, LOW>), grid, block, 0, a, (unsigned)tiles_n, ts);
    return 0;
}

template <typename T, bool KN, int LOW>
static int rows_t(lnasr_ctx* ctx, const RowsArgs& a, const char* name) {
    if (a.N <= 32) return launch_tile<T, 128, 32, 4, 1, KN, LOW>(ctx, a, name);
    if (a.N <= 64) return launch_tile<T, 128, 64, 4, 1, KN, LOW>(ctx, a, name);
    if constexpr (sizeof(T) == 2) {
        if (a.sg.rows / 256 * (a.N / 256) >= 256) return launch_tile<T, 256, 256, 2, 4, KN, LOW>(ctx, a, name);
        return launch_tile<T, 128, 128, 2, 2, KN, LOW>(ctx, a, name);
    } else if constexpr (sizeof(T) == 4) {
        return launch_tile<T, 128, 128, 2, 2, KN, LOW>(ctx, a, name);
    } else {
        return launch_tile<T, 128, 128, 2, 4, KN, LOW>(ctx, a, name);
    }
}

template <typename T, bool KN>
static int rows_kn(lnasr_ctx* ctx, const RowsArgs& a, const char* name) {
    if (a.w_stride) return rows_t<T, KN, 0>(ctx, a, name);
    if (a.sg.rows / a.sg.S >= 64) return rows_t<T, KN, 1>(ctx, a, name);
    return launch_tile<T, 64, 64, 2, 2, KN, 2>(ctx, a, name);
}

template <typename T>
static int rows_any(lnasr_ctx* ctx, const RowsArgs& a, const char* name) {
    return a.kn ? rows_kn<T, true>(ctx, a, name) : rows_kn<T, false>(ctx, a, name);
}

int transform_rows(lnasr_ctx* ctx, int dtype, const RowsArgs& a, const char* name) {
    if (a.sg.rows == 0 || a.sg.S == 0 || a.N == 0) return 0;
    if (rows_narrow_ok(a)) return transform_rows_narrow(ctx, dtype, a, name);
    switch (dtype) {
        case LNASR_F64: return rows_any<double>(ctx, a, name);
        case LNASR_F32: return rows_any<float>(ctx, a, name);
        case LNASR_F16: return rows_any<_Float16>(ctx, a, name);
        default: return rows_any<__bf16>(ctx, a, name);
    }
}

}  // namespace lnasr
