// Feature transforms, products with one result row per feature row (transform.h: RowsArgs).
#include <algorithm>

#include "transform.h"

namespace lnasr {

// acc[n][m] += p L_k' for the rows row0 + 16 m + (lane & 15) < row1 and the columns c0 + 16 n .., segment by segment with the
// adapter of each (those numbered `turn` modulo `turns`).  64 segments are looked up at a time, a lane each; fragments come straight
// from memory: for segments of a few rows every adapter is read once and there is nothing to share.
template <typename T, bool KN, int MR, int NR>
__device__ __forceinline__ void add_adapters(const RowsArgs& a, int64_t row0, int64_t row1, int c0, int turn, int turns,
                                             typename Mat<T>::Acc (&acc)[NR][MR]) {
    using U = Mid<T>;                                     // (the adapters' matrices, too, are multiplied as values of this type)
    constexpr int E = Mat<U>::E;
    const int lane = threadIdx.x & 63, l15 = lane & 15, kk = lane >> 4;
    if (row0 >= row1) return;
    const int last = (int)(row1 - 1 - row0);
    const U* p = (const U*)a.p + row0 * a.ldp;
    int count = 0;
    for (int s = max(0, wave_search(a.sg.S, row0, [&](int i) { return seg_off(a.sg, i); })); s < a.sg.S; s += 64) {
        const int mine = min(s + lane, a.sg.S - 1);
        const int64_t lo = seg_off(a.sg, mine), hi = seg_off(a.sg, mine + 1);
        const int slot = seg_slot(a.sg, mine);
        const int from = (int)(max(lo, row0) - row0), to = (int)max((int64_t)0, min(hi, row1) - row0);     // (from may lie past `last`)
        for (uint64_t todo = __ballot(s + lane < a.sg.S && lo < row1 && from < to && slot >= 0); todo; todo &= todo - 1) {
            if (count++ % turns != turn) continue;
            const int b = __builtin_ctzll(todo), f = __builtin_amdgcn_readlane(from, b), t = __builtin_amdgcn_readlane(to, b);
            const T* low = (const T*)a.low + __builtin_amdgcn_readlane(slot, b) * a.low_stride;
            for (int k0 = 0; k0 < a.R; k0 += 4 * E) {
                const int k = k0 + kk * E;
                u32x4 wf[NR];
#pragma unroll
                for (int n = 0; n < NR; ++n) {
                    const int c = min(c0 + 16 * n + l15, a.N - 1);
                    if (KN) {
                        U e[E];
#pragma unroll
                        for (int j = 0; j < E; ++j) e[j] = k + j < a.R ? (U)low[(int64_t)(k + j) * a.N + c] : (U)0;
                        __builtin_memcpy(&wf[n], e, 16);
                    } else {
                        wf[n] = load_as<U>(low + (int64_t)c * a.R, k, a.R);
                    }
                }
#pragma unroll
                for (int m = 0; m < MR; ++m) {
                    if (t <= 16 * m || f >= 16 * m + 16) continue;
                    const int row = 16 * m + l15;
                    const u32x4 pf = load_piece(p + (int64_t)min(row, last) * a.ldp, k, a.R);
                    const bool in = row >= f && row < t;
#pragma unroll
                    for (int n = 0; n < NR; ++n) {
                        // chosen, not masked by a product with zero: another row's adapter may hold a NaN
                        const typename Mat<U>::Acc d = mma<U>(wf[n], pf, acc[n][m]);
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[n][m][r] = in ? d[r] : acc[n][m][r];
                    }
                }
            }
        }
        if (seg_off(a.sg, min(s + 64, a.sg.S)) >= row1) break;
    }
}

// Writes acc (times scale, plus bias) to the rows row0 + 16 m + (lane & 15) < row1, columns c0 + 16 n ..  Sixteen rows at a time pass
// through `scratch` (the wave's own put_scratch bytes of LDS), so that a row's results leave as whole runs of 16-byte pieces: as the
// matrix instruction leaves them, 32 bytes of a row at a time, twice the bytes went out to memory.
// Y: the type of the results.
template <typename Y, int NR>
constexpr int put_scratch() {
    return 16 * (NR * 16 * (int)sizeof(Y) + 16);
}
template <typename T, typename Y, int MR, int NR>
__device__ __forceinline__ void put_tile(const RowsArgs& a, int64_t row0, int64_t row1, int c0, typename Mat<T>::Sum scale, const T* bias,
                                         const typename Mat<T>::Acc (&acc)[NR][MR], char* scratch) {
    using M = Mat<T>;
    using Sum = typename M::Sum;
    constexpr int SZ = (int)sizeof(Y), E = 16 / SZ, PITCH = NR * 16 * SZ + 16, PER = NR * SZ;    // bytes, pieces of a row
    const int lane = threadIdx.x & 63, l15 = lane & 15, kk = lane >> 4;
    Sum bv[NR][4];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int c = c0 + 16 * n + M::row(r, kk);
            bv[n][r] = bias && c < a.N ? (Sum)bias[c] : (Sum)0;
        }
#pragma unroll
    for (int m = 0; m < MR; ++m) {
        if (row0 + 16 * m >= row1) break;
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            Y v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = (Y)(acc[n][m][r] * scale + bv[n][r]);             // the one rounding of the result
            if constexpr (SZ != 8) {
                __builtin_memcpy(scratch + l15 * PITCH + (16 * n + 4 * kk) * SZ, v, 4 * SZ);
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r) *(Y*)(scratch + l15 * PITCH + (16 * n + M::row(r, kk)) * SZ) = v[r];
            }
        }
        wave_lds_order();
#pragma unroll
        for (int i = 0; i < (16 * PER + 63) / 64; ++i) {
            const int q = lane + 64 * i, row = q / PER, c = c0 + q % PER * E;
            if (q >= 16 * PER || row0 + 16 * m + row >= row1 || c >= a.N) continue;
            const char* from = scratch + row * PITCH + q % PER * 16;
            Y* y = (Y*)a.y + (row0 + 16 * m + row) * a.ldy + c;
            if (c + E <= a.N) {
                const u32x4 v = *(const u32x4*)from;
                __builtin_memcpy(y, &v, 16);
            } else {
                for (int j = 0; j < a.N - c; ++j) y[j] = *(const Y*)(from + j * SZ);
            }
        }
        wave_lds_order();
    }
}

// ------------------------------------------------------------------------------------------
// A few rows: 16 MR rows x 16 results a block, its eight waves divide k between them.  Bound by the latency of memory and, with many
// groups, by the matrices read once: fragments go from memory to registers, many at a time, and meet in LDS at the end.
// bf16 64 single rows x 2048 -> 2048, 48 adapters of rank 16: 5.5 us for the middle and 12 for the rest, 15 MB, a pass 19; through
// the tiles below a pass takes 45.
// ------------------------------------------------------------------------------------------
template <typename T, typename Y, bool KN, int MR, int LOW>
__global__ __launch_bounds__(512) void rows_few(RowsArgs a, unsigned tiles_n, int ts) {
    using M = Mat<T>;
    using Acc = typename M::Acc;
    constexpr int E = M::E, WAVES = 8, DEEP = MR == 1 ? 8 : MR == 2 ? 4 : 2;
    __shared__ Acc part[WAVES - 1][MR][64];
    __shared__ __attribute__((aligned(16))) char scratch[put_scratch<Y, 1>()];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l15 = lane & 15, kk = lane >> 4;
    const int c0 = (int)(block_id() % tiles_n) * 16;
    int64_t r0, r1;
    int slot = 0;
    if (LOW == 0) {
        const int s = find_span(a.sg.off, a.sg.S, a.sg.rows, block_id() / tiles_n, ts, &r0, &r1);
        if (s < 0) return;
        slot = seg_slot(a.sg, s);
        if (slot < 0) return;
    } else {
        r0 = seg_off(a.sg, 0) + (int64_t)(block_id() / tiles_n) * (16 * MR);
        r1 = min(seg_off(a.sg, a.sg.S), r0 + 16 * MR);
        if (r0 >= r1) return;
    }
    const T* w = (const T*)a.w + (LOW ? 0 : slot * a.w_stride);
    const T* x[MR];
#pragma unroll
    for (int m = 0; m < MR; ++m) x[m] = (const T*)a.x + min(r0 + 16 * m + l15, r1 - 1) * a.ldx;
    const int c = min(c0 + l15, a.N - 1);
    Acc acc[1][MR];
#pragma unroll
    for (int m = 0; m < MR; ++m) acc[0][m] = Acc{0, 0, 0, 0};
    for (int k0 = wave * (4 * E * DEEP); k0 < a.K; k0 += WAVES * 4 * E * DEEP) {
        u32x4 wf[DEEP], xf[DEEP][MR];
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            const int k = k0 + (4 * d + kk) * E;
            if (KN) {
                T e[E];
#pragma unroll
                for (int j = 0; j < E; ++j) e[j] = k + j < a.K ? w[(int64_t)(k + j) * a.N + c] : (T)0;
                __builtin_memcpy(&wf[d], e, 16);
            } else {
                wf[d] = load_piece(w + (int64_t)c * a.K, k, a.K);
            }
#pragma unroll
            for (int m = 0; m < MR; ++m) xf[d][m] = load_piece(x[m], k, a.K);
        }
#pragma unroll
        for (int d = 0; d < DEEP; ++d)
#pragma unroll
            for (int m = 0; m < MR; ++m) acc[0][m] = mma<T>(wf[d], xf[d][m], acc[0][m]);
    }
    if (LOW) add_adapters<T, KN, MR, 1>(a, r0, r1, c0, wave, WAVES, acc);
    if (wave) {
#pragma unroll
        for (int m = 0; m < MR; ++m) part[wave - 1][m][lane] = acc[0][m];
    }
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int i = 0; i < WAVES - 1; ++i)
#pragma unroll
        for (int m = 0; m < MR; ++m) acc[0][m] += part[i][m][lane];
    const typename M::Sum scale = LOW == 0 && a.scale ? (typename M::Sum)a.scale[slot] : (typename M::Sum)1;
    put_tile<T, Y, MR, 1>(a, r0, r1, c0, scale, a.bias ? (const T*)a.bias + (LOW ? 0 : slot * a.bias_stride) : nullptr, acc, scratch);
}

// ------------------------------------------------------------------------------------------
// Tiles of TM rows x TN results, WM x WN waves.  Both operands pass through LDS in steps of 128 bytes of k, two steps ahead, as
// 16-byte pieces in the order of the threads that bring them (LDS-DMA, buffer_load ... lds, needs just that; its addresses need
// no alignment, so rows of 351 values take it too).  Which piece a thread brings is chosen so that the reads of a fragment spread
// over the banks:
//   k contiguous (x, and w [n, k]): rows of 8 pieces; place p of row r holds piece p ^ (r & 7)
//   k strided (w [k, n]): lines of k (spread, strided_fragment)
// The first `full` steps go by LDS-DMA, the rest -- a last step that ends inside a piece -- through registers.
// LOW: 0 tiles are spans of one segment, with its matrix.  One matrix for all rows, tiles of rows that lie together, and the
// adapters of the segments that a tile meets join in: 1 through LDS, a step for each; 2 straight from memory (add_adapters): rows_kn.
// f32 and f64 are bound by the matrix cores, and by the uneven last turn of the CUs: f32 120,011 x 351 x 128 with adapters of rank 8
// 122 us, 88 TFLOP/s of the 153 of a large library product; 20,011 x 512 x 429 95 us, cores busy 59 % of the time.  With few results
// they wait for memory: f32 200,003 x 351 x 40 95 us, 3.3 TB/s (rows of 351 values begin off any alignment: 352 take a fifth less).
// ------------------------------------------------------------------------------------------
template <typename T, typename Y, int TM, int TN, int WM, int WN, bool KN, int LOW>
__global__ __launch_bounds__(64 * WM * WN, 2) void rows_tile(RowsArgs a, unsigned tiles_n, int ts, int full) {
    using M = Mat<T>;
    using Acc = typename M::Acc;
    constexpr int SZ = (int)sizeof(T), E = M::E, KB = 128 / SZ, NT = 64 * WM * WN, MR = TM / WM / 16, NR = TN / WN / 16;
    constexpr int XB = TM * 128, WB = TN * 128, XI = TM * 8 / NT, WI = (TN * 8 + NT - 1) / NT;
    constexpr int LINE = TN * SZ / 16;                                                // pieces of a line of w [k, n]
    static_assert(TM * 8 % NT == 0 && TN * 8 % 64 == 0, "whole waves of pieces");
    // Three buffers for 16 bits, whose products are over before a step's bytes come; two for the others and for the large tile, which
    // gain more from the blocks that then fit beside each other (f32 120,011 x 351 x 128 with adapters: 137 against 128 us).
    // (variables of their own, not one array: the compiler then knows that reading one does not wait for what is brought into another)
    constexpr bool THREE = SZ == 2 && 3 * (XB + WB) <= (160 << 10) / 3;
    __shared__ __attribute__((aligned(1024))) char l0[XB + WB], l1[XB + WB], l2[THREE ? XB + WB : 16];
    constexpr int PUTS = (XB + WB) / put_scratch<Y, NR>();                            // put_tile's rows: waves a buffer has room for
    static_assert((THREE ? 3 : 2) * PUTS >= WM * WN && PUTS > 0, "put_tile's rows");
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l15 = lane & 15, kk = lane >> 4;
    const int wm = wave / WN * (TM / WM), wn = wave % WN * (TN / WN);
    const unsigned id = die_order(block_id(), block_count());
    const int n0 = (int)(id % tiles_n) * TN;
    const int64_t t = id / tiles_n;
    auto brings_w = [&](int i) { return TN * 8 % NT == 0 || wave * 64 + NT * i < TN * 8; };

    int64_t r0, r1;
    int slot = 0;
    if (LOW == 0) {
        const int s = find_span(a.sg.off, a.sg.S, a.sg.rows, t, ts, &r0, &r1);
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

    Acc acc[NR][MR];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int m = 0; m < MR; ++m) acc[n][m] = Acc{0, 0, 0, 0};

    // acc += X W' over the 128 bytes of k, values of type U, in a buffer; with SOME only for the rows from .. to - 1 of the wave's
    auto multiply = [&](auto type, const char* xs, auto some, int from, int to, int left = 1 << 20) {
        using U = decltype(type);
        constexpr bool SOME = decltype(some)::value;
        const char* ws = xs + XB;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (SOME && h && left <= 64 / (int)sizeof(U)) break;                      // (an adapter of a low rank)
            u32x4 xf[MR], wf[NR];
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                const int c = wn + 16 * n;
                if constexpr (KN) wf[n] = strided_fragment<U, TN>(ws, h, c);
                else wf[n] = *(const u32x4*)(ws + (c + l15) * 128 + (((4 * h + kk) ^ (l15 & 7)) << 4));
            }
#pragma unroll
            for (int m = 0; m < MR; ++m) xf[m] = *(const u32x4*)(xs + (wm + 16 * m + l15) * 128 + (((4 * h + kk) ^ (l15 & 7)) << 4));
            if constexpr (!SOME) mma_all<U>(wf, xf, acc);
            else
#pragma unroll
            for (int m = 0; m < MR; ++m) {
                if (to <= 16 * m || from >= 16 * m + 16) continue;
                if (from > 16 * m || to < 16 * m + 16) {
                    // chosen, not masked by a product with zero: another row's adapter may hold a NaN
                    const bool in = 16 * m + l15 >= from && 16 * m + l15 < to;
#pragma unroll
                    for (int n = 0; n < NR; ++n) {
                        const Acc d = mma<U>(wf[n], xf[m], acc[n][m]);
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[n][m][r] = in ? d[r] : acc[n][m][r];
                    }
                } else {
#pragma unroll
                    for (int n = 0; n < NR; ++n) acc[n][m] = mma<U>(wf[n], xf[m], acc[n][m]);
                }
            }
        }
    };

    // a step through registers, w as values of x's type: what lies past klen (or, in a line of w, past N) is 0
    struct Pieces {
        u32x4 x[XI], w[WI];
    };
    auto fetch = [&](Pieces& p, auto x, int64_t ldx, const T* w, int64_t ldw, int k0, int klen) {
        using U = std::remove_const_t<std::remove_pointer_t<decltype(x)>>;
        constexpr int E = Mat<U>::E, LINE = TN * (int)sizeof(U) / 16;
#pragma unroll
        for (int i = 0; i < XI; ++i) {
            const int q = tid + NT * i, row = q >> 3;
            p.x[i] = load_piece(x + (int64_t)min(row, nrow - 1) * ldx, k0 + ((q ^ row) & 7) * E, klen);
        }
#pragma unroll
        for (int i = 0; i < WI; ++i) {
            if (!brings_w(i)) break;
            const int q = tid + NT * i;
            if (KN) {
                const int k = q / LINE, c = (q % LINE ^ spread<U, TN>(k) * (int)sizeof(U)) * E;
                p.w[i] = k0 + k < klen ? load_as<U>(w + (int64_t)(k0 + k) * ldw, n0 + c, a.N) : u32x4{0, 0, 0, 0};
            } else {
                const int row = q >> 3;
                p.w[i] = load_as<U>(w + (int64_t)min(n0 + row, a.N - 1) * ldw, k0 + ((q ^ row) & 7) * E, klen);
            }
        }
    };
    auto apply = [&](auto type, const Pieces& p, auto some, int from, int to, int left = 1 << 20) {
#pragma unroll
        for (int i = 0; i < XI; ++i) *(u32x4*)(l0 + (tid + NT * i) * 16) = p.x[i];
#pragma unroll
        for (int i = 0; i < WI; ++i)
            if (brings_w(i)) *(u32x4*)(l0 + XB + (tid + NT * i) * 16) = p.w[i];
        __syncthreads();
        multiply(type, l0, some, from, to, left);
        __syncthreads();
    };

    const T* x = (const T*)a.x + r0 * a.ldx;
    const T* w = (const T*)a.w + (LOW ? 0 : slot * a.w_stride);
    const int64_t ldw = KN ? a.N : a.K;
    // what comes behind the steps of the LDS-DMA, asked for before them: the last, uneven step, and the first adapter's first
    Pieces rest, first;
    if (full * KB < a.K) fetch(rest, x, a.ldx, w, ldw, full * KB, a.K);
    // the first segment of the tile from s on that has rows in it and an adapter; a.sg.S: none
    auto next_adapter = [&](int s, int64_t* lo, int64_t* hi, int* k) {
        for (; s < a.sg.S; ++s) {
            *lo = seg_off(a.sg, s);
            *hi = seg_off(a.sg, s + 1);
            if (*lo >= r1) break;
            *k = seg_slot(a.sg, s);
            if (*hi > r0 && *lo < *hi && *k >= 0) return s;
        }
        return a.sg.S;
    };
    using U = Mid<T>;                                                                 // (the adapters' products are of this type)
    constexpr int KU = 128 / (int)sizeof(U);
    const U* p = (const U*)a.p + r0 * a.ldp;
    int64_t lo = 0, hi = 0;
    int s = 0, k = 0;
    if (LOW == 1) {
        s = next_adapter(max(0, wave_search(a.sg.S, r0, [&](int i) { return seg_off(a.sg, i); })), &lo, &hi, &k);
        if (s < a.sg.S) fetch(first, p, a.ldp, (const T*)a.low + k * a.low_stride, KN ? a.N : a.R, 0, a.R);
    }
    if (full > 0) {
        // offsets of this lane's pieces from the step's first; out of range (nothing is read, LDS gets zeros) past the last column
        unsigned xo[XI], wo[WI];
        const int xk = ((tid ^ tid >> 3) & 7) * 16;
#pragma unroll
        for (int i = 0; i < XI; ++i) xo[i] = (unsigned)min((tid + NT * i) >> 3, nrow - 1) * (unsigned)(a.ldx * SZ) + xk;
#pragma unroll
        for (int i = 0; i < WI; ++i) {
            const int q = tid + NT * i;
            if (KN) {
                const int k = q / LINE, c = (q % LINE ^ spread<T, TN>(k) * SZ) * E;
                wo[i] = n0 + c < a.N ? (unsigned)k * (unsigned)(ldw * SZ) + c * SZ : 0xffffffffu;
            } else {
                wo[i] = (unsigned)min(q >> 3, a.N - 1 - n0) * (unsigned)(ldw * SZ) + xk;
            }
        }
        const char* xb = (const char*)x;
        const char* wb = (const char*)(KN ? w + n0 : w + (int64_t)n0 * ldw);
        auto bring = [&](char* xs) {
#pragma unroll
            for (int i = 0; i < XI; ++i) bring_piece(xb, xo[i], xs + (wave * 64 + NT * i) * 16);
#pragma unroll
            for (int i = 0; i < WI; ++i)
                if (brings_w(i)) bring_piece(wb, wo[i], xs + XB + (wave * 64 + NT * i) * 16);
            xb += KB * SZ;
            wb += KN ? KB * ldw * SZ : KB * SZ;
        };
        bring(l0);
        if (THREE && full > 1) bring(l1);
        // At the barrier this step has arrived for every wave, and every wave is done with the step before, whose buffer takes the
        // step after next; the next one's requests (a wave's XI of x, and its WI of w) may still be out.  (Two buffers: the next
        // step is asked for only here, and waited for whole.)
        auto turn = [&](int i, const char* now, char* free) {
            if (!THREE || i + 1 >= full) __builtin_amdgcn_s_waitcnt(0x0070);          // vmcnt(0) lgkmcnt(0)
            else if (brings_w(WI - 1)) __builtin_amdgcn_s_waitcnt(0x0070 | (XI + WI));
            else __builtin_amdgcn_s_waitcnt(0x0070 | (XI + WI - 1));
            __builtin_amdgcn_s_barrier();
            if (i + (THREE ? 2 : 1) < full) bring(free);
            multiply(T{}, now, std::false_type{}, 0, 0);
        };
        static_assert(XI + WI < 16, "a wait's low counter");
        if constexpr (THREE) {
            for (int i = 0; i < full; i += 3) {
                turn(i, l0, l2);
                if (i + 1 < full) turn(i + 1, l1, l0);
                if (i + 2 < full) turn(i + 2, l2, l1);
            }
        } else {
            for (int i = 0; i < full; i += 2) {
                turn(i, l0, l1);
                if (i + 1 < full) turn(i + 1, l1, l0);
            }
        }
        __syncthreads();
    }
    for (int k0 = full * KB; k0 < a.K; k0 += KB) {
        if (k0 > full * KB) fetch(rest, x, a.ldx, w, ldw, k0, a.K);
        apply(T{}, rest, std::false_type{}, 0, 0);
    }
    if (LOW == 1) {
        for (bool waits = true; s < a.sg.S; waits = false, s = next_adapter(s + 1, &lo, &hi, &k)) {
            const int from = lo > r0 ? (int)(lo - r0) - wm : 0, to = hi < r1 ? (int)(hi - r0) - wm : TM;
            for (int k0 = 0; k0 < a.R; k0 += KU) {
                if (!waits || k0 > 0) fetch(first, p, a.ldp, (const T*)a.low + k * a.low_stride, KN ? a.N : a.R, k0, a.R);
                apply(U{}, first, std::true_type{}, from, to, a.R - k0);
            }
        }
    }
    if (LOW == 2) add_adapters<T, KN, MR, NR>(a, r0 + wm, r1, n0 + wn, 0, 1, acc);

    const typename M::Sum scale = LOW == 0 && a.scale ? (typename M::Sum)a.scale[slot] : (typename M::Sum)1;
    put_tile<T, Y, MR, NR>(a, r0 + wm, r1, n0 + wn, scale, a.bias ? (const T*)a.bias + (LOW ? 0 : slot * a.bias_stride) : nullptr, acc,
                           (wave < PUTS ? l0 : wave < 2 * PUTS ? l1 : l2) + wave % PUTS * put_scratch<Y, NR>());
}

// ------------------------------------------------------------------------------------------
// The same for 16-bit types and wide matrices: 256 x 256 results, eight waves of 128 x 64, steps of 64 k through a ring of five LDS
// buffers of 32 KB (x and w of a step take two).  While half a step multiplies, the fragments of the next half are read; w of the
// step after next and x of the one behind it are asked for in the middle of each step, where its own buffers fall free: the matrix
// cores, the LDS and the memory each work ahead of one another, with one barrier a step and a wait that counts (the newest four
// requests, x of the step after next, may be out).
// bf16 65,536 x 2048 x 2048 in 32 equal groups: 500-520 us, 1060-1100 TFLOP/s (a library's product of 8192^3: 1270-1310); in ragged
// ones 515-535, 8.5 turns of the CUs taking nine.  16,384 x 1024 x 1024: 36 us, 960; with adapters of rank 16 47, a step each through
// registers and 32-bit instructions, of a sixteenth of the rate.
// ------------------------------------------------------------------------------------------
// Up to 64 segments, a lane each: the tiles of 256 rows numbered without gaps (find_span leaves some), so that the dies get equally
// many: 16,384 x 1024 x 1024 of one group 55 -> 36 us.  (All whole tiles before the segments' last ones, for a shorter last turn of
// the CUs, gained nothing: those then fetch their matrices again.)  False: no tile for this block.
__device__ __forceinline__ bool exact_tile(const Segments& sg, unsigned id, unsigned tiles_n, unsigned* tn, int* slot, int64_t* r0, int64_t* r1) {
    const int lane = threadIdx.x & 63, s = min(lane, sg.S - 1);
    const int64_t lo = seg_off(sg, s), n = max((int64_t)0, seg_off(sg, s + 1) - lo);
    const int k = lane < sg.S ? seg_slot(sg, s) : -1, mine = k < 0 ? 0 : (int)((n + 255) >> 8);
    int sum = mine;                                                                   // running sum over the segments
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int v = __shfl_up(sum, d);
        sum += lane >= d ? v : 0;
    }
    const unsigned tiles = (unsigned)__builtin_amdgcn_readlane(sum, 63);
    if (id >= tiles * tiles_n) return false;
    unsigned tm;
    tile_order(die_order(id, tiles * tiles_n), tiles, tiles_n, &tm, tn);
    const int from = __builtin_ctzll(__ballot(sum > (int)tm));
    *slot = __builtin_amdgcn_readlane(k, from);
    *r0 = seg_off(sg, from) + (int64_t)(tm - (unsigned)__builtin_amdgcn_readlane(sum - mine, from)) * 256;
    *r1 = min(*r0 + 256, max(*r0, seg_off(sg, from + 1)));
    return true;
}

template <typename T, bool KN, int LOW>
__global__ __launch_bounds__(512, 2) void rows_deep(RowsArgs a, unsigned tiles_m, unsigned tiles_n, int full) {
    using M = Mat<T>;
    using Acc = typename M::Acc;
    constexpr int SZ = 2, E = 8, KB = 64, NT = 512, MR = 8, NR = 4, TM = 256, TN = 256, LINE = TN * SZ / 16;
    static_assert(sizeof(T) == 2, "16-bit types");
    // (five variables, not one array: the compiler then knows that reading one does not wait for what is brought into another)
    __shared__ __attribute__((aligned(1024))) char u0[TM * 128], u1[TM * 128], u2[TM * 128], u3[TM * 128], u4[TM * 128];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l15 = lane & 15, kk = lane >> 4;
    const int wm = wave / 4 * 128, wn = wave % 4 * 64;
    unsigned tm, tn;
    int64_t r0, r1;
    int slot = 0;
    if (LOW == 0 && a.sg.S <= 64) {
        if (!exact_tile(a.sg, block_id(), tiles_n, &tn, &slot, &r0, &r1)) return;
    } else {
        if (block_id() >= tiles_m * tiles_n) return;
        tile_order(die_order(block_id(), tiles_m * tiles_n), tiles_m, tiles_n, &tm, &tn);
    }
    const int n0 = (int)tn * TN;
    if (LOW == 0 && a.sg.S > 64) {
        const int s = find_span(a.sg.off, a.sg.S, a.sg.rows, tm, 8, &r0, &r1);
        if (s < 0) return;
        slot = seg_slot(a.sg, s);
        if (slot < 0) return;
    } else if (LOW) {
        r0 = seg_off(a.sg, 0) + (int64_t)tm * TM;
        r1 = seg_off(a.sg, a.sg.S);
        if (r1 > r0 + TM) r1 = r0 + TM;
        if (r0 >= r1) return;
    }
    const int nrow = (int)(r1 - r0);

    Acc acc[NR][MR];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int m = 0; m < MR; ++m) acc[n][m] = Acc{0, 0, 0, 0};
    struct Frags {
        u32x4 x[MR], w[NR];
    };
    auto read_as = [&](auto type, const char* xs, const char* ws, int h, Frags& f) {
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const int c = wn + 16 * n;
            if constexpr (KN) f.w[n] = strided_fragment<decltype(type), TN>(ws, h, c);
            else f.w[n] = *(const u32x4*)(ws + (c + l15) * 128 + (((4 * h + kk) ^ (l15 & 7)) << 4));
        }
#pragma unroll
        for (int m = 0; m < MR; ++m) f.x[m] = *(const u32x4*)(xs + (wm + 16 * m + l15) * 128 + (((4 * h + kk) ^ (l15 & 7)) << 4));
    };
    auto read = [&](const char* xs, const char* ws, int h, Frags& f) { read_as(T{}, xs, ws, h, f); };
    // (a fragment of x meets its four of w and is done with: the next one can take its registers)
    auto multiply = [&](const Frags& f) {
#pragma unroll
        for (int m = 0; m < MR; ++m)
#pragma unroll
            for (int n = 0; n < NR; ++n) acc[n][m] = mma<T>(f.w[n], f.x[m], acc[n][m]);
    };
    // an adapter's: rows from .. to - 1 of the wave's only
    using U = Mid<T>;
    constexpr int KU = 128 / (int)sizeof(U);
    auto multiply_some = [&](const Frags& f, int from, int to) {
#pragma unroll
        for (int m = 0; m < MR; ++m) {
            if (to <= 16 * m || from >= 16 * m + 16) continue;
            if (from > 16 * m || to < 16 * m + 16) {
                // chosen, not masked by a product with zero: another row's adapter may hold a NaN
                const bool in = 16 * m + l15 >= from && 16 * m + l15 < to;
#pragma unroll
                for (int n = 0; n < NR; ++n) {
                    const Acc d = mma<U>(f.w[n], f.x[m], acc[n][m]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[n][m][r] = in ? d[r] : acc[n][m][r];
                }
            } else {
#pragma unroll
                for (int n = 0; n < NR; ++n) acc[n][m] = mma<U>(f.w[n], f.x[m], acc[n][m]);
            }
        }
    };
    const T* x = (const T*)a.x + r0 * a.ldx;
    const T* w = (const T*)a.w + (LOW ? 0 : slot * a.w_stride);
    const int64_t ldw = KN ? a.N : a.K;
    if (full > 0) {
        unsigned xo[4], wo[4];
        const int xk = ((tid ^ tid >> 3) & 7) * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i) xo[i] = (unsigned)min((tid + NT * i) >> 3, nrow - 1) * (unsigned)(a.ldx * SZ) + xk;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int q = tid + NT * i;
            if (KN) {
                const int k = q / LINE, c = (q % LINE ^ spread<T, TN>(k) * SZ) * E;
                wo[i] = n0 + c < a.N ? (unsigned)k * (unsigned)(ldw * SZ) + c * SZ : 0xffffffffu;
            } else {
                wo[i] = (unsigned)min(q >> 3, a.N - 1 - n0) * (unsigned)(ldw * SZ) + xk;
            }
        }
        const char* xb = (const char*)x;
        const char* wb = (const char*)(KN ? w + n0 : w + (int64_t)n0 * ldw);
        auto bring_x = [&](char* u) {
#pragma unroll
            for (int i = 0; i < 4; ++i) bring_piece(xb, xo[i], u + (wave * 64 + NT * i) * 16);
            xb += KB * SZ;
        };
        auto bring_w = [&](char* u) {
#pragma unroll
            for (int i = 0; i < 4; ++i) bring_piece(wb, wo[i], u + (wave * 64 + NT * i) * 16);
            wb += KN ? KB * ldw * SZ : KB * SZ;
        };
        constexpr int VM0 = 0x0f70, VM4 = 0x0f74;                                     // s_waitcnt vmcnt(n), the other counters free
        bring_x(u0);
        bring_w(u1);
        if (full > 1) {
            bring_x(u2);
            bring_w(u3);
        }
        if (full > 2) bring_x(u4);
        __builtin_amdgcn_s_waitcnt(VM0);
        __builtin_amdgcn_s_barrier();
        Frags f0, f1;
        read(u0, u1, 0, f0);
        // One step: its x and w in xs, ws; the next one's in xn, wn.  At the barrier the next step has arrived for every wave, and
        // every wave has read all of this one, whose buffers take w of the step after next and x of the one behind.
        auto run = [&](char* xs, char* ws, const char* xn, const char* wn_) {
            auto interleave = [&]() {                                                 // a read behind every two or three products
                if constexpr (KN) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x008, 3, 0);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            };
            read(xs, ws, 1, f1);
            multiply(f0);
            interleave();
            __builtin_amdgcn_s_waitcnt(VM4 & 0xf0ff);                                 // vmcnt(4) lgkmcnt(0)
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
            bring_w(xs);
            bring_x(ws);
            read(xn, wn_, 0, f0);
            multiply(f1);
            __builtin_amdgcn_sched_group_barrier(0x020, 8, 0);
            interleave();
        };
        auto turn = [&](int s, char* xs, char* ws, const char* xn, const char* wn_) {
            read(xs, ws, 1, f1);
            multiply(f0);
            __builtin_amdgcn_s_waitcnt(VM0 & 0xf0ff);
            __builtin_amdgcn_s_barrier();
            if (s + 2 < full) bring_w(xs);
            if (s + 3 < full) bring_x(ws);
            if (s + 1 < full) read(xn, wn_, 0, f0);
            multiply(f1);
        };
        int s = 0;
        for (; s + 8 <= full; s += 5) {
            run(u0, u1, u2, u3);
            run(u2, u3, u4, u0);
            run(u4, u0, u1, u2);
            run(u1, u2, u3, u4);
            run(u3, u4, u0, u1);
        }
        for (; s < full; s += 5) {
            turn(s, u0, u1, u2, u3);
            if (s + 1 < full) turn(s + 1, u2, u3, u4, u0);
            if (s + 2 < full) turn(s + 2, u4, u0, u1, u2);
            if (s + 3 < full) turn(s + 3, u1, u2, u3, u4);
            if (s + 4 < full) turn(s + 4, u3, u4, u0, u1);
        }
        __syncthreads();
    }
    // one step through registers, w as values of x's type: what lies past klen (or, in a line of w, past N) is 0
    auto step = [&](auto x, int64_t ldx, const T* w, int64_t ldw, int k0, int klen, auto some, int from, int to) {
        using V = std::remove_const_t<std::remove_pointer_t<decltype(x)>>;
        constexpr int E = Mat<V>::E, LINE = TN * (int)sizeof(V) / 16;
        u32x4 xr[4], wr[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int q = tid + NT * i, row = q >> 3;
            xr[i] = load_piece(x + (int64_t)min(row, nrow - 1) * ldx, k0 + ((q ^ row) & 7) * E, klen);
            if (KN) {
                const int k = q / LINE, c = (q % LINE ^ spread<V, TN>(k) * (int)sizeof(V)) * E;
                wr[i] = k0 + k < klen ? load_as<V>(w + (int64_t)(k0 + k) * ldw, n0 + c, a.N) : u32x4{0, 0, 0, 0};
            } else {
                wr[i] = load_as<V>(w + (int64_t)min(n0 + row, a.N - 1) * ldw, k0 + ((q ^ row) & 7) * E, klen);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            *(u32x4*)(u0 + (tid + NT * i) * 16) = xr[i];
            *(u32x4*)(u1 + (tid + NT * i) * 16) = wr[i];
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (h && klen - k0 <= 64 / (int)sizeof(V)) break;
            Frags f;
            read_as(V{}, u0, u1, h, f);
            if constexpr (decltype(some)::value) multiply_some(f, from, to);
            else multiply(f);
        }
        __syncthreads();
    };
    for (int k0 = full * KB; k0 < a.K; k0 += KB) step(x, a.ldx, w, ldw, k0, a.K, std::false_type{}, 0, 0);
    if (LOW == 1) {
        const U* p = (const U*)a.p + r0 * a.ldp;
        for (int s = max(0, wave_search(a.sg.S, r0, [&](int i) { return seg_off(a.sg, i); })); s < a.sg.S; ++s) {
            const int64_t lo = seg_off(a.sg, s), hi = seg_off(a.sg, s + 1);
            if (lo >= r1) break;
            const int k = seg_slot(a.sg, s);
            if (hi <= r0 || lo >= hi || k < 0) continue;
            const T* low = (const T*)a.low + k * a.low_stride;
            const int from = lo > r0 ? (int)(lo - r0) - wm : 0, to = hi < r1 ? (int)(hi - r0) - wm : TM;
            for (int k0 = 0; k0 < a.R; k0 += KU) step(p, a.ldp, low, KN ? a.N : a.R, k0, a.R, std::true_type{}, from, to);
        }
    }
    const typename M::Sum scale = LOW == 0 && a.scale ? (typename M::Sum)a.scale[slot] : (typename M::Sum)1;
    put_tile<T, T, MR, NR>(a, r0 + wm, r1, n0 + wn, scale, a.bias ? (const T*)a.bias + (LOW ? 0 : slot * a.bias_stride) : nullptr, acc,
                           (wave < 4 ? u0 : u1) + wave % 4 * put_scratch<T, NR>());
}

constexpr int log2_of(int v) { return v <= 1 ? 0 : 1 + log2_of(v / 2); }

template <typename T, int TM, int TN, int WM, int WN, bool KN, int LOW, typename Y = T>
static int launch_tile(lnasr_ctx* ctx, const RowsArgs& a, const char* name) {
    static_assert(TM == 1 << log2_of(TM), "tile heights");
    constexpr int KB = 128 / (int)sizeof(T), E = Mat<T>::E;
    const int64_t tiles_n = (a.N + TN - 1) / TN, tiles_m = LOW == 0 ? a.sg.rows / TM + a.sg.S : (a.sg.rows + TM - 1) / TM;
    LN_REQUIRE(tiles_n * tiles_m < (1ll << 31), "%lld rows x %d results are too many for one call", (long long)a.sg.rows, a.N);
    // Steps for the LDS-DMA: whole ones; not the last line of w [k, n] where a piece would run past its end (elsewhere it runs
    // into the next line); none where a tile's offsets pass 31 bits
    const int64_t ldw = KN ? a.N : a.K;
    int full = KN && a.N % E ? (a.K - 1) / KB : a.K / KB;
    if (a.ldx * TM * (int64_t)sizeof(T) >= (1ll << 31) || ldw * std::max(TN, KB) * (int64_t)sizeof(T) >= (1ll << 31)) full = 0;
    LN_LAUNCH(ctx, name, (rows_tile<T, Y, TM, TN, WM, WN, KN, LOW>), transform_grid(tiles_n * tiles_m, 64 * WM * WN), dim3(64 * WM * WN), 0, a,
              (unsigned)tiles_n, log2_of(TM), full);
    return 0;
}

template <typename T, bool KN, int LOW>
static int launch_deep(lnasr_ctx* ctx, const RowsArgs& a, const char* name) {
    const int64_t tiles_n = (a.N + 255) / 256, tiles_m = LOW == 0 ? a.sg.rows / 256 + a.sg.S : (a.sg.rows + 255) / 256;
    LN_REQUIRE(tiles_n * tiles_m < (1ll << 31) && tiles_m < (1ll << 24), "%lld rows x %d results are too many for one call",
               (long long)a.sg.rows, a.N);
    int full = KN && a.N % 8 ? (a.K - 1) / 64 : a.K / 64;                             // as in launch_tile
    if (a.ldx * 512 >= (1ll << 31) || (KN ? a.N : a.K) * 512ll >= (1ll << 31)) full = 0;
    LN_LAUNCH(ctx, name, (rows_deep<T, KN, LOW>), transform_grid(tiles_n * tiles_m, 512), dim3(512), 0, a, (unsigned)tiles_m, (unsigned)tiles_n, full);
    return 0;
}

template <typename T, bool KN, int MR, int LOW>
static int launch_few(lnasr_ctx* ctx, const RowsArgs& a, const char* name) {
    const int64_t tiles_n = (a.N + 15) / 16, tiles_m = LOW == 0 ? a.sg.rows / (16 * MR) + a.sg.S : (a.sg.rows + 16 * MR - 1) / (16 * MR);
    LN_REQUIRE(tiles_n * tiles_m < (1ll << 31), "%lld rows x %d results are too many for one call", (long long)a.sg.rows, a.N);
    const dim3 grid = transform_grid(tiles_n * tiles_m, 512);
    if constexpr (LOW == 0 && !std::is_same<T, Mid<T>>::value)
        if (a.mid) {
            LN_LAUNCH(ctx, name, (rows_few<T, Mid<T>, KN, MR, LOW>), grid, dim3(512), 0, a, (unsigned)tiles_n, log2_of(16 * MR));
            return 0;
        }
    LN_LAUNCH(ctx, name, (rows_few<T, T, KN, MR, LOW>), grid, dim3(512), 0, a, (unsigned)tiles_n, log2_of(16 * MR));
    return 0;
}

template <typename T, bool KN, int LOW>
static int rows_t(lnasr_ctx* ctx, const RowsArgs& a, const char* name) {
    const int64_t cus = ctx->prop.multiProcessorCount, rows = a.sg.rows;
    if constexpr (LOW == 0 && !std::is_same<T, Mid<T>>::value) {                      // a middle: narrow, in a type of its own
        if (a.mid) {
            if (a.N <= 16) return launch_tile<T, 64, 16, 4, 1, KN, LOW, Mid<T>>(ctx, a, name);
            if (a.N <= 32) return launch_tile<T, 64, 32, 4, 1, KN, LOW, Mid<T>>(ctx, a, name);
            if (a.N <= 48) return launch_tile<T, 64, 48, 4, 1, KN, LOW, Mid<T>>(ctx, a, name);
            return launch_tile<T, 64, 64, 2, 2, KN, LOW, Mid<T>>(ctx, a, name);
        }
    }
    // (16-bit adapters from memory: short segments, whose time the adapters are)
    if constexpr (LOW != 2 || sizeof(T) != 2) {
        // few results: us, 64 x 64 / as wide as they are: f32 200,003 x 351 -> 8 99 / 57, -> 24 98 / 72, -> 48 104 / 90; f64 60,001 x
        // 351 -> 16 50 / 29; bf16 200,003 x 512 -> 16 38 / 32, -> 48 39 / 39
        if (a.N <= 16) return launch_tile<T, 64, 16, 4, 1, KN, LOW>(ctx, a, name);
        if (a.N <= 32) return launch_tile<T, 64, 32, 4, 1, KN, LOW>(ctx, a, name);
        if (a.N <= 48) return launch_tile<T, 64, 48, 4, 1, KN, LOW>(ctx, a, name);
        // 16 bits: the larger the tile the less it asks of the memory for its products (us, 64 x 64 / 128 x 128 / 256 x 256: 65,536 x
        // 2048 x 2048 1185 / 634 / 496; 16,384 x 1024 x 1024 65 / 47 / 36), as long as there is one for every CU.  32 and 64 bits
        // have time for that: 64 x 64 leaves the least over at the ends (f32 120,011 x 351 x 128 105 against 142 us, f64 16,384 x
        // 1024 x 1024 609 against 640; f32 65,536 x 1024 x 1024 1169 against 1165).
        // Tiles of one segment's rows want segments about as long: 256 of 192 rows x 2048 -> 2048 1002 / 620 / 556, 512 of 96 1125 / 763 /
        // 866, 1024 of 32 1184 / 1134 / 1581; 4096 of 4 x 1024 -> 256 231 / 268 / -, x 1000 -> 64 67 / 138 / -.
        if constexpr (sizeof(T) == 2) {
            if (rows / 256 * (a.N / 256) >= cus && (LOW || rows / a.sg.S >= 192)) return launch_deep<T, KN, LOW>(ctx, a, name);
            if (a.N > 64 && (LOW || rows / a.sg.S >= 32) && (rows / 128 + a.sg.S / 2) * ((a.N + 127) / 128) >= 2 * cus) return launch_tile<T, 128, 128, 2, 2, KN, LOW>(ctx, a, name);
        }
    }
    return launch_tile<T, 64, 64, 2, 2, KN, LOW>(ctx, a, name);
}

// The mean rows of a segment up to which rows_few, which divides k, is faster than the tiles at any number of segments; 0: at none.
// us, few / tile: f64 2048 -> 16, 4096 of 2 rows 167 / 266, 1024 of 12 74 / 100; 1024 -> 256, 4096 of 4 1513 / 1847, 1024 of 12 506 / 498
// (dx 403 / 532); 351 -> 40, 4096 of 4 137 / 146; 351 -> 128, 2048 of 8 204 / 191.  f32 2048 -> 16, 1024 of 12 44 / 53; 1024 -> 256, 8192 of 1
// 1742 / 1903, 4096 of 4 943 / 958, 1024 of 12 310 / 273; 512 -> 64, 4096 of 2 145 / 139; 351 -> 8, 8192 of 1 66 / 68.  bf16 2048 -> 8, 8192 of
// 1 83 / 98, 4096 of 4 49 / 55, 1024 of 12 21 / 19; -> 16, 8192 of 1 103 / 98; dx 15 <- 1823, 8192 of 1 114 / 205, 1024 of 12 33 / 46; 16 <-
// 2048, 8192 of 1 104 / 98.
template <typename T, bool KN>
static int few_mean(const RowsArgs& a) {
    const int64_t line = a.K * (int64_t)sizeof(T);
    if (sizeof(T) == 2) return a.K < 1024 ? 0 : KN ? (a.N <= 16 && a.N % 8 ? 12 : 0) : a.N <= 8 ? 4 : 0;
    if (a.N <= 32) return line >= 2048 ? 12 : 0;
    return line >= 4000 ? (sizeof(T) == 8 ? 12 : 4) : sizeof(T) == 8 && line >= 2048 ? 4 : 0;
}

template <typename T, bool KN>
static int rows_kn(lnasr_ctx* ctx, const RowsArgs& a, const char* name) {
    const int64_t cus = ctx->prop.multiProcessorCount, rows = a.sg.rows, mean = rows / a.sg.S;
    if (a.w_stride) {
        // Short segments, as long as the blocks of 16 x 16 find room on the CUs; past that each block's pass over x and W by itself
        // costs more than the tiles' empty rows, all the more where the mean hides a long segment.  us, few / tile (S segments of the
        // mean): bf16 512 -> 256, 64 of 1 12.0 / 12.0, 256 of 1 23 / 13; 2048 -> 2048, 1024 of 1 1498 / 1067; f64 351 -> 128, 64 of 1
        // 11.7 / 17.4, 256 of 1 25 / 40, 512 of 8 54 / 51; f32 512 -> 512, 64 of 24 33 / 30; bf16 1024 -> 1024, 10,000 of 1 and one of
        // 100,000 8500 / 2930.
        const int64_t blocks = (rows / 16 + a.sg.S) * ((a.N + 15) / 16);
        if (mean <= 16 && (mean <= few_mean<T, KN>(a) || blocks <= (sizeof(T) == 2 ? 4 : 12) * cus)) return launch_few<T, KN, 1, 0>(ctx, a, name);
        if (mean <= 32 && blocks <= 4 * cus) return launch_few<T, KN, 2, 0>(ctx, a, name);
        return rows_t<T, KN, 0>(ctx, a, name);
    }
    // Up to two blocks of 64 x 16 for every CU; lower ones where that leaves CUs without, and for 64 bits, whose 64 rows find no
    // registers.  us, tiles / 16 / 32 / 64 rows a block, adapters of rank 16 or 8: bf16 2048 -> 2048, 64 single rows 45 / 20.0 / 19.4 / 26.5,
    // 256 53 / 52 / 42 / 47, 512 59 / 94 / 73 / 84; segments of 64 rows, 128 rows 27 / 30 / 26 / 24, 256 33 / 45 / 37 / 35; f32 1024 -> 1024,
    // 256 rows 36 / 32 / 28 / 26; 351 -> 128, 64 single rows 48 / 16.8 / 17.2 / 21.5, 4096 78 / 68 / 62 / 66; f64 351 -> 128, 1000 rows 31 /
    // 18.1 / 18.2 / 21.5.
    if (rows * a.N <= 64 * 16 * 2 * cus) {
        const int64_t wide = (a.N + 15) / 16;
        if (rows <= 16 || (rows + 31) / 32 * wide < cus / 2) return launch_few<T, KN, 1, 2>(ctx, a, name);
        if constexpr (sizeof(T) < 8)
            if (rows > 32 && (rows + 63) / 64 * wide >= cus) return launch_few<T, KN, 4, 2>(ctx, a, name);
        return launch_few<T, KN, 2, 2>(ctx, a, name);
    }
    // Adapters through LDS or straight from memory: us, f16 16,384 x 1024 -> 2048, rank 32, segments of 16 rows 221 / 245, of 32 161 /
    // 204, of 512 100 / 160; bf16 16,384 x 1024 -> 1024, rank 16, of 16 125 / 99, of 32 91 / 87, of 64 72 / 80; f32 120,011 x 351 -> 128,
    // rank 8, of 16 272 / 247, of 128 155 / 146, of 512 147 / 142, rank 64, of 64 232 / 228; f64 20,011 x 351 -> 128, rank 16, of 32 81 /
    // 77, of 512 61 / 59.
    if constexpr (sizeof(T) == 2)
        if (mean >= 32) return rows_t<T, KN, 1>(ctx, a, name);
    return rows_t<T, KN, 2>(ctx, a, name);
}

template <typename T>
static int rows_any(lnasr_ctx* ctx, const RowsArgs& a, const char* name) {
    return a.kn ? rows_kn<T, true>(ctx, a, name) : rows_kn<T, false>(ctx, a, name);
}

int transform_rows(lnasr_ctx* ctx, int dtype, const RowsArgs& a, const char* name) {
    if (a.sg.rows == 0 || a.sg.S == 0 || a.N == 0) return 0;
    const int size = (int)transform_size(dtype);
    if (rows_narrow_ok(a, size) && !(a.mid && size == 2)) return transform_rows_narrow(ctx, dtype, a, name);
    switch (dtype) {
        case LNASR_F64: return rows_any<double>(ctx, a, name);
        case LNASR_F32: return rows_any<float>(ctx, a, name);
        case LNASR_F16: return rows_any<_Float16>(ctx, a, name);
        default: return rows_any<__bf16>(ctx, a, name);
    }
}

}  // namespace lnasr
