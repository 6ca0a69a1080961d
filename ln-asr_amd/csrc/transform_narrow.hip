// Feature transforms of a few dozen values a row: MFCC frames (39) and the like, their gradients.  Such a product is bound by the memory it moves (39 x 39 in fp64: 5 operations a byte), so rows are read and written as the contiguous
// bytes they are, whatever their width, and the matrix stays in registers.
#include <algorithm>
#include <type_traits>

#include "transform.h"

namespace lnasr {

// `bytes` (a multiple of 16, at most 1024 HF) from src to the wave's LDS, 16 a lane; lanes past the end load nothing.  No branches:
// the wait for the loads can then be told from that for stores that came after them.
template <typename T, int HF>
struct Chunk {
    u32x4 v[HF];
    __device__ __forceinline__ void load(const char* src, int bytes) {
        const __amdgpu_buffer_rsrc_t d = __builtin_amdgcn_make_buffer_rsrc((void*)src, 0, (unsigned)bytes, 0x00027000);
        const int at = (threadIdx.x & 63) * 16;
#pragma unroll
        for (int i = 0; i < HF; ++i) v[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(d, at + 1024 * i, 0, 0));
    }
    // the same for values first, first + 1, .. of src up to value c of the chunk, second + c, .. up to value `live`, then zeros
    __device__ __forceinline__ void load_two(const T* src, int64_t first, int64_t second, int c, int live) {
        constexpr int E = Mat<T>::E;
#pragma unroll
        for (int i = 0; i < HF; ++i) {
            T e[E];
#pragma unroll
            for (int j = 0; j < E; ++j) {
                const int at = ((threadIdx.x & 63) + 64 * i) * E + j;
                e[j] = src[at < c ? first + at : at < live ? second + at : first];
                if (at >= live) e[j] = (T)0;
            }
            __builtin_memcpy(&v[i], e, 16);
        }
    }
    // the same where the array ends after `room` bytes
    __device__ __forceinline__ void load_end(const char* src, int64_t room) {
#pragma unroll
        for (int i = 0; i < HF; ++i)
            v[i] = load_piece((const T*)src, ((threadIdx.x & 63) + 64 * i) * Mat<T>::E, room > 0 ? room / (int)sizeof(T) : 0);
    }
    __device__ __forceinline__ void store(char* lds, int bytes) const {
        const int at = (threadIdx.x & 63) * 16;
#pragma unroll
        for (int i = 0; i < HF; ++i)
            if (at + 1024 * i < bytes) *(u32x4*)(lds + at + 1024 * i) = v[i];
    }
};
// values of a small array; 0 where `live` does not hold
template <typename T>
struct Words {
    __amdgpu_buffer_rsrc_t d;
    __device__ __forceinline__ Words(const T* p, int n) : d(__builtin_amdgcn_make_buffer_rsrc((void*)p, 0, n * (unsigned)sizeof(T), 0x00027000)) {}
    __device__ __forceinline__ T get(int i, bool live) const {
        const unsigned at = live ? i * (unsigned)sizeof(T) : 0xffffffffu;
        if constexpr (sizeof(T) == 8) return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b64(d, at, 0, 0));
        else if constexpr (sizeof(T) == 4) return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(d, at, 0, 0));
        else return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b16(d, at, 0, 0));
    }
};
// 16-byte pieces of the wave's LDS to memory, the counterpart of Chunk
template <int HF>
__device__ __forceinline__ void put_chunk(char* to, const char* lds, int bytes) {
    const __amdgpu_buffer_rsrc_t d = __builtin_amdgcn_make_buffer_rsrc((void*)to, 0, (unsigned)bytes, 0x00027000);
    const int at = (threadIdx.x & 63) * 16;
    u32x4 v[HF];
#pragma unroll
    for (int i = 0; i < HF; ++i) v[i] = *(const u32x4*)(lds + at + 1024 * i);
#pragma unroll
    for (int i = 0; i < HF; ++i) __builtin_amdgcn_raw_buffer_store_b128(v[i], d, at + 1024 * i, 0, 0);
}

// ------------------------------------------------------------------------------------------
// y[r] = scale (W x[r]) + bias: the four waves of a block share a span of rows, each takes 16 at a time.  The next 16 rows are on
// their way while the current ones multiply, and the stores of the last ones are not waited for.  N <= 16 NF, K sizeof(T) <= 64
// HF; with a bias K + 1 values fit: the bias is a column of W that meets a one behind each row (and takes no scale: no call has both).
// fp64 1,024,000 x 39 x 39: 145-155 us, 4.2-4.4 TB/s of the 5.2 of a large copy; 64 single rows: 6.4 us, three
// latencies of memory.
// ------------------------------------------------------------------------------------------
template <typename T, int NF, int HF>
__global__ __launch_bounds__(256, 3) void rows_narrow(RowsArgs a, int ts, int wave_lds) {
    using M = Mat<T>;
    using Sum = typename M::Sum;
    constexpr int SZ = (int)sizeof(T), E = M::E, HO = (16 * 16 * NF * SZ + 1023) / 1024;
    extern __shared__ __attribute__((aligned(16))) char lds_all[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l15 = lane & 15, kk = lane >> 4;
    char* lds = lds_all + wave * wave_lds;
    int64_t r0, r1;
    const int s = find_span(a.sg.off, a.sg.S, a.sg.rows, die_order(block_id(), block_count()), ts, &r0, &r1);
    if (s < 0) return;
    const int slot = seg_slot(a.sg, s);
    if (slot < 0) return;
    r0 += wave * 16;
    if (r0 >= r1) return;

    const int K = a.K, N = a.N, in_bytes = 16 * K * SZ, out_bytes = 16 * N * SZ;
    const char* x = (const char*)a.x + r0 * K * SZ;
    char* y = (char*)a.y + r0 * N * SZ;
    Chunk<T, HF> next;
    // (rows past the span may be read, past the array not: its last, uneven rows are loaded when their turn comes)
    auto fetch = [&](int64_t r) {
        next.load(x, r < r1 && r + 16 <= a.sg.rows ? in_bytes : 0);
        x += 64 * K * SZ;
    };
    fetch(r0);

    // (32-bit offsets and zeros for what lies outside, without a branch or an address in registers)
    const Words<T> w((const T*)a.w + slot * a.w_stride, K * N), bias((const T*)a.bias + slot * a.bias_stride, a.bias ? N : 0);
    const int wc = a.kn ? 1 : K, wk = a.kn ? N : 1;
    u32x4 wf[NF][HF];
#pragma unroll
    for (int n = 0; n < NF; ++n) {
        const int c = min(16 * n + l15, N - 1);
#pragma unroll
        for (int h = 0; h < HF; ++h) {
            T e[E];
#pragma unroll
            for (int j = 0; j < E; ++j) {
                const int k = (4 * h + kk) * E + j;
                e[j] = w.get(c * wc + k * wk, k < K);
                if ((4 * h + 4) * E > K) {                                    // (the same for every lane)
                    const T b = bias.get(c, k == K);
                    e[j] = k == K ? b : e[j];
                }
            }
            __builtin_memcpy(&wf[n][h], e, 16);
        }
    }
    const Sum scale = a.scale ? (Sum)a.scale[slot] : (Sum)1;

    // 16 rows in LDS -> their results in LDS
    auto multiply = [&]() {
        u32x4 xf[HF];
#pragma unroll
        for (int h = 0; h < HF; ++h) {
            const int k = (4 * h + kk) * E;
            T e[E];
            __builtin_memcpy(e, lds + (l15 * K + k) * SZ, 16);                // (past a row's end: the next row, or what lies behind)
            if ((4 * h + 4) * E > K)                                          // (the same for every lane)
#pragma unroll
                for (int j = 0; j < E; ++j) e[j] = k + j < K ? e[j] : k + j == K ? (T)1 : (T)0;
            __builtin_memcpy(&xf[h], e, 16);
        }
        wave_lds_order();
#pragma unroll
        for (int n = 0; n < NF; ++n) {
            typename M::Acc acc = typename M::Acc{0, 0, 0, 0};
#pragma unroll
            for (int h = 0; h < HF; ++h) acc = mma<T>(wf[n][h], xf[h], acc);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int c = 16 * n + M::row(r, kk);
                if (c < N) *(T*)(lds + (l15 * N + c) * SZ) = (T)(acc[r] * scale);     // the one rounding of the result
            }
        }
        wave_lds_order();
    };
    for (; r0 + 16 <= r1; r0 += 64) {
        next.store(lds, in_bytes);
        wave_lds_order();
        fetch(r0 + 64);
        multiply();
        put_chunk<HO>(y, lds, out_bytes);
        y += 64 * N * SZ;
        wave_lds_order();
    }
    if (r0 < r1) {                                                            // the span's last rows
        if (r0 + 16 > a.sg.rows) next.load_end(x - 64 * K * SZ, (a.sg.rows - r0) * K * SZ);
        next.store(lds, in_bytes);
        wave_lds_order();
        multiply();
        const int bytes = (int)(r1 - r0) * N * SZ;
        for (int at = lane * 16; at < bytes; at += 1024) {
            if (at + 16 <= bytes) {
                const u32x4 v = *(const u32x4*)(lds + at);
                __builtin_memcpy(y + at, &v, 16);
            } else {
                for (int b = at; b < bytes; b += SZ) *(T*)(y + b) = *(const T*)(lds + b);
            }
        }
    }
}

// LDS of a wave: fragments read 64 HF bytes from the start of each of the 16 rows, past the last one's end where K is not as wide;
// put_chunk reads to the end of its last kilobyte
constexpr int narrow_lds(int size, int NF, int HF, int K) {
    const int in = (15 * K * size + 64 * HF + 15) / 16 * 16, out = (16 * 16 * NF * size + 1023) / 1024 * 1024;
    return in > out ? in : out;
}
// every K up to 64 HF bytes: rows and what is read behind the last of them lie in the wave's own LDS
constexpr bool narrow_lds_holds(int size, int NF, int HF) {
    for (int K = 1; K * size <= 64 * HF; ++K)
        for (int h = 0; h < HF; ++h)
            for (int kk = 0; kk < 4; ++kk) {
                const int end = (15 * K + (4 * h + kk) * (16 / size)) * size + 16, lds = narrow_lds(size, NF, HF, K);
                if (end > lds || 16 * K * size > lds || 16 * 16 * NF * size > lds || lds % 16) return false;
            }
    return true;
}

template <typename T, int NF, int HF>
static int launch_narrow(lnasr_ctx* ctx, const RowsArgs& a, const char* name) {
    // spans: long ones spread the cost of fetching the matrix, but every CU should have a few blocks
    int ts = 6;
    while (ts < 10 && (a.sg.rows >> ts) > 8 * ctx->prop.multiProcessorCount) ++ts;
    const int64_t spans = (a.sg.rows >> ts) + a.sg.S;
    LN_REQUIRE(spans < (1ll << 31), "%lld rows in %d segments are too many for one call", (long long)a.sg.rows, a.sg.S);
    static_assert(narrow_lds_holds((int)sizeof(T), NF, HF), "fragments of rows_narrow");
    const int wave_lds = narrow_lds((int)sizeof(T), NF, HF, a.K);
    LN_LAUNCH(ctx, name, (rows_narrow<T, NF, HF>), transform_grid(spans, 256), dim3(256), 4 * wave_lds, a, ts, wave_lds);
    return 0;
}

template <typename T, int HF>
static int narrow_n(lnasr_ctx* ctx, const RowsArgs& a, const char* name) {
    if (a.N <= 16) return launch_narrow<T, 1, HF>(ctx, a, name);
    if constexpr (sizeof(T) == 2)
        if (a.N > 48) return launch_narrow<T, 4, HF>(ctx, a, name);
    return launch_narrow<T, 3, HF>(ctx, a, name);
}

// bytes of a row (and the one behind it that meets the bias) that fragments hold
constexpr int narrow_row(int size) { return size == 8 ? 320 : size == 4 ? 192 : 128; }

template <typename T>
static int narrow_t(lnasr_ctx* ctx, const RowsArgs& a, const char* name) {
    const int bytes = (a.K + (a.bias ? 1 : 0)) * (int)sizeof(T);
    constexpr int HF = narrow_row((int)sizeof(T)) / 64, LOW = sizeof(T) == 8 ? 2 : 1;
    return bytes <= 64 * LOW ? narrow_n<T, LOW>(ctx, a, name) : narrow_n<T, HF>(ctx, a, name);
}

// Up to 40 fp64, 48 fp32 or 64 16-bit values, and as many results (fp64: 48); but not rows of whole 128 bytes, which begin in the same
// banks of the LDS, nor, where W is read across its lines (y = W x) in fewer bits than 64, of whole 32 bytes: the tiles then have
// aligned pieces.  us, tiles / this, 300,007 rows: y with a bias, fp64 39 -> 39 50 / 48, 32 -> 32 30 / 53, 41 -> 41 56 / 73, 51 -> 51 73 /
// 116; fp32 39 -> 39 40 / 36, 40 -> 40 39 / 48, 48 -> 48 39 / 55, 51 -> 51 51 / 54; bf16 39 -> 39 40 / 31, 48 -> 48 36 / 53, 51 -> 51 62 / 45,
// 56 -> 56 44 / 44; dx, fp64 40 -> 40 50 / 42, 32 -> 32 29 / 47; fp32 32 -> 32 20 / 32, 48 -> 48 37 / 28; bf16 48 -> 48 29 / 24, 51 -> 51
// 58 / 34, 64 -> 64 28 / 32.
bool rows_narrow_ok(const RowsArgs& a, int size) {
    const int row = a.K * size, whole = a.kn || size == 8 ? 128 : 32;
    return a.w_stride && (a.K + (a.bias ? 1 : 0)) * size <= narrow_row(size) && a.N <= (size == 2 ? 64 : 48) && a.ldx == a.K && a.ldy == a.N &&
           (row % whole != 0 || row <= 32);
}

int transform_rows_narrow(lnasr_ctx* ctx, int dtype, const RowsArgs& a, const char* name) {
    switch (dtype) {
        case LNASR_F64: return narrow_t<double>(ctx, a, name);
        case LNASR_F32: return narrow_t<float>(ctx, a, name);
        case LNASR_F16: return narrow_t<_Float16>(ctx, a, name);
        default: return narrow_t<__bf16>(ctx, a, name);
    }
}

// ------------------------------------------------------------------------------------------
// out = sum over the rows of a span of a[r]^T b[r], up to 48 x 48: each of the four waves sums its own chunks of R rows (the k of
// one matrix instruction's piece, or two), whole, and the block adds the four at the end.  The column sums of a come with the
// product: b has a column of ones behind its last.  Rows of two segments, and a span's last ones, come ahead as whole chunks do:
// looked up one by one when their turn came, each such chunk held its block up (fp64 300,007 x 39 x 39 in 300 segments 77 us, so
// 60).  187 MB take 36 us at a large copy's rate; the rest is the blocks' start and end, eight to sixteen chunks a wave.
// ------------------------------------------------------------------------------------------
template <typename T, int IF, int JF, int HA, int HB>
__global__ __launch_bounds__(256, 2) void sum_narrow(SumArgs a, int ts, typename Mat<T>::Sum* parts,
                                                                                    typename Mat<T>::Sum* col_parts, int wave_lds) {
    using M = Mat<T>;
    using Sum = typename M::Sum;
    constexpr int SZ = (int)sizeof(T), E = M::E, R = SZ == 2 ? 32 : 16, H = R / (4 * E);
    extern __shared__ __attribute__((aligned(16))) char lds_all[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l15 = lane & 15, kk = lane >> 4;
    const int I = a.I, J = a.J, a_bytes = R * I * SZ, b_bytes = R * J * SZ;
    char* as = lds_all + wave * wave_lds;
    char* bs = as + (a_bytes + 15) / 16 * 16;
    const int64_t t = die_order(block_id(), block_count());
    int g, n;
    int64_t q0, place;
    bool whole;
    if (!sum_span(a, t, ts, &g, &q0, &n, &whole, &place)) return;

    typename M::Acc acc[IF][JF];
#pragma unroll
    for (int i = 0; i < IF; ++i)
#pragma unroll
        for (int j = 0; j < JF; ++j) acc[i][j] = typename M::Acc{0, 0, 0, 0};

    Chunk<T, HA> an;
    Chunk<T, HB> bn;
    // the segment (of the sorted ones) of the place looked at last, and of the one after that
    int seg = a.place ? max(0, wave_search(a.sg.S, q0, [&](int j) { return a.place[j]; })) : 0;
    auto row_at = [&](int64_t q, int i) -> int64_t {
        if (!a.place) return q;
        while (i + 1 < a.sg.S && a.place[i + 1] <= q) ++i;
        return seg_off(a.sg, a.ord[i]) + min(q, a.place[i + 1]) - a.place[i];
    };
    // The R rows from place k of the span on, as many as there are (the same for every lane): true if they come from one or two
    // segments, and then asks for them
    auto fetch = [&](int k) {
        const int live = min(R, n - k);
        int64_t first = q0 + k, second = 0;
        int c = live;                                      // rows of the first segment
        if (a.place) {
            while (seg + 1 < a.sg.S && a.place[seg + 1] <= q0 + k) ++seg;
            first += seg_off(a.sg, a.ord[seg]) - a.place[seg];
            const int64_t left = a.place[seg + 1] - (q0 + k);
            if (left < live) {
                c = (int)left;
                int i = seg + 1;
                while (i + 1 < a.sg.S && a.place[i + 1] <= q0 + k + c) ++i;
                if (i >= a.sg.S || a.place[i + 1] < q0 + k + live) return false;
                second = seg_off(a.sg, a.ord[i]) - c;
            }
        }
        if (c == R) {                                      // (R rows of the array: nothing past its end)
            an.load((const char*)a.a + first * I * SZ, a_bytes);
            bn.load((const char*)a.b + first * J * SZ, b_bytes);
        } else {
            an.load_two((const T*)a.a, first * I, second * I, c * I, live * I);
            bn.load_two((const T*)a.b, first * J, second * J, c * J, live * J);
        }
        return true;
    };
    int k0 = wave * R;
    bool came = k0 < n && fetch(k0);
    int here = seg;
    for (; k0 < n; k0 += 4 * R) {
        if (came) {
            an.store(as, a_bytes);
            bn.store(bs, b_bytes);
        } else {                                           // rows of three segments and more: one value at a time
            for (int e = lane; e < R * I; e += 64) {
                const int k = e / I;
                const int64_t at = k0 + k < n ? row_at(q0 + k0 + k, here) : -1;
                *(T*)(as + e * SZ) = at >= 0 ? ((const T*)a.a)[at * I + e - k * I] : (T)0;
            }
            for (int e = lane; e < R * J; e += 64) {
                const int k = e / J;
                const int64_t at = k0 + k < n ? row_at(q0 + k0 + k, here) : -1;
                *(T*)(bs + e * SZ) = at >= 0 ? ((const T*)a.b)[at * J + e - k * J] : (T)0;
            }
        }
        wave_lds_order();
        const int k1 = k0 + 4 * R;
        if (k1 < n) {
            came = fetch(k1);
            here = seg;
        }
#pragma unroll
        for (int h = 0; h < H; ++h) {
            u32x4 af[IF], bf[JF];
#pragma unroll
            for (int i = 0; i < IF; ++i) {
                T e[E];
                const int c = min(16 * i + l15, I - 1);
#pragma unroll
                for (int j = 0; j < E; ++j) e[j] = *(const T*)(as + (((4 * h + kk) * E + j) * I + c) * SZ);
                __builtin_memcpy(&af[i], e, 16);
            }
#pragma unroll
            for (int i = 0; i < JF; ++i) {
                T e[E];
                const int c = min(16 * i + l15, J - 1);
#pragma unroll
                for (int j = 0; j < E; ++j) e[j] = *(const T*)(bs + (((4 * h + kk) * E + j) * J + c) * SZ);
                if (i == J >> 4)
#pragma unroll
                    for (int j = 0; j < E; ++j) e[j] = l15 == (J & 15) ? (T)1 : e[j];
                __builtin_memcpy(&bf[i], e, 16);
            }
            mma_all<T>(af, bf, acc);
        }
        wave_lds_order();
    }

    // the four waves' sums, in their order
    Sum* sum = (Sum*)lds_all;
    constexpr int W = 16 * JF;
    for (int turn = 0; turn < 4; ++turn) {
        __syncthreads();
        if (wave == turn) {
#pragma unroll
            for (int i = 0; i < IF; ++i)
#pragma unroll
                for (int j = 0; j < JF; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int at = (16 * i + M::row(r, kk)) * W + 16 * j + l15;
                        sum[at] = turn ? sum[at] + acc[i][j][r] : acc[i][j][r];
                    }
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < I * J; e += 256) {
        const Sum v = sum[e / J * W + e % J];
        if (whole) ((T*)a.out)[(int64_t)g * I * J + e] = (T)v;
        else parts[place * I * J + e] = v;
    }
    if (a.cols)
        for (int i = threadIdx.x; i < I; i += 256) {
            const Sum v = sum[i * W + J];
            if (whole) ((T*)a.cols)[(int64_t)g * I + i] = (T)v;
            else col_parts[place * I + i] = v;
        }
}

template <typename T, int IF, int JF>
static int launch_sum_narrow(lnasr_ctx* ctx, const SumArgs& a, const char* name) {
    using Sum = typename Mat<T>::Sum;
    constexpr int SZ = (int)sizeof(T), R = SZ == 2 ? 32 : 16;
    constexpr int HA = R * 16 * IF * SZ / 1024, HB = R * 16 * JF * SZ / 1024;
    const int64_t size = (int64_t)a.I * a.J + a.I;
    int ts = 8;
    // spans: as many as the CUs hold blocks of 64-bit sums (fp64 300,007 x 39 x 39 with the join: 68 us; twice as many 71, four times 73),
    // and no more than 256 MB of sums
    const int64_t most = 2 * ctx->prop.multiProcessorCount;
    while (ts < 40 && ((a.sg.rows >> ts) > most || (a.sg.rows >> ts) * size * (int64_t)sizeof(Sum) > (256ll << 20))) ++ts;
    const int64_t spans = (a.sg.rows >> ts) + a.groups;
    LN_REQUIRE(spans < (1ll << 31), "%lld rows in %d groups are too many for one call", (long long)a.sg.rows, a.groups);
    void* parts = nullptr;
    const bool split = a.sg.rows > (1ll << ts);
    const int64_t places = sum_places(a, ts);
    if (split) LN_TRY(transform_ws(ctx, kTrPart, (size_t)places * size * sizeof(Sum), &parts));
    Sum* cp = (Sum*)parts + places * a.I * a.J;
    const int wave_lds = (R * a.I * SZ + 15) / 16 * 16 + (R * a.J * SZ + 15) / 16 * 16;
    const int lds = std::max(4 * wave_lds, 16 * IF * 16 * JF * (int)sizeof(Sum));
    LN_LAUNCH(ctx, name, (sum_narrow<T, IF, JF, HA, HB>), transform_grid(spans, 256), dim3(256), lds, a, ts, (Sum*)parts, cp, wave_lds);
    constexpr int dtype = SZ == 8 ? LNASR_F64 : SZ == 4 ? LNASR_F32 : std::is_same<T, _Float16>::value ? LNASR_F16 : LNASR_BF16;
    return split ? transform_join(ctx, a, dtype, ts, parts, cp) : 0;
}

template <typename T>
static int sum_narrow_t(lnasr_ctx* ctx, const SumArgs& a, const char* name) {
    const int j = a.J + (a.cols ? 1 : 0);              // columns of b, and the ones
    if (a.I <= 16) return launch_sum_narrow<T, 1, 3>(ctx, a, name);
    return j <= 16 ? launch_sum_narrow<T, 3, 1>(ctx, a, name) : launch_sum_narrow<T, 3, 3>(ctx, a, name);
}

// us, tiles / this, 300,007 rows in 300 segments of 64 groups: fp64 39 x 39 83 / 67, 48 x 48 82 / 70, 49 x 49 87 / 133; fp32 39 x 39 58 / 46,
// 49 x 49 58 / 62; bf16 39 x 39 36 / 32, 32 x 32 27 / 31, 49 x 49 37 / 62
bool sum_narrow_ok(const SumArgs& a) {
    return a.I <= 48 && a.J + (a.cols ? 1 : 0) <= 48 && a.lda == a.I && a.ldb == a.J;
}

int transform_sum_narrow(lnasr_ctx* ctx, int dtype, const SumArgs& a, const char* name) {
    switch (dtype) {
        case LNASR_F64: return sum_narrow_t<double>(ctx, a, name);
        case LNASR_F32: return sum_narrow_t<float>(ctx, a, name);
        case LNASR_F16: return sum_narrow_t<_Float16>(ctx, a, name);
        default: return sum_narrow_t<__bf16>(ctx, a, name);
    }
}

}  // namespace lnasr
