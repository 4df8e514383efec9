// Orthogonalisation of matrices by Newton-Schulz products, and the Muon step around it.
//
// Mathematics.  X_0 = G / max(|G|_F, eps), the shorter side m as rows, the longer n as columns.  A step of the quintic iteration is
//     A = X X^T,   Q = a I + b A + c A^2,   X <- Q X,
// which takes every singular value s to p(s) = a s + b s^3 + c s^5.  Steps are taken on the Gram side: all of these m x m matrices are
// polynomials of A, so X_L = (Q_{L-1} ... Q_0) X_0 with A_{k+1} = Q_k A_k Q_k, and a segment of L steps reads the large matrix twice
// (its Gram product and the product with P = Q_{L-1} ... Q_0) instead of 2 L times.  Rounding in A_k acts on the SQUARES of
// the singular values and is amplified by a^2 a step, so X is formed and its Gram matrix taken anew after segments of 2 and 1 steps.
// A segment of one step leaves the identity out of the product, X <- a X + (b A + c A^2) X: the part that carries small
// singular values is then not rounded through a matrix whose entries are as large as a.  Median distance from 64-bit results relative to the
// fp32 iteration's, noise with strong directions 128 x 128 / 64 x 128, low rank 256 x 512: five steps as 2 + 1 + 2: 1.8 / 1.06 /
// 1.5, one by one: 1.07 / 1.05 / 1.1, 1 + 2 + 2: 2.4 / 2.3 / 2.1, 3 + 2: 3.6 / 6.1 / 1.2.  One by one needs 15 m^2 n + 5 m^3 operations
// (symmetric products halved), 2 + 1 + 2 9 m^2 n + 11 m^3: the same for square matrices, which therefore go one by one up to
// n < 2 m, and fewer the wider they are.
//
// Arithmetic.  Every matrix is held as hi + lo, two fp16 numbers of one value scaled by a power of two (22 - 23 significant bits; fp32
// has 24), and a product is hi hi + hi lo + lo hi on v_mfma_f32_32x32x16_f16 with fp32 accumulators.  The dropped lo lo term and the
// split are 2^-22 relative, and the same measurement puts the whole iteration at the distance of the fp32 one, at a third
// of the fp16 rate = 5 times the fp32 matrix rate.  fp16's range is no obstacle here: the iterates' singular values are bounded by
// intervals that follow from the coefficients (`Bounds` below), so each matrix gets the scale that puts its bound below 2^15; what is
// lost below fp16's subnormal step is at most 2^-25 / 2^14 = 2^-39 of the largest possible entry.  fp32 would keep the relative accuracy of small
// values: rows (or columns) from 1 down to 1e-4 come out as in fp32, in 1e-6 the worst row is off by 4e-5 (64 x 576), 1.1e-4 (256 x 1024), 2.5e-4 (300 x
// 5000), fp32's by 3e-6 - 1e-5, in 1e-8 by 4e-3, 9e-3, 2e-2.
//
// Symmetric products compute the tiles on and below the diagonal and store each twice.
//
// Up to 16 rows are another matter (see TINY): small_matrix and ns_thin take their Gram matrix and Q in 64 bits.
//
// Layout.  A line is 16 consecutive values of a row as 16 fp16 hi followed by 16 fp16 lo, 64 bytes: one matrix instruction's K, one
// DMA row of LDS.  64 rows form a panel, in which line q of all 64 rows is one 4 KiB run, so that what a workgroup requests per step is
// contiguous.  Both dimensions are padded to 64 with zeros: no kernel but the first and the last knows a border.
#include "segmi_common.h"
#include "lds_dma.h"
#include <algorithm>
#include <cmath>
#include <memory>
#include <mutex>
#include <new>
#include <type_traits>

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr int BATCH = 60;            // matrices per launch: their descriptors travel as kernel arguments (< 4 KiB, asserted at each)
static_assert(BATCH <= 64, "a lane looks at a matrix");
constexpr int MAX_GROUPS = 8;
constexpr unsigned LINE = 64, LINE_K = 16;   // bytes, values

enum Buf { X = 0, T0, T1, A, Q, W, P0, P1 };

// one matrix as the products see it: m <= n, both unpadded; its buffers start `base` * 256 bytes into the workspace
struct Item {
    unsigned first;                  // first workgroup of the launch that works on it
    int m, n;
    unsigned base;
};
struct Batch {
    char* ws;
    int count;
    Item item[BATCH];
};

__host__ __device__ inline unsigned pad64(unsigned v) { return (v + 63u) & ~63u; }
__host__ __device__ inline size_t big_bytes(int m, int n) { return (size_t)pad64(m) * pad64(n) * 4; }
__host__ __device__ inline size_t square_bytes(int m) { return (size_t)pad64(m) * pad64(m) * 4; }
__host__ __device__ inline size_t buffer_offset(int buf, int m, int n) {
    return buf < A ? (size_t)buf * big_bytes(m, n) : 3 * big_bytes(m, n) + (size_t)(buf - A) * square_bytes(m);
}

// lane l looks at item l: one load and one ballot instead of a search.  (Workgroups are dealt to the XCDs within each matrix, by
// xcd_swizzle of the number inside it: an XCD gets a run of neighbouring tiles of EVERY matrix, however unequal their sums are.)
template <typename B>
__device__ __forceinline__ int find_item(const B& b, unsigned wg) {
    const int lane = threadIdx.x & 63;
    const unsigned first = lane < b.count ? b.item[lane].first : 0xFFFFFFFFu;
    return __builtin_amdgcn_readfirstlane((int)__popcll(__ballot(first <= wg)) - 1);
}

// hi = v rounded, lo = the rest rounded.  The empty statement makes v one fp32 number: the compiler may otherwise round the expression
// behind v straight to fp16 for hi, in one step, and take the rest from v, rounded in two, which now and then is a neighbour's.
__device__ __forceinline__ void split(float v, _Float16& hi, _Float16& lo) {
    asm("" : "+v"(v));
    hi = (_Float16)v;
    lo = (_Float16)__builtin_fmaf((float)hi, -1.f, v);
}
__device__ __forceinline__ float join(_Float16 hi, _Float16 lo) { return __builtin_fmaf((float)lo, 1.f, (float)hi); }
__device__ __forceinline__ unsigned pair_word(float v) {
    _Float16 h, l;
    split(v, h, l);
    return __builtin_bit_cast(unsigned, f16x2{h, l});
}
// where value k of a row lies
__device__ __forceinline__ size_t at_line(unsigned lines, unsigned row, unsigned k) {
    return ((size_t)((row >> 6) * lines + k / LINE_K) * 64 + (row & 63)) * LINE + k % LINE_K * 2;
}
// values k .. k+3 (k % 4 == 0) of a row
__device__ __forceinline__ void store4(char* buf, unsigned lines, unsigned row, unsigned k, const float* v) {
    f16x4 hi, lo;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        _Float16 h, l;
        split(v[x], h, l);
        hi[x] = h;
        lo[x] = l;
    }
    char* p = buf + at_line(lines, row, k);
    *reinterpret_cast<f16x4*>(p) = hi;
    *reinterpret_cast<f16x4*>(p + LINE / 2) = lo;
}
__device__ __forceinline__ void store1(char* buf, unsigned lines, unsigned row, unsigned k, float v) {
    _Float16 h, l;
    split(v, h, l);
    char* p = buf + at_line(lines, row, k);
    *reinterpret_cast<_Float16*>(p) = h;
    *reinterpret_cast<_Float16*>(p + LINE / 2) = l;
}
// ------------------------------------------------------------------------------------------------ reading the updates
// An update is seen as outer x inner with the inner dimension the contiguous one where there is one.
struct Source {
    unsigned first;                  // workgroup of the current launch
    unsigned base;                   // as in Item
    const void* src;                 // MUON: the gradient
    float* mom;                      // MUON: the momentum buffer (same order)
    long so, si;                     // strides in elements
    int outer, inner;
    unsigned part, parts;            // its partial sums of squares
    signed char dtype;               // 0 fp32, 1 bf16
    signed char inner_is_n;          // 1: the inner dimension is the longer side
    signed char group;
};
static_assert(sizeof(Source) == 64, "sixty of them fit the kernel arguments");
struct SourceBatch {
    char* ws;
    double* partial;
    double eps;
    float scale;                     // of X_0
    int count;
    int nesterov;
    Source item[BATCH];
};
struct Hyper {
    float lr[MAX_GROUPS], wd[MAX_GROUPS], mom[MAX_GROUPS];
};
// descriptors, by-value hyper-parameters and the pointer to those on the device, with eight bytes of padding
template <typename B>
constexpr bool fits_arguments = sizeof(B) + sizeof(Hyper) + 2 * sizeof(void*) < 4096;
static_assert(fits_arguments<SourceBatch>, "kernel arguments");

__device__ __forceinline__ float bf16_to_f32(unsigned short u) { return __uint_as_float((unsigned)u << 16); }
__device__ __forceinline__ unsigned short f32_to_bf16(float f) {
    const unsigned u = __float_as_uint(f);
    const unsigned nearest = (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;                        // ties to even
    return (unsigned short)(f != f ? (u >> 16) | 0x40u : nearest);                          // NaN stays NaN
}

__device__ __forceinline__ float source_at(const Source& s, long off) {
    return s.dtype ? bf16_to_f32(static_cast<const unsigned short*>(s.src)[off]) : static_cast<const float*>(s.src)[off];
}
// four neighbours of the inner dimension in one load
__device__ __forceinline__ bool by_fours(const Source& s) {
    return s.si == 1 && (s.so & 3) == 0 && (s.inner & 3) == 0 && ((size_t)s.src & (s.dtype ? 7 : 15)) == 0 && ((size_t)s.mom & 15) == 0;
}
__device__ __forceinline__ float4 source_four(const Source& s, long off) {
    if (!s.dtype) return ld4(static_cast<const float*>(s.src) + off);
    const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const unsigned short*>(s.src) + off);
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xFFFF0000u));
}

// Sum of squares of every update in fp64 (a gradient of 1e-25 or 1e25 must not vanish or overflow), one partial per 64 x 256
// elements, summed later in a fixed order.  MUON also advances the momentum buffer: mom = mu mom + g.
// HBM-bound: 4 B (MUON 12 B) per element.  A wave has four rows under way at a time: one, and bf16 by single elements,
// took 9.9 instead of 6.6 us for 1024 x 4608 and 37 instead of 14 us for 13 M elements in bf16.
template <bool MUON>
__global__ __launch_bounds__(256) void ns_sum_squares(SourceBatch b, Hyper h, const Hyper* __restrict__ hd) {
    const int it = find_item(b, blockIdx.x);
    const Source& s = b.item[it];
    const unsigned unit = blockIdx.x - s.first;
    const unsigned across = (unsigned)(s.inner + 255) / 256;
    const long o0 = (long)(unit / across) * 64, i0 = (long)(unit % across) * 256;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const float mu = MUON ? (hd ? hd->mom[s.group] : h.mom[s.group]) : 0.f;
    const bool nest = MUON && b.nesterov;
    double sum = 0.0;
    const bool vec = by_fours(s);
    const auto add = [&](float g, float& m) {            // the update's square; the momentum advanced
        if (MUON) {
            m = fmaf(mu, m, g);
            g = nest ? fmaf(mu, m, g) : m;
        }
        sum = fma((double)g, (double)g, sum);
    };
#pragma unroll 1
    for (int r0 = wave; r0 < 64 && o0 + r0 < s.outer; r0 += 16) {
        if (vec) {
            const long i = i0 + lane * 4;
            float4 g[4], m[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const long o = o0 + r0 + 4 * k;
                const bool in = o < s.outer && i < s.inner;
                g[k] = in ? source_four(s, o * s.so + i) : zero4();
                m[k] = MUON && in ? ld4(s.mom + o * s.so + i) : zero4();
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                add(g[k].x, m[k].x);
                add(g[k].y, m[k].y);
                add(g[k].z, m[k].z);
                add(g[k].w, m[k].w);
                const long o = o0 + r0 + 4 * k;
                if (MUON && o < s.outer && i < s.inner) st4(s.mom + o * s.so + i, m[k]);
            }
        } else {
            float g[4][4], m[4][4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const long o = o0 + r0 + 4 * k, i = i0 + x * 64 + lane;
                    const bool in = o < s.outer && i < s.inner;
                    g[k][x] = in ? source_at(s, o * s.so + i * s.si) : 0.f;
                    m[k][x] = MUON && in ? s.mom[o * s.so + i * s.si] : 0.f;
                }
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    add(g[k][x], m[k][x]);
                    const long o = o0 + r0 + 4 * k, i = i0 + x * 64 + lane;
                    if (MUON && o < s.outer && i < s.inner) s.mom[o * s.so + i * s.si] = m[k][x];
                }
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    __shared__ double red[4];
    if (lane == 0) red[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) b.partial[s.part + unit] = (red[0] + red[1]) + (red[2] + red[3]);
}

// X_0 = u / max(|u|, eps), scaled and split, in both orders (rows along n for the Gram product, rows along m for the
// product with P), zeros in the padding; 64 x 64 elements a workgroup, turned round in LDS.
// HBM-bound: reads 4 B (MUON 8 B with nesterov), writes 8 B per element; 47 M elements 140 us = 4.0 TB/s.
template <bool MUON>
__global__ __launch_bounds__(256) void ns_normalise(SourceBatch b, Hyper h, const Hyper* __restrict__ hd) {
    const int it = find_item(b, blockIdx.x);
    const Source& s = b.item[it];
    const unsigned tile = blockIdx.x - s.first;
    const int tid = threadIdx.x;
    __shared__ double red[4];
    __shared__ float turn[64][65];

    double sum = 0.0;
    for (unsigned i = tid; i < s.parts; i += 256) sum += b.partial[s.part + i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if ((tid & 63) == 0) red[tid >> 6] = sum;
    __syncthreads();
    const double norm = sqrt((red[0] + red[1]) + (red[2] + red[3]));
    const double inv = (double)b.scale / (norm <= b.eps ? b.eps : norm);       // (a NaN norm stays)

    const unsigned across = pad64(s.inner) / 64;
    const int o0 = (int)(tile / across) * 64, i0 = (int)(tile % across) * 64;
    const int m = s.inner_is_n ? s.outer : s.inner, n = s.inner_is_n ? s.inner : s.outer;
    char* const base = b.ws + (size_t)s.base * 256;
    char* const direct = base + buffer_offset(s.inner_is_n ? X : T0, m, n);
    char* const turned = base + buffer_offset(s.inner_is_n ? T0 : X, m, n);
    const unsigned lines_inner = pad64(s.inner) / LINE_K, lines_outer = pad64(s.outer) / LINE_K;
    const float mu = MUON ? (hd ? hd->mom[s.group] : h.mom[s.group]) : 0.f;
    const bool nest = MUON && b.nesterov;
    const int r0 = tid >> 4, c4 = (tid & 15) * 4, i = i0 + c4;
    float u[4][4];                                       // all loads first: behind a store they would wait for it
    if (by_fours(s)) {
        float4 g[4], m[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int o = o0 + r0 + 16 * k;
            const bool in = o < s.outer && i < s.inner;
            const long off = (long)o * s.so + i;
            g[k] = in && (!MUON || nest) ? source_four(s, off) : zero4();
            m[k] = in && MUON ? ld4(s.mom + off) : zero4();
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float gv[4] = {g[k].x, g[k].y, g[k].z, g[k].w}, mv[4] = {m[k].x, m[k].y, m[k].z, m[k].w};
#pragma unroll
            for (int x = 0; x < 4; ++x) u[k][x] = !MUON ? gv[x] : nest ? fmaf(mu, mv[x], gv[x]) : mv[x];
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int o = o0 + r0 + 16 * k;
                const bool in = o < s.outer && i + x < s.inner;
                const long off = (long)o * s.so + (long)(i + x) * s.si;
                const float g = in && (!MUON || nest) ? source_at(s, off) : 0.f, m = in && MUON ? s.mom[off] : 0.f;
                u[k][x] = !MUON ? g : nest ? fmaf(mu, m, g) : m;
            }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int r = r0 + 16 * k;
        float v[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            v[x] = (float)((double)u[k][x] * inv);
            turn[r][c4 + x] = v[x];
        }
        store4(direct, lines_inner, o0 + r, i, v);
    }
    __syncthreads();
    for (int r = tid >> 4; r < 64; r += 16) {
        float v[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) v[x] = turn[c4 + x][r];
        store4(turned, lines_outer, i0 + r, o0 + c4, v);
    }
}

// ------------------------------------------------------------------------------------------------ products
// One workgroup's BT x BT tile of L R^T over the lines q0 .. q1-1 of both operands: 4 waves in 2 x 2.  A step is U lines; one is
// multiplied while the copies of the next STAGES - 1 are on their way.
// LDS chunk c (16 B) of a row sits at c ^ ((row >> 2) & 3): 16 consecutive rows, which one ds_read_b128 phase reads, then cover all 64 banks;
// the permutation is applied to the copy's source address.
// Per step: the wave waits for ITS copies of the step (those of STAGES - 2 later ones may be in flight), the barrier makes all waves'
// visible and the step before it free, and the copies of the step STAGES - 1 ahead go there, one every few products: requested in one go the copies of
// the waves keep each of them from issuing products for the 16 cycles a copy occupies the CU's address path.
// What bounds a product: MFMA-bound it would take 384 cycles per 128 x 128 tile and line on a CU; LDS serves 32 KiB of reads and 16 KiB of
// copies in about as many, L2 delivers those 16 KiB in 315 (its limit, 52 B a cycle and CU) to 680 (behind HBM), and the three meet: 800 - 900
// cycles measured.  Short sums (m = 512 is 32 lines) add the tile's two stores, 128 KiB, at what HBM takes (4 TB/s).  512 x 36864: product
// with P 92 us, of which 225 MB of HBM 50, the Gram product 38 us = 0.31 of the matrix rate.  Slower were: registers loaded a line ahead
// (2 - 5 %), 64 x 64 tiles of 8 waves with half the lines each (10 %), both stores through LDS (7 - 10 %), five stages for two workgroups a CU
// (0 - 3 %), tiles on XCDs in blocks (0).
struct Wide { static constexpr int BT = 128, U = 1, PER_CU = 3; static constexpr unsigned STAGES = 3; };
struct Many { static constexpr int BT = 64, U = 1, PER_CU = 4; static constexpr unsigned STAGES = 4; };
struct Few { static constexpr int BT = 64, U = 2, PER_CU = 1; static constexpr unsigned STAGES = 8; };

template <typename C>
struct Tile {
    static constexpr int BT = C::BT, U = C::U;           // U: lines per step
    static constexpr int S = BT / 64;                    // 32 x 32 subtiles per wave and dimension
    static constexpr unsigned ROWS = BT * LINE;          // bytes of an operand's line
    static constexpr unsigned STAGE = 2 * ROWS * U, STAGES = C::STAGES;
    static constexpr int PIECES = BT / 64;               // 1 KiB copies (16 rows) per wave, operand and line
    static constexpr int PER = 2 * PIECES * U;           // copies per wave and step
    static constexpr int PITCH = S * 32 + 8;             // see store_rows
    static constexpr unsigned SMEM = STAGES * STAGE;
    static_assert(SMEM >= 4 * 32 * PITCH * 4, "four waves turn 32 rows each");
    f32x16 acc[S][S];

    // This wave's LDS reads are back and at most N of its copies are in flight; then every wave's are.  The builtin, not asm: the
    // compiler counts the LDS reads with it and puts no second wait before their uses.
    template <int N>
    __device__ __forceinline__ static void wait_all() {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4));
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }

    // The two mixed products have an accumulator of their own, added at the end: the large sum is rounded a third as often.
    __device__ __forceinline__ void run(char* smem, const char* L, unsigned rows_l, const char* R, unsigned rows_r, unsigned lines,
                                        unsigned l0, unsigned r0, unsigned q0, unsigned q1) {
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int wr = wave >> 1, wc = wave & 1;
        const i32x4 rsl = make_rsrc(L, rows_l * lines * LINE), rsr = make_rsrc(R, rows_r * lines * LINE);
        unsigned off_l[PIECES], off_r[PIECES];
        const unsigned lds = lds_addr(smem);
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const unsigned row = (wave * PIECES + p) * 16 + (lane >> 2);
            const unsigned chunk = (lane & 3) ^ ((row >> 2) & 3);
            off_l[p] = (unsigned)at_line(lines, l0 + row, 0) + chunk * 16;      // beyond the last panel: beyond the range, zeros
            off_r[p] = (unsigned)at_line(lines, r0 + row, 0) + chunk * 16;
        }
        // copy c of step k into `stage`
        auto copy = [&](unsigned k, unsigned stage, int c) {
            const int u = c / (2 * PIECES), o = c / PIECES % 2, p = c % PIECES;
            const unsigned at = lds + stage * STAGE + (2 * u + o) * ROWS + (wave * PIECES + p) * 1024, q = (q0 + k * U + u) * (64 * LINE);
            if (o == 0) dma16s(rsl, off_l[p], q, at);
            else dma16s(rsr, off_r[p], q, at);
        };
        f32x16 mix[S][S];
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
            for (int j = 0; j < S; ++j)
#pragma unroll
                for (int x = 0; x < 16; ++x) acc[i][j][x] = mix[i][j][x] = 0.f;
        const unsigned n = (q1 - q0) / U;                // >= 2
#pragma unroll
        for (unsigned k = 0; k < STAGES - 1; ++k)
            if (k < n)
#pragma unroll
                for (int c = 0; c < PER; ++c) copy(k, k, c);
        const int fr = lane & 31, fk = lane >> 5;
        const int sw = (fr >> 2) & 3;                    // row bases are multiples of 32: the permutation depends on the lane alone
        const int hi = (fk ^ sw) * 16, lo = ((fk + 2) ^ sw) * 16;
        const char* const sl = smem + (wr * S * 32 + fr) * LINE;
        const char* const sr = smem + ROWS + (wc * S * 32 + fr) * LINE;
        auto step = [&](unsigned k, unsigned stage, unsigned into, auto more) {
            const unsigned at = stage * STAGE;
            f16x8 lh[U][S], ll[U][S], rh[U][S], rl[U][S];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < S; ++i) {
                    const unsigned o = at + 2 * u * ROWS + i * 32 * LINE;
                    lh[u][i] = *reinterpret_cast<const f16x8*>(sl + o + hi);
                    rh[u][i] = *reinterpret_cast<const f16x8*>(sr + o + hi);
                    ll[u][i] = *reinterpret_cast<const f16x8*>(sl + o + lo);
                    rl[u][i] = *reinterpret_cast<const f16x8*>(sr + o + lo);
                }
            __builtin_amdgcn_sched_barrier(0);
            constexpr int EACH = 3 * S * S * U / PER;
            int done = 0;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int t = 0; t < 3; ++t)
#pragma unroll
                    for (int i = 0; i < S; ++i)
#pragma unroll
                        for (int j = 0; j < S; ++j) {
                            if (t == 0) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(lh[u][i], rh[u][j], acc[i][j], 0, 0, 0);
                            if (t == 1) mix[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ll[u][i], rh[u][j], mix[i][j], 0, 0, 0);
                            if (t == 2) mix[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(lh[u][i], rl[u][j], mix[i][j], 0, 0, 0);
                            if (decltype(more)::value && (((u * 3 + t) * S + i) * S + j) % EACH == 0 && done < PER) {
                                __builtin_amdgcn_sched_barrier(0);
                                copy(k + STAGES - 1, into, done++);
                                __builtin_amdgcn_sched_barrier(0);
                            }
                        }
        };
        unsigned k = 0, stage = 0, before = STAGES - 1;
        for (; k + STAGES - 1 < n; ++k) {
            wait_all<(STAGES - 2) * PER>();
            step(k, stage, before, std::true_type{});
            before = stage;
            stage = stage + 1 == STAGES ? 0 : stage + 1;
        }
        for (; k < n; ++k) {                             // everything is under way or here
            switch (n - 1 - k < STAGES - 2 ? n - 1 - k : STAGES - 2) {
                case 0: wait_all<0>(); break;
                case 1: wait_all<PER>(); break;
                case 2: wait_all<2 * PER>(); break;
                case 3: wait_all<3 * PER>(); break;
                case 4: wait_all<4 * PER>(); break;
                case 5: wait_all<5 * PER>(); break;
                default: wait_all<6 * PER>(); break;
            }
            step(k, stage, 0, std::false_type{});
            stage = stage + 1 == STAGES ? 0 : stage + 1;
        }
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
            for (int j = 0; j < S; ++j)
#pragma unroll
                for (int x = 0; x < 16; ++x) acc[i][j][x] += mix[i][j][x];
    }

    // f(row, col, v, at) per 32 x 32 subtile: v[4 g + x] is row `row` + 8 g + x of column `col` (tile-relative); what f makes of v
    // stays; at: see Columns
    template <typename F>
    __device__ __forceinline__ void each(F f) {
        const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
            for (int j = 0; j < S; ++j) {
                float v[16];
#pragma unroll
                for (int x = 0; x < 16; ++x) v[x] = acc[i][j][x];
                f(((wave >> 1) * S + i) * 32 + 4 * (lane >> 5), ((wave & 1) * S + j) * 32 + (lane & 31), v, i * 2 * 64 * LINE + j * 32 * LINE);
#pragma unroll
                for (int x = 0; x < 16; ++x) acc[i][j][x] = v[x];
            }
    }

    // Stores the tile, pairs in one word, by rows.  A lane holds runs of rows of one column, a row's line wants runs of columns: each wave turns its own part
    // round in LDS, 32 rows at a time, and writes them 16 B a lane.  Pitch: 4 rows apart is 32 banks apart.
    __device__ __forceinline__ void store_rows(char* smem, char* out, unsigned lines, unsigned r0, unsigned c0, unsigned rows, unsigned cols) {
        constexpr int PER_ROW = S * 4;                   // lanes
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = (lane % PER_ROW) * 8;
        unsigned* const words = reinterpret_cast<unsigned*>(smem) + wave * 32 * PITCH;
        __syncthreads();                                 // the stages are done with
#pragma unroll
        for (int i = 0; i < S; ++i) {
#pragma unroll
            for (int j = 0; j < S; ++j)
#pragma unroll
                for (int x = 0; x < 16; ++x) words[(4 * (lane >> 5) + 8 * (x >> 2) + (x & 3)) * PITCH + j * 32 + (lane & 31)] = __float_as_uint(acc[i][j][x]);
            __builtin_amdgcn_wave_barrier();             // (a wave's LDS operations run in their order)
#pragma unroll
            for (int r = lane / PER_ROW; r < 32; r += 64 / PER_ROW) {
                const unsigned row = r0 + ((wave >> 1) * S + i) * 32 + r, col = c0 + (wave & 1) * S * 32 + c;
                const uint4 p = *reinterpret_cast<const uint4*>(words + r * PITCH + c), q = *reinterpret_cast<const uint4*>(words + r * PITCH + c + 4);
                if (row >= rows || col >= cols) continue;
                uint4 hi, lo;
                hi.x = (p.x & 0xFFFFu) | p.y << 16; hi.y = (p.z & 0xFFFFu) | p.w << 16; hi.z = (q.x & 0xFFFFu) | q.y << 16; hi.w = (q.z & 0xFFFFu) | q.w << 16;
                lo.x = p.x >> 16 | (p.y & 0xFFFF0000u); lo.y = p.z >> 16 | (p.w & 0xFFFF0000u); lo.z = q.x >> 16 | (q.y & 0xFFFF0000u); lo.w = q.z >> 16 | (q.w & 0xFFFF0000u);
                char* const at = out + at_line(lines, row, col);
                *reinterpret_cast<uint4*>(at) = hi;
                *reinterpret_cast<uint4*>(at + LINE / 2) = lo;
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
};

// A matrix whose rows are a tile's columns (the transpose, or a symmetric one).  A lane's place in it is computed once; the subtiles and register
// groups lie at distances that are the same for all lanes.  Loads from beyond the buffer give zeros; what lies beyond the last row is not stored.
struct Columns {
    i32x4 rsrc;
    unsigned at;
    template <typename C>
    static __device__ __forceinline__ Columns of(const Tile<C>&, const char* buf, unsigned rows, unsigned lines, unsigned r0, unsigned c0) {
        constexpr int S = Tile<C>::S;
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        return Columns{make_rsrc(buf, rows * lines * LINE),
                       (unsigned)at_line(lines, c0 + (wave & 1) * S * 32 + (lane & 31), r0 + (wave >> 1) * S * 32 + 4 * (lane >> 5))};
    }
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer() const {
        return __builtin_amdgcn_make_buffer_rsrc((void*)((unsigned long long)(unsigned)rsrc.x | (unsigned long long)(unsigned)rsrc.y << 32), 0, rsrc.z, rsrc.w);
    }
    // rows 8 g .. 8 g + 3 of a subtile, as pairs in one word
    __device__ __forceinline__ void store(unsigned sub, int g, const float* v) const {
        unsigned w[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) w[x] = __float_as_uint(v[x]);
        const u32x2 hi = {(w[0] & 0xFFFFu) | w[1] << 16, (w[2] & 0xFFFFu) | w[3] << 16};
        const u32x2 lo = {w[0] >> 16 | (w[1] & 0xFFFF0000u), w[2] >> 16 | (w[3] & 0xFFFF0000u)};
        const unsigned to = at + (g & 1) * 16, up = sub + (g >> 1) * 64 * LINE;
        __builtin_amdgcn_raw_buffer_store_b64(hi, buffer(), to, up, 0);
        __builtin_amdgcn_raw_buffer_store_b64(lo, buffer(), to + LINE / 2, up, 0);
    }
    __device__ __forceinline__ void load(unsigned sub, int g, float* v) const {
        const unsigned from = at + (g & 1) * 16, up = sub + (g >> 1) * 64 * LINE;
        const f16x4 hi = __builtin_bit_cast(f16x4, __builtin_amdgcn_raw_buffer_load_b64(buffer(), from, up, 0));
        const f16x4 lo = __builtin_bit_cast(f16x4, __builtin_amdgcn_raw_buffer_load_b64(buffer(), from + LINE / 2, up, 0));
#pragma unroll
        for (int x = 0; x < 4; ++x) v[x] = join(hi[x], lo[x]);
    }
};

// t-th tile on or below the diagonal, row by row
__device__ __forceinline__ void lower_tile(unsigned t, unsigned& i, unsigned& j) {
    i = (unsigned)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while ((i + 1) * (i + 2) / 2 <= t) ++i;
    while (i * (i + 1) / 2 > t) --i;
    j = t - i * (i + 1) / 2;
}

// a symmetric result: rows r .. r+3 of column c, stored as values r .. r+3 of row c, and off the diagonal tiles also as themselves
__device__ __forceinline__ void store_symmetric(char* out, unsigned lines, unsigned r, unsigned c, const float* v, bool mirror) {
    store4(out, lines, c, r, v);
    if (mirror) {
#pragma unroll
        for (int x = 0; x < 4; ++x) store1(out, lines, r + x, c, v[x]);
    }
}

struct Product {
    int l, r, out;
    float scale;                     // fp32 sum -> stored result
    float ident, lin;                // out = ident I + lin A + scale L R^T (POLY only; A in its stored scale)
};
static_assert(sizeof(Batch) + sizeof(Product) < 4096, "kernel arguments");

// m x m products (all operands symmetric): A^2 with the polynomial's epilogue, Q A, W Q, P Q.
template <typename C, bool POLY>
__global__ __launch_bounds__(256, C::PER_CU) void ns_square_product(Batch b, Product pr) {
    constexpr int BT = C::BT;
    __shared__ __attribute__((aligned(1024))) char smem[Tile<C>::SMEM];
    const Item s = b.item[find_item(b, blockIdx.x)];
    char* const base = b.ws + (size_t)s.base * 256;
    const unsigned M = pad64(s.m), lines = M / LINE_K, rows = (M + BT - 1) / BT;
    unsigned ti, tj;
    lower_tile(xcd_swizzle(blockIdx.x - s.first, rows * (rows + 1) / 2), ti, tj);
    Tile<C> t;
    t.run(smem, base + buffer_offset(pr.l, s.m, s.n), M, base + buffer_offset(pr.r, s.m, s.n), M, lines, ti * BT, tj * BT, 0, lines);
    char* const out = base + buffer_offset(pr.out, s.m, s.n);
    const Columns a = Columns::of(t, base + buffer_offset(A, s.m, s.n), M, lines, ti * BT, tj * BT), o = Columns::of(t, out, M, lines, ti * BT, tj * BT);
    const bool mirror = ti != tj;
    t.each([&](int row, int col, float* v, unsigned at) {
        const unsigned r = ti * BT + row, c = tj * BT + col;
        float av[16];
        if (POLY)
#pragma unroll
            for (int g = 0; g < 4; ++g) a.load(at, g, av + 4 * g);
#pragma unroll
        for (int x = 0; x < 16; ++x) {
            v[x] *= pr.scale;
            if (POLY) v[x] += pr.lin * av[x] + (r + 8 * (x >> 2) + (x & 3) == c && c < (unsigned)s.m ? pr.ident : 0.f);
            v[x] = __uint_as_float(pair_word(v[x]));
        }
        if (r < M && c < M)                              // (all 32 rows of a subtile or none)
#pragma unroll
            for (int g = 0; g < 4; ++g) o.store(at, g, v + 4 * g);
    });
    if (mirror) t.store_rows(smem, out, lines, ti * BT, tj * BT, M, M);
}

// Gram products A = X X^T: few tiles, long sums.  The sum is cut into `splits` runs of lines, each workgroup leaves its fp32 tile in
// the workspace (as its registers lie, 16 B per lane), and ns_gram_reduce adds the runs in their order.
struct GramItem {
    unsigned first, part;            // workgroup of the launch; first tile slot in the partial region
    int m, n;
    unsigned base, tiles, splits, run;
};
struct GramBatch {
    char* ws;
    float* partial;
    int count;
    float scale;
    GramItem item[BATCH];
};
static_assert(sizeof(GramBatch) < 4096, "kernel arguments");

template <typename C>
__global__ __launch_bounds__(256, C::PER_CU) void ns_gram(GramBatch b) {
    constexpr int BT = C::BT;
    __shared__ __attribute__((aligned(1024))) char smem[Tile<C>::SMEM];
    const GramItem s = b.item[find_item(b, blockIdx.x)];
    const char* const x = b.ws + (size_t)s.base * 256;
    const unsigned M = pad64(s.m), lines = pad64(s.n) / LINE_K;
    const unsigned u = xcd_swizzle(blockIdx.x - s.first, s.tiles * s.splits), k = u / s.tiles, tile = u - k * s.tiles;      // the tiles of one run are neighbours: they share its lines
    unsigned ti, tj;
    lower_tile(tile, ti, tj);
    Tile<C> t;
    const unsigned q0 = k * s.run, q1 = q0 + s.run < lines ? q0 + s.run : lines;
    t.run(smem, x, M, x, M, lines, ti * BT, tj * BT, q0, q1);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    constexpr int S = Tile<C>::S;
    float* const out = b.partial + ((size_t)s.part + (size_t)tile * s.splits + k) * (BT * BT);
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int j = 0; j < S; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int sub = ((wave >> 1) * S + i) * (BT / 32) + (wave & 1) * S + j;
                st4(out + (((size_t)sub * 4 + g) * 64 + lane) * 4,
                    make_float4(t.acc[i][j][4 * g], t.acc[i][j][4 * g + 1], t.acc[i][j][4 * g + 2], t.acc[i][j][4 * g + 3]));
            }
}

// one workgroup per 32 x 32 subtile; wave w adds the runs w, w + 4, ... and the four sums are joined in order
template <int BT>
__global__ __launch_bounds__(256) void ns_gram_reduce(GramBatch b) {
    constexpr unsigned SUBS = (BT / 32) * (BT / 32);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    // `first` counts the product's workgroups (tiles * splits): this launch has tiles * SUBS per item, so the item is found by walking
    unsigned wg = blockIdx.x;
    int it = 0;
    while (wg >= b.item[it].tiles * SUBS) wg -= b.item[it++].tiles * SUBS;
    const GramItem s = b.item[it];
    const unsigned tile = wg / SUBS, sub = wg - tile * SUBS;
    const float* const in = b.partial + ((size_t)s.part + (size_t)tile * s.splits) * (BT * BT) + (size_t)sub * 1024 + lane * 4;
    float4 v[4] = {zero4(), zero4(), zero4(), zero4()};
    for (unsigned k = wave; k < s.splits; k += 4)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float4 p = ld4(in + (size_t)k * (BT * BT) + g * 256);
            v[g].x += p.x; v[g].y += p.y; v[g].z += p.z; v[g].w += p.w;
        }
    __shared__ float4 red[4][4][64];
#pragma unroll
    for (int g = 0; g < 4; ++g) red[wave][g][lane] = v[g];
    __syncthreads();
    const int g = wave;                                  // wave g joins and stores register group g
    const float4 a = red[0][g][lane], c = red[1][g][lane], d = red[2][g][lane], e = red[3][g][lane];
    const float r4[4] = {((a.x + c.x) + (d.x + e.x)) * b.scale, ((a.y + c.y) + (d.y + e.y)) * b.scale,
                         ((a.z + c.z) + (d.z + e.z)) * b.scale, ((a.w + c.w) + (d.w + e.w)) * b.scale};
    unsigned ti, tj;
    lower_tile(tile, ti, tj);
    const unsigned M = pad64(s.m);
    const unsigned row = ti * BT + (sub / (BT / 32)) * 32 + 8 * g + 4 * (lane >> 5), col = tj * BT + (sub % (BT / 32)) * 32 + (lane & 31);
    if (row >= M || col >= M) return;
    store_symmetric(b.ws + (size_t)s.base * 256 + buffer_offset(A, s.m, s.n), M / LINE_K, row, col, r4, ti != tj);
}

// The tiles of a product with P in strips of 8 rows of tiles, column by column: what an XCD works on at a time (32 tiles of 128) is then
// nearly square, and its L2 serves every panel to several workgroups (4096 x 4096: 409 -> 257 us for the copies alone).
__device__ __forceinline__ void big_tile(unsigned u, unsigned down, unsigned across, unsigned& ti, unsigned& tj) {
    u = xcd_swizzle(u, down * across);
    const unsigned g = u / (8 * across), left = down - 8 * g, h = left < 8 ? left : 8, v = u - 8 * g * across;
    tj = v / h;
    ti = 8 * g + v - tj * h;
}

// X <- alpha X + P X between segments (alpha = 0 where P holds the identity's part): both orders again (T1 from T0, X in place:
// no workgroup reads X)
template <typename C>
__global__ __launch_bounds__(256, C::PER_CU) void ns_apply(Batch b, int p, int tin, int tout, float scale, float alpha) {
    constexpr int BT = C::BT;
    __shared__ __attribute__((aligned(1024))) char smem[Tile<C>::SMEM];
    const Item s = b.item[find_item(b, blockIdx.x)];
    char* const base = b.ws + (size_t)s.base * 256;
    const unsigned M = pad64(s.m), N = pad64(s.n);
    unsigned ti, tj;
    big_tile(blockIdx.x - s.first, (M + BT - 1) / BT, (N + BT - 1) / BT, ti, tj);
    Tile<C> t;
    t.run(smem, base + buffer_offset(p, s.m, s.n), M, base + buffer_offset(tin, s.m, s.n), N, M / LINE_K, ti * BT, tj * BT, 0, M / LINE_K);
    const Columns to = Columns::of(t, base + buffer_offset(tout, s.m, s.n), N, M / LINE_K, ti * BT, tj * BT);
    const Columns from = Columns::of(t, base + buffer_offset(tin, s.m, s.n), N, M / LINE_K, ti * BT, tj * BT);
    t.each([&](int row, int col, float* v, unsigned at) {
        if (alpha != 0.f) {
            float old[16];
#pragma unroll
            for (int g = 0; g < 4; ++g) from.load(at, g, old + 4 * g);
#pragma unroll
            for (int x = 0; x < 16; ++x) v[x] = fmaf(alpha, old[x], v[x] * scale);
        } else {
#pragma unroll
            for (int x = 0; x < 16; ++x) v[x] *= scale;
        }
#pragma unroll
        for (int x = 0; x < 16; ++x) v[x] = __uint_as_float(pair_word(v[x]));
        if (ti * BT + row < M && tj * BT + col < N)      // (all 32 rows of a subtile or none)
#pragma unroll
            for (int g = 0; g < 4; ++g) to.store(at, g, v + 4 * g);
    });
    t.store_rows(smem, base, N / LINE_K, ti * BT, tj * BT, M, N);
}

// the last product goes straight to where the caller wants it
struct Target {
    unsigned first, base;
    void* dst;
    long si, sj;                     // strides of X's rows (m) and columns (n) in the destination
    int m, n;
    float factor;                    // MUON: the shape's factor on lr
    int dtype, group;
    int turned;                      // 1: the lanes of a wave run along m (si == 1)
};
struct TargetBatch {
    char* ws;
    int count;
    int p, tin;
    float scale, alpha;              // of the stored sum, of the stored X (as in ns_apply)
    Target item[BATCH];
};
static_assert(fits_arguments<TargetBatch>, "kernel arguments");

// MUON: param = param (1 - lr wd) - lr factor O, else dst = O
template <typename C, bool MUON>
__global__ __launch_bounds__(256, C::PER_CU) void ns_finish(TargetBatch b, Hyper h, const Hyper* __restrict__ hd) {
    constexpr int BT = C::BT;
    __shared__ __attribute__((aligned(1024))) char smem[Tile<C>::SMEM];
    const Target s = b.item[find_item(b, blockIdx.x)];
    const char* const base = b.ws + (size_t)s.base * 256;
    const unsigned M = pad64(s.m), N = pad64(s.n);
    unsigned ti, tj;
    big_tile(blockIdx.x - s.first, (M + BT - 1) / BT, (N + BT - 1) / BT, ti, tj);
    const char* const P = base + buffer_offset(b.p, s.m, s.n);
    const char* const T = base + buffer_offset(b.tin, s.m, s.n);
    Tile<C> t;
    if (s.turned) t.run(smem, T, N, P, M, M / LINE_K, tj * BT, ti * BT, 0, M / LINE_K);
    else t.run(smem, P, M, T, N, M / LINE_K, ti * BT, tj * BT, 0, M / LINE_K);
    const unsigned r0 = (s.turned ? tj : ti) * BT, c0 = (s.turned ? ti : tj) * BT;
    const unsigned rows = s.turned ? s.n : s.m, cols = s.turned ? s.m : s.n;
    const long sr = s.turned ? s.sj : s.si, sc = s.turned ? s.si : s.sj;
    float keep = 1.f, step = 0.f;
    if (MUON) {
        const float lr = hd ? hd->lr[s.group] : h.lr[s.group], wd = hd ? hd->wd[s.group] : h.wd[s.group];
        keep = 1.f - lr * wd;
        step = lr * s.factor;
    }
    // row c of it, values r .. r+3: X's own order, or the other one
    const Columns old = Columns::of(t, s.turned ? base : T, s.turned ? M : N, (s.turned ? N : M) / LINE_K, r0, c0);
    t.each([&](int row, int col, float* v, unsigned sub) {
        const unsigned c = c0 + col, r = r0 + row;
        if (c >= cols || r >= rows) return;              // (r is the lane's first row)
        if (b.alpha != 0.f) {
            float old4[16];
#pragma unroll
            for (int g = 0; g < 4; ++g) old.load(sub, g, old4 + 4 * g);
#pragma unroll
            for (int x = 0; x < 16; ++x) v[x] = fmaf(b.alpha, old4[x], v[x] * b.scale);
        } else {
#pragma unroll
            for (int x = 0; x < 16; ++x) v[x] *= b.scale;
        }
        const long at = (long)r * sr + (long)c * sc;     // and uniform distances from there
        const auto rows_of = [&](auto* const dst, auto make) {
            if ((r & ~31u) + 32 <= rows) {               // all of a subtile's rows, for the wave
#pragma unroll
                for (int x = 0; x < 16; ++x) make(dst + (8 * (x >> 2) + (x & 3)) * sr, x);
            } else {
#pragma unroll
                for (int x = 0; x < 16; ++x)
                    if (r + 8 * (x >> 2) + (x & 3) < rows) make(dst + (8 * (x >> 2) + (x & 3)) * sr, x);
            }
        };
        if (MUON) {
            float before[16];                            // all loads first: behind a store they would wait for it
            rows_of(static_cast<float*>(s.dst) + at, [&](float* p, int x) { before[x] = *p; });
            rows_of(static_cast<float*>(s.dst) + at, [&](float* p, int x) { *p = fmaf(-step, v[x], before[x] * keep); });
        } else if (s.dtype) {
            rows_of(static_cast<unsigned short*>(s.dst) + at, [&](unsigned short* p, int x) { *p = f32_to_bf16(v[x]); });
        } else {
            rows_of(static_cast<float*>(s.dst) + at, [&](float* p, int x) { *p = v[x]; });
        }
    });
}

// ------------------------------------------------------------------------------------------------ small matrices
// One workgroup does the whole iteration of a matrix whose X fits its registers: m <= 32 R rows, n <= 256 G columns; one launch instead of 22.
// Wave w of 8 owns the 32-column slices w, w + 8, ...; a lane holds one column of each, in the order of a matrix
// instruction's result (rows 8 e + 4 (lane / 32) + 0 .. 3 of each 32).  Steps one by one:
//     A = X X^T    each wave turns its slices in LDS (words hi | lo << 16) and sums its columns' products; the 8 sums are added in order
//     Q = b A + c A^2
//     X <- a X + Q X    X goes into the instruction as it lies in the registers: the sum over rows may run in any order, so Q's words
//                       are read in the order in which a lane holds the rows
// Bound by latency: 64 x 576 is 25 MFLOP a step on one CU (2.7 us at its peak rate) plus four barriers.
enum Class { SMALL_1_1, SMALL_1_3, SMALL_1_9, SMALL_2_1, SMALL_2_3, THIN, SQUARE, WIDE_MATRIX, CLASSES };    // SMALL_R_G
struct SmallItem {
    const void* src;                 // MUON: the gradient
    void* dst;                       // MUON: the parameter
    float* mom;
    long si, sj, di, dj;             // strides of X's rows and columns in src (and mom), and in dst
    int m, n;
    float factor;
    int dtype, group, cls;
    unsigned src_bytes, dst_bytes;   // up to the last element
};
struct SmallStep {
    float gram, quad, lin, apply;    // fp32 sums to the next stored scale; X <- a X + Q X keeps X's scale `apply` folded in
    float alpha, ident;
};
constexpr int SMALL_BATCH = 32;
struct SmallBatch {
    double eps;
    float scale, unscale;            // of the first X, and of the last one's inverse
    int steps, nesterov;
    SmallStep step[SEGMI_NS_MAX_STEPS];
    SmallItem item[SMALL_BATCH];
};
static_assert(fits_arguments<SmallBatch>, "kernel arguments");

// two values' pairs: hi of both in one register, lo of both in another; the mixed-precision instructions take the halves as they lie
struct Pair2 {
    unsigned hi, lo;
    __device__ __forceinline__ void set(float a, float b) {
        asm("" : "+v"(a), "+v"(b));                      // as in `split`
        hi = __builtin_bit_cast(unsigned, f16x2{(_Float16)a, (_Float16)b});
        asm("v_fma_mixlo_f16 %0, %1, -1.0, %2 op_sel:[0,0,0] op_sel_hi:[1,0,0]\n\t"
            "v_fma_mixhi_f16 %0, %1, -1.0, %3 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=&v"(lo) : "v"(hi), "v"(a), "v"(b));
    }
    // f * value
    __device__ __forceinline__ float times(int which, float f) const {
        float v;
        if (which)
            asm("v_fma_mix_f32 %0, %1, %3, 0 op_sel:[1,0,0] op_sel_hi:[1,0,0]\n\t"
                "v_fma_mix_f32 %0, %2, %3, %0 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=&v"(v) : "v"(lo), "v"(hi), "v"(f));
        else
            asm("v_fma_mix_f32 %0, %1, %3, 0 op_sel:[0,0,0] op_sel_hi:[1,0,0]\n\t"
                "v_fma_mix_f32 %0, %2, %3, %0 op_sel:[0,0,0] op_sel_hi:[1,0,0]" : "=&v"(v) : "v"(lo), "v"(hi), "v"(f));
        return v;
    }
    __device__ __forceinline__ unsigned word(int which) const { return __builtin_amdgcn_perm(lo, hi, which ? 0x07060302u : 0x05040100u); }
};
struct PairFrag {
    f16x8 hi, lo;
    __device__ __forceinline__ void from_words(uint4 p, uint4 q) {
        const uint4 h = make_uint4(__builtin_amdgcn_perm(p.y, p.x, 0x05040100u), __builtin_amdgcn_perm(p.w, p.z, 0x05040100u),
                                   __builtin_amdgcn_perm(q.y, q.x, 0x05040100u), __builtin_amdgcn_perm(q.w, q.z, 0x05040100u));
        const uint4 l = make_uint4(__builtin_amdgcn_perm(p.y, p.x, 0x07060302u), __builtin_amdgcn_perm(p.w, p.z, 0x07060302u),
                                   __builtin_amdgcn_perm(q.y, q.x, 0x07060302u), __builtin_amdgcn_perm(q.w, q.z, 0x07060302u));
        hi = __builtin_bit_cast(f16x8, h);
        lo = __builtin_bit_cast(f16x8, l);
    }
    __device__ __forceinline__ void from_pairs(const Pair2* p) {
        hi = __builtin_bit_cast(f16x8, make_uint4(p[0].hi, p[1].hi, p[2].hi, p[3].hi));
        lo = __builtin_bit_cast(f16x8, make_uint4(p[0].lo, p[1].lo, p[2].lo, p[3].lo));
    }
};
// a symmetric 32 R x 32 R matrix in LDS as two planes; the pitch lets ds_read_b128 of 16 rows cover all 64 banks
template <int R>
struct PairPlanes {
    static constexpr int PITCH = 32 * R + 8;
    _Float16 hi[32 * R][PITCH], lo[32 * R][PITCH];
    // values (row .. row + 3, col), and their mirror images if `mirror`
    __device__ __forceinline__ void store(int row, int col, const float* v, bool mirror) {
        Pair2 p[2];
        p[0].set(v[0], v[1]);
        p[1].set(v[2], v[3]);
        *reinterpret_cast<uint2*>(&hi[col][row]) = make_uint2(p[0].hi, p[1].hi);
        *reinterpret_cast<uint2*>(&lo[col][row]) = make_uint2(p[0].lo, p[1].lo);
        if (mirror)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                hi[row + x][col] = __builtin_bit_cast(f16x2, p[x >> 1].hi)[x & 1];
                lo[row + x][col] = __builtin_bit_cast(f16x2, p[x >> 1].lo)[x & 1];
            }
    }
    __device__ __forceinline__ void load(int row, int col, float f, float* v) const {       // f times the values
        Pair2 p[2];
        const uint2 h = *reinterpret_cast<const uint2*>(&hi[col][row]), l = *reinterpret_cast<const uint2*>(&lo[col][row]);
        p[0].hi = h.x; p[1].hi = h.y; p[0].lo = l.x; p[1].lo = l.y;
#pragma unroll
        for (int x = 0; x < 4; ++x) v[x] = p[x >> 1].times(x & 1, f);
    }
    // eight values of a row from k on, and two times four
    __device__ __forceinline__ PairFrag frag(int row, int k) const {
        return PairFrag{*reinterpret_cast<const f16x8*>(&hi[row][k]), *reinterpret_cast<const f16x8*>(&lo[row][k])};
    }
    __device__ __forceinline__ PairFrag frag(int row, int k0, int k1) const {
        const uint2 a = *reinterpret_cast<const uint2*>(&hi[row][k0]), b = *reinterpret_cast<const uint2*>(&hi[row][k1]);
        const uint2 c = *reinterpret_cast<const uint2*>(&lo[row][k0]), d = *reinterpret_cast<const uint2*>(&lo[row][k1]);
        return PairFrag{__builtin_bit_cast(f16x8, make_uint4(a.x, a.y, b.x, b.y)), __builtin_bit_cast(f16x8, make_uint4(c.x, c.y, d.x, d.y))};
    }
};
__device__ __forceinline__ void pair_product(const PairFrag& l, const PairFrag& r, f32x16& acc, f32x16& mix) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(l.hi, r.hi, acc, 0, 0, 0);
    mix = __builtin_amdgcn_mfma_f32_32x32x16_f16(l.lo, r.hi, mix, 0, 0, 0);
    mix = __builtin_amdgcn_mfma_f32_32x32x16_f16(l.hi, r.lo, mix, 0, 0, 0);
}
__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int x = 0; x < 16; ++x) z[x] = 0.f;
    return z;
}

// Up to this many rows a rounding of A or Q is not averaged over many directions: it moves all singular values near 1, where the
// terms of the polynomial cancel (0.7 = 3.44 - 4.77 + 2.03), ten times its size.  There A^2 and Q are taken in 64 bits and Q enters the product
// as three fp16 numbers: median distance of 5 x 162 from 64-bit results 9.7e-7 -> 4.7e-7, of 16 x 200 8.2e-7 -> 4.6e-7 (the fp32 iteration
// 6.9e-7, 6.6e-7), at no measurable time.
constexpr int TINY = 16;

template <int R>
struct SmallShared {
    static constexpr int SUBS = R * (R + 1) / 2;         // 32 x 32 subtiles on and below the diagonal
    static constexpr int XP = 36;                        // row pitch in words: ds_read_b128 of 16 rows covers all 64 banks
    union {
        unsigned x[8][32 * R][XP];                       // a wave's slice, turned
        float4 part[8][SUBS][4][64];                     // the waves' sums
    } u;
    PairPlanes<R> A, Q;
    double red[8];
    // R == 1, m <= TINY: A in 64 bits, and what Q's pairs leave of it
    double a64[R == 1 ? TINY : 1][TINY + 1];
    _Float16 rest[R == 1 ? 32 : 1][PairPlanes<R>::PITCH];
};

template <int R, int G, bool MUON>
__device__ __forceinline__ void small_matrix(const SmallBatch& b, const SmallItem& s, SmallShared<R>& sh, const Hyper& h, const Hyper* __restrict__ hd) {
    constexpr int SUBS = SmallShared<R>::SUBS;
    auto& u = sh.u;
    PairPlanes<R>&A = sh.A, &Q = sh.Q;
    double* const red = sh.red;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, half = lane >> 5;
    const int m = s.m, n = s.n;
    const int slices = (n + 31) / 32, waves = slices < 8 ? slices : 8;
    const float mu = MUON ? (hd ? hd->mom[s.group] : h.mom[s.group]) : 0.f;
    const bool nest = MUON && b.nesterov;
    const bool tiny = R == 1 && m <= TINY;
    if (tiny)                                            // Q and its rest stay zero beyond the 16 rows and columns
        for (int i = tid; i < 32 * PairPlanes<R>::PITCH; i += 512) (&Q.hi[0][0])[i] = (&Q.lo[0][0])[i] = (&sh.rest[0][0])[i] = (_Float16)0.f;

    // An element's byte offset is a lane's part (column, half of the rows) plus a uniform part (the row in the half): the instruction
    // adds the two.  A lane outside the matrix gets an offset beyond the buffer, which reads as 0 and drops what is written.
    const unsigned size = s.dtype ? 2 : 4;
    const auto lane_offset = [&](int g, long si, long sj) {
        const int j = (g * 8 + wave) * 32 + col;
        return j < n ? ((unsigned)j * (unsigned)sj + 4u * half * (unsigned)si) * size : 0xFFFFFFFFu;
    };
    // f(r, e, lane's part, uniform part) for the elements of a slice; the uniform part never leaves the buffer
    const auto each = [&](unsigned at, long si, auto f) {
        int rows = m - 4 * half;                         // the comparisons are made anew each time: kept, their masks would fill the registers
        asm volatile("" : "+v"(rows));
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const unsigned i = 32 * r + 8 * (e >> 2) + (e & 3);
                f(r, e, (int)i < rows ? at : 0xFFFFFFFFu, (int)i < m ? i * (unsigned)si * size : 0u);
            }
        __builtin_amdgcn_sched_barrier(0);
    };
    const __amdgpu_buffer_rsrc_t src = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(s.src), 0, s.src_bytes, 0x00020000);
    const __amdgpu_buffer_rsrc_t mom = __builtin_amdgcn_make_buffer_rsrc(s.mom, 0, MUON ? s.src_bytes : 0, 0x00020000);
    const __amdgpu_buffer_rsrc_t dst = __builtin_amdgcn_make_buffer_rsrc(s.dst, 0, s.dst_bytes, 0x00020000);
    const auto load = [](__amdgpu_buffer_rsrc_t b, unsigned lane_part, unsigned part) {
        return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(b, lane_part, part, 0));
    };

    float x[G][R][16];
    Pair2 w[G][R][8];                                    // X as pairs, from the first step on: rows 2 p, 2 p + 1 of the order above
    double sum = 0.0;
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const unsigned at = lane_offset(g, s.si, s.sj);
        if (s.dtype)
            each(at, s.si, [&](int r, int e, unsigned lp, unsigned up) { x[g][r][e] = bf16_to_f32(__builtin_amdgcn_raw_buffer_load_b16(src, lp, up, 0)); });
        else
            each(at, s.si, [&](int r, int e, unsigned lp, unsigned up) { x[g][r][e] = load(src, lp, up); });
    }
    if (MUON)
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const unsigned at = lane_offset(g, s.si, s.sj);
            float v[R][16];                              // all loads first: behind a store they would wait for it
            each(at, s.si, [&](int r, int e, unsigned lp, unsigned up) { v[r][e] = fmaf(mu, load(mom, lp, up), x[g][r][e]); });
            each(at, s.si, [&](int r, int e, unsigned lp, unsigned up) {
                __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v[r][e]), mom, lp, up, 0);
                x[g][r][e] = nest ? fmaf(mu, v[r][e], x[g][r][e]) : v[r][e];
            });
        }
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < 16; ++e) sum = fma((double)x[g][r][e], (double)x[g][r][e], sum);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (lane == 0) red[wave] = sum;
    __syncthreads();
    const double norm = sqrt(((red[0] + red[1]) + (red[2] + red[3])) + ((red[4] + red[5]) + (red[6] + red[7])));
    // In 64 bits: the factor may lie outside fp32's range, and its rounding would be an error of all singular values at once, which the
    // iteration enlarges tenfold near 1 (a NaN norm stays)
    const double factor = (double)b.scale / (norm <= b.eps ? b.eps : norm);
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int p = 0; p < 8; ++p)
                w[g][r][p].set((float)((double)x[g][r][2 * p] * factor), (float)((double)x[g][r][2 * p + 1] * factor));

    for (int step = 0; step < b.steps; ++step) {
        SmallStep k = b.step[step];
        // One singular value, 1 from the start, is where a and Q cancel (0.7 = 3.44 - 2.74): there the sum is taken before it is rounded.
        if (m == 1) k.alpha = 0.f;
        else k.ident = 0.f;
        {   // A = X X^T
            f32x16 acc[SUBS], mix[SUBS];
#pragma unroll
            for (int t = 0; t < SUBS; ++t) acc[t] = mix[t] = zero16();
#pragma unroll
            for (int g = 0; g < G; ++g) {
                if (g * 8 + wave >= slices) continue;
                // (a wave's own LDS: its reads follow its writes in order, no barrier)
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int e = 0; e < 16; ++e) u.x[wave][32 * r + 8 * (e >> 2) + 4 * half + (e & 3)][col] = w[g][r][e >> 1].word(e & 1);
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    PairFrag f[R];
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const uint4* const p = reinterpret_cast<const uint4*>(&u.x[wave][32 * r + col][ks * 16 + half * 8]);
                        f[r].from_words(p[0], p[1]);
                    }
#pragma unroll
                    for (int i = 0; i < R; ++i)
#pragma unroll
                        for (int j = 0; j <= i; ++j) pair_product(f[i], f[j], acc[i * (i + 1) / 2 + j], mix[i * (i + 1) / 2 + j]);
                    __builtin_amdgcn_sched_barrier(0);   // (slices and steps one after the other: all at once do not fit the registers)
                }
            }
            __syncthreads();
            if (wave < waves)
#pragma unroll
                for (int t = 0; t < SUBS; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        u.part[wave][t][e][lane] = make_float4(acc[t][4 * e] + mix[t][4 * e], acc[t][4 * e + 1] + mix[t][4 * e + 1],
                                                           acc[t][4 * e + 2] + mix[t][4 * e + 2], acc[t][4 * e + 3] + mix[t][4 * e + 3]);
            __syncthreads();
            for (int p = tid; p < SUBS * 256; p += 512) {
                const int t = p >> 8, e = (p >> 6) & 3, l = p & 63;
                float4 q[8];                             // all reads first; a wave without columns counts as zeros
#pragma unroll
                for (int i = 0; i < 8; ++i) q[i] = u.part[i < waves ? i : 0][t][e][l];
                float4 v = q[0];
#pragma unroll
                for (int i = 1; i < 8; ++i) {
                    const float in = i < waves ? 1.f : 0.f;
                    v.x = fmaf(in, q[i].x, v.x); v.y = fmaf(in, q[i].y, v.y); v.z = fmaf(in, q[i].z, v.z); v.w = fmaf(in, q[i].w, v.w);
                }
                const int ti = t == 0 ? 0 : 1, tj = t == 2 ? 1 : 0;
                const int row = 32 * ti + 8 * e + 4 * (l >> 5), c = 32 * tj + (l & 31);
                if (tiny) {
                    if (row < TINY && c < TINY) {
                        double d[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (i < waves) { d[0] += q[i].x; d[1] += q[i].y; d[2] += q[i].z; d[3] += q[i].w; }
#pragma unroll
                        for (int x = 0; x < 4; ++x) sh.a64[row + x][c] = d[x] * k.gram;
                    }
                    continue;
                }
                const float a4[4] = {v.x * k.gram, v.y * k.gram, v.z * k.gram, v.w * k.gram};
                A.store(row, c, a4, ti != tj);
            }
        }
        __syncthreads();
        if (tiny) {          // Q = b A + c A^2, a thread per element
            const int i = (tid >> 4) & 15, j = tid & 15;
            if (tid < 256) {
                double q = 0.0;
#pragma unroll
                for (int y = 0; y < TINY; ++y) q = fma(sh.a64[i][y], sh.a64[y][j], q);
                q = fma(q, (double)k.quad, fma(sh.a64[i][j], (double)k.lin, i == j ? (double)k.ident : 0.0));
                const _Float16 hi = (_Float16)(float)q;
                const double left = q - (double)(float)hi;
                const _Float16 lo = (_Float16)(float)left;
                Q.hi[i][j] = hi;
                Q.lo[i][j] = lo;
                sh.rest[i][j] = (_Float16)(float)(left - (double)(float)lo);
            }
        } else if (wave < SUBS) {   // a wave per subtile
            const int ti = wave == 0 ? 0 : 1, tj = wave == 2 ? 1 : 0;
            f32x16 acc = zero16(), mix = zero16(), mix2 = zero16();
            PairFrag l[2 * R], r[2 * R];                 // all reads first
#pragma unroll
            for (int ks = 0; ks < 2 * R; ++ks) {
                l[ks] = A.frag(32 * ti + col, ks * 16 + half * 8);
                r[ks] = A.frag(32 * tj + col, ks * 16 + half * 8);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int ks = 0; ks < 2 * R; ++ks) pair_product(l[ks], r[ks], acc, ks & 1 ? mix2 : mix);
#pragma unroll
            for (int y = 0; y < 16; ++y) mix[y] += mix2[y];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = 32 * ti + 8 * e + 4 * half, c = 32 * tj + col;
                float v[4];
                A.load(row, c, k.lin, v);
#pragma unroll
                for (int y = 0; y < 4; ++y) v[y] = fmaf(acc[4 * e + y] + mix[4 * e + y], k.quad, v[y] + (row + y == c ? k.ident : 0.f));
                Q.store(row, c, v, ti != tj);
            }
        }
        __syncthreads();
        // X <- a X + Q X, Q's rows one block of 16 columns ahead of the products (behind the last block comes the first again)
        PairFrag q[R];
        const auto q_block = [&](int t) {
#pragma unroll
            for (int r = 0; r < R; ++r) q[r] = Q.frag(32 * r + col, 16 * t + 4 * half, 16 * t + 8 + 4 * half);
        };
        q_block(0);
        f16x8 rest = {0, 0, 0, 0, 0, 0, 0, 0};
        if (tiny) {
            const uint2 a = *reinterpret_cast<const uint2*>(&sh.rest[col][4 * half]), b2 = *reinterpret_cast<const uint2*>(&sh.rest[col][8 + 4 * half]);
            rest = __builtin_bit_cast(f16x8, make_uint4(a.x, a.y, b2.x, b2.y));
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            if (g * 8 + wave >= slices) continue;
            f32x16 acc[R];                               // (at most 64 products: no accumulator of their own for the mixed ones)
#pragma unroll
            for (int r = 0; r < R; ++r) acc[r] = zero16();
#pragma unroll
            for (int t = 0; t < 2 * R; ++t) {            // rows 16 t .. 16 t + 15 of X
                PairFrag xf, now[R];
                xf.from_pairs(&w[g][t >> 1][4 * (t & 1)]);
#pragma unroll
                for (int r = 0; r < R; ++r) now[r] = q[r];
                q_block((t + 1) % (2 * R));
                __builtin_amdgcn_sched_barrier(0);
                if (t == 0 && tiny) acc[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(rest, xf.hi, acc[0], 0, 0, 0);
#pragma unroll
                for (int r = 0; r < R; ++r) acc[r] = __builtin_amdgcn_mfma_f32_32x32x16_f16(now[r].lo, xf.hi, acc[r], 0, 0, 0);
#pragma unroll
                for (int r = 0; r < R; ++r) acc[r] = __builtin_amdgcn_mfma_f32_32x32x16_f16(now[r].hi, xf.lo, acc[r], 0, 0, 0);
#pragma unroll
                for (int r = 0; r < R; ++r) acc[r] = __builtin_amdgcn_mfma_f32_32x32x16_f16(now[r].hi, xf.hi, acc[r], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int p = 0; p < 8; ++p)
                    w[g][r][p].set(fmaf(acc[r][2 * p], k.apply, w[g][r][p].times(0, k.alpha)), fmaf(acc[r][2 * p + 1], k.apply, w[g][r][p].times(1, k.alpha)));
            __builtin_amdgcn_sched_barrier(0);
        }
        // (the next step's first barrier lies behind its turning of X, which touches neither A nor Q)
    }

    float keep = 1.f, rate = 0.f;
    if (MUON) {
        const float lr = hd ? hd->lr[s.group] : h.lr[s.group], wd = hd ? hd->wd[s.group] : h.wd[s.group];
        keep = 1.f - lr * wd;
        rate = lr * s.factor;
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const unsigned at = lane_offset(g, s.di, s.dj);
        if (MUON) {
            float v[R][16];
            each(at, s.di, [&](int r, int e, unsigned lp, unsigned up) { v[r][e] = load(dst, lp, up); });
            each(at, s.di, [&](int r, int e, unsigned lp, unsigned up) {
                __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(fmaf(-rate, w[g][r][e >> 1].times(e & 1, b.unscale), v[r][e] * keep)), dst, lp, up, 0);
            });
        } else if (s.dtype) {
            each(at, s.di, [&](int r, int e, unsigned lp, unsigned up) {
                __builtin_amdgcn_raw_buffer_store_b16(f32_to_bf16(w[g][r][e >> 1].times(e & 1, b.unscale)), dst, lp, up, 0);
            });
        } else {
            each(at, s.di, [&](int r, int e, unsigned lp, unsigned up) {
                __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(w[g][r][e >> 1].times(e & 1, b.unscale)), dst, lp, up, 0);
            });
        }
    }
}

// CLS: the class of all matrices of the launch, or CLASSES: mixed, then it lasts as long as the longest of them (a kernel of its
// own per class needs fewer registers: 64 x 576 45 us instead of 50)
template <int CLS, bool MUON>
__global__ __launch_bounds__(512, 2) void ns_small(SmallBatch b, Hyper h, const Hyper* __restrict__ hd) {
    constexpr bool SMALL_LDS = CLS == SMALL_1_1 || CLS == SMALL_1_3 || CLS == SMALL_1_9;
    __shared__ __attribute__((aligned(16))) char smem[SMALL_LDS ? sizeof(SmallShared<1>) : sizeof(SmallShared<2>)];
    const SmallItem& s = b.item[blockIdx.x];
    SmallShared<1>& one = *reinterpret_cast<SmallShared<1>*>(smem);
    SmallShared<2>& two = *reinterpret_cast<SmallShared<2>*>(smem);
    switch (CLS == CLASSES ? s.cls : CLS) {
        case SMALL_1_1: small_matrix<1, 1, MUON>(b, s, one, h, hd); break;
        case SMALL_1_3: small_matrix<1, 3, MUON>(b, s, one, h, hd); break;
        case SMALL_1_9: small_matrix<1, 9, MUON>(b, s, one, h, hd); break;
        case SMALL_2_1: small_matrix<2, 1, MUON>(b, s, two, h, hd); break;
        default: small_matrix<2, 3, MUON>(b, s, two, h, hd); break;
    }
}

// ------------------------------------------------------------------------------------------------ thin matrices
// Up to TINY rows that small_matrix does not take (more than 2304 columns, or a span beyond its 32-bit offsets).  For the reason given at TINY
// the Gram matrix, A^2, Q and the products with Q are all taken in 64 bits; X is held in fp32, [row][column].  A launch per step: a workgroup adds
// the Gram matrix's parts, one per workgroup of the launch before, in their order, makes Q of them, takes its columns through
// X <- (a I + b A + c A^2) X, one column a thread, and leaves its part of the new Gram matrix, one element a thread.
// Distance from 64-bit results (root mean square of 16 matrices): 16 x 4608 6e-8, noise with strong directions 1.6e-7; as fp16 pairs through the
// products above 1.3e-6, the fp32 iteration 1.0e-6.  Time, here / there: 3 x 5000 57 / 94 us, 16 x 36864 113 / 152, 16 x 10^6 656 / 1046, 32 of
// 8 x 10000 168 / 358; 16 x 4608 beside 256 x 1024, which it no longer shares launches with, 188 / 134, beside a network's filters nothing.
// Bound by latency: seven launches, of 9 us each for 3 x 5000 and 19 for 16 x 36864, and from some 10^5 columns on that of the 64-bit products of four
// waves a CU, whose operands come from LDS (16 x 16 000 000: 1.4 ms a step for 2 GB of X, 1.5 TB/s; without the Gram matrix no less).
struct ThinItem {
    const void* src;                 // MUON: the gradient
    void* dst;                       // MUON: the parameter
    float* mom;
    long si, sj, di, dj;             // strides of X's rows and columns in src (and mom), and in dst
    size_t x;                        // X in the batch's X region
    unsigned first;                  // first workgroup of a launch; also the first part of the Gram matrix
    unsigned part, parts;            // its partial sums of squares
    int m, n;
    float factor;                    // MUON
    short dtype, group;
};
constexpr int THIN_BATCH = 32;
struct ThinBatch {
    float* x;
    const double* partial;
    double* gram[2];                 // parts of 256 values, read and written in turns
    double a, b, c, eps;
    int count, nesterov;
    ThinItem item[THIN_BATCH];
};
static_assert(THIN_BATCH <= BATCH && fits_arguments<ThinBatch>, "kernel arguments");
constexpr int THIN_TILE = 256;       // columns at a time
// Columns per workgroup: at most 256 workgroups a matrix, so that adding their parts stays short.
__host__ __device__ inline unsigned thin_columns(int n) { return THIN_TILE * (((unsigned)n + 256u * THIN_TILE - 1) / (256u * THIN_TILE)); }
__host__ __device__ inline unsigned thin_groups(int n) { return ((unsigned)n + thin_columns(n) - 1) / thin_columns(n); }

enum ThinStage { THIN_FIRST, THIN_NEXT, THIN_LAST };     // source to X; X to X; X to the destination

template <int STAGE, bool MUON>
__global__ __launch_bounds__(256) void ns_thin(ThinBatch b, int from, Hyper h, const Hyper* __restrict__ hd) {
    __shared__ double red[4];
    __shared__ double gram[TINY][TINY + 1], q[TINY][TINY];
    __shared__ __attribute__((aligned(16))) float tile[TINY][THIN_TILE + 4];        // ds_read_b128 of 16 rows covers all 64 banks
    const ThinItem s = b.item[find_item(b, blockIdx.x)];
    const int tid = threadIdx.x, gi = tid >> 4, gj = tid & 15;
    const unsigned part = blockIdx.x - s.first, groups = thin_groups(s.n), cols = thin_columns(s.n);
    const size_t pitch = pad64(s.n);
    float* const x = b.x + s.x;
    double inv = 0.0;
    if (STAGE == THIN_FIRST) {
        double sum = 0.0;
        for (unsigned i = tid; i < s.parts; i += 256) sum += b.partial[s.part + i];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        if ((tid & 63) == 0) red[tid >> 6] = sum;
        __syncthreads();
        const double norm = sqrt((red[0] + red[1]) + (red[2] + red[3]));
        inv = 1.0 / (norm <= b.eps ? b.eps : norm);      // (a NaN norm stays)
    } else {
        const double* const in = b.gram[from] + (size_t)s.first * 256 + tid;
        double v = 0.0;
#pragma unroll 8
        for (unsigned g = 0; g < groups; ++g) v += in[(size_t)g * 256];
        gram[gi][gj] = v;
        __syncthreads();
        double sq = 0.0;
#pragma unroll
        for (int y = 0; y < TINY; ++y) sq = fma(gram[gi][y], gram[y][gj], sq);
        q[gi][gj] = fma(b.c, sq, fma(b.b, v, gi == gj ? b.a : 0.0));
        __syncthreads();
    }
    const float mu = MUON ? (hd ? hd->mom[s.group] : h.mom[s.group]) : 0.f;
    const bool nest = MUON && b.nesterov;
    float keep = 1.f, rate = 0.f;
    if (MUON && STAGE == THIN_LAST) {
        const float lr = hd ? hd->lr[s.group] : h.lr[s.group], wd = hd ? hd->wd[s.group] : h.wd[s.group];
        keep = 1.f - lr * wd;
        rate = lr * s.factor;
    }
    double acc = 0.0;
    const unsigned end = part * cols + cols < (unsigned)s.n ? part * cols + cols : (unsigned)s.n;
#pragma unroll 1
    for (unsigned c0 = part * cols; c0 < end; c0 += THIN_TILE) {
        const unsigned col = c0 + tid;
        const bool in = col < end;
        float v[TINY];
#pragma unroll
        for (int r = 0; r < TINY; ++r) v[r] = 0.f;
        if (in) {                                        // all loads first
#pragma unroll
            for (int r = 0; r < TINY; ++r) {
                if (r >= s.m) continue;
                if (STAGE != THIN_FIRST) {
                    v[r] = x[r * pitch + col];
                    continue;
                }
                const long off = (long)r * s.si + (long)col * s.sj;
                const float g = !MUON || nest ? (s.dtype ? bf16_to_f32(static_cast<const unsigned short*>(s.src)[off]) : static_cast<const float*>(s.src)[off]) : 0.f;
                const float m = MUON ? s.mom[off] : 0.f;             // already advanced
                v[r] = !MUON ? g : nest ? fmaf(mu, m, g) : m;
            }
        }
        if (STAGE == THIN_FIRST) {
#pragma unroll
            for (int r = 0; r < TINY; ++r)
                if (in && r < s.m) v[r] = (float)((double)v[r] * inv);
        } else {
            double w[TINY];
#pragma unroll
            for (int r = 0; r < TINY; ++r) {
                w[r] = 0.0;
                if (r >= s.m) continue;
#pragma unroll
                for (int k = 0; k < TINY; ++k) w[r] = fma(q[r][k], (double)v[k], w[r]);
            }
#pragma unroll
            for (int r = 0; r < TINY; ++r) v[r] = in ? (float)w[r] : 0.f;
        }
        if (STAGE == THIN_LAST) {
            if (!in) continue;
#pragma unroll
            for (int r = 0; r < TINY; ++r) {
                if (r >= s.m) continue;
                const long off = (long)r * s.di + (long)col * s.dj;
                if (MUON) {
                    float* const p = static_cast<float*>(s.dst) + off;
                    *p = fmaf(-rate, v[r], *p * keep);
                } else if (s.dtype) {
                    static_cast<unsigned short*>(s.dst)[off] = f32_to_bf16(v[r]);
                } else {
                    static_cast<float*>(s.dst)[off] = v[r];
                }
            }
        } else {
#pragma unroll
            for (int r = 0; r < TINY; ++r) {
                if (in && r < s.m) x[r * pitch + col] = v[r];
                tile[r][tid] = v[r];
            }
            __syncthreads();
            if (gi < s.m && gj < s.m)
                for (int k = 0; k < THIN_TILE; k += 4) {
                    const float4 l = *reinterpret_cast<const float4*>(&tile[gi][k]), r = *reinterpret_cast<const float4*>(&tile[gj][k]);
                    acc = fma((double)l.x, (double)r.x, acc);
                    acc = fma((double)l.y, (double)r.y, acc);
                    acc = fma((double)l.z, (double)r.z, acc);
                    acc = fma((double)l.w, (double)r.w, acc);
                }
            __syncthreads();
        }
    }
    if (STAGE != THIN_LAST) b.gram[STAGE == THIN_FIRST ? from : 1 - from][(size_t)(s.first + part) * 256 + tid] = acc;
}

// ------------------------------------------------------------------------------------------------ host side
// Largest value of |f| on [0, s] for the polynomials of the iteration, and the power-of-two scale that keeps such entries below 2^15
// (fp16 ends at 65504; a matrix's entries are bounded by its spectral norm).
struct Bounds {
    double a, b, c;
    static float scale_for(double bound) {
        int e;
        std::frexp(32768.0 / bound, &e);                 // 32768 / bound in [2^(e-1), 2^e)
        return (float)std::ldexp(1.0, e - 1);
    }
    double p(double s) const { return std::fabs(s * (a + s * s * (b + s * s * c))); }
    double q(double s) const { return std::fabs(a + s * s * (b + s * s * c)); }
    double r(double s) const { return std::fabs(s * s * (b + s * s * c)); }
    double max_r(double s) const {
        double v = std::fmax(r(s), 1e-6);
        if (c != 0.0) {
            const double y = -b / (2.0 * c);
            if (y > 0.0 && y < s * s) v = std::fmax(v, r(std::sqrt(y)));
        }
        return v;
    }
    double max_p(double s) const {
        double v = p(s);
        // p' = a + 3 b y + 5 c y^2, y = s^2
        double y[2];
        int k = 0;
        if (c != 0.0) {
            const double d = 9.0 * b * b - 20.0 * a * c;
            if (d >= 0.0) {
                y[k++] = (-3.0 * b + std::sqrt(d)) / (10.0 * c);
                y[k++] = (-3.0 * b - std::sqrt(d)) / (10.0 * c);
            }
        } else if (b != 0.0) {
            y[k++] = -a / (3.0 * b);
        }
        while (k-- > 0)
            if (y[k] > 0.0 && y[k] < s * s) v = std::fmax(v, p(std::sqrt(y[k])));
        return v;
    }
    double max_q(double s) const {
        double v = std::fmax(q(0.0), q(s));
        if (c != 0.0) {
            const double y = -b / (2.0 * c);
            if (y > 0.0 && y < s * s) v = std::fmax(v, q(std::sqrt(y)));
        }
        return v;
    }
};
constexpr double SLACK = 1.0 + 1e-5;                     // what rounding may add to a bound
constexpr double MAX_BOUND = 4096.0;                     // coefficients whose iterates grow beyond this are refused

// Steps between Gram products: one by one for matrices of nearly square shape and for small ones, else 2, 1, 2, 1, ... (see the head
// of this file)
int segment_length(bool wide, int index, int left) { return wide && (index & 1) == 0 && left >= 2 ? 2 : 1; }
bool is_wide(int m, int n) { return n / 2 >= m; }
// `span`: bytes from the first to behind the last element; small_matrix addresses with 32 bits
Class class_of(int rows, int cols, size_t span) {
    const int m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
    if (span < ((size_t)1 << 31)) {
        if (m <= 32 && n <= 2304) return n <= 256 ? SMALL_1_1 : n <= 768 ? SMALL_1_3 : SMALL_1_9;
        if (m <= 64 && n <= 768) return n <= 256 ? SMALL_2_1 : SMALL_2_3;
    }
    if (m <= TINY) return THIN;
    return is_wide(m, n) ? WIDE_MATRIX : SQUARE;
}
size_t span_of(const segmi_ns_matrix& a) {
    constexpr size_t FAR = (size_t)1 << 62;              // a negative stride, or no sum of 64 bits: not for 32-bit offsets
    const auto end = [&](long rs, long cs) {
        if (rs < 0 || cs < 0 || (double)(a.rows - 1) * (double)rs + (double)(a.cols - 1) * (double)cs > 1e15) return FAR;
        return ((size_t)(a.rows - 1) * rs + (size_t)(a.cols - 1) * cs + 1) * (a.dtype ? 2 : 4);
    };
    return std::max(end(a.src_rs, a.src_cs), end(a.dst_rs, a.dst_cs));
}
size_t span_of(const segmi_muon_matrix& a) { return (size_t)a.rows * a.cols * 4; }
template <typename M>
Class class_of(const M& a) { return class_of(a.rows, a.cols, span_of(a)); }

bool iteration_ok(const Bounds& f, int steps) {
    double s = SLACK;
    for (int left = steps, seg = 0; left > 0; ++seg) {
        double P = 1.0;
        for (int i = segment_length(true, seg, left); i > 0; --i, --left) {
            P *= f.max_q(s) * SLACK;
            if (!(f.max_r(s) < MAX_BOUND)) return false;
            s = f.max_p(s) * SLACK;
            if (!(P > 1e-6 && P < MAX_BOUND && s > 1e-6 && s < MAX_BOUND)) return false;
        }
    }
    return true;
}

struct Shape {
    int m, n;                        // m <= n
    int outer, inner;                // as the source lies
};

struct Plan {
    size_t partial_at, gram_at, mats_at, bytes;
};

unsigned tiles_of(int m, int bt) { return (pad64(m) + bt - 1) / bt; }
unsigned low_tiles(int m, int bt) { const unsigned t = tiles_of(m, bt); return t * (t + 1) / 2; }
unsigned big_tiles(const Shape& s, int bt) { return tiles_of(s.m, bt) * tiles_of(s.n, bt); }

// Which tiles a launch runs on (see Tile).  128 x 128 copy half as much per product, 64 x 64 spread better: in us, WIDE / MANY, products of
// m x m matrices with 408 tiles of 128 (3 of 2048 x 2048) 103 / 122, 288 (8 of 1024) 55 / 54, 257 (fifty filters) 34 / 31; with P 392 tiles
// 27.7 / 29.7, 288 tiles 48 / 46.  Fewer 64s than CUs run one to a CU with a longer pipeline: 1024 x 1024 (136) 12.2 instead of 14.1.
enum Config { WIDE, MANY, FEW };
int tile_of(Config c) { return c == WIDE ? 128 : 64; }
template <typename F>
Config config_of(const Shape* s, int count, F tiles) {
    size_t wide = 0, many = 0;
    for (int i = 0; i < count; ++i) {
        wide += tiles(s[i], 128);
        many += tiles(s[i], 64);
    }
    return 4 * wide >= 5 * SEGMI_NUM_CU ? WIDE : many > SEGMI_NUM_CU ? MANY : FEW;
}
#define NS_LAUNCH(config, kernel, grid, ...)                                                                               \
    do {                                                                                                                   \
        if ((config) == WIDE) hipLaunchKernelGGL((kernel(Wide)), dim3(grid), dim3(256), 0, st, __VA_ARGS__);               \
        else if ((config) == MANY) hipLaunchKernelGGL((kernel(Many)), dim3(grid), dim3(256), 0, st, __VA_ARGS__);          \
        else hipLaunchKernelGGL((kernel(Few)), dim3(grid), dim3(256), 0, st, __VA_ARGS__);                                 \
    } while (0)
#define NS_GRAM(C) ns_gram<C>
#define NS_POLY(C) ns_square_product<C, true>
#define NS_SQUARE(C) ns_square_product<C, false>
#define NS_APPLY(C) ns_apply<C>
#define NS_FINISH(C) ns_finish<C, MUON>

struct GramPlan {
    Config config;
    int bt;
    unsigned run;
};
GramPlan gram_plan(const Shape* s, int count) {
    double work128 = 0.0, work64 = 0.0;
    for (int i = 0; i < count; ++i) {
        work128 += (double)low_tiles(s[i].m, 128) * (pad64(s[i].n) / LINE_K);
        work64 += (double)low_tiles(s[i].m, 64) * (pad64(s[i].n) / LINE_K);
    }
    GramPlan g;
    g.config = work128 / 16.0 >= 512.0 ? WIDE : work64 / 16.0 > SEGMI_NUM_CU ? MANY : FEW;
    g.bt = tile_of(g.config);
    if (g.config != WIDE) {
        const double run = std::ceil(work64 / 1024.0 / 4.0) * 4.0;
        g.run = run < 16.0 ? 16u : (unsigned)run;        // whole steps of a tile
        return g;
    }
    // All workgroups are on the card at once, so the CU with one more of them than the others decides: the shortest run that leaves at most
    // two a CU, or three where that is less work for the fullest one.  (Runs of a 512th of all lines: 2048 x 36864 in 544 workgroups 552 us, in
    // 680 477; fifty filters of a network 123 -> 108 us.)
    unsigned longest = 16;
    for (int i = 0; i < count; ++i) longest = std::max(longest, pad64(s[i].n) / LINE_K);
    const auto groups = [&](unsigned run) {
        size_t w = 0;
        for (int i = 0; i < count; ++i) w += (size_t)low_tiles(s[i].m, 128) * segmi_cdiv(pad64(s[i].n) / LINE_K, run);
        return w;
    };
    double best = 0.0;
    for (unsigned per = 2; per <= 3; ++per) {
        unsigned lo = 4, hi = longest / 4;               // the shortest run in units of four lines, if any
        while (lo < hi) {
            const unsigned mid = (lo + hi) / 2;
            if (groups(4 * mid) <= (size_t)per * SEGMI_NUM_CU) hi = mid;
            else lo = mid + 1;
        }
        const double cost = 4.0 * lo * (double)segmi_cdiv((long)groups(4 * lo), SEGMI_NUM_CU);
        if (best == 0.0 || cost < best) {
            best = cost;
            g.run = 4 * lo;
        }
    }
    return g;
}

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

Plan plan_batch(const Shape* s, int count) {
    Plan p;
    size_t parts = 0, slots = 0, mats = 0;
    const GramPlan g = gram_plan(s, count);
    for (int i = 0; i < count; ++i) {
        const unsigned lines = pad64(s[i].n) / LINE_K;
        parts += (size_t)segmi_cdiv(s[i].outer, 64) * segmi_cdiv(s[i].inner, 256);
        slots += (size_t)low_tiles(s[i].m, g.bt) * segmi_cdiv(lines, g.run);
        mats += 3 * big_bytes(s[i].m, s[i].n) + 5 * square_bytes(s[i].m);
    }
    p.partial_at = 0;
    p.gram_at = align256(parts * sizeof(double));
    p.mats_at = p.gram_at + align256(slots * g.bt * g.bt * sizeof(float));
    p.bytes = p.mats_at + mats;
    return p;
}

// runs the whole iteration of up to BATCH matrices; `src` and `dst` carry the callers' pointers, the rest is filled in here
template <bool MUON>
int run_batch(bool wide, const Shape* shapes, SourceBatch& src, TargetBatch& dst, int count, const Bounds& f, int steps, char* ws,
              const Hyper& h, const Hyper* hd, hipStream_t st) {
    const Plan plan = plan_batch(shapes, count);
    const GramPlan gp = gram_plan(shapes, count);
    const Config c_sq = config_of(shapes, count, [](const Shape& x, int bt) { return low_tiles(x.m, bt); });
    const Config c_big = config_of(shapes, count, big_tiles);
    const int bt_sq = tile_of(c_sq), bt_big = tile_of(c_big);
    Batch sq, big;
    GramBatch gram;
    src.ws = dst.ws = sq.ws = big.ws = gram.ws = ws + plan.mats_at;
    src.partial = reinterpret_cast<double*>(ws + plan.partial_at);
    gram.partial = reinterpret_cast<float*>(ws + plan.gram_at);
    src.count = dst.count = sq.count = big.count = gram.count = count;

    unsigned g_sum = 0, g_norm = 0, g_sq = 0, g_gram = 0, g_red = 0, g_big = 0, parts = 0, slots = 0;
    size_t base = 0;
    for (int i = 0; i < count; ++i) {
        const Shape& s = shapes[i];
        const unsigned lines = pad64(s.n) / LINE_K, low = low_tiles(s.m, gp.bt), splits = segmi_cdiv(lines, gp.run);
        const unsigned b256 = (unsigned)(base / 256);
        const unsigned units = segmi_cdiv(s.outer, 64) * segmi_cdiv(s.inner, 256);
        src.item[i].base = dst.item[i].base = b256;
        src.item[i].first = g_sum;
        src.item[i].part = parts;
        src.item[i].parts = units;
        sq.item[i] = Item{g_sq, s.m, s.n, b256};
        gram.item[i] = GramItem{g_gram, slots, s.m, s.n, b256, low, splits, gp.run};
        big.item[i] = Item{g_big, s.m, s.n, b256};
        dst.item[i].first = g_big;
        g_sum += units;
        parts += units;
        g_norm += (pad64(s.outer) / 64) * (pad64(s.inner) / 64);
        g_sq += low_tiles(s.m, bt_sq);
        g_gram += low * splits;
        g_red += low * (gp.bt / 32) * (gp.bt / 32);
        slots += low * splits;
        g_big += big_tiles(s, bt_big);
        base += 3 * big_bytes(s.m, s.n) + 5 * square_bytes(s.m);
    }
    hipLaunchKernelGGL((ns_sum_squares<MUON>), dim3(g_sum), dim3(256), 0, st, src, h, hd);
    unsigned at = 0;
    for (int i = 0; i < count; ++i) {
        src.item[i].first = at;
        at += (pad64(shapes[i].outer) / 64) * (pad64(shapes[i].inner) / 64);
    }
    double s = SLACK;                                    // bound of X's singular values
    double sx = Bounds::scale_for(s);
    src.scale = (float)sx;
    hipLaunchKernelGGL((ns_normalise<MUON>), dim3(g_norm), dim3(256), 0, st, src, h, hd);

    int tin = T0;
    for (int left = steps, seg = 0; left > 0; ++seg) {
        const int len = segment_length(wide, seg, left);
        double sa = Bounds::scale_for(s * s);
        gram.scale = (float)(sa / (sx * sx));
        NS_LAUNCH(gp.config, NS_GRAM, g_gram, gram);
        if (gp.bt == 128) hipLaunchKernelGGL((ns_gram_reduce<128>), dim3(g_red), dim3(256), 0, st, gram);
        else hipLaunchKernelGGL((ns_gram_reduce<64>), dim3(g_red), dim3(256), 0, st, gram);
        const auto product = [&](int l, int r, int out, double so, double sl, double sr) { return Product{l, r, out, (float)(so / (sl * sr)), 0.f, 0.f}; };
        const auto square = [&](int out, double so, double ident) {      // out = ident I + b A + c A^2
            const Product pr{A, A, out, (float)(f.c * so / (sa * sa)), (float)(ident * so), (float)(f.b * so / sa)};
            NS_LAUNCH(c_sq, NS_POLY, g_sq, sq, pr);
        };
        const double s1 = f.max_p(s) * SLACK;            // bound after the segment's first step
        double sp, alpha = 0.0;
        int p = P0;
        if (len == 1) {
            sp = Bounds::scale_for(f.max_r(s) * SLACK);
            square(P0, sp, 0.0);
            alpha = f.a;
            s = s1;
        } else {
            // P0 = Q(A), W = P0 A, A <- W P0, Q = Q(A), P1 = P0 Q
            const double bq0 = f.max_q(s) * SLACK, bq1 = f.max_q(s1) * SLACK;
            const double sq0 = Bounds::scale_for(bq0), sw = Bounds::scale_for(s * s1), san = Bounds::scale_for(s1 * s1), sq1 = Bounds::scale_for(bq1);
            square(P0, sq0, f.a);
            NS_LAUNCH(c_sq, NS_SQUARE, g_sq, sq, product(P0, A, W, sw, sq0, sa));
            NS_LAUNCH(c_sq, NS_SQUARE, g_sq, sq, product(W, P0, A, san, sw, sq0));
            sa = san;
            square(Q, sq1, f.a);
            sp = Bounds::scale_for(bq0 * bq1);
            NS_LAUNCH(c_sq, NS_SQUARE, g_sq, sq, product(P0, Q, P1, sp, sq0, sq1));
            p = P1;
            s = f.max_p(s1) * SLACK;
        }
        left -= len;
        if (left > 0) {
            const double nsx = Bounds::scale_for(s);
            const int tout = tin == T0 ? T1 : T0;
            NS_LAUNCH(c_big, NS_APPLY, g_big, big, p, tin, tout, (float)(nsx / (sp * sx)), (float)(alpha * nsx / sx));
            tin = tout;
            sx = nsx;
        } else {
            dst.p = p;
            dst.tin = tin;
            dst.scale = (float)(1.0 / (sp * sx));
            dst.alpha = (float)(alpha / sx);
            NS_LAUNCH(c_big, NS_FINISH, g_big, dst, h, hd);
        }
    }
    return segmi_launch_status();
}

struct ThinPlan {
    size_t gram_at, x_at, bytes;
    unsigned groups;
};
ThinPlan thin_plan(const Shape* s, int count) {
    ThinPlan p{};
    size_t parts = 0, x = 0;
    for (int i = 0; i < count; ++i) {
        parts += (size_t)segmi_cdiv(s[i].outer, 64) * segmi_cdiv(s[i].inner, 256);
        p.groups += thin_groups(s[i].n);
        x += (size_t)s[i].m * pad64(s[i].n);
    }
    p.gram_at = align256(parts * sizeof(double));
    p.x_at = p.gram_at + 2 * (size_t)p.groups * 256 * sizeof(double);
    p.bytes = p.x_at + x * sizeof(float);
    return p;
}

// `src` and `dst` carry the callers' pointers, as in run_batch
template <bool MUON>
int run_thin(const Shape* shapes, SourceBatch& src, const TargetBatch& dst, int count, const Bounds& f, int steps, char* ws, const Hyper& h,
             const Hyper* hd, hipStream_t st) {
    const ThinPlan plan = thin_plan(shapes, count);
    src.ws = ws;
    src.partial = reinterpret_cast<double*>(ws);
    src.count = count;
    ThinBatch b{};
    b.x = reinterpret_cast<float*>(ws + plan.x_at);
    b.partial = src.partial;
    b.gram[0] = reinterpret_cast<double*>(ws + plan.gram_at);
    b.gram[1] = b.gram[0] + (size_t)plan.groups * 256;
    b.a = f.a;
    b.b = f.b;
    b.c = f.c;
    b.eps = src.eps;
    b.count = count;
    b.nesterov = src.nesterov;
    unsigned g_sum = 0, grid = 0;
    size_t x = 0;
    for (int i = 0; i < count; ++i) {
        const Shape& s = shapes[i];
        Source& o = src.item[i];
        const Target& t = dst.item[i];
        o.first = o.part = g_sum;
        o.parts = segmi_cdiv(s.outer, 64) * segmi_cdiv(s.inner, 256);
        b.item[i] = ThinItem{o.src, t.dst, o.mom, o.inner_is_n ? o.so : o.si, o.inner_is_n ? o.si : o.so, t.si, t.sj, x, grid, o.part, o.parts,
                             s.m, s.n, t.factor, (short)t.dtype, (short)t.group};
        g_sum += o.parts;
        grid += thin_groups(s.n);
        x += (size_t)s.m * pad64(s.n);
    }
    hipLaunchKernelGGL((ns_sum_squares<MUON>), dim3(g_sum), dim3(256), 0, st, src, h, hd);
    hipLaunchKernelGGL((ns_thin<THIN_FIRST, MUON>), dim3(grid), dim3(256), 0, st, b, 0, h, hd);
    for (int i = 0; i + 1 < steps; ++i) hipLaunchKernelGGL((ns_thin<THIN_NEXT, MUON>), dim3(grid), dim3(256), 0, st, b, i & 1, h, hd);
    hipLaunchKernelGGL((ns_thin<THIN_LAST, MUON>), dim3(grid), dim3(256), 0, st, b, (steps - 1) & 1, h, hd);
    return segmi_launch_status();
}

// `b` carries the callers' pointers; the steps' scales are filled in here
template <bool MUON>
int run_small(SmallBatch& b, int count, const Bounds& f, int steps, const Hyper& h, const Hyper* hd, hipStream_t st) {
    double s = SLACK, sx = Bounds::scale_for(s);
    b.scale = (float)sx;
    b.steps = steps;
    for (int i = 0; i < steps; ++i) {
        const double sa = Bounds::scale_for(s * s), sq = Bounds::scale_for(std::fmax(f.max_r(s), f.max_q(s)) * SLACK);
        s = f.max_p(s) * SLACK;
        const double nsx = Bounds::scale_for(s);
        b.step[i] = SmallStep{(float)(sa / (sx * sx)), (float)(f.c * sq / (sa * sa)), (float)(f.b * sq / sa), (float)(nsx / (sq * sx)), (float)(f.a * nsx / sx), (float)(f.a * sq)};
        sx = nsx;
    }
    b.unscale = (float)(1.0 / sx);
    int cls = b.item[0].cls;
    for (int i = 1; i < count; ++i)
        if (b.item[i].cls != cls) cls = CLASSES;
    const dim3 grid(count), threads(512);
    switch (cls) {
        case SMALL_1_1: hipLaunchKernelGGL((ns_small<SMALL_1_1, MUON>), grid, threads, 0, st, b, h, hd); break;
        case SMALL_1_3: hipLaunchKernelGGL((ns_small<SMALL_1_3, MUON>), grid, threads, 0, st, b, h, hd); break;
        case SMALL_1_9: hipLaunchKernelGGL((ns_small<SMALL_1_9, MUON>), grid, threads, 0, st, b, h, hd); break;
        case SMALL_2_1: hipLaunchKernelGGL((ns_small<SMALL_2_1, MUON>), grid, threads, 0, st, b, h, hd); break;
        case SMALL_2_3: hipLaunchKernelGGL((ns_small<SMALL_2_3, MUON>), grid, threads, 0, st, b, h, hd); break;
        default: hipLaunchKernelGGL((ns_small<CLASSES, MUON>), grid, threads, 0, st, b, h, hd); break;
    }
    return segmi_launch_status();
}

// Small matrices take one CU each for as long as a third of a network's whole step, so next to others they run (and thin ones with them) on a stream of
// their own, which waits for the caller's and is waited for by it (a whole Muon step of PSPNet's filters 1777 -> 1728 us, of UNet's 1194 -> 1130;
// five small ones beside 150 x 257 and 333 x 65 242 -> 210 us for a call alone.  The two waits cost the host 25 us.)
// Inside a capture everything stays on the captured stream: this one may be at work for another thread.
class Aside {
    static constexpr int DEVICES = 64;
    struct Side {
        hipStream_t stream = nullptr;
        hipEvent_t event = nullptr;      // recorded and waited for under the lock: a wait keeps the record it saw
    };
    static std::mutex& lock() { static std::mutex m; return m; }
    static Side* sides() { static Side s[DEVICES]; return s; }
    hipStream_t caller;
    Side* side = nullptr;

    static bool pass(hipStream_t from, hipEvent_t event, hipStream_t to) {
        return hipEventRecord(event, from) == hipSuccess && hipStreamWaitEvent(to, event, 0) == hipSuccess;
    }

public:
    Aside(hipStream_t st, bool wanted) : caller(st) {
        int dev = -1;
        hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
        if (!wanted) return;
        if (hipStreamIsCapturing(st, &capture) != hipSuccess || capture != hipStreamCaptureStatusNone || hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= DEVICES) {
            (void)hipGetLastError();
            return;
        }
        const std::lock_guard<std::mutex> hold(lock());
        Side& s = sides()[dev];
        if (!s.event && hipEventCreateWithFlags(&s.event, hipEventDisableTiming) != hipSuccess) s.event = nullptr;
        if (s.event && !s.stream && hipStreamCreateWithFlags(&s.stream, hipStreamNonBlocking) != hipSuccess) s.stream = nullptr;
        if (s.stream && pass(st, s.event, s.stream)) side = &s;
        else (void)hipGetLastError();                    // then everything runs on the caller's
    }
    hipStream_t stream() const { return side ? side->stream : caller; }
    // the caller's stream goes on behind both
    int join(int rc) {
        if (!side) return rc;
        const std::lock_guard<std::mutex> hold(lock());
        const bool ok = pass(side->stream, side->event, caller);
        return rc != SEGMI_OK ? rc : ok ? SEGMI_OK : SEGMI_ERR_LAUNCH;
    }
};

template <typename M>
bool mixed(const M* mats, int count) {
    int small = 0;
    for (int i = 0; i < count; ++i) small += class_of(mats[i]) < THIN;
    return small && small < count;
}

bool shape_ok(int rows, int cols) {
    return rows > 0 && cols > 0 && big_bytes(rows < cols ? rows : cols, rows < cols ? cols : rows) < ((size_t)1 << 32);
}

// `inner` = the contiguous dimension
Shape shape_of(int rows, int cols, bool cols_inner) {
    return Shape{rows <= cols ? rows : cols, rows <= cols ? cols : rows, cols_inner ? rows : cols, cols_inner ? cols : rows};
}

Shape shape_of(const segmi_ns_matrix& a) { return shape_of(a.rows, a.cols, a.src_cs == 1 || a.src_rs != 1); }

// Wide matrices next to square ones go step by step with them while a second chain of 22 launches costs more than their two additional products
// each: 150 x 257 with 512 x 2048 175 instead of 288 us, with 1024 x 2048 263 / 360, with 1024 x 4608 436 / 467, with 4 of 512 x 4608
// 441 / 455.
constexpr size_t JOIN_WORK = (size_t)1 << 32;            // sum of m^2 n

// The matrices of a call in batches of one kind (small, thin, square, wide), those with the longest sums first (what is started last should be short):
// f(class, indices, how many) in order, until it returns something other than SEGMI_OK.  Batches of one stream run one after the other and
// share their part of the workspace.
template <typename M, typename F>
int for_batches(const M* mats, int count, F f) {
    const auto side = [&](int i) { return mats[i].rows < mats[i].cols ? mats[i].rows : mats[i].cols; };
    const std::unique_ptr<int[]> order(new (std::nothrow) int[count]);      // (no exception leaves a C entry)
    if (!order) return SEGMI_ERR_BADARG;
    size_t square = 0, wide_work = 0;
    for (int i = 0; i < count; ++i) {
        const Class c = class_of(mats[i]);
        square += c == SQUARE;
        if (c == WIDE_MATRIX) wide_work += (size_t)pad64(side(i)) * pad64(side(i)) * pad64(std::max(mats[i].rows, mats[i].cols));
    }
    const bool join = square && wide_work <= JOIN_WORK;
    for (int c = SMALL_2_3; c < CLASSES; ++c) {          // SMALL_2_3 stands for all small classes
        int k = 0;
        for (int i = 0; i < count; ++i) {
            const Class own = std::max(class_of(mats[i]), SMALL_2_3);
            if ((join && own == WIDE_MATRIX ? SQUARE : own) == c) order[k++] = i;
        }
        std::sort(order.get(), order.get() + k, [&](int a, int b) { return side(a) != side(b) ? side(a) > side(b) : a < b; });
        const int most = c < THIN ? SMALL_BATCH : c == THIN ? THIN_BATCH : BATCH;
        for (int at = 0; at < k; at += most) {
            const int rc = f((Class)c, order.get() + at, k - at < most ? k - at : most);
            if (rc != SEGMI_OK) return rc;
        }
    }
    return SEGMI_OK;
}

// The workspace: `thin` bytes that the thin batches share, which may run beside the others, and `rest` that those share.
struct Need {
    size_t thin, rest;
    size_t bytes() const { return rest ? thin + rest : 0; }
};
template <typename M, typename F>
Need need_of(const M* mats, int count, F shape) {
    Need need{0, 256};                                   // (small matrices need none; 0 means refused)
    const int rc = for_batches(mats, count, [&](Class c, const int* index, int k) {
        if (c < THIN) return (int)SEGMI_OK;
        Shape s[BATCH];
        for (int i = 0; i < k; ++i) s[i] = shape(mats[index[i]]);
        if (c == THIN) need.thin = std::max(need.thin, align256(thin_plan(s, k).bytes));
        else need.rest = std::max(need.rest, plan_batch(s, k).bytes);
        return (int)SEGMI_OK;
    });
    return rc == SEGMI_OK ? need : Need{0, 0};
}
Need need_of(const segmi_ns_matrix* mats, int count) { return need_of(mats, count, [](const segmi_ns_matrix& a) { return shape_of(a); }); }
Need need_of(const segmi_muon_matrix* mats, int count) { return need_of(mats, count, [](const segmi_muon_matrix& a) { return shape_of(a.rows, a.cols, true); }); }

}  // namespace

extern "C" {

size_t segmi_ns_workspace(const segmi_ns_matrix* mats_host, int count) {
    if (!mats_host || count <= 0) return 0;
    for (int i = 0; i < count; ++i)
        if (!shape_ok(mats_host[i].rows, mats_host[i].cols)) return 0;
    return need_of(mats_host, count).bytes();
}

int segmi_ns_coefficients_ok(const double* coefficients_host, int steps) {
    if (!coefficients_host || steps < 1 || steps > SEGMI_NS_MAX_STEPS) return 0;
    return iteration_ok(Bounds{coefficients_host[0], coefficients_host[1], coefficients_host[2]}, steps) ? 1 : 0;
}

int segmi_ns_orthogonalize(const segmi_ns_matrix* mats_host, int count, const double* coefficients_host, int steps, double eps,
                           void* workspace, size_t workspace_bytes, segmi_stream_t stream) {
    if (!mats_host || count <= 0 || !(eps > 0.0) || !workspace || !segmi_ns_coefficients_ok(coefficients_host, steps)) return SEGMI_ERR_BADARG;
    for (int i = 0; i < count; ++i) {
        const segmi_ns_matrix& a = mats_host[i];
        if (!a.src || !a.dst || !shape_ok(a.rows, a.cols) || a.dtype < 0 || a.dtype > 1) return SEGMI_ERR_BADARG;
    }
    if ((size_t)workspace & 255) return SEGMI_ERR_ALIGN;
    const Need need = need_of(mats_host, count);
    if (!need.bytes() || workspace_bytes < need.bytes()) return SEGMI_ERR_WORKSPACE;
    char* const thin = static_cast<char*>(workspace);
    char* const rest = thin + need.thin;
    const Bounds f{coefficients_host[0], coefficients_host[1], coefficients_host[2]};
    Aside aside((hipStream_t)stream, mixed(mats_host, count));
    return aside.join(for_batches(mats_host, count, [&](Class cls, const int* index, int k) {
        if (cls < THIN) {
            SmallBatch b{};
            b.eps = eps;
            for (int i = 0; i < k; ++i) {
                const segmi_ns_matrix& a = mats_host[index[i]];
                const bool wide = a.rows <= a.cols;
                b.item[i] = SmallItem{a.src, a.dst, nullptr, wide ? a.src_rs : a.src_cs, wide ? a.src_cs : a.src_rs, wide ? a.dst_rs : a.dst_cs,
                                      wide ? a.dst_cs : a.dst_rs, wide ? a.rows : a.cols, wide ? a.cols : a.rows, 0.f, a.dtype, 0, class_of(a), (unsigned)span_of(a), (unsigned)span_of(a)};
            }
            return run_small<false>(b, k, f, steps, Hyper{}, nullptr, aside.stream());
        }
        Shape shapes[BATCH];
        SourceBatch src{};
        TargetBatch dst{};
        src.eps = eps;
        for (int i = 0; i < k; ++i) {
            const segmi_ns_matrix& a = mats_host[index[i]];
            const Shape s = shapes[i] = shape_of(a);
            const bool cols_inner = a.src_cs == 1 || a.src_rs != 1, wide = a.rows <= a.cols;
            Source& o = src.item[i];
            o.src = a.src;
            o.so = cols_inner ? a.src_rs : a.src_cs;
            o.si = cols_inner ? a.src_cs : a.src_rs;
            o.outer = s.outer;
            o.inner = s.inner;
            o.dtype = (signed char)a.dtype;
            o.inner_is_n = cols_inner == wide;
            Target& t = dst.item[i];
            t.dst = a.dst;
            t.si = wide ? a.dst_rs : a.dst_cs;
            t.sj = wide ? a.dst_cs : a.dst_rs;
            t.m = s.m;
            t.n = s.n;
            t.dtype = a.dtype;
            t.turned = t.si == 1 && t.sj != 1;
        }
        if (cls == THIN) return run_thin<false>(shapes, src, dst, k, f, steps, thin, Hyper{}, nullptr, aside.stream());
        return run_batch<false>(cls == WIDE_MATRIX, shapes, src, dst, k, f, steps, rest, Hyper{}, nullptr, (hipStream_t)stream);
    }));
}

size_t segmi_muon_workspace(const segmi_muon_matrix* mats_host, int count) {
    if (!mats_host || count <= 0) return 0;
    for (int i = 0; i < count; ++i)
        if (!shape_ok(mats_host[i].rows, mats_host[i].cols)) return 0;
    return need_of(mats_host, count).bytes();
}

int segmi_muon_step(const segmi_muon_matrix* mats_host, int count, const float* lr_host, const float* weight_decay_host,
                    const float* momentum_host, int ngroups, const float* hyper_dev, int nesterov, const double* coefficients_host, int steps,
                    double eps, void* workspace, size_t workspace_bytes, segmi_stream_t stream) {
    if (!mats_host || count <= 0 || !(eps > 0.0) || !workspace || !segmi_ns_coefficients_ok(coefficients_host, steps)) return SEGMI_ERR_BADARG;
    if (!hyper_dev && (!lr_host || !weight_decay_host || !momentum_host)) return SEGMI_ERR_BADARG;
    if (ngroups <= 0 || ngroups > MAX_GROUPS) return SEGMI_ERR_BADARG;
    for (int i = 0; i < count; ++i) {
        const segmi_muon_matrix& a = mats_host[i];
        if (!a.param || !a.grad || !a.momentum || !shape_ok(a.rows, a.cols) || a.group < 0 || a.group >= ngroups) return SEGMI_ERR_BADARG;
    }
    if ((size_t)workspace & 255) return SEGMI_ERR_ALIGN;
    const Need need = need_of(mats_host, count);
    if (!need.bytes() || workspace_bytes < need.bytes()) return SEGMI_ERR_WORKSPACE;
    char* const thin = static_cast<char*>(workspace);
    char* const rest = thin + need.thin;
    const Bounds f{coefficients_host[0], coefficients_host[1], coefficients_host[2]};
    Hyper h{};
    if (!hyper_dev)
        for (int i = 0; i < ngroups; ++i) {
            h.lr[i] = lr_host[i];
            h.wd[i] = weight_decay_host[i];
            h.mom[i] = momentum_host[i];
        }
    Aside aside((hipStream_t)stream, mixed(mats_host, count));
    return aside.join(for_batches(mats_host, count, [&](Class cls, const int* index, int k) {
        if (cls < THIN) {
            SmallBatch b{};
            b.eps = eps;
            b.nesterov = nesterov;
            for (int i = 0; i < k; ++i) {
                const segmi_muon_matrix& a = mats_host[index[i]];
                const bool wide = a.rows <= a.cols;
                const long si = wide ? a.cols : 1, sj = wide ? 1 : a.cols;
                b.item[i] = SmallItem{a.grad, a.param, a.momentum, si, sj, si, sj, wide ? a.rows : a.cols, wide ? a.cols : a.rows, a.factor, 0, a.group,
                                      class_of(a), (unsigned)span_of(a), (unsigned)span_of(a)};
            }
            return run_small<true>(b, k, f, steps, h, reinterpret_cast<const Hyper*>(hyper_dev), aside.stream());
        }
        Shape shapes[BATCH];
        SourceBatch src{};
        TargetBatch dst{};
        src.eps = eps;
        src.nesterov = nesterov;
        for (int i = 0; i < k; ++i) {
            const segmi_muon_matrix& a = mats_host[index[i]];
            const Shape s = shapes[i] = shape_of(a.rows, a.cols, true);
            const bool wide = a.rows <= a.cols;
            Source& o = src.item[i];
            o.src = a.grad;
            o.mom = a.momentum;
            o.so = a.cols;
            o.si = 1;
            o.outer = s.outer;
            o.inner = s.inner;
            o.inner_is_n = wide;
            o.group = (signed char)a.group;
            Target& t = dst.item[i];
            t.dst = a.param;
            t.si = wide ? a.cols : 1;
            t.sj = wide ? 1 : a.cols;
            t.m = s.m;
            t.n = s.n;
            t.factor = a.factor;
            t.group = a.group;
            t.turned = !wide;
        }
        if (cls == THIN)
            return run_thin<true>(shapes, src, dst, k, f, steps, thin, h, reinterpret_cast<const Hyper*>(hyper_dev), aside.stream());
        return run_batch<true>(cls == WIDE_MATRIX, shapes, src, dst, k, f, steps, rest, h, reinterpret_cast<const Hyper*>(hyper_dev), (hipStream_t)stream);
    }));
}

}  // extern "C"
