// Newton-Schulz orthogonalisation of many matrices at once, and the Muon update.
//
//   A = Y Y^T,  B = b A + c A A,  Y <- a Y + B Y          (Y is [m, n], m <= n)
//
// Numbers.  Y, A and B live between launches as sums of two fp16 planes, value * 2^e = hi + lo,
// which together carry 22 bits or more: hi is the value rounded to 11 bits and lo its remainder
// rounded to 11 more.  The exponents e are powers of two taken from the range that the polynomial
// can reach, so hi neither overflows nor loses bits to subnormals where it matters.  A product
// multiplies the hi planes alone ("narrow": relative 2^-12 per factor) or adds hi*lo + lo*hi
// ("wide": 2^-22), always with fp32 accumulators.  The diagonals of A and B never enter a product:
// with A = D + O and B = E + P (D, E diagonal, fp32)
//
//     (A A)_ij = (O O)_ij + (d_i + d_j) O_ij + [i = j] d_i^2,     (a Y + B Y)_i = (a + e_i) Y_i + (P Y)_i
//
// Late in the iteration A is close to the identity, so the large part of both products is exact
// and only the small off-diagonal part carries the narrow factors' rounding (measured against 64
// bits on [512, 4608]: 1e-4 of the result's norm; with the diagonals left in, 3e-3).
#include <algorithm>
#include <cmath>
#include <limits>
#include <stdexcept>
#include <string>
#include <tuple>
#include <type_traits>
#include <utility>

#include "dml_common.h"
#include "dml_newton_schulz.h"

namespace dml {
namespace {

typedef _Float16 f16_t;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((address_space(3))) void* lds_ptr;
typedef const __attribute__((address_space(1))) void* global_ptr;
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;

constexpr int kMaxProblems = 24;        // per launch: the table has to fit the kernel arguments
constexpr int kPad = 64;                // planes are zero-padded to multiples of this
constexpr int kMaxPartials = 1024;      // blocks (partial sums of squares) per matrix
constexpr int kMaxSteps = 64;
constexpr int kCus = 256;

// Products: A = Y Y^T; P = b A + c A A, its diagonal with the a; Y <- P Y.
enum NsPhase { GRAM, SQUARE, APPLY };

struct NsProblem {
    int rows, cols, m, n, mp, np, batch;
    int trans;                          // Y is the transpose of the matrix in memory (rows > cols)
    long long src, ld, stride;
    long long out, out_ld, out_stride;
    long long ws, ws_stride;            // bytes
    int part, parts;                    // partial sums: first index, count per matrix
    float lr;
    int tiles;                          // of one matrix, in the launch at hand
    int begin;                          // first tile of this entry, counted over the batch
    int splits;                         // blocks that share a tile's summed index (1: none)
    int slab;                           // first of their partial tiles in the slab
};
struct NsTable {
    int count;
    int whole;                          // blocks that own a whole tile; the split ones follow
    int first[kMaxProblems + 1];        // first block of each problem, in the launch at hand
    NsProblem p[kMaxProblems];
};
static_assert(sizeof(NsTable) <= 3900, "kernel arguments");

// Row pitch of a plane: an odd number of 128-byte lines, so that the rows of a tile spread over the
// memory channels (with a power of two they all meet in a few).
__host__ __device__ inline int ns_pitch(int padded) { return (padded / 64) % 2 ? padded : padded + 64; }

// Workspace of one matrix: Y twice (this step's and the next one's) as [mp, np] planes, the diagonals of
// A and P and their off-diagonal parts as [mp, mp] planes.  The hi plane comes first.
enum NsSquare { MAT_A = 0, MAT_P = 1, kSquares = 2 };
struct NsPlanes {
    uint16_t *y, *squares;
    float* diagonals;
    size_t yplane, aplane;              // elements of a plane
    int yld, ald, mp;                   // pitches
    __device__ __forceinline__ uint16_t* square(int i) const { return squares + (size_t)i * 2 * aplane; }
    __device__ __forceinline__ float* diagonal(int i) const { return diagonals + i * mp; }
};
inline size_t ns_matrix_bytes(int mp, int np) {
    return 8 * (size_t)mp * ns_pitch(np) + kSquares * (4 * (size_t)mp + 4 * (size_t)mp * ns_pitch(mp));
}
__device__ __forceinline__ NsPlanes ns_planes(const NsProblem& q, char* ws, int b, int buffer) {
    NsPlanes r;
    uint16_t* base = (uint16_t*)(ws + q.ws + (size_t)b * q.ws_stride);
    r.mp = q.mp;
    r.yld = ns_pitch(q.np);
    r.ald = ns_pitch(q.mp);
    r.yplane = (size_t)q.mp * r.yld;
    r.aplane = (size_t)q.mp * r.ald;
    r.y = base + (size_t)buffer * 2 * r.yplane;
    r.diagonals = (float*)(base + 4 * r.yplane);
    r.squares = (uint16_t*)(r.diagonals + kSquares * q.mp);
    return r;
}

// The problem a block works on: one load per lane and a vote instead of a chain of dependent loads.
static_assert(kMaxProblems < 64, "one lane per problem");
__device__ __forceinline__ int ns_find(const NsTable& t, int block) {
    const int lane = threadIdx.x & 63;
    const bool past = lane < t.count && block >= t.first[lane];
    return __popcll(__ballot(past)) - 1;
}

__device__ __forceinline__ uint16_t f16_bits(f16_t v) { return __builtin_bit_cast(uint16_t, v); }
__device__ __forceinline__ float f16_value(uint16_t v) { return (float)__builtin_bit_cast(f16_t, v); }
__device__ __forceinline__ void split_f16(float v, uint16_t& hi, uint16_t& lo) {
    const f16_t h = (f16_t)v;
    hi = f16_bits(h);
    lo = f16_bits((f16_t)(v - (float)h));
}

__device__ __forceinline__ float ns_elem(float v) { return v; }
__device__ __forceinline__ float ns_elem(bf16_t v) { return (float)v; }
__device__ __forceinline__ float ns_elem(f16_t v) { return (float)v; }

// Sum over the 256 threads of a block in a fixed order.
__device__ __forceinline__ double block_sum(double v, double* smem) {
    smem[threadIdx.x] = v;
    __syncthreads();
    for (int k = 128; k > 0; k >>= 1) {
        if ((int)threadIdx.x < k) smem[threadIdx.x] += smem[threadIdx.x + k];
        __syncthreads();
    }
    const double r = smem[0];
    __syncthreads();
    return r;
}

struct NsUpdate {           // the momentum part of the update
    const float* g;
    float* m;
    float mu, grad_scale;
    int nesterov;
};
struct NsSegments {
    int count;
    NsSegment s[64];
};

// Eight consecutive elements as floats; `wide`: the address is a multiple of the vector's size.
template <typename T>
__device__ __forceinline__ void ns_load8(const T* p, bool wide, float (&v)[8]) {
    if (wide) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = ((const float4*)p)[0], b = ((const float4*)p)[1];
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const uint4 a = *(const uint4*)p;
            const T* e = (const T*)&a;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = ns_elem(e[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = ns_elem(p[j]);
    }
}

// Partial sums of squares in 64 bits: squares of fp32 values neither overflow nor vanish there.  A
// wave takes 2048 consecutive elements of a row at a time, and a matrix without gaps between its
// rows is one long row; 16-byte loads wherever the addresses allow them.  In the update the same
// pass moves the momentum on.  Memory-bound: 240 MB of a 20 M parameter update in 50 us, 4.8 TB/s (a
// large copy: 5.2).
template <typename T, bool MUON>
__global__ __launch_bounds__(256) void ns_norm_kernel(NsTable tab, const T* __restrict__ x, NsUpdate u,
                                                      double* __restrict__ partials) {
    __shared__ double smem[256];
    const int i = ns_find(tab, blockIdx.x);
    const NsProblem& q = tab.p[i];
    const int local = blockIdx.x - tab.first[i];
    const int b = local / q.parts, part = local % q.parts;
    const bool flat = q.ld == q.cols;
    const long long cols = flat ? (long long)q.rows * q.cols : q.cols;
    const long long per_row = (cols + 2047) / 2048, units = per_row * (flat ? 1 : q.rows);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    double sum = 0.0;
    for (long long t = (long long)part * 4 + wave; t < units; t += (long long)q.parts * 4) {
        const long long r = flat ? 0 : t / per_row;
        const long long c0 = (flat ? t : t % per_row) * 2048;
        const long long at0 = q.src + b * q.stride + r * q.ld + c0;
        const bool full = c0 + 2048 <= cols;
        if constexpr (MUON) {
            if (full && (at0 & 3) == 0) {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const long long at = at0 + k * 256 + lane * 4;
                    const float4 g4 = *(const float4*)(u.g + at);
                    float4 m4 = *(const float4*)(u.m + at);
                    float v4[4];
                    const float* g = (const float*)&g4;
                    float* m = (float*)&m4;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float gj = g[j] * u.grad_scale;
                        m[j] = u.mu * m[j] + gj;
                        v4[j] = u.nesterov ? gj + u.mu * m[j] : m[j];
                    }
                    *(float4*)(u.m + at) = m4;
#pragma unroll
                    for (int j = 0; j < 4; ++j) sum += (double)v4[j] * (double)v4[j];
                }
            } else {
                for (int k = lane; k < 2048 && c0 + k < cols; k += 64) {
                    const float g = u.g[at0 + k] * u.grad_scale;
                    const float m = u.mu * u.m[at0 + k] + g;
                    u.m[at0 + k] = m;
                    const float v = u.nesterov ? g + u.mu * m : m;
                    sum += (double)v * (double)v;
                }
            }
        } else if (full) {
            const bool wide = ((uintptr_t)(x + at0) & 15) == 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float v[8];
                ns_load8(x + at0 + k * 512 + lane * 8, wide, v);
#pragma unroll
                for (int j = 0; j < 8; ++j) sum += (double)v[j] * (double)v[j];
            }
        } else {
            for (int k = lane; k < 2048 && c0 + k < cols; k += 64) {
                const float v = ns_elem(x[at0 + k]);
                sum += (double)v * (double)v;
            }
        }
    }
    sum = block_sum(sum, smem);
    if (threadIdx.x == 0) partials[q.part + (size_t)b * q.parts + part] = sum;
}

// Y_0 = X / (||X|| + eps) as planes, zeros in the padding.  64 x 64 tiles of the matrix in memory,
// transposed through LDS where Y is its transpose.  Memory-bound like the pass before (50 us there).
template <typename T, bool MUON>
__global__ __launch_bounds__(256) void ns_load_kernel(NsTable tab, const T* __restrict__ x, NsUpdate u,
                                                      const double* __restrict__ partials, char* ws,
                                                      double eps, float scale) {
    __shared__ double smem[256];
    __shared__ float tile[64][65];
    const int i = ns_find(tab, blockIdx.x);
    const NsProblem& q = tab.p[i];
    const int local = blockIdx.x - tab.first[i];
    const int b = local / q.tiles, t = local % q.tiles;
    double sum = 0.0;
    for (int k = threadIdx.x; k < q.parts; k += 256) sum += partials[q.part + (size_t)b * q.parts + k];
    const double inv = (double)scale / (sqrt(block_sum(sum, smem)) + eps);

    const int tiles_c = (q.trans ? q.mp : q.np) / 64;
    const int r0 = (t / tiles_c) * 64, c0 = (t % tiles_c) * 64;
    const NsPlanes w = ns_planes(q, ws, b, 0);
    const long long at0 = q.src + b * q.stride + (long long)r0 * q.ld + c0;
    const bool full = r0 + 64 <= q.rows && c0 + 64 <= q.cols;
#pragma unroll
    for (int k = threadIdx.x; k < 512; k += 256) {
        const int r = k >> 3, c = (k & 7) * 8;
        const long long at = at0 + r * q.ld + c;
        float v[8];
        if (full) {
            if constexpr (MUON) {
                const bool wide = (at & 3) == 0;
                float m[8];
                ns_load8(u.m + at, wide, m);
                if (u.nesterov) {
                    ns_load8(u.g + at, wide, v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = v[j] * u.grad_scale + u.mu * m[j];
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = m[j];
                }
            } else {
                ns_load8(x + at, ((uintptr_t)(x + at) & 15) == 0, v);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = 0.f;
                if (r0 + r < q.rows && c0 + c + j < q.cols) {
                    if constexpr (MUON) {
                        const float m = u.m[at + j];
                        v[j] = u.nesterov ? u.g[at + j] * u.grad_scale + u.mu * m : m;
                    } else {
                        v[j] = ns_elem(x[at + j]);
                    }
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)((double)v[j] * inv);
        if (q.trans) {
#pragma unroll
            for (int j = 0; j < 8; ++j) tile[r][c + j] = v[j];
        } else {
            uint16_t hi[8], lo[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) split_f16(v[j], hi[j], lo[j]);
            const size_t to = (size_t)(r0 + r) * w.yld + c0 + c;
            *(uint4*)(w.y + to) = *(const uint4*)hi;
            *(uint4*)(w.y + w.yplane + to) = *(const uint4*)lo;
        }
    }
    if (!q.trans) return;
    __syncthreads();
#pragma unroll
    for (int k = threadIdx.x; k < 512; k += 256) {
        const int r = k >> 3, c = (k & 7) * 8;
        uint16_t hi[8], lo[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) split_f16(tile[c + j][r], hi[j], lo[j]);
        const size_t to = (size_t)(c0 + r) * w.yld + r0 + c;
        *(uint4*)(w.y + to) = *(const uint4*)hi;
        *(uint4*)(w.y + w.yplane + to) = *(const uint4*)lo;
    }
}

// SGD with momentum over the segments that are no matrices: g' = g + wd p, m = mu m + g', p -= lr m.
__global__ __launch_bounds__(256) void ns_segments_kernel(NsSegments segs, float* __restrict__ p,
                                                          const float* __restrict__ g,
                                                          float* __restrict__ m, float lr, float mu,
                                                          float wd, float grad_scale) {
    const NsSegment s = segs.s[blockIdx.y];
    for (long long k = (long long)blockIdx.x * 256 + threadIdx.x; k < s.count; k += (long long)gridDim.x * 256) {
        const long long at = s.offset + k;
        const float pv = p[at];
        const float mv = mu * m[at] + (g[at] * grad_scale + wd * pv);
        m[at] = mv;
        p[at] = pv - lr * mv;
    }
}

// Tile shapes of the products, and their measured times in microseconds with n blocks on a CU: a step
// of the summed index takes step + step_more * n, what comes before and after the sum about
// tile[phase] + tile_more[phase] * n.
struct TileTimes {
    double wide_step, narrow_step, step_more;
    double tile[3], tile_more[3];       // GRAM, SQUARE, APPLY
};
// Only for narrow B Y: 149 us for 4096 x 4096, BigTile 169, since it reads three quarters as much LDS for
// a product.  Wide it is the slower one (8192 x 2048, four of them: 1613 us against 1529), and the
// symmetric products have too few tiles of this size and more epilogue than registers.
struct HugeTile {       // 8 waves of 128 x 64 in two halves, one stage in flight
    static constexpr bool kRing = true;
    static constexpr int kGroups = 1, kParts = 2;
    static constexpr int kM = 256, kN = 256, kWavesM = 2, kWavesN = 4, kStages = 2, kBlocksPerCu = 1;
    static constexpr bool kTurns = true;
    static constexpr TileTimes kTimes = {0, 1.55, 0.0, {0, 0, 20}, {0, 0, 0}};
};
struct BigTile {        // 8 waves of 64 x 64, two stages in flight
    static constexpr bool kRing = true;
    static constexpr int kGroups = 1, kParts = 1;
    static constexpr int kM = 128, kN = 256, kWavesM = 2, kWavesN = 4, kStages = 3, kBlocksPerCu = 1;
    static constexpr bool kTurns = true;
    static constexpr TileTimes kTimes = {1.0, 0.85, 0.0, {15, 20, 14}, {0, 0, 0}};
};
struct MidTile {        // 4 waves of 64 x 64, one stage in flight
    static constexpr bool kRing = true;
    static constexpr int kGroups = 1, kParts = 1;
    static constexpr int kM = 128, kN = 128, kWavesM = 2, kWavesN = 2, kStages = 2, kBlocksPerCu = 2;
    static constexpr bool kTurns = false;
    static constexpr TileTimes kTimes = {0.85, 0.7, 0.25, {8, 12, 8}, {0, 0, 0}};
};
struct SmallTile {      // 4 waves of 32 x 32, two stages in flight
    static constexpr bool kRing = true;
    static constexpr int kGroups = 1, kParts = 1;
    static constexpr int kM = 64, kN = 64, kWavesM = 2, kWavesN = 2, kStages = 3, kBlocksPerCu = 3;
    static constexpr bool kTurns = false;
    static constexpr TileTimes kTimes = {0.2, 0.18, 0.13, {4, 5, 3}, {1.5, 2, 1}};
};

// Where tiles are few, a CU's only block takes two steps at once: 0.25 us a step against 0.33 with one
// group (three SmallTile blocks on a CU: 0.2).
struct PairTile {       // two groups of 4 waves of 32 x 32, each with half of the summed index
    static constexpr bool kRing = true;
    static constexpr int kGroups = 2, kParts = 1;
    static constexpr int kM = 64, kN = 64, kWavesM = 2, kWavesN = 2, kStages = 3, kBlocksPerCu = 1;
    static constexpr bool kTurns = false;
    static constexpr TileTimes kTimes = {0.5, 0.46, 0.0, {4.8, 5, 3.5}, {0, 0, 0}};
};
struct ShortTile {      // 8 waves, each with an eighth of the summed index; a step is 8 x 64 of it
    static constexpr int kM = 32, kN = 32, kWaves = 8, kBlocksPerCu = 2;
    static constexpr bool kRing = false;
    static constexpr int kGroups = 1;
    static constexpr TileTimes kTimes = {2.0, 0.3, 1.5, {2.5, 3, 0}, {0.5, 0.5, 0}};
};

// This wave's loads but the last N have landed and its LDS reads are done, then so for all waves.
template <int N>
__device__ __forceinline__ void await_stage() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}
__device__ __forceinline__ void turn() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
// Where the 32-byte pair p of a row of COLS fp16 with summed index k lies: at p ^ pair_swizzle(k).
template <int COLS>
__device__ __forceinline__ int pair_swizzle(int k) {
    if (COLS >= 128) return (k & 3) | ((k >> 1) & 4);
    return ((k >> 1) & 1) | ((k >> 2) & 2);         // two rows share the banks' 256 bytes
}
// Consecutive blocks go to the 8 XCDs in turn; with this numbering each XCD gets consecutive tiles,
// which share rows of an operand in its L2.
__device__ __forceinline__ int xcd_order(int block, int blocks) {
    const int each = blocks >> 3, rest = blocks & 7, x = block & 7;
    return x * each + (x < rest ? x : rest) + (block >> 3);
}

// Fragments of an operand that runs across the summed index: for each of FN column groups (LDS address
// at[y]) the rows OFFSET bytes on and the rows STRIDE bytes further.  The reads and the wait for them
// are one block of assembly: the compiler would put a wait for ALL loads in flight before the builtin,
// since it cannot tell the stage that is read from those that are being filled.
template <int FN, int OFFSET, int STRIDE>
__device__ __forceinline__ void read_across(const unsigned (&at)[FN], f16x8 (&out)[FN]) {
    static_assert(FN == 2 || FN == 4, "column groups");
    f16x4 a[FN], b[FN];
    if constexpr (FN == 4) {
        asm volatile(
            "ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %4, %8 offset:%13\n\t"
            "ds_read_b64_tr_b16 %1, %9 offset:%12\n\tds_read_b64_tr_b16 %5, %9 offset:%13\n\t"
            "ds_read_b64_tr_b16 %2, %10 offset:%12\n\tds_read_b64_tr_b16 %6, %10 offset:%13\n\t"
            "ds_read_b64_tr_b16 %3, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
            "s_waitcnt lgkmcnt(0)"
            : "=&v"(a[0]), "=&v"(a[1]), "=&v"(a[2]), "=&v"(a[3]), "=&v"(b[0]), "=&v"(b[1]), "=&v"(b[2]),
              "=&v"(b[3])
            : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(OFFSET), "n"(OFFSET + STRIDE)
            : "memory");
    } else {
        asm volatile(
            "ds_read_b64_tr_b16 %0, %4 offset:%6\n\tds_read_b64_tr_b16 %2, %4 offset:%7\n\t"
            "ds_read_b64_tr_b16 %1, %5 offset:%6\n\tds_read_b64_tr_b16 %3, %5 offset:%7\n\t"
            "s_waitcnt lgkmcnt(0)"
            : "=&v"(a[0]), "=&v"(a[1]), "=&v"(b[0]), "=&v"(b[1])
            : "v"(at[0]), "v"(at[1]), "n"(OFFSET), "n"(OFFSET + STRIDE)
            : "memory");
    }
#pragma unroll
    for (int y = 0; y < FN; ++y)
        out[y] = f16x8{a[y][0], a[y][1], a[y][2], a[y][3], b[y][0], b[y][1], b[y][2], b[y][3]};
}

struct NsItem {
    int problem, b, ti, tj, split, slab;     // split < 0: the block owns the tile
};

// Tiles of the symmetric products: those that touch the upper triangle, column by column.  A column
// of tiles is kN / kM as wide as it is high, so column j has kN / kM * (j + 1) of them.
template <typename G>
inline long long triangle_tiles(int mp) {
    constexpr int R = G::kN / G::kM;
    const long long rows = (mp + G::kM - 1) / G::kM, cols = (mp + G::kN - 1) / G::kN;
    return R * cols * (cols - 1) / 2 + rows;
}
template <typename G, int PHASE>
__device__ __forceinline__ void tile_of(const NsProblem& q, int t, int& ti, int& tj) {
    if (PHASE == APPLY) {
        // groups of eight tile rows, column by column: neighbours share both operands
        const int rows = (q.mp + G::kM - 1) / G::kM, cols = (q.np + G::kN - 1) / G::kN;
        const int g = t / (8 * cols), in = t - g * 8 * cols;
        const int high = rows - g * 8 < 8 ? rows - g * 8 : 8;
        tj = in / high;
        ti = g * 8 + in % high;
    } else {
        constexpr int R = G::kN / G::kM;
        tj = 0;
        while (R * (tj + 1) * (tj + 2) / 2 <= t) ++tj;
        ti = t - R * tj * (tj + 1) / 2;
    }
}
template <typename G, int PHASE>
__device__ __forceinline__ NsItem item_of(const NsTable& tab, int block, int blocks) {
    NsItem it;
    const bool whole = block < tab.whole;
    const int id = whole ? xcd_order(block, tab.whole) : tab.whole + xcd_order(block - tab.whole, blocks - tab.whole);
    it.problem = ns_find(tab, id);
    const NsProblem& q = tab.p[it.problem];
    int local = id - tab.first[it.problem];
    it.split = -1;
    if (q.splits > 1) {
        it.split = local % q.splits;
        it.slab = q.slab + local;
        local /= q.splits;
    }
    local += q.begin;
    it.b = local / q.tiles;
    tile_of<G, PHASE>(q, local % q.tiles, it.ti, it.tj);
    return it;
}

struct NsStep {
    float inv;                  // accumulator -> value
    float sy;                   // Y's planes hold value * sy
    float ia;                   // SQUARE: planes of A -> value
    float sz;                   // GRAM, SQUARE: value -> planes of A or P
    float a, b, c;              // SQUARE: P = a + b A + c A A
    int buffer;                 // planes of Y that are read
    int last;                   // APPLY: write the result instead of the next planes
};
struct NsResult {
    void* out;                  // orthogonalize
    float* p;                   // update
    float lr, decay;            // decay = 1 - lr * weight decay
};

__device__ __forceinline__ void store_planes(uint16_t* hi_plane, size_t plane, const float (&z)[8]) {
    uint16_t hi[8], lo[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) split_f16(z[j], hi[j], lo[j]);
    *(uint4*)hi_plane = *(const uint4*)hi;
    *(uint4*)(hi_plane + plane) = *(const uint4*)lo;
}
// Eight consecutive elements of a thread in each of its turns over a tile, requested all at once and
// before the accumulators go to LDS.  Stores count as loads in flight, so a load between the stores of
// two turns would wait for the first of them to reach memory (3300 clocks a turn instead of 500).
template <int M, int N, int THREADS>
struct NsOperand {
    static constexpr int kVec = N / 8, kTurns = M * kVec / THREADS;
    static_assert(M * kVec % THREADS == 0 && THREADS % kVec == 0, "whole turns");
    uint4 hi[kTurns], lo[kTurns];

    __device__ __forceinline__ void load(const uint16_t* src, size_t plane, int ld, int rows, int cols, int i0, int j0) {
#pragma unroll
        for (int n = 0; n < kTurns; ++n) {
            const int v = threadIdx.x + n * THREADS, gi = i0 + v / kVec, gj = j0 + v % kVec * 8;
            const uint16_t* at = src + (gi < rows && gj < cols ? (size_t)gi * ld + gj : 0);
            hi[n] = *(const uint4*)at;
            lo[n] = *(const uint4*)(at + plane);
        }
    }
    __device__ __forceinline__ void value(int n, float (&z)[8]) const {
        const uint16_t *h = (const uint16_t*)&hi[n], *l = (const uint16_t*)&lo[n];
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = f16_value(h[j]) + f16_value(l[j]);
    }
};

// What follows a product.  `put` writes the M x N values of the tile (accumulators times s.inv) to
// E in LDS, row pitch LD; rows / cols hold the diagonals of the operands along the tile's sides; the
// tile starts at row i0, column j0.
template <int M, int N, int LD, int THREADS, int BLOCK, int PHASE, typename OUT, typename PUT>
__device__ __forceinline__ void ns_epilogue(float* E, const float* rows, const float* cols, const NsProblem& q,
                                            const NsPlanes& w, char* ws, int b, int i0, int j0, const NsStep& s,
                                            const NsResult& res, const PUT& put) {
    constexpr int kVec = N / 8, kTurns = M * kVec / THREADS;
    if constexpr (PHASE == APPLY) {
        NsOperand<M, N, THREADS> y;
        y.load(w.y, w.yplane, w.yld, q.mp, q.np, i0, j0);
        put();
        const float un = 1.f / s.sy;
        uint16_t* next = ns_planes(q, ws, b, s.buffer ^ 1).y;
        if (!s.last) {
#pragma unroll
            for (int n = 0; n < kTurns; ++n) {
                const int v = threadIdx.x + n * THREADS, r = v / kVec, c = v % kVec * 8, gi = i0 + r, gj = j0 + c;
                if (gi >= q.mp || gj >= q.np) continue;
                float z[8];
                y.value(n, z);
#pragma unroll
                for (int j = 0; j < 8; ++j) z[j] = rows[r] * z[j] + E[r * LD + c + j] * s.sy;
                store_planes(next + (size_t)gi * w.yld + gj, w.yplane, z);
            }
            return;
        }
#pragma unroll
        for (int n = 0; n < kTurns; ++n) {
            const int v = threadIdx.x + n * THREADS, r = v / kVec, c = v % kVec * 8;
            float z[8];
            y.value(n, z);
#pragma unroll
            for (int j = 0; j < 8; ++j) E[r * LD + c + j] += rows[r] * (z[j] * un);
        }
        __syncthreads();
        // Consecutive threads along the rows of the matrix in memory, four elements each; where Y is
        // its transpose those are Y's columns.
        const int wide = q.trans ? M : N;
        const int rest = q.trans ? q.m - i0 : q.n - j0, deep = q.trans ? q.n - j0 : q.m - i0;
        const long long ld = res.p ? q.ld : q.out_ld;
        const long long base = (res.p ? q.src + b * q.stride : q.out + b * q.out_stride) +
                               (q.trans ? (long long)j0 * ld + i0 : (long long)i0 * ld + j0);
        const float lr = res.lr * q.lr;
#pragma unroll 2
        for (int v = threadIdx.x; v < M * N / 4; v += THREADS) {
            const int c = v % (wide / 4) * 4, r = v / (wide / 4);
            if (r >= deep || c >= rest) continue;
            float z[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) z[j] = q.trans ? E[(c + j) * LD + r] : E[r * LD + c + j];
            const long long to = base + r * ld + c;
            const bool all = c + 4 <= rest;
            if (res.p) {
                float* at = res.p + to;
                if (all && ((uintptr_t)at & 15) == 0) {
                    float4 p4 = *(float4*)at;
                    p4.x = res.decay * p4.x - lr * z[0];
                    p4.y = res.decay * p4.y - lr * z[1];
                    p4.z = res.decay * p4.z - lr * z[2];
                    p4.w = res.decay * p4.w - lr * z[3];
                    *(float4*)at = p4;
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (c + j < rest) at[j] = res.decay * at[j] - lr * z[j];
                }
            } else {
                struct alignas(4 * sizeof(OUT)) Four { OUT e[4]; } o;
#pragma unroll
                for (int j = 0; j < 4; ++j) o.e[j] = (OUT)z[j];
                OUT* at = (OUT*)res.out + to;
                if (all && ((uintptr_t)at & (sizeof(Four) - 1)) == 0) {
                    *(Four*)at = o;
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (c + j < rest) at[j] = o.e[j];
                }
            }
        }
    } else {
        // Squares of BLOCK above the diagonal are written twice, mirrored the second time; those below
        // it not at all.
        NsOperand<M, N, THREADS> a;
        if constexpr (PHASE == SQUARE) a.load(w.square(MAT_A), w.aplane, w.ald, q.mp, q.mp, i0, j0);
        put();
        constexpr int kTo = PHASE == GRAM ? MAT_A : MAT_P;
        uint16_t* dst = w.square(kTo);
        float* diag = w.diagonal(kTo);
#pragma unroll
        for (int n = 0; n < kTurns; ++n) {
            const int v = threadIdx.x + n * THREADS, r = v / kVec, c = v % kVec * 8, gi = i0 + r, gj = j0 + c;
            if (gi >= q.mp || gj >= q.mp || gj / BLOCK < gi / BLOCK) continue;
            float z[8], a8[8];
            if (PHASE == SQUARE) a.value(n, a8);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                z[j] = E[r * LD + c + j];
                if (PHASE == SQUARE) {
                    const float di = rows[r], dj = cols[c + j], o = a8[j] * s.ia;
                    z[j] = gi == gj + j ? s.c * (z[j] + di * di) + (s.b * di + s.a)
                                        : s.c * (z[j] + (di + dj) * o) + s.b * o;
                }
                if (gi == gj + j) {
                    diag[gi] = z[j];
                    z[j] = 0.f;
                }
                z[j] *= s.sz;
                E[r * LD + c + j] = z[j];
            }
            store_planes(dst + (size_t)gi * w.ald + gj, w.aplane, z);
        }
        if ((j0 + N - 1) / BLOCK <= i0 / BLOCK) return;
        __syncthreads();
        // eight lanes to a row of 64 values, eight rows to a wave
#pragma unroll 2
        for (int v = threadIdx.x; v < M * N / 8; v += THREADS) {
            const int group = v >> 6, r = (group % (M / 64)) * 64 + (v & 7) * 8;
            const int c = (group / (M / 64)) * 8 + (v >> 3 & 7), gi = i0 + r, gj = j0 + c;
            if (gi >= q.mp || gj >= q.mp || gj / BLOCK <= gi / BLOCK) continue;
            float z[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) z[j] = E[(r + j) * LD + c];
            store_planes(dst + (size_t)gj * w.ald + gi, w.aplane, z);
        }
    }
}
// The operands' diagonals along a tile's sides: requested first of all, put to LDS last of all.
template <int M, int N, int PHASE>
struct NsSides {
    float row = 0.f, col = 0.f;
    __device__ __forceinline__ void load(const NsPlanes& w, int i0, int j0) {
        const int t = threadIdx.x;
        if (PHASE != GRAM && t < M && i0 + t < w.mp) row = w.diagonal(PHASE == SQUARE ? MAT_A : MAT_P)[i0 + t];
        if (PHASE == SQUARE && t < N && j0 + t < w.mp) col = w.diagonal(MAT_A)[j0 + t];
    }
    __device__ __forceinline__ void put(float* rows, float* cols) const {
        const int t = threadIdx.x;
        if (PHASE != GRAM && t < M) rows[t] = row;
        if (PHASE == SQUARE && t < N) cols[t] = col;
    }
};

// One tile of a product, or a part of its summed index.  64 fp16 of every row are staged per step,
// either 64 consecutive hi values (narrow) or 32 hi and the same 32 lo values (wide), straight from
// memory into a ring of LDS stages with counted waits and one barrier per step.
//   * An operand whose rows run along the summed index: rows of 128 bytes, 16-byte piece p of row r at
//     p ^ (r & 7), which spreads a fragment read (16 rows, same piece) over the banks.
//   * Y in B Y runs across it: rows of one summed index, kN columns wide, read with the transposing
//     LDS read (per 16 lanes a 4 x 16 block).  32-byte pair p of row k sits at p ^ pair_swizzle(k): the
//     eight rows that half a wave reads at once meet different banks.
// The columns' operand is the first of the MFMA, so a lane ends with four consecutive columns of a row.
//
// What bounds it: the matrix units with large tiles (wide, eight of [8192, 2048]: Y Y^T 1.02, A A 0.89,
// B Y 1.08 PFLOP/s, where a large library product reaches 1.24; counters at 4096 x 4096: busy in 62 to 65 %
// of a CU's cycles, waves waiting in 25 %); narrow, a third of the instructions for the same bytes, B Y of
// 4096 x 4096 reaches 0.9 PFLOP/s.  With 64 x 64 tiles it is latency: 16 x 512 x 512 keeps the matrix units
// busy in 19 to 26 % and the LDS in 21 to 27 % of the cycles, and waves wait at barriers and for loads in
// 35 to 43 %; one 512 x 512 has only 36 tiles for 256 CUs (11.5 us for 8 steps of PairTile).
template <typename G, bool WIDE, int PHASE, typename OUT>
__global__ __launch_bounds__(G::kGroups * G::kWavesM * G::kWavesN * 64, G::kBlocksPerCu) void ns_product_kernel(
    NsTable tab, char* ws, float* slab, NsStep s, NsResult res) {
    constexpr int kWaves = G::kWavesM * G::kWavesN, kThreads = G::kGroups * kWaves * 64;
    static_assert(G::kParts == 1 || G::kParts == G::kWavesM, "a part of the rows is a row of waves");
    constexpr int WM = G::kM / G::kWavesM, WN = G::kN / G::kWavesN, FM = WM / 16, FN = WN / 16;
    constexpr int kStage = (G::kM + G::kN) * 128, LD = G::kN + 4;
    constexpr int kRing = G::kStages * kStage, kRings = G::kGroups * kRing;
    constexpr int kRows = G::kM / G::kParts, kTile = kRows * LD * 4;      // rows that are finished at a time
    constexpr int FP = FM / G::kParts;
    constexpr int kLoads = kStage / 1024 / kWaves;      // per wave and stage
    constexpr int kStep = WIDE ? 32 : 64;
    __shared__ __attribute__((aligned(1024))) char smem[kRings > kTile ? kRings : kTile];
    __shared__ float rows[G::kM], cols[G::kN];
    static_assert(kThreads >= G::kM && kThreads >= G::kN, "one thread per row and column");

    const NsItem it = item_of<G, PHASE>(tab, blockIdx.x, gridDim.x);
    const NsProblem& q = tab.p[it.problem];
    const NsPlanes w = ns_planes(q, ws, it.b, s.buffer);
    const int group = G::kGroups > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / kWaves : 0;
    const int wave = (threadIdx.x >> 6) - group * kWaves, lane = threadIdx.x & 63;
    char* ring = smem + group * kRing;
    const int i0 = it.ti * G::kM, j0 = it.tj * G::kN;
    // rows' operand, columns' operand
    const uint16_t* rp = PHASE == GRAM ? w.y : w.square(PHASE == SQUARE ? MAT_A : MAT_P);
    const uint16_t* cp = PHASE == SQUARE ? w.square(MAT_A) : w.y;
    const size_t rplane = PHASE == GRAM ? w.yplane : w.aplane, cplane = PHASE == SQUARE ? w.aplane : w.yplane;
    const int rld = PHASE == GRAM ? w.yld : w.ald, cld = PHASE == SQUARE ? w.ald : w.yld;
    const int depth = PHASE == GRAM ? q.np : q.mp;
    NsSides<G::kM, G::kN, PHASE> sides;
    sides.load(w, i0, j0);

    int from = 0, to = depth / kStep;
    if (it.split >= 0) {
        const int all = to;
        from = (int)((long long)all * it.split / q.splits);
        to = (int)((long long)all * (it.split + 1) / q.splits);
    }
    // `mine` of the steps are this group's; a group may have one less than another
    const int steps = (to - from + G::kGroups - 1) / G::kGroups;
    int mine = steps;
    if (G::kGroups > 1) {
        from += group * steps;
        mine = min(steps, to - from);
    }

    // Addresses of this lane's pieces in the first stage; a stage on, they move by a fixed distance.
    const char* src[kLoads];
    long long hop[2];
    hop[0] = kStep * 2;
    hop[1] = PHASE == APPLY ? (long long)kStep * cld * 2 : kStep * 2;
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
        const int kb = wave + l * kWaves;           // KB of the stage
        if (kb < G::kM / 8) {
            const int r = kb * 8 + (lane >> 3), piece = (lane & 7) ^ (lane >> 3);
            int gi = i0 + r;
            gi = gi < q.mp ? gi : q.mp - 1;
            const int k = from * kStep + (WIDE ? (piece & 3) * 8 : piece * 8);
            src[l] = (const char*)(rp + (WIDE && piece >= 4 ? rplane : 0) + (size_t)gi * rld + k);
        } else if (PHASE != APPLY) {
            const int r = (kb - G::kM / 8) * 8 + (lane >> 3), piece = (lane & 7) ^ (lane >> 3);
            int gj = j0 + r;
            gj = gj < q.mp ? gj : q.mp - 1;
            const int k = from * kStep + (WIDE ? (piece & 3) * 8 : piece * 8);
            src[l] = (const char*)(cp + (WIDE && piece >= 4 ? cplane : 0) + (size_t)gj * cld + k);
        } else {
            constexpr int kRowPieces = G::kN / 8;   // 16-byte pieces of a row
            const int at = (kb - G::kM / 8) * 64 + lane;
            const int row = at / kRowPieces, phys = at % kRowPieces;
            const int k = WIDE ? row & 31 : row;
            const int piece = phys ^ (pair_swizzle<G::kN>(k) * 2);
            int gj = j0 + piece * 8;
            gj = gj < q.np ? gj : q.np - 8;
            src[l] = (const char*)(cp + (WIDE && row >= 32 ? cplane : 0) + (size_t)(from * kStep + k) * cld + gj);
        }
    }
    auto stage = [&](int n) {
        char* dst = ring + (n % G::kStages) * kStage;
#pragma unroll
        for (int l = 0; l < kLoads; ++l) {
            const int kb = wave + l * kWaves;
            __builtin_amdgcn_global_load_lds((global_ptr)src[l], (lds_ptr)(dst + kb * 1024), 16, 0, 0);
            src[l] += kb < G::kM / 8 ? hop[0] : hop[1];
        }
    };

    f32x4 acc[FM][FN];
#pragma unroll
    for (int x = 0; x < FM; ++x)
#pragma unroll
        for (int y = 0; y < FN; ++y) acc[x][y] = f32x4{0.f, 0.f, 0.f, 0.f};

    const int wi = (wave / G::kWavesN) * WM, wj = (wave % G::kWavesN) * WN;
    const int l15 = lane & 15, lq = lane >> 4;
    unsigned across[FN];        // row lq*8 + l15/4, columns 4*(l15 & 3) of 16
    if constexpr (PHASE == APPLY) {
        const int row = lq * 8 + (l15 >> 2);
#pragma unroll
        for (int y = 0; y < FN; ++y) {
            const int pair = ((wj + y * 16) >> 4) ^ pair_swizzle<G::kN>(row);
            across[y] = (unsigned)(size_t)(lds_char*)ring + G::kM * 128 + row * (G::kN * 2) + pair * 32 + (l15 & 3) * 8;
        }
    }
#pragma unroll
    for (int n = 0; n < G::kStages - 1; ++n)
        if (n < mine) stage(n);
    struct Fragments { f16x8 r[2][FP], c[2][FN]; };
    auto read = [&](int k, int part, Fragments& f) {
        const char* sr = ring + (k % G::kStages) * kStage;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int x = 0; x < FP; ++x) {
                const int r = wi + (part * FP + x) * 16 + l15;
                f.r[h][x] = *(const f16x8*)(sr + r * 128 + (((h * 4 + lq) ^ (r & 7)) * 16));
            }
        if (part) return;
        if constexpr (PHASE == APPLY) {
            unsigned at[FN];
#pragma unroll
            for (int y = 0; y < FN; ++y) at[y] = across[y] + (unsigned)(k % G::kStages) * kStage;
            read_across<FN, 0, 4 * G::kN * 2>(at, f.c[0]);
            read_across<FN, 32 * G::kN * 2, 4 * G::kN * 2>(at, f.c[1]);
        } else {
            const char* sc = sr + G::kM * 128;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int y = 0; y < FN; ++y) {
                    const int r = wj + y * 16 + l15;
                    f.c[h][y] = *(const f16x8*)(sc + r * 128 + (((h * 4 + lq) ^ (r & 7)) * 16));
                }
        }
    };
    auto multiply = [&](const Fragments& f, int part) {
#pragma unroll
        for (int n = 0; n < (WIDE ? 3 : 2); ++n)        // hi hi, hi lo, lo hi; or two halves of the step
#pragma unroll
            for (int x = 0; x < FP; ++x)
#pragma unroll
                for (int y = 0; y < FN; ++y)
                    acc[part * FP + x][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                        f.c[WIDE ? n >> 1 : n][y], f.r[WIDE ? n & 1 : n][x], acc[part * FP + x][y], 0, 0, 0);
    };
    auto await = [&](int k) {
        if (k + G::kStages - 2 < mine) await_stage<(G::kStages - 2) * kLoads>();
        else await_stage<0>();
    };
    if constexpr (G::kTurns) {
        // The two waves of a SIMD take turns: half a step apart, one reads its fragments while the
        // products of the other one run, and neither the LDS nor the matrix unit waits for the
        // other.  The second half of the waves is one barrier behind; a stage has landed before the
        // first half reads it and is refilled after the second half has.
        Fragments f;
        const bool second = __builtin_amdgcn_readfirstlane(wave) >= kWaves / 2;
        if (second) await(0);
        for (int k = 0; k < steps; ++k) {
#pragma unroll
            for (int part = 0; part < G::kParts; ++part) {
                if (second || part) turn();
                else await(k);
                read(k, part, f);
                if (!part && k + G::kStages - 1 < steps) stage(k + G::kStages - 1);
                if (second && part == G::kParts - 1) await(k + 1);
                else turn();
                multiply(f, part);
            }
        }
        if (!second) turn();
    } else if constexpr (PHASE != APPLY) {
        // A wave reads the fragments of a step while the products of the step before run.  All waves
        // have read stage k when they pass the barrier of step k, so it is refilled at once.
        Fragments f0, f1;
        if (G::kStages - 1 < mine) stage(G::kStages - 1);
        await(0);
        read(0, 0, f0);
        auto step = [&](int k, const Fragments& now, Fragments& next) {
            if (k + 1 < steps) {
                await(k + 1);
                if (k + G::kStages < mine) stage(k + G::kStages);
                read(k + 1, 0, next);
            }
            if (G::kGroups == 1 || k < mine) multiply(now, 0);
        };
        for (int k = 0; k < steps; k += 2) {
            step(k, f0, f1);
            if (k + 1 < steps) step(k + 1, f1, f0);
        }
    } else {
        Fragments f;
        for (int k = 0; k < steps; ++k) {
            await(k);
            if (k + G::kStages - 1 < mine) stage(k + G::kStages - 1);
            read(k, 0, f);
            if (G::kGroups == 1 || k < mine) multiply(f, 0);
        }
    }
    if constexpr (G::kGroups == 2) {        // the second group's sums to the first
        static_assert(kWaves * FM * FN * 1024 <= kRing, "the sums fit the first ring");
        f32x4* over = (f32x4*)smem + (wave * FM * FN) * 64 + lane;
        __syncthreads();
#pragma unroll
        for (int x = 0; x < FM * FN; ++x)
            if (group) over[x * 64] = acc[x / FN][x % FN];
        __syncthreads();
#pragma unroll
        for (int x = 0; x < FM * FN; ++x)
            if (!group) acc[x / FN][x % FN] += over[x * 64];
    }
    if (it.split >= 0) {        // fragments of 16 x 16, lane by lane
        if (group) return;
        float* to_slab = slab + (size_t)it.slab * G::kM * G::kN;
#pragma unroll
        for (int x = 0; x < FM; ++x)
#pragma unroll
            for (int y = 0; y < FN; ++y)
                *(f32x4*)(to_slab + ((size_t)((wi / 16 + x) * (G::kN / 16) + wj / 16 + y) * 64 + lane) * 4) = acc[x][y];
        return;
    }
    float* E = (float*)smem;
#pragma unroll
    for (int part = 0; part < G::kParts; ++part) {
        auto put = [&]() {
            if (part == 0) sides.put(rows, cols);
            __syncthreads();    // the ring's last stage has been read, or the rows before these
            if (group == 0 && wi / kRows == part)
#pragma unroll
                for (int x = 0; x < FM; ++x)
#pragma unroll
                    for (int y = 0; y < FN; ++y)
                        *(f32x4*)(E + (wi % kRows + x * 16 + l15) * LD + wj + y * 16 + lq * 4) = acc[x][y] * s.inv;
            __syncthreads();
        };
        ns_epilogue<kRows, G::kN, LD, kThreads, G::kM, PHASE, OUT>(E, rows + part * kRows, cols, q, w, ws, it.b,
                                                                   i0 + part * kRows, j0, s, res, put);
    }
}

// Adds the parts of split tiles in the order of the summed index and finishes them, a 64 x 64 piece of
// a tile per block.  Latency of one trip to memory and one back: 6 to 8 us for 36 to 250 tiles of 64 x 64.
template <typename G, int PHASE, typename OUT>
__global__ __launch_bounds__(256) void ns_join_kernel(NsTable tab, char* ws, const float* __restrict__ slab,
                                                      NsStep s, NsResult res) {
    constexpr int kPieces = (G::kM / 64) * (G::kN / 64), LD = 68;
    __shared__ float E[64 * LD], rows[64], cols[64];
    const int id = blockIdx.x / kPieces, piece = blockIdx.x % kPieces;
    const int p = ns_find(tab, id);
    const NsProblem& q = tab.p[p];
    const int local = id - tab.first[p];
    const int b = (q.begin + local) / q.tiles;
    int ti, tj;
    tile_of<G, PHASE>(q, (q.begin + local) % q.tiles, ti, tj);
    const int pi = (piece / (G::kN / 64)) * 64, pj = (piece % (G::kN / 64)) * 64;
    const int i0 = ti * G::kM + pi, j0 = tj * G::kN + pj;
    if (i0 >= q.mp || j0 >= (PHASE == APPLY ? q.np : q.mp)) return;
    if (PHASE != APPLY && j0 / G::kM < i0 / G::kM) return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l15 = lane & 15, lq = lane >> 4;
    const NsPlanes w = ns_planes(q, ws, b, s.buffer);
    NsSides<64, 64, PHASE> sides;
    sides.load(w, i0, j0);
    auto put = [&]() {
        f32x4 sum[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) sum[y] = f32x4{0.f, 0.f, 0.f, 0.f};
        const float* from = slab + (size_t)(q.slab + (size_t)local * q.splits) * G::kM * G::kN +
                            ((size_t)((pi / 16 + wave) * (G::kN / 16) + pj / 16) * 64 + lane) * 4;
        constexpr int kBatch = 4;       // parts in flight; one at a time is a chain of memory latencies
        for (int k = 0; k < q.splits; k += kBatch) {
            f32x4 part[kBatch][4];
#pragma unroll
            for (int n = 0; n < kBatch; ++n) {
                const float* at = from + (size_t)(k + n < q.splits ? k + n : q.splits - 1) * G::kM * G::kN;
#pragma unroll
                for (int y = 0; y < 4; ++y) part[n][y] = *(const f32x4*)(at + y * 256);
            }
#pragma unroll
            for (int n = 0; n < kBatch; ++n)
                if (k + n < q.splits)
#pragma unroll
                    for (int y = 0; y < 4; ++y) sum[y] += part[n][y];
        }
        sides.put(rows, cols);
#pragma unroll
        for (int y = 0; y < 4; ++y)
            *(f32x4*)(E + (wave * 16 + l15) * LD + y * 16 + lq * 4) = sum[y] * s.inv;
        __syncthreads();
    };
    ns_epilogue<64, 64, LD, 256, G::kM, PHASE, OUT>(E, rows, cols, q, w, ws, b, i0, j0, s, res, put);
}

// The symmetric products where their sums are short.  A 64 x 64 tile of 512 summed values spends its
// time on 16 barriers one after another; here the 8 waves of a block take 64 of the summed values each,
// straight from memory to registers with every load in flight at once, and add their 32 x 32 parts in
// LDS, in the order of the waves: 8.5 us instead of 13 for 512 x 512.  Each operand is read twice as
// often as by 64 x 64 tiles, and that bounds it from about 700 values on (777 x 777: 18 us, PairTile 14).
template <bool WIDE, int PHASE>
__global__ __launch_bounds__(ShortTile::kWaves * 64, 4) void ns_short_kernel(NsTable tab, char* ws, NsStep s) {
    static_assert(PHASE == GRAM || PHASE == SQUARE, "operands along the summed index");
    typedef ShortTile G;
    constexpr int LD = 36, kPlanes = WIDE ? 2 : 1, kTo = PHASE == GRAM ? MAT_A : MAT_P;
    __shared__ __attribute__((aligned(16))) f32x4 parts[G::kWaves][256];
    __shared__ __attribute__((aligned(16))) float E[32 * LD];
    const NsItem it = item_of<G, PHASE>(tab, blockIdx.x, gridDim.x);
    const NsProblem& q = tab.p[it.problem];
    const NsPlanes w = ns_planes(q, ws, it.b, s.buffer);
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63, l15 = lane & 15, lq = lane >> 4;
    const int i0 = it.ti * 32, j0 = it.tj * 32;
    const uint16_t* x = PHASE == GRAM ? w.y : w.square(MAT_A);
    const size_t plane = PHASE == GRAM ? w.yplane : w.aplane;
    const int ld = PHASE == GRAM ? w.yld : w.ald, depth = PHASE == GRAM ? q.np : q.mp;

    // of the first four waves, thread t finishes row fr, columns fc .. fc + 3 (as its accumulators lie)
    const int fr = (t >> 7 & 1) * 16 + l15, fc = (t >> 6 & 1) * 16 + lq * 4;
    uint2 ah, al;
    float di = 0.f;
    f32x4 dj;
    if (PHASE == SQUARE && t < 256) {
        const size_t at = (size_t)(i0 + fr) * ld + j0 + fc;
        ah = *(const uint2*)(x + at);
        al = *(const uint2*)(x + plane + at);
        di = w.diagonal(MAT_A)[i0 + fr];
        dj = *(const f32x4*)(w.diagonal(MAT_A) + j0 + fc);
    }
    f32x4 acc[2][2] = {};
    for (int k = wave * 64; k < depth; k += G::kWaves * 64) {
        f16x8 r[2][2][kPlanes], c[2][2][kPlanes];       // half of the 64 values, 16 rows, plane
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int f = 0; f < 2; ++f)
#pragma unroll
                for (int l = 0; l < kPlanes; ++l) {
                    const size_t in = (size_t)l * plane + k + h * 32 + lq * 8;
                    r[h][f][l] = *(const f16x8*)(x + (size_t)(i0 + f * 16 + l15) * ld + in);
                    c[h][f][l] = *(const f16x8*)(x + (size_t)(j0 + f * 16 + l15) * ld + in);
                }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int f = 0; f < 2; ++f)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    acc[f][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(c[h][y][0], r[h][f][0], acc[f][y], 0, 0, 0);
                    if constexpr (WIDE) {
                        acc[f][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(c[h][y][0], r[h][f][1], acc[f][y], 0, 0, 0);
                        acc[f][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(c[h][y][1], r[h][f][0], acc[f][y], 0, 0, 0);
                    }
                }
    }
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int y = 0; y < 2; ++y) parts[wave][(f * 2 + y) * 64 + lane] = acc[f][y];
    __syncthreads();
    if (t < 256) {
        f32x4 z = parts[0][t];
#pragma unroll
        for (int k = 1; k < G::kWaves; ++k) z += parts[k][t];
        z *= s.inv;
        const int gi = i0 + fr, gj = j0 + fc;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (PHASE == SQUARE) {
                const float o = (f16_value(((const uint16_t*)&ah)[j]) + f16_value(((const uint16_t*)&al)[j])) * s.ia;
                z[j] = gi == gj + j ? s.c * (z[j] + di * di) + (s.b * di + s.a)
                                    : s.c * (z[j] + (di + dj[j]) * o) + s.b * o;
            }
            if (gi == gj + j) {
                w.diagonal(kTo)[gi] = z[j];
                z[j] = 0.f;
            }
        }
        *(f32x4*)(E + fr * LD + fc) = z * s.sz;
    }
    __syncthreads();
    // the first four waves write the tile, the others its mirror image
    const bool mirror = t >= 256;
    if (mirror && i0 == j0) return;
    const int r = (t & 255) >> 3, c = (t & 7) * 4;
    uint16_t hi[4], lo[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) split_f16(mirror ? E[(c + j) * LD + r] : E[r * LD + c + j], hi[j], lo[j]);
    uint16_t* at = w.square(kTo) + (size_t)((mirror ? j0 : i0) + r) * w.ald + (mirror ? i0 : j0) + c;
    *(uint2*)at = *(const uint2*)hi;
    *(uint2*)(at + w.aplane) = *(const uint2*)lo;
}

// ------------------------------------------------------------------ one block per matrix
// Where Y and one m x m matrix fit a CU's LDS, a block runs the whole chain of a matrix by itself:
// one launch instead of 12 or more, no memory traffic but the matrix itself.  Rows are padded to
// multiples of 32, pitches by 8 elements so that the 16 rows of a fragment meet different banks.
// Latency bounds it: of the 51000 clocks of 64 x 27 waves spend 62 % waiting at barriers and for LDS and
// memory and 17 % waiting to issue; the matrix units are busy in 2 % and 6 instruction cache lines are
// missed.  64 x 27 takes 21 us (2.5 a step, 8.8 for launch, norm and planes), 10 x 512 25, 64 x 448 57
// (grouped launches: 64 x 520 81), 32 x 1056 54 (32 x 1200 89), 128 x 128 86 (128 x 192 85).
constexpr int kSoloThreads = 1024, kSoloWaves = kSoloThreads / 64;
constexpr size_t kSoloLds = 156 * 1024;
constexpr int kSoloRows = 128;              // largest m
constexpr int kSoloMost = 1 << 21;          // blocks of a launch: it has fewer than 2^32 threads
static_assert((unsigned long long)kSoloMost * kSoloThreads < 1ULL << 32, "threads of a launch");

// A matrix in LDS: hi plane, then lo plane.  Addresses are a part that is the same for the wave and one
// of the lane; `lanes` makes the latter anew, for kept over the steps they crowd out the registers.
struct SoloPlanes {
    uint16_t* hi;
    int plane, ld, of_rows, of_across, of_four;
    __device__ __forceinline__ void lanes(int lane) {
        asm volatile("" : "+v"(lane));
        of_rows = (lane & 15) * ld + (lane >> 4) * 8;
        of_across = ((lane >> 4) * 8 + ((lane & 15) >> 2)) * ld + (lane & 3) * 4;
        of_four = (lane & 15) * ld + (lane >> 4) * 4;
    }
    // 16 x 16 tile from (i, j): row lane % 16, four columns from 4 (lane / 16)
    __device__ __forceinline__ f32x4 four(int i, int j) const {
        const uint16_t* at = hi + (i * ld + j + of_four);
        return __builtin_convertvector(*(const f16x4*)at, f32x4) + __builtin_convertvector(*(const f16x4*)(at + plane), f32x4);
    }
    __device__ __forceinline__ void put(int i, int j, f32x4 v) const {
        uint16_t h[4], l[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) split_f16(v[r], h[r], l[r]);
        uint16_t* at = hi + (i * ld + j + of_four);
        *(uint2*)at = *(const uint2*)h;
        *(uint2*)(at + plane) = *(const uint2*)l;
    }
    // 16 rows from i, 32 columns from k: this lane's eight
    __device__ __forceinline__ f16x8 rows(int i, int k, int lo) const {
        return *(const f16x8*)(hi + (lo * plane + i * ld + k + of_rows));
    }
    // 32 rows from k, 16 columns from j, transposed
    __device__ __forceinline__ f16x8 across(int k, int j, int lo) const {
        const uint16_t* at = hi + (lo * plane + k * ld + j + of_across);
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 4 * ld));
        const s16x8 v = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        return __builtin_bit_cast(f16x8, v);
    }
};
__host__ __device__ inline int solo_pad(int v) { return (v + 31) / 32 * 32; }
__host__ __device__ inline size_t solo_lds(int m, int n) {
    const size_t mp = solo_pad(m), np = solo_pad(n);
    return 4 * mp * (np + 8) + 4 * mp * (mp + 8) + 8 * mp + kSoloWaves * 1024;
}
// A 16 x 16 tile of a wide product.  The columns' operand comes first: a lane ends with columns
// 4 (lane / 16) .. + 3 of row lane % 16.  Two sums, for the chain of one is all latency.
struct SoloSum {
    f32x4 high = {0.f, 0.f, 0.f, 0.f}, low = {0.f, 0.f, 0.f, 0.f};
    __device__ __forceinline__ void add(f16x8 ch, f16x8 cl, f16x8 rh, f16x8 rl) {
        high = __builtin_amdgcn_mfma_f32_16x16x32_f16(ch, rh, high, 0, 0, 0);
        low = __builtin_amdgcn_mfma_f32_16x16x32_f16(ch, rl, low, 0, 0, 0);
        low = __builtin_amdgcn_mfma_f32_16x16x32_f16(cl, rh, low, 0, 0, 0);
    }
    // rows i, columns j of X X^T over 32-column steps from .. to
    __device__ __forceinline__ void gram(const SoloPlanes& x, int i, int j, int from, int to) {
#pragma unroll 2
        for (int k = from * 32; k < to * 32; k += 32)
            add(x.rows(j, k, 0), x.rows(j, k, 1), x.rows(i, k, 0), x.rows(i, k, 1));
    }
    __device__ __forceinline__ f32x4 sum() const { return high + low; }
};

// A power of two near the square root of v, so that v is the product of two floats of modest size.
__device__ __forceinline__ float solo_power(double v) {
    const int e = v > 0.0 && v < 1e300 ? ilogb(v) / 2 : 0;
    return ldexpf(1.f, e);
}

struct SoloSteps {
    int steps;
    float sy, sa, sp;               // scales of the planes of Y, A, P
    float k[3 * kMaxSteps];         // (a, b, c) per step
};
static_assert(sizeof(NsTable) + sizeof(SoloSteps) <= 4000, "kernel arguments");

// One loop for both passes over the matrix, and one tile of A to a wave where ROWS is 64: more copies of
// the code took the same time.
template <typename T, bool MUON, int ROWS>
__global__ __launch_bounds__(kSoloThreads) void ns_solo_kernel(NsTable tab, const T* __restrict__ x, NsUpdate u,
                                                               double eps, SoloSteps st, NsResult res) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int problem = ns_find(tab, blockIdx.x);
    const NsProblem& q = tab.p[problem];
    const int b = blockIdx.x - tab.first[problem];
    const int mp = solo_pad(q.m), np = solo_pad(q.n);
    SoloPlanes y, sq;
    y.hi = (uint16_t*)smem;
    y.ld = np + 8;
    y.plane = mp * y.ld;
    sq.hi = y.hi + 2 * y.plane;
    sq.ld = mp + 8;
    sq.plane = mp * sq.ld;
    float* d = (float*)(sq.hi + 2 * sq.plane);      // diagonal of A
    float* e = d + mp;                              // diagonal of P
    float* parts = e + mp;
    const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, lq = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);     // tiles by scalar arithmetic

    // The norm, and in the update the momentum, then the planes.  A lane takes four consecutive elements of
    // a row where all of them allow a vector load, else one; a wave takes 64 such groups of a row or, where
    // rows are shorter, several rows, so that no element needs a division.
    const long long src = q.src + b * q.stride;
    for (int k = tid; k < (y.plane + sq.plane) / 4; k += kSoloThreads) ((uint4*)y.hi)[k] = uint4{0, 0, 0, 0};
    const int sr = q.trans ? 1 : y.ld, sc = q.trans ? y.ld : 1;
    auto read = [&](auto vector) {
        constexpr int V = decltype(vector)::value, kBatch = V == 4 ? 4 : 8;     // loads in flight
        const int groups = q.cols / V;
        const int shift = groups >= 64 ? 6 : 32 - __clz(groups - 1);        // (one group: __clz(0) is 32)
        const int high = 64 >> shift, chunks = (groups + 63) >> 6;
        const int units = (q.rows + high - 1) / high * chunks;
        const int turns = (units - wave + kSoloWaves - 1) / kSoloWaves;     // of this wave
        const int lr = lane >> shift, lc = (lane & ((1 << shift) - 1)) * V;
        const int down = kSoloWaves / chunks, right = kSoloWaves % chunks;
        const long long lane_at = (long long)lr * q.ld + lc;
        struct Place { int row, col; };
        auto inside = [&](const Place& p) { return p.row + lr < q.rows && p.col + lc < q.cols; };
        auto advance = [&](Place& p) {
            p.row += down * high;
            p.col += right * 64 * V;
            if (p.col >= chunks * 64 * V) {
                p.col -= chunks * 64 * V;
                p.row += high;
            }
        };
        auto load = [&](const auto* from, float (&v)[V]) {
            typedef typename std::remove_cv<typename std::remove_pointer<decltype(from)>::type>::type E;
            struct alignas(V * sizeof(E)) Group { E e[V]; };
            const Group w = *(const Group*)from;
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = ns_elem(w.e[j]);
        };
        double sum = 0.0;
        float power = 0.f, scale = 0.f;
#pragma unroll 1
        for (int pass = 0; pass < 2; ++pass) {
            Place p{wave / chunks * high, wave % chunks * 64 * V};
#pragma unroll 1
            for (int n0 = 0; n0 < turns; n0 += kBatch) {
                float v[kBatch][V], m[kBatch][V];
                Place at = p;
#pragma unroll
                for (int n = 0; n < kBatch; ++n) {
                    const long long from = src + (long long)at.row * q.ld + at.col;
#pragma unroll
                    for (int j = 0; j < V; ++j) v[n][j] = m[n][j] = 0.f;
                    if (inside(at)) {
                        if constexpr (MUON) {
                            load(u.g + from + lane_at, v[n]);
                            load((const float*)u.m + from + lane_at, m[n]);
                        } else {
                            load(x + from + lane_at, v[n]);
                        }
                    }
                    advance(at);
                }
#pragma unroll
                for (int n = 0; n < kBatch; ++n) {
                    const bool in = inside(p);
                    if constexpr (MUON) {
#pragma unroll
                        for (int j = 0; j < V; ++j) {
                            const float g = v[n][j] * u.grad_scale;
                            if (pass == 0) m[n][j] = u.mu * m[n][j] + g;
                            v[n][j] = u.nesterov ? g + u.mu * m[n][j] : m[n][j];
                        }
                        if (pass == 0 && in) {
                            struct alignas(V * 4) Group { float e[V]; } w;
#pragma unroll
                            for (int j = 0; j < V; ++j) w.e[j] = m[n][j];
                            *(Group*)(u.m + (src + (long long)p.row * q.ld + p.col) + lane_at) = w;
                        }
                    }
                    if (pass == 0) {
#pragma unroll
                        for (int j = 0; j < V; ++j) sum += (double)v[n][j] * (double)v[n][j];
                    } else if (in) {
                        uint16_t h[V], l[V];
#pragma unroll
                        for (int j = 0; j < V; ++j) split_f16(v[n][j] * power * scale, h[j], l[j]);
                        uint16_t* to = y.hi + (p.row * sr + p.col * sc + lr * sr + lc * sc);
                        if (V == 4 && !q.trans) {
                            *(uint2*)to = *(const uint2*)h;
                            *(uint2*)(to + y.plane) = *(const uint2*)l;
                        } else {
#pragma unroll
                            for (int j = 0; j < V; ++j) {
                                to[j * sc] = h[j];
                                to[j * sc + y.plane] = l[j];
                            }
                        }
                    }
                    advance(p);
                }
            }
            if (pass == 0) {
                double* sums = (double*)parts;
#pragma unroll
                for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
                if (lane == 0) sums[wave] = sum;
                __syncthreads();
                sum = sums[0];
#pragma unroll
                for (int k = 1; k < kSoloWaves; ++k) sum += sums[k];
                // 1 / norm may be out of fp32's range: it is applied as two factors, neither of which is
                const double inv = (double)st.sy / (sqrt(sum) + eps);
                power = solo_power(inv);
                scale = (float)(inv / (double)power);
            }
        }
    };
    const int esize = MUON ? 4 : (int)sizeof(T);
    const size_t at0 = (MUON ? (size_t)u.g | (size_t)u.m : (size_t)x) + (size_t)src * esize;
    if (q.cols % 4 == 0 && q.ld % 4 == 0 && at0 % (4 * esize) == 0) read(std::integral_constant<int, 4>{});
    else read(std::integral_constant<int, 1>{});
    __syncthreads();

    // All tiles of the symmetric matrices: no more rounds of the 16 waves than their upper triangle
    // takes (one more from 81 rows on), and no mirrored writes.  Rows are padded to 16 here, sums over
    // rows to 32 by zeros that nothing overwrites.
    constexpr int kOwn = (ROWS / 16) * (ROWS / 16) / kSoloWaves;        // tiles of a wave
    const int tm = (q.m + 15) / 16, tiles = tm * tm, ksteps = np / 32;
    const int cuts = tiles >= kSoloWaves ? 1 : min(kSoloWaves / tiles, ksteps);
    const float inv_a = 1.f / (st.sy * st.sy), inv_p = 1.f / (st.sa * st.sa), inv_y = 1.f / (st.sp * st.sy);
    const float un_a = 1.f / st.sa, un_y = 1.f / st.sy;
    for (int step = 0; step < st.steps; ++step) {
        y.lanes(lane);
        sq.lanes(lane);
        const float ka = st.k[3 * step], kb = st.k[3 * step + 1], kc = st.k[3 * step + 2];
        f32x4 acc[kOwn];
        // A = Y Y^T: a wave takes whole tiles or, where they are few, a part of one's sum
#pragma unroll
        for (int n = 0; n < kOwn; ++n) {
            int t = cuts > 1 ? wave / cuts : wave + n * kSoloWaves;
            if (cuts == 1 ? t >= tiles : n > 0) break;
            const int cut = cuts > 1 ? wave % cuts : 0;
            f32x4 z = {0.f, 0.f, 0.f, 0.f};
            if (t < tiles) {
                SoloSum a;
                a.gram(y, t / tm * 16, t % tm * 16, ksteps * cut / cuts, ksteps * (cut + 1) / cuts);
                z = a.sum();
            }
            if (cuts > 1) {
                *(f32x4*)(parts + (wave * 64 + lane) * 4) = z;
                __syncthreads();
                t = wave;
                if (t >= tiles) break;
                z = *(const f32x4*)(parts + (t * cuts * 64 + lane) * 4);
#pragma unroll 4
                for (int k = 1; k < cuts; ++k) z += *(const f32x4*)(parts + ((t * cuts + k) * 64 + lane) * 4);
            }
            const int ti = t / tm * 16, tj = t % tm * 16, i = ti + l15, j = tj + lq * 4;
            z *= inv_a;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (i == j + r) {
                    d[i] = z[r];
                    z[r] = 0.f;
                }
            sq.put(ti, tj, z * st.sa);
        }
        __syncthreads();
        // P = b A + c A A in place of A, its diagonal with the a
#pragma unroll
        for (int n = 0; n < kOwn; ++n) {
            const int t = wave + n * kSoloWaves;
            if (t >= tiles) break;
            const int ti = t / tm * 16, tj = t % tm * 16, i = ti + l15, j = tj + lq * 4;
            const f32x4 o = sq.four(ti, tj) * un_a, dj = *(const f32x4*)(d + j);
            const float di = d[i];
            SoloSum a;
            a.gram(sq, ti, tj, 0, mp / 32);
            const f32x4 z = a.sum() * inv_p;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                acc[n][r] = i == j + r ? kc * (z[r] + di * di) + (kb * di + ka)
                                       : kc * (z[r] + (di + dj[r]) * o[r]) + kb * o[r];
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < kOwn; ++n) {
            const int t = wave + n * kSoloWaves;
            if (t >= tiles) break;
            const int ti = t / tm * 16, tj = t % tm * 16, i = ti + l15, j = tj + lq * 4;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (i == j + r) {
                    e[i] = acc[n][r];
                    acc[n][r] = 0.f;
                }
            sq.put(ti, tj, acc[n] * st.sp);
        }
        __syncthreads();
        // Y <- P Y: a wave takes columns, whose old values it has read before it writes the new ones
        const bool last = step == st.steps - 1;
#pragma unroll 1
        for (int tj = wave; tj < np / 16; tj += kSoloWaves) {
            f16x8 ch[ROWS / 32], cl[ROWS / 32];
#pragma unroll
            for (int k = 0; k < ROWS / 32; ++k)
                if (k < mp / 32) {
                    ch[k] = y.across(k * 32, tj * 16, 0);
                    cl[k] = y.across(k * 32, tj * 16, 1);
                }
#pragma unroll 1
            for (int ti = 0; ti < tm; ++ti) {
                const int i = ti * 16 + l15, j = tj * 16 + lq * 4;
                const f32x4 old = y.four(ti * 16, tj * 16) * un_y;
                const float ei = e[i];
                SoloSum a;
#pragma unroll
                for (int k = 0; k < ROWS / 32; ++k)
                    if (k < mp / 32) a.add(ch[k], cl[k], sq.rows(ti * 16, k * 32, 0), sq.rows(ti * 16, k * 32, 1));
                const f32x4 z = old * ei + a.sum() * inv_y;
                if (!last) {
                    y.put(ti * 16, tj * 16, z * st.sy);
                    continue;
                }
                if (!q.trans && i < q.m && j + 4 <= q.n) {
                    if constexpr (MUON) {
                        float* at = res.p + src + (long long)i * q.ld + j;
                        if (((uintptr_t)at & 15) == 0) {
                            *(f32x4*)at = res.decay * *(f32x4*)at - res.lr * q.lr * z;
                            continue;
                        }
                    } else {
                        T* at = (T*)res.out + q.out + b * q.out_stride + (long long)i * q.out_ld + j;
                        struct alignas(4 * sizeof(T)) Four { T e[4]; };
                        if (((uintptr_t)at & (sizeof(Four) - 1)) == 0) {
                            *(Four*)at = Four{{(T)z[0], (T)z[1], (T)z[2], (T)z[3]}};
                            continue;
                        }
                    }
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (i >= q.m || j + r >= q.n) continue;
                    const long long row = q.trans ? j + r : i, col = q.trans ? i : j + r;
                    if (MUON) {
                        float* at = res.p + src + row * q.ld + col;
                        *at = res.decay * *at - res.lr * q.lr * z[r];
                    } else {
                        ((T*)res.out)[q.out + b * q.out_stride + row * q.out_ld + col] = (T)z[r];
                    }
                }
            }
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------ A A and B Y in one launch
// Where A is small, a block that makes a 64 x 64 tile of the next Y first makes the 64 rows of P that it
// needs: 64 m^2 multiplications next to the tile's 64^2 m, and one launch less per step.  A block fills
// its CU's LDS, so this pays for one round of blocks (96 x 320: 80 us against 92, 128 x 8192: 157 against
// 172) and not for several (24 of 128 x 1024, 768 blocks: 198 against 151).
constexpr int kFusedRows = 128;             // largest padded m
constexpr double kFusedUs = 8;              // of a block; one to a CU
template <typename OUT>
__global__ __launch_bounds__(512) void ns_fused_kernel(NsTable tab, char* ws, NsStep sq, NsStep s, NsResult res) {
    constexpr int R = kFusedRows, LD = 68;
    __shared__ __attribute__((aligned(16))) uint16_t amem[2 * R * (R + 8)], pmem[2 * 64 * (R + 8)], ymem[2 * R * 72];
    __shared__ __attribute__((aligned(16))) float d[R], e[64];
    const NsItem it = item_of<SmallTile, APPLY>(tab, blockIdx.x, gridDim.x);
    const NsProblem& q = tab.p[it.problem];
    const NsPlanes w = ns_planes(q, ws, it.b, s.buffer);
    const int t = threadIdx.x, lane = t & 63, l15 = lane & 15, lq = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int i0 = it.ti * 64, j0 = it.tj * 64, mp = q.mp;
    SoloPlanes a, p, y;
    a.hi = amem; a.ld = mp + 8; a.plane = mp * a.ld;
    p.hi = pmem; p.ld = mp + 8; p.plane = 64 * p.ld;
    y.hi = ymem; y.ld = 72; y.plane = mp * 72;
    a.lanes(lane);
    p.lanes(lane);
    y.lanes(lane);

    // A and a column of Y's tiles to LDS, all loads in flight at once
    constexpr int kA = R * R / 4 / 512, kY = R * 16 / 512;
    const uint16_t* from = w.square(MAT_A);
    typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
    const int shift = mp == 64 ? 3 : 4;         // 8 or 16 pieces of 16 bytes in a row of A
    u32x4 va[kA], vy[kY];
#pragma unroll
    for (int n = 0; n < kA; ++n) {
        const int at = t + n * 512, r = at >> shift, c = (at & ((1 << shift) - 1)) * 8;
        const int row = r < 2 * mp ? r : 0;     // rows of the hi, then of the lo plane
        va[n] = *(const u32x4*)(from + (row >= mp ? w.aplane : 0) + (row >= mp ? row - mp : row) * w.ald + c);
    }
#pragma unroll
    for (int n = 0; n < kY; ++n) {
        const int at = t + n * 512, r = at >> 3, c = (at & 7) * 8, row = r < 2 * mp ? r : 0;
        vy[n] = *(const u32x4*)(w.y + (row >= mp ? w.yplane : 0) + (size_t)(row >= mp ? row - mp : row) * w.yld + j0 + c);
    }
    const float dt = w.diagonal(MAT_A)[t < mp ? t : 0];
#pragma unroll
    for (int n = 0; n < kA; ++n) {
        const int at = t + n * 512, row = at >> shift, c = (at & ((1 << shift) - 1)) * 8;
        if (row < 2 * mp) *(u32x4*)(amem + row * a.ld + c) = va[n];
    }
#pragma unroll
    for (int n = 0; n < kY; ++n) {
        const int at = t + n * 512, row = at >> 3, c = (at & 7) * 8;
        if (row < 2 * mp) *(u32x4*)(ymem + row * 72 + c) = vy[n];
    }
    if (t < mp) d[t] = dt;
    __syncthreads();

    // rows i0 .. i0 + 63 of P: a wave takes 32 of them and a quarter of the columns
    const int wr = (wave >> 2) * 32, quarter = wave & 3;
    for (int c = quarter * (mp / 4); c < (quarter + 1) * (mp / 4); c += 16) {
        SoloSum sum[2];
#pragma unroll 2
        for (int k = 0; k < mp; k += 32) {
            const f16x8 ch = a.rows(c, k, 0), cl = a.rows(c, k, 1);
#pragma unroll
            for (int x = 0; x < 2; ++x) sum[x].add(ch, cl, a.rows(i0 + wr + x * 16, k, 0), a.rows(i0 + wr + x * 16, k, 1));
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int i = i0 + wr + x * 16 + l15, j = c + lq * 4;
            const f32x4 o = a.four(i0 + wr + x * 16, c) * sq.ia, dj = *(const f32x4*)(d + j);
            const float di = d[i];
            f32x4 z = sum[x].sum() * sq.inv;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                z[r] = i == j + r ? sq.c * (z[r] + di * di) + (sq.b * di + sq.a)
                                  : sq.c * (z[r] + (di + dj[r]) * o[r]) + sq.b * o[r];
                if (i == j + r) {
                    e[i - i0] = z[r];
                    z[r] = 0.f;
                }
            }
            p.put(wr + x * 16, c, z * sq.sz);
        }
    }
    __syncthreads();
    SoloSum sum[2];
    const int wc = quarter * 16;
#pragma unroll 2
    for (int k = 0; k < mp; k += 32) {
        const f16x8 ch = y.across(k, wc, 0), cl = y.across(k, wc, 1);
#pragma unroll
        for (int x = 0; x < 2; ++x) sum[x].add(ch, cl, p.rows(wr + x * 16, k, 0), p.rows(wr + x * 16, k, 1));
    }
    float* E = (float*)amem;        // A has been read before the last barrier
    auto put = [&]() {
#pragma unroll
        for (int x = 0; x < 2; ++x)
            *(f32x4*)(E + (wr + x * 16 + l15) * LD + wc + lq * 4) = sum[x].sum() * s.inv;
        __syncthreads();
    };
    ns_epilogue<64, 64, LD, 512, 64, APPLY, OUT>(E, e, nullptr, q, w, ws, it.b, i0, j0, s, res, put);
}

int round_up(int v, int to) { return (v + to - 1) / to * to; }

// Largest |a x + b x^3 + c x^5| over [0, r].
double poly_max(double a, double b, double c, double r) {
    auto f = [&](double x) { return std::fabs(x * (a + x * x * (b + c * x * x))); };
    double best = f(r);
    // critical points: a + 3 b z + 5 c z^2 = 0 with z = x^2
    const double disc = 9 * b * b - 20 * a * c;
    if (c != 0.0 && disc >= 0.0) {
        for (double sg : {-1.0, 1.0}) {
            const double z = (-3 * b + sg * std::sqrt(disc)) / (10 * c);
            if (z > 0 && z < r * r) best = std::max(best, f(std::sqrt(z)));
        }
    } else if (c == 0.0 && b != 0.0) {
        const double z = -a / (3 * b);
        if (z > 0 && z < r * r) best = std::max(best, f(std::sqrt(z)));
    }
    return best;
}
// Largest |a + b z + c z^2| over [0, r].
double factor_max(double a, double b, double c, double r) {
    double best = std::max(std::fabs(a), std::fabs(a + r * (b + c * r)));
    if (c != 0.0) {
        const double z = -b / (2 * c);
        if (z > 0 && z < r) best = std::max(best, std::fabs(a + z * (b + c * z)));
    }
    return best;
}
// e with v * 2^e in [2^14, 2^15): half of fp16's range stays free for rounding.  Values under 2^-96
// are scaled like it (their planes keep fewer bits): 2^e times another scale stays in the range of fp32.
int scale_exp(double v) {
    int e;
    std::frexp(std::max(v, 0x1p-96), &e);       // v = f * 2^e, f in [0.5, 1)
    return 15 - e;
}

// One launch: its table and how many blocks it takes.
struct NsLaunch {
    NsTable tab, join;          // `join`: the split entries, counted in tiles
    unsigned blocks = 0, join_tiles = 0;
    int tile = 0;               // 0 big, 1 mid, 2 small, 3 pair, 4 huge, 5 short
    double cost = 0;            // estimate, us
    size_t slab_bytes = 0;

    // A launch has fewer than 2^32 threads, 512 to a block at most (the solo kernel's are counted apart).
    // No matrices whose workspace a GPU could hold come near it with 64 x 64 tiles.
    static constexpr long long kMost = (1LL << 23) - 1;
    static int checked(long long blocks) {
        if (blocks > kMost) throw std::invalid_argument("newton_schulz: too many blocks for one launch");
        return (int)blocks;
    }
    template <typename F>
    static NsLaunch simple(const std::vector<NsProblem>& ps, const F& blocks_of) {
        NsLaunch l{};
        long long at = 0;
        for (const NsProblem& p : ps) {
            NsProblem& e = l.tab.p[l.tab.count];
            e = p;
            e.tiles = checked(blocks_of(p));
            l.tab.first[l.tab.count++] = checked(at);
            at += blocks_of(p) * p.batch;
        }
        l.tab.first[l.tab.count] = checked(at);
        l.blocks = (unsigned)at;
        return l;
    }

    template <typename G>
    static long long tiles_of(const NsProblem& p, int phase) {
        if (phase != APPLY) return triangle_tiles<G>(p.mp);
        return (long long)((p.mp + G::kM - 1) / G::kM) * ((p.np + G::kN - 1) / G::kN);
    }
    // Tiles fill the chip a round of kCus * kBlocksPerCu at a time.  Where they fill less than three
    // quarters of the last round, its tiles' summed index may be divided until they do; whether it is
    // goes by the estimate in microseconds that is left in `cost`.
    template <typename G>
    static NsLaunch tiled(const std::vector<NsProblem>& ps, int phase, bool wide, double& cost) {
        constexpr int kSlots = kCus * G::kBlocksPerCu;
        constexpr int kShortest = 4;            // steps of the shortest part
        const int step = wide ? 32 : 64;
        NsLaunch l{};
        struct Entry { NsProblem p; long long begin, count; int splits; };
        std::vector<Entry> whole, split;
        long long total = 0;
        int longest = 0;
        auto steps_of = [&](const NsProblem& p) {
            const int depth = phase == GRAM ? p.np : p.mp;
            return G::kRing ? depth / step : (depth + 511) / 512;
        };
        for (const NsProblem& p : ps) {
            const long long each = tiles_of<G>(p, phase);
            if (each > (kMost - total) / p.batch) {     // (too small a tile for matrices of this size)
                cost = std::numeric_limits<double>::infinity();
                return l;
            }
            total += each * p.batch;
            longest = std::max(longest, steps_of(p));
        }
        // one round of `blocks` with sums of `steps`, `finish`: the share of the tile's own time
        auto round_us = [&](long long blocks, double steps, double finish) {
            const TileTimes& t = G::kTimes;
            const double n = (double)std::min<long long>(G::kBlocksPerCu, (blocks + kCus - 1) / kCus);
            return steps / G::kGroups * ((wide ? t.wide_step : t.narrow_step) + t.step_more * n) +
                   finish * (t.tile[phase] + t.tile_more[phase] * n);
        };
        // the joining launch: its latency, a tile's parts, and all parts written and read at 4 TB/s
        auto join_us = [&](long long items, int parts) {
            return (phase == SQUARE ? 8.5 : 7.0) + 0.2 * parts + (double)items * G::kM * G::kN * 8 / 4e6;
        };
        const long long rest = total % kSlots;
        const double full = (total / kSlots) * round_us(kSlots, longest, 1);
        long long keep = total;         // tiles that stay whole
        cost = full + (rest ? round_us(rest, longest, 1) : 0);
        if (G::kRing && rest && rest * 4 <= kSlots * 3) {
            if (total < kSlots) {       // one round: parts of equal length, of all that are longer
                int part = longest;
                for (int n = kShortest; n < longest; ++n) {
                    long long items = 0;
                    for (const NsProblem& p : ps)
                        items += tiles_of<G>(p, phase) * p.batch * ((steps_of(p) + n - 1) / n);
                    if (items > kSlots) continue;
                    const double divided = round_us(items, n, 0.5) + join_us(items, (longest + n - 1) / n);
                    if (divided < cost) {
                        cost = divided;
                        part = n;
                    }
                }
                if (part < longest) {
                    keep = 0;
                    for (const NsProblem& p : ps) {
                        const long long n = tiles_of<G>(p, phase) * p.batch;
                        const int parts = (steps_of(p) + part - 1) / part;
                        (parts > 1 ? split : whole).push_back({p, 0, n, parts});
                    }
                }
            } else {
                const int parts = (int)std::min<long long>(kSlots / rest, steps_of(ps.back()) / kShortest);
                if (parts > 1) {
                    const double divided = full + round_us(rest * parts, (double)longest / parts, 0.5) + join_us(rest * parts, parts);
                    if (divided < cost) {
                        cost = divided;
                        keep = total - rest;
                    }
                }
            }
        }
        if (keep) {
            long long at = 0;
            for (const NsProblem& p : ps) {
                const long long n = tiles_of<G>(p, phase) * p.batch, w = std::max(0LL, std::min(n, keep - at));
                if (w) whole.push_back({p, 0, w, 1});
                if (w < n) {
                    const int parts = (int)std::min<long long>(kSlots / rest, std::max(1, steps_of(p) / kShortest));
                    (parts > 1 ? split : whole).push_back({p, w, n - w, parts});
                }
                at += n;
            }
        }
        long long at = 0, tiles = 0, slab = 0;
        for (const std::vector<Entry>* list : {&whole, &split})
            for (const Entry& e : *list) {
                NsProblem& p = l.tab.p[l.tab.count];
                p = e.p;
                p.tiles = checked(tiles_of<G>(e.p, phase));
                p.begin = checked(e.begin);
                p.splits = e.splits;
                p.slab = checked(slab);
                l.tab.first[l.tab.count++] = checked(at);
                at += e.count * e.splits;
                if (list == &whole) {
                    l.tab.whole = checked(at);
                } else {
                    slab += e.count * e.splits;
                    l.join.p[l.join.count] = p;
                    l.join.first[l.join.count++] = checked(tiles);
                    tiles += e.count;
                }
            }
        l.tab.first[l.tab.count] = l.blocks = (unsigned)checked(at);
        l.join.first[l.join.count] = l.join_tiles = (unsigned)checked(tiles);
        l.slab_bytes = (size_t)slab * G::kM * G::kN * sizeof(float);
        return l;
    }
    // A A and B Y in one launch, where every A fits it
    static NsLaunch fused(const std::vector<NsProblem>& ps) {
        NsLaunch l{};
        for (const NsProblem& p : ps)
            if (p.mp > kFusedRows) return l;
        double cost;
        l = tiled<SmallTile>(ps, APPLY, true, cost);
        if (l.join_tiles || std::isinf(cost)) return NsLaunch{};
        l.cost = kFusedUs * ((l.blocks + kCus - 1) / kCus) + 2.5;
        return l;
    }
    static NsLaunch product(const std::vector<NsProblem>& ps, int phase, bool wide) {
        double cost[6];
        NsLaunch l[6] = {tiled<BigTile>(ps, phase, wide, cost[0]),   tiled<MidTile>(ps, phase, wide, cost[1]),
                         tiled<SmallTile>(ps, phase, wide, cost[2]), tiled<PairTile>(ps, phase, wide, cost[3]),
                         tiled<HugeTile>(ps, phase, wide, cost[4]),  tiled<ShortTile>(ps, phase, wide, cost[5])};
        int best = 0;
        for (int i = 0; i < 6; ++i) {
            if (i == 4 && (wide || phase != APPLY)) continue;
            if (i == 5 && phase == APPLY) continue;
            l[i].tile = i;
            if (cost[i] < cost[best]) best = i;
        }
        if (std::isinf(cost[best])) throw std::invalid_argument("newton_schulz: too many blocks for one launch");
        l[best].cost = cost[best] + 2.5 + (l[best].join_tiles ? 1.0 : 0.0);
        return l[best];
    }
};

}  // namespace

struct NewtonSchulzPlan::Group {
    NsLaunch norm, load, product[3], fused, solo;
    // The workspace of the problem whose partial sums start at `part`, in every table.
    void place(int part, long long ws, long long stride) {
        for (NsTable* t : {&norm.tab, &load.tab, &product[0].tab, &product[1].tab, &product[2].tab,
                           &product[0].join, &product[1].join, &product[2].join, &fused.tab})
            for (int i = 0; i < t->count; ++i)
                if (t->p[i].part == part) {
                    t->p[i].ws = ws;
                    t->p[i].ws_stride = stride;
                }
    }
};
struct NewtonSchulzPlan::Solo {
    SoloSteps steps{};
    size_t lds = 0;
    int rows = 0;               // the most of a matrix's smaller side
};
struct NewtonSchulzPlan::Op {
    int phase;
    NsStep step;
};

NewtonSchulzPlan::NewtonSchulzPlan(const std::vector<NsShape>& shapes,
                                   const std::vector<NsSegment>& segments,
                                   const std::vector<float>& coefficients, double eps,
                                   bool wide_products)
    : segs_(segments), coef_(coefficients), eps_(eps), wide_(wide_products) {
    if (coef_.empty() || coef_.size() % 3 || coef_.size() > 3 * kMaxSteps)
        throw std::invalid_argument("newton_schulz: one (a, b, c) per step, at most 64");
    if (!(eps >= 0) || !std::isfinite(eps)) throw std::invalid_argument("newton_schulz: bad eps");
    // Ranges from ||Y_0|| <= 1 on: the singular values before each step, and the polynomial's factor.
    const int steps = (int)coef_.size() / 3;
    std::vector<double> sigma{1.0}, factor;
    for (int k = 0; k < steps; ++k) {
        const double a = coef_[3 * k], b = coef_[3 * k + 1], c = coef_[3 * k + 2], r = sigma.back();
        factor.push_back(factor_max(a, b, c, r * r));
        sigma.push_back(poly_max(a, b, c, r));
        if (!(sigma.back() <= 8.0) || !(factor.back() <= 1024.0))
            throw std::invalid_argument("newton_schulz: step " + std::to_string(k) +
                                        " of these coefficients lets singular values grow past 8");
    }
    x_exp_ = scale_exp(*std::max_element(sigma.begin(), sigma.end()));

    // Problems by falling length of their sums: a launch's last blocks are then its cheapest.
    std::vector<NsShape> order = shapes;
    for (const NsShape& s : shapes) {
        if (s.rows <= 0 || s.cols <= 0 || s.batch <= 0 || s.ld < s.cols || s.offset < 0 || s.stride < 0 ||
            s.out_offset < 0)
            throw std::invalid_argument("newton_schulz: bad matrix");
        if (std::max(s.rows, s.cols) > (1 << 24)) throw std::invalid_argument("newton_schulz: dimension over 2^24");
    }
    std::stable_sort(order.begin(), order.end(), [](const NsShape& x, const NsShape& y) {
        return std::max(x.rows, x.cols) > std::max(y.rows, y.cols);
    });
    std::vector<std::vector<NsProblem>> sets;
    long long partials = 0;
    bool solo = !shapes.empty();
    size_t lds = 0;
    for (const NsShape& s : order) {
        // (a set may need one entry more than it has problems: see NsLaunch::tiled)
        if (sets.empty() || sets.back().size() == kMaxProblems - 1) sets.emplace_back();
        NsProblem p{};
        p.rows = s.rows; p.cols = s.cols; p.batch = s.batch;
        p.m = std::min(s.rows, s.cols);
        p.n = std::max(s.rows, s.cols);
        p.mp = round_up(p.m, kPad);
        p.np = round_up(p.n, kPad);
        p.trans = s.rows > s.cols;
        p.src = s.offset; p.ld = s.ld; p.stride = s.stride;
        p.out = s.out_offset; p.out_ld = s.out_ld; p.out_stride = s.out_stride;
        p.lr = s.lr;
        p.splits = 1;
        const bool flat = p.ld == p.cols;
        const long long cols = flat ? (long long)p.rows * p.cols : p.cols;
        const long long units = (cols + 2047) / 2048 * (flat ? 1 : p.rows);
        p.parts = (int)std::min<long long>((units + 3) / 4, kMaxPartials);
        p.part = (int)partials;
        partials += (long long)p.batch * p.parts;
        if (partials > 0x7fffffffLL) throw std::invalid_argument("newton_schulz: too many matrices");
        sets.back().push_back(p);
        solo = solo && p.m <= kSoloRows && solo_lds(p.m, p.n) <= kSoloLds;
        if (solo) lds = std::max(lds, solo_lds(p.m, p.n));
    }

    // One block per matrix where all of them fit one (next to larger ones they cost nothing extra).
    if (solo) {
        solo_ = std::make_shared<Solo>();
        solo_->lds = lds;
        for (const auto& ps : sets)
            for (const NsProblem& p : ps) solo_->rows = std::max(solo_->rows, p.m);
        SoloSteps& st = solo_->steps;
        st.steps = steps;
        double amax = 1e-3;
        for (int k = 0; k < steps; ++k) amax = std::max(amax, sigma[k] * sigma[k]);
        st.sy = std::ldexp(1.f, x_exp_);
        st.sa = std::ldexp(1.f, scale_exp(amax));
        st.sp = std::ldexp(1.f, scale_exp(*std::max_element(factor.begin(), factor.end())));
        std::copy(coef_.begin(), coef_.end(), st.k);
        // a large batch takes several launches
        std::vector<std::vector<NsProblem>> launches;
        int blocks = kSoloMost;
        for (const auto& ps : sets)
            for (const NsProblem& p : ps)
                for (int b = 0; b < p.batch;) {
                    if (blocks == kSoloMost || launches.back().size() == kMaxProblems) {
                        launches.emplace_back();
                        blocks = 0;
                    }
                    NsProblem part = p;
                    part.batch = std::min(p.batch - b, kSoloMost - blocks);
                    part.src += b * p.stride;
                    part.out += b * p.out_stride;
                    launches.back().push_back(part);
                    b += part.batch;
                    blocks += part.batch;
                }
        for (const auto& ps : launches) {
            groups_.push_back(std::make_shared<Group>());
            groups_.back()->solo = NsLaunch::simple(ps, [](const NsProblem&) { return 1LL; });
        }
        return;
    }

    double single_us = 0, fused_us = 0;
    bool can_fuse = wide_;
    size_t slab = 0;
    for (const auto& ps : sets) {
        groups_.push_back(std::make_shared<Group>());
        Group& g = *groups_.back();
        g.norm = NsLaunch::simple(ps, [](const NsProblem& p) { return (long long)p.parts; });
        g.load = NsLaunch::simple(ps, [](const NsProblem& p) { return (long long)(p.mp / 64) * (p.np / 64); });
        for (int phase : {(int)GRAM, (int)SQUARE, (int)APPLY}) {
            g.product[phase] = NsLaunch::product(ps, phase, wide_);
            slab = std::max(slab, g.product[phase].slab_bytes);
        }
        single_us += g.product[SQUARE].cost + g.product[APPLY].cost;
        g.fused = NsLaunch::fused(ps);
        can_fuse = can_fuse && g.fused.blocks;
        fused_us += g.fused.cost;
    }
    fused_ = can_fuse && fused_us < single_us;

    // Every step multiplies its own Y.  (Two or three steps could share one A = Y Y^T, carried on as
    // Q A Q: fewer products where n is several times m, but the rounding of A then grows by a^2 a step
    // beside a Y that never had it.  With one dominant column that is 2 to 4 times the error of fp32
    // products for two steps and 10 to 25 times for three; single steps stay at 0.3 to 2.2 times.)
    for (int k = 0; k < steps; ++k) {
        const int ea = scale_exp(std::max(sigma[k] * sigma[k], 1e-3)), ep = scale_exp(factor[k]);
        NsStep s{};
        s.sy = std::ldexp(1.f, x_exp_);
        s.buffer = k & 1;
        s.inv = std::ldexp(1.f, -2 * x_exp_);
        s.sz = std::ldexp(1.f, ea);
        ops_.push_back(std::make_shared<Op>(Op{GRAM, s}));
        s.inv = std::ldexp(1.f, -2 * ea);
        s.ia = std::ldexp(1.f, -ea);
        s.sz = std::ldexp(1.f, ep);
        s.a = coef_[3 * k];
        s.b = coef_[3 * k + 1];
        s.c = coef_[3 * k + 2];
        ops_.push_back(std::make_shared<Op>(Op{SQUARE, s}));
        s.inv = std::ldexp(1.f, -x_exp_ - ep);
        s.last = k == steps - 1;
        ops_.push_back(std::make_shared<Op>(Op{APPLY, s}));
    }

    // workspace: the matrices' planes, the partial sums, the parts of divided tiles
    size_t at = 0;
    for (size_t i = 0; i < sets.size(); ++i)
        for (size_t j = 0; j < sets[i].size(); ++j) {
            const NsProblem& p = sets[i][j];
            const size_t each = (ns_matrix_bytes(p.mp, p.np) + 255) & ~(size_t)255;
            groups_[i]->place(p.part, (long long)at, (long long)each);
            at += each * p.batch;
        }
    partials_ = at;
    at += ((size_t)partials * sizeof(double) + 255) & ~(size_t)255;
    slab_ = at;
    ws_bytes_ = at + slab;
}

std::vector<NsLaunchInfo> NewtonSchulzPlan::launches() const {
    static const struct { const char* name; unsigned threads; } kTiles[6] = {
        {"128x256", 512}, {"128x128", 256}, {"64x64", 256}, {"64x64 in pairs", 512}, {"256x256", 512}, {"32x32", 512}};
    std::vector<NsLaunchInfo> out;
    for (const auto& g : groups_) {
        if (solo_) {
            out.push_back({"solo", solo_->rows <= 64 ? "64" : "128", g->solo.blocks, kSoloThreads, 0, 0});
            continue;
        }
        out.push_back({"norm", "", g->norm.blocks, 256, 0, 0});
        out.push_back({"load", "64x64", g->load.blocks, 256, 0, 0});
        static const char* const kPhases[3] = {"gram", "square", "apply"};
        for (int phase = 0; phase < (fused_ ? 1 : 3); ++phase) {
            const NsLaunch& l = g->product[phase];
            out.push_back({kPhases[phase], kTiles[l.tile].name, l.blocks, kTiles[l.tile].threads,
                           (unsigned)l.tab.whole, l.join_tiles});
        }
        if (fused_) out.push_back({"square and apply", "64x64", g->fused.blocks, 512, g->fused.blocks, 0});
    }
    return out;
}

void NewtonSchulzPlan::check_workspace(const void* ws, size_t ws_bytes) const {
    if (ws_bytes < ws_bytes_ || ((uintptr_t)ws & 255) || (!ws && ws_bytes_))
        throw std::invalid_argument("newton_schulz: workspace too small or not 256-byte aligned");
}

namespace {

// Launches with the kernel's own parameter types; a launch that is refused raises.
template <typename... P, typename... A>
void ns_launch(void (*kernel)(P...), dim3 blocks, unsigned threads, size_t lds, hipStream_t stream, A&&... values) {
    std::tuple<P...> own(std::forward<A>(values)...);
    const hipError_t e = std::apply(
        [&](auto&... v) {
            void* at[] = {(void*)&v...};
            return hipLaunchKernel((const void*)kernel, blocks, dim3(threads), at, lds, stream);
        },
        own);
    if (e == hipSuccess) return;
    (void)hipGetLastError();        // reported here, not by the next call that looks
    throw std::runtime_error(std::string("newton_schulz: launch: ") + hipGetErrorString(e));
}

template <typename G, bool WIDE, int PHASE, typename OUT>
void launch_product(const NsLaunch& l, char* ws, float* slab, const NsStep& s, const NsResult& r,
                    hipStream_t stream) {
    ns_launch(ns_product_kernel<G, WIDE, PHASE, OUT>, l.blocks, G::kGroups * G::kWavesM * G::kWavesN * 64, 0, stream,
              l.tab, ws, slab, s, r);
    if (l.join_tiles)
        ns_launch(ns_join_kernel<G, PHASE, OUT>, l.join_tiles * (G::kM / 64) * (G::kN / 64), 256, 0, stream, l.join, ws,
                  slab, s, r);
}
template <typename G, bool WIDE>
void launch_apply(const NsLaunch& l, NsType type, char* ws, float* slab, const NsStep& s, const NsResult& r,
                  hipStream_t stream) {
    if (type == NS_BF16) launch_product<G, WIDE, APPLY, bf16_t>(l, ws, slab, s, r, stream);
    else if (type == NS_F16) launch_product<G, WIDE, APPLY, f16_t>(l, ws, slab, s, r, stream);
    else launch_product<G, WIDE, APPLY, float>(l, ws, slab, s, r, stream);
}
template <typename G, bool WIDE>
void launch_phase(const NsLaunch& l, int phase, NsType type, char* ws, float* slab, const NsStep& s,
                  const NsResult& r, hipStream_t stream) {
    if (phase == GRAM) launch_product<G, WIDE, GRAM, float>(l, ws, slab, s, r, stream);
    else if (phase == SQUARE) launch_product<G, WIDE, SQUARE, float>(l, ws, slab, s, r, stream);
    else launch_apply<G, WIDE>(l, type, ws, slab, s, r, stream);
}
void launch_fused(const NsLaunch& l, NsType type, char* ws, const NsStep& square, const NsStep& s, const NsResult& r,
                  hipStream_t stream) {
    auto go = [&](auto kernel) { ns_launch(kernel, l.blocks, 512, 0, stream, l.tab, ws, square, s, r); };
    if (type == NS_BF16) go(ns_fused_kernel<bf16_t>);
    else if (type == NS_F16) go(ns_fused_kernel<f16_t>);
    else go(ns_fused_kernel<float>);
}
void launch_short(const NsLaunch& l, int phase, bool wide, char* ws, const NsStep& s, hipStream_t stream) {
    auto go = [&](auto kernel) { ns_launch(kernel, l.blocks, ShortTile::kWaves * 64, 0, stream, l.tab, ws, s); };
    if (phase == GRAM) go(wide ? ns_short_kernel<true, GRAM> : ns_short_kernel<false, GRAM>);
    else go(wide ? ns_short_kernel<true, SQUARE> : ns_short_kernel<false, SQUARE>);
}

}  // namespace

template <typename T, bool MUON, int ROWS>
void NewtonSchulzPlan::launch_solo_rows(const Group& g, const void* x, const void* update, const void* result,
                                   hipStream_t stream) const {
    // (more than the default 64 KB of LDS has to be allowed once per device)
    const auto kernel = ns_solo_kernel<T, MUON, ROWS>;
    if (hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)kSoloLds) != hipSuccess)
        throw std::runtime_error("newton_schulz: hipFuncSetAttribute");
    ns_launch(kernel, g.solo.blocks, kSoloThreads, solo_->lds, stream, g.solo.tab, (const T*)x,
              *(const NsUpdate*)update, eps_, solo_->steps, *(const NsResult*)result);
}

template <typename T, bool MUON>
void NewtonSchulzPlan::launch_solo(const Group& g, const void* x, const void* update, const void* result,
                                   hipStream_t stream) const {
    if (solo_->rows <= 64) launch_solo_rows<T, MUON, 64>(g, x, update, result, stream);
    else launch_solo_rows<T, MUON, kSoloRows>(g, x, update, result, stream);
}

template <typename Prepare, typename SoloRun>
void NewtonSchulzPlan::chain(char* ws, NsType type, const Prepare& prepare, const SoloRun& solo, void* out,
                             float* p, float lr, float decay, hipStream_t stream) const {
    const NsResult r{out, p, lr, decay};
    float* slab = (float*)(ws + slab_);
    for (const auto& g : groups_) {
        if (solo_) {
            solo(*g, r);
            continue;
        }
        prepare(*g, (double*)(ws + partials_), std::ldexp(1.f, x_exp_));
        const NsStep* before = nullptr;
        for (const auto& op : ops_) {
            if (fused_ && op->phase != GRAM) {
                if (op->phase == APPLY) launch_fused(g->fused, type, ws, *before, op->step, r, stream);
                before = &op->step;
                continue;
            }
            const NsLaunch& l = g->product[op->phase];
            auto go = [&](auto tile) {
                typedef decltype(tile) G;
                if (wide_) launch_phase<G, true>(l, op->phase, type, ws, slab, op->step, r, stream);
                else launch_phase<G, false>(l, op->phase, type, ws, slab, op->step, r, stream);
            };
            if (l.tile == 0) go(BigTile{});
            else if (l.tile == 1) go(MidTile{});
            else if (l.tile == 2) go(SmallTile{});
            else if (l.tile == 3) go(PairTile{});
            else if (l.tile == 4) launch_apply<HugeTile, false>(l, type, ws, slab, op->step, r, stream);
            else launch_short(l, op->phase, wide_, ws, op->step, stream);
        }
    }
}

void NewtonSchulzPlan::orthogonalize(const void* x, void* out, NsType type, void* ws, size_t ws_bytes,
                                     hipStream_t stream) const {
    if (groups_.empty()) return;
    check_workspace(ws, ws_bytes);
    if (!x || !out) throw std::invalid_argument("newton_schulz: null matrix");
    auto prepare = [&](const Group& g, double* partials, float scale) {
        auto go = [&](auto elem) {
            typedef decltype(elem) T;
            ns_launch(ns_norm_kernel<T, false>, g.norm.blocks, 256, 0, stream, g.norm.tab, (const T*)x, NsUpdate{},
                      partials);
            ns_launch(ns_load_kernel<T, false>, g.load.blocks, 256, 0, stream, g.load.tab, (const T*)x, NsUpdate{},
                      partials, (char*)ws, eps_, scale);
        };
        if (type == NS_BF16) go(bf16_t{});
        else if (type == NS_F16) go(f16_t{});
        else go(0.f);
    };
    auto solo = [&](const Group& g, const NsResult& r) {
        const NsUpdate none{};
        if (type == NS_BF16) launch_solo<bf16_t, false>(g, x, &none, &r, stream);
        else if (type == NS_F16) launch_solo<f16_t, false>(g, x, &none, &r, stream);
        else launch_solo<float, false>(g, x, &none, &r, stream);
    };
    chain((char*)ws, type, prepare, solo, out, nullptr, 0.f, 0.f, stream);
}

void NewtonSchulzPlan::muon(float* p, const float* g, float* m, const MuonArgs& a, void* ws,
                            size_t ws_bytes, hipStream_t stream) const {
    if (!p || !g || !m) throw std::invalid_argument("muon: null buffer");
    if (((uintptr_t)p | (uintptr_t)g | (uintptr_t)m) & 15)
        throw std::invalid_argument("muon: buffers must be 16-byte aligned");
    check_workspace(ws, ws_bytes);
    for (size_t lo = 0; lo < segs_.size(); lo += 64) {
        NsSegments segs;
        segs.count = (int)std::min<size_t>(64, segs_.size() - lo);
        long long most = 0;
        for (int i = 0; i < segs.count; ++i) {
            segs.s[i] = segs_[lo + i];
            most = std::max(most, segs.s[i].count);
        }
        const unsigned bx = (unsigned)std::min<long long>((most + 255) / 256, 256);
        if (bx == 0) continue;
        ns_launch(ns_segments_kernel, dim3(bx, (unsigned)segs.count), 256, 0, stream, segs, p, g, m, a.sgd_lr,
                  a.sgd_momentum, a.sgd_weight_decay, a.grad_scale);
    }
    if (groups_.empty()) return;
    NsUpdate u{g, m, a.momentum, a.grad_scale, a.nesterov ? 1 : 0};
    auto prepare = [&](const Group& gr, double* partials, float scale) {
        ns_launch(ns_norm_kernel<float, true>, gr.norm.blocks, 256, 0, stream, gr.norm.tab, (const float*)nullptr, u,
                  partials);
        ns_launch(ns_load_kernel<float, true>, gr.load.blocks, 256, 0, stream, gr.load.tab, (const float*)nullptr, u,
                  partials, (char*)ws, eps_, scale);
    };
    auto solo = [&](const Group& gr, const NsResult& r) { launch_solo<float, true>(gr, nullptr, &u, &r, stream); };
    chain((char*)ws, NS_F32, prepare, solo, nullptr, p, a.lr, 1.f - a.lr * a.weight_decay, stream);
}

}  // namespace dml
