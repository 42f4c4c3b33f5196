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
#include <cmath>
#include <stdexcept>
#include <string>

#include "dml_common.h"
#include "dml_newton_schulz.h"

namespace dml {
namespace {

typedef _Float16 f16_t;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((address_space(3))) void* lds_ptr;
typedef const __attribute__((address_space(1))) void* global_ptr;

constexpr int kMaxProblems = 32;        // per launch: the table has to fit the kernel arguments
constexpr int kPad = 64;                // planes are zero-padded to multiples of this
constexpr int kMaxPartials = 256;       // blocks (partial sums of squares) per matrix

struct NsProblem {
    int rows, cols, m, n, mp, np, batch;
    int trans;                          // Y is the transpose of the matrix in memory (rows > cols)
    long long src, ld, stride;
    long long out, out_ld, out_stride;
    long long ws, ws_stride;            // bytes
    int part, parts;                    // partial sums: first index, count per matrix
    float lr;
    int tiles;                          // of one matrix, in the launch at hand
};
struct NsTable {
    int count;
    int first[kMaxProblems + 1];        // first block of each problem, in the launch at hand
    NsProblem p[kMaxProblems];
};
static_assert(sizeof(NsTable) <= 3800, "kernel arguments");

// Workspace of one matrix: Y twice (this step's and the next one's) as [mp, np] planes and as
// [np, mp] planes, the off-diagonal parts of A and B as [mp, mp] planes, their diagonals.
struct NsPlanes {
    uint16_t *y, *yt, *o, *p;           // hi plane; the lo plane follows it
    float *d, *e;
    size_t yplane, aplane;
};
__host__ __device__ inline size_t ns_matrix_bytes(size_t mp, size_t np) {
    return 16 * mp * np + 8 * mp * mp + 8 * mp;
}
__device__ __forceinline__ NsPlanes ns_planes(const NsProblem& q, char* ws, int b, int buffer) {
    NsPlanes r;
    uint16_t* base = (uint16_t*)(ws + q.ws + (size_t)b * q.ws_stride);
    r.yplane = (size_t)q.mp * q.np;
    r.aplane = (size_t)q.mp * q.mp;
    r.y = base + (size_t)buffer * 2 * r.yplane;
    r.yt = base + (size_t)(4 + buffer * 2) * r.yplane;
    r.o = base + 8 * r.yplane;
    r.p = r.o + 2 * r.aplane;
    r.d = (float*)(r.p + 2 * r.aplane);
    r.e = r.d + q.mp;
    return r;
}

__device__ __forceinline__ int ns_find(const NsTable& t, int block) {
    int i = 0;
    while (i + 1 < t.count && block >= t.first[i + 1]) ++i;
    return i;
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

// The update direction of one element (its momentum already updated).
__device__ __forceinline__ float ns_direction(const NsUpdate& u, long long at) {
    const float m = u.m[at];
    return u.nesterov ? u.g[at] * u.grad_scale + u.mu * m : m;
}

// Partial sums of squares in 64 bits: squares of fp32 values neither overflow nor vanish there.
// A block takes 64 x 256 tiles.  In the update it first moves the momentum on.
template <typename T, bool MUON>
__global__ __launch_bounds__(256) void ns_norm_kernel(NsTable tab, const T* __restrict__ x, NsUpdate u,
                                                      double* __restrict__ partials) {
    __shared__ double smem[256];
    const int i = ns_find(tab, blockIdx.x);
    const NsProblem& q = tab.p[i];
    const int local = blockIdx.x - tab.first[i];
    const int b = local / q.parts, part = local % q.parts;
    const int tiles_c = (q.cols + 255) / 256;
    const long long tiles = (long long)((q.rows + 63) / 64) * tiles_c;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    double sum = 0.0;
    for (long long t = part; t < tiles; t += q.parts) {
        const int r0 = (int)(t / tiles_c) * 64, c0 = (int)(t % tiles_c) * 256;
        for (int r = r0 + wave; r < r0 + 64 && r < q.rows; r += 4) {
            const long long row = q.src + b * q.stride + r * q.ld;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int c = c0 + k * 64 + lane;
                if (c >= q.cols) continue;
                float v;
                if constexpr (MUON) {
                    const float g = u.g[row + c] * u.grad_scale;
                    const float m = u.mu * u.m[row + c] + g;
                    u.m[row + c] = m;
                    v = u.nesterov ? g + u.mu * m : m;
                } else {
                    v = ns_elem(x[row + c]);
                }
                sum += (double)v * (double)v;
            }
        }
    }
    sum = block_sum(sum, smem);
    if (threadIdx.x == 0) partials[q.part + (size_t)b * q.parts + part] = sum;
}

// Y_0 = X / (||X|| + eps) as planes in both orientations, zeros in the padding.  64 x 64 tiles of
// the matrix in memory, transposed through LDS.
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

    const int colsp = q.trans ? q.mp : q.np;
    const int tiles_c = colsp / 64;
    const int r0 = (t / tiles_c) * 64, c0 = (t % tiles_c) * 64;
    for (int k = threadIdx.x; k < 4096; k += 256) {
        const int r = r0 + (k >> 6), c = c0 + (k & 63);
        float v = 0.f;
        if (r < q.rows && c < q.cols) {
            const long long at = q.src + b * q.stride + r * q.ld + c;
            if constexpr (MUON) v = ns_direction(u, at);
            else v = ns_elem(x[at]);
            v = (float)((double)v * inv);
        }
        tile[k >> 6][k & 63] = v;
    }
    __syncthreads();
    const NsPlanes w = ns_planes(q, ws, b, 0);
    // `same` has the orientation of the memory matrix, `flip` the other one
    uint16_t* same = q.trans ? w.yt : w.y;
    uint16_t* flip = q.trans ? w.y : w.yt;
    const size_t same_ld = q.trans ? q.mp : q.np, flip_ld = q.trans ? q.np : q.mp;
    for (int k = threadIdx.x; k < 512; k += 256) {
        const int r = k >> 3, c = (k & 7) * 8;
        uint16_t hi[8], lo[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) split_f16(tile[r][c + j], hi[j], lo[j]);
        const size_t at = (size_t)(r0 + r) * same_ld + c0 + c;
        *(uint4*)(same + at) = *(const uint4*)hi;
        *(uint4*)(same + w.yplane + at) = *(const uint4*)lo;
#pragma unroll
        for (int j = 0; j < 8; ++j) split_f16(tile[c + j][r], hi[j], lo[j]);
        const size_t ft = (size_t)(c0 + r) * flip_ld + r0 + c;
        *(uint4*)(flip + ft) = *(const uint4*)hi;
        *(uint4*)(flip + w.yplane + ft) = *(const uint4*)lo;
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

enum NsPhase { GRAM, POLY, APPLY };

struct NsStep {
    float a, b, c;
    float sx, sa, sb;           // plane scales 2^e
    float inv;                  // accumulator -> value
    int buffer;                 // planes of this step's Y
    int last;                   // APPLY: write the result instead of the next planes
};
struct NsResult {
    void* out;                  // orthogonalize
    float* p;                   // update
    float lr, decay;            // decay = 1 - lr * weight decay
};

// One T x T tile of a product of two matrices whose rows both run along the summed index.  The
// four waves own quarters of the tile; 64 fp16 of every row are staged per step, either 64
// consecutive hi values (narrow) or 32 hi and the same 32 lo values (wide), straight from memory
// into LDS.  16-byte pieces of a row sit at (piece ^ (row & 7)), which spreads a fragment read
// (16 rows, same piece) over the banks.
template <int T, bool WIDE, int PHASE, typename OUT>
__global__ __launch_bounds__(256, 2) void ns_product_kernel(NsTable tab, char* ws, NsStep s, NsResult res) {
    constexpr int W = T / 2, N = W / 16;            // wave tile, fragments per side
    constexpr int kStage = 2 * T * 128;
    constexpr int kEld = T + 4;
    constexpr int kSmem = 2 * kStage > T * kEld * 4 ? 2 * kStage : T * kEld * 4;
    __shared__ __attribute__((aligned(1024))) char smem[kSmem];

    const int i = ns_find(tab, blockIdx.x);
    const NsProblem& q = tab.p[i];
    const int local = blockIdx.x - tab.first[i];
    const int b = local / q.tiles;
    int t = local % q.tiles, ti, tj;
    if (PHASE == APPLY) {
        const int tiles_n = (q.np + T - 1) / T;
        ti = t / tiles_n;
        tj = t % tiles_n;
    } else {        // upper triangle, row by row
        const int tiles_m = (q.mp + T - 1) / T;
        ti = 0;
        while (t >= tiles_m - ti) { t -= tiles_m - ti; ++ti; }
        tj = ti + t;
    }
    const NsPlanes w = ns_planes(q, ws, b, s.buffer);
    const uint16_t *ah, *al, *bh, *bl;
    int ld, depth, rows_b;
    if (PHASE == GRAM) {
        ah = bh = w.y; al = bl = w.y + w.yplane; ld = depth = q.np; rows_b = q.mp;
    } else if (PHASE == POLY) {
        ah = bh = w.o; al = bl = w.o + w.aplane; ld = depth = q.mp; rows_b = q.mp;
    } else {
        ah = w.p; al = w.p + w.aplane; bh = w.yt; bl = w.yt + w.yplane; ld = depth = q.mp; rows_b = q.np;
    }
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int i0 = ti * T, j0 = tj * T;

    auto stage = [&](int k0, int buf) {
        char* dst = smem + buf * kStage;
        const int piece = (lane & 7) ^ (lane >> 3);
        const int kk = WIDE ? k0 + (piece & 3) * 8 : k0 + piece * 8;
#pragma unroll
        for (int r = wave * 8; r < T; r += 32) {
            const int ra = i0 + r + (lane >> 3), rb = j0 + r + (lane >> 3);
            const uint16_t* pa = (WIDE && piece >= 4 ? al : ah) + (size_t)(ra < q.mp ? ra : q.mp - 1) * ld + kk;
            const uint16_t* pb = (WIDE && piece >= 4 ? bl : bh) + (size_t)(rb < rows_b ? rb : rows_b - 1) * ld + kk;
            __builtin_amdgcn_global_load_lds((global_ptr)pa, (lds_ptr)(dst + r * 128), 16, 0, 0);
            __builtin_amdgcn_global_load_lds((global_ptr)pb, (lds_ptr)(dst + T * 128 + r * 128), 16, 0, 0);
        }
    };

    f32x4 acc[N][N];
#pragma unroll
    for (int x = 0; x < N; ++x)
#pragma unroll
        for (int y = 0; y < N; ++y) acc[x][y] = f32x4{0.f, 0.f, 0.f, 0.f};

    const int wi = (wave >> 1) * W, wj = (wave & 1) * W;
    const int l15 = lane & 15, lq = lane >> 4;
    constexpr int kStep = WIDE ? 32 : 64;
    const int steps = depth / kStep;
    stage(0, 0);
    for (int k = 0; k < steps; ++k) {
        __syncthreads();
        if (k + 1 < steps) stage((k + 1) * kStep, (k + 1) & 1);
        const char* sa = smem + (k & 1) * kStage;
        const char* sb = sa + T * 128;
        f16x8 fa[2][N], fb[2][N];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int x = 0; x < N; ++x) {
                const int ra = wi + x * 16 + l15, rb = wj + x * 16 + l15;
                fa[h][x] = *(const f16x8*)(sa + ra * 128 + (((h * 4 + lq) ^ (ra & 7)) * 16));
                fb[h][x] = *(const f16x8*)(sb + rb * 128 + (((h * 4 + lq) ^ (rb & 7)) * 16));
            }
#pragma unroll
        for (int x = 0; x < N; ++x)
#pragma unroll
            for (int y = 0; y < N; ++y) {
                acc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa[0][x], fb[0][y], acc[x][y], 0, 0, 0);
                if (WIDE) {
                    acc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa[0][x], fb[1][y], acc[x][y], 0, 0, 0);
                    acc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa[1][x], fb[0][y], acc[x][y], 0, 0, 0);
                } else {
                    acc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa[1][x], fb[1][y], acc[x][y], 0, 0, 0);
                }
            }
    }
    __syncthreads();
    float* E = (float*)smem;
#pragma unroll
    for (int x = 0; x < N; ++x)
#pragma unroll
        for (int y = 0; y < N; ++y)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                E[(wi + x * 16 + lq * 4 + r) * kEld + wj + y * 16 + l15] = acc[x][y][r] * s.inv;
    __syncthreads();

    if (PHASE == APPLY) {
        const NsPlanes nx = ns_planes(q, ws, b, s.buffer ^ 1);
        for (int v = threadIdx.x; v < T * T / 8; v += 256) {
            const int r = v / (T / 8), c = (v % (T / 8)) * 8;
            const int gi = i0 + r, gj = j0 + c;
            if (gi >= q.mp || gj >= q.np) continue;
            const float k = s.a + w.e[gi];
            const size_t at = (size_t)gi * q.np + gj;
            uint16_t hi[8], lo[8];
            *(uint4*)hi = *(const uint4*)(w.y + at);
            *(uint4*)lo = *(const uint4*)(w.y + w.yplane + at);
            float z[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                z[j] = k * ((f16_value(hi[j]) + f16_value(lo[j])) / s.sx) + E[r * kEld + c + j];
                E[r * kEld + c + j] = z[j];
            }
            if (!s.last) {
#pragma unroll
                for (int j = 0; j < 8; ++j) split_f16(z[j] * s.sx, hi[j], lo[j]);
                *(uint4*)(nx.y + at) = *(const uint4*)hi;
                *(uint4*)(nx.y + nx.yplane + at) = *(const uint4*)lo;
            }
        }
        __syncthreads();
        if (!s.last) {
            for (int v = threadIdx.x; v < T * T / 8; v += 256) {
                const int c = v / (T / 8), r = (v % (T / 8)) * 8;
                const int gi = i0 + r, gj = j0 + c;
                if (gi >= q.mp || gj >= q.np) continue;
                uint16_t hi[8], lo[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) split_f16(E[(r + j) * kEld + c] * s.sx, hi[j], lo[j]);
                const size_t at = (size_t)gj * q.mp + gi;
                *(uint4*)(nx.yt + at) = *(const uint4*)hi;
                *(uint4*)(nx.yt + nx.yplane + at) = *(const uint4*)lo;
            }
            return;
        }
        for (int v = threadIdx.x; v < T * T; v += 256) {
            // consecutive threads along the rows of the matrix in memory
            const int r = q.trans ? v % T : v / T, c = q.trans ? v / T : v % T;
            const int gi = i0 + r, gj = j0 + c;
            if (gi >= q.m || gj >= q.n) continue;
            const float z = E[r * kEld + c];
            const long long row = q.trans ? gj : gi, col = q.trans ? gi : gj;
            if (res.p) {
                float* at = res.p + q.src + b * q.stride + row * q.ld + col;
                *at = res.decay * *at - res.lr * q.lr * z;
            } else {
                ((OUT*)res.out)[q.out + b * q.out_stride + row * q.out_ld + col] = (OUT)z;
            }
        }
        return;
    }

    // GRAM: A = E.  POLY: A A = E + (d_i + d_j) O + [i = j] d_i^2, B = b A + c A A.
    uint16_t* dst = PHASE == GRAM ? w.o : w.p;
    float* diag = PHASE == GRAM ? w.d : w.e;
    const float sc = PHASE == GRAM ? s.sa : s.sb;
    for (int v = threadIdx.x; v < T * T / 8; v += 256) {
        const int r = v / (T / 8), c = (v % (T / 8)) * 8;
        const int gi = i0 + r, gj = j0 + c;
        if (gi >= q.mp || gj >= q.mp) continue;
        const size_t at = (size_t)gi * q.mp + gj;
        uint16_t hi[8], lo[8];
        float di = 0.f;
        if (PHASE == POLY) {
            *(uint4*)hi = *(const uint4*)(w.o + at);
            *(uint4*)lo = *(const uint4*)(w.o + w.aplane + at);
            di = w.d[gi];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float z = E[r * kEld + c + j];
            if (PHASE == POLY) {
                const float dj = w.d[gj + j];
                const float o = (f16_value(hi[j]) + f16_value(lo[j])) / s.sa;
                z = gi == gj + j ? s.b * di + s.c * (z + di * di)
                                 : s.b * o + s.c * (z + (di + dj) * o);
            }
            if (gi == gj + j) {
                diag[gi] = z;
                z = 0.f;
            }
            z *= sc;
            E[r * kEld + c + j] = z;
            split_f16(z, hi[j], lo[j]);
        }
        *(uint4*)(dst + at) = *(const uint4*)hi;
        *(uint4*)(dst + w.aplane + at) = *(const uint4*)lo;
    }
    if (ti == tj) return;
    __syncthreads();
    for (int v = threadIdx.x; v < T * T / 8; v += 256) {
        const int c = v / (T / 8), r = (v % (T / 8)) * 8;
        const int gi = i0 + r, gj = j0 + c;
        if (gi >= q.mp || gj >= q.mp) continue;
        const size_t at = (size_t)gj * q.mp + gi;
        uint16_t hi[8], lo[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) split_f16(E[(r + j) * kEld + c], hi[j], lo[j]);
        *(uint4*)(dst + at) = *(const uint4*)hi;
        *(uint4*)(dst + w.aplane + at) = *(const uint4*)lo;
    }
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
// Largest |b z + c z^2| over [0, r].
double poly2_max(double b, double c, double r) {
    double best = std::fabs(r * (b + c * r));
    if (c != 0.0) {
        const double z = -b / (2 * c);
        if (z > 0 && z < r) best = std::max(best, std::fabs(z * (b + c * z)));
    }
    return best;
}
// e with v * 2^e in (2^14, 2^15]: half of fp16's range stays free for rounding
int scale_exp(double v) {
    int e;
    std::frexp(v, &e);          // v = f * 2^e, f in [0.5, 1)
    return 15 - e;
}

}  // namespace

NewtonSchulzPlan::NewtonSchulzPlan(const std::vector<NsShape>& shapes,
                                   const std::vector<NsSegment>& segments,
                                   const std::vector<float>& coefficients, double eps,
                                   bool wide_products)
    : segs_(segments), coef_(coefficients), eps_(eps), wide_(wide_products) {
    if (coef_.empty() || coef_.size() % 3)
        throw std::invalid_argument("newton_schulz: one (a, b, c) per step");
    if (!(eps >= 0) || !std::isfinite(eps)) throw std::invalid_argument("newton_schulz: bad eps");
    // The range of the singular values after each step, from ||Y_0|| <= 1.
    double r = 1.0, ymax = 1.0, amax = 1.0, bmax = 0.0;
    for (size_t k = 0; k < coef_.size(); k += 3) {
        const double a = coef_[k], b = coef_[k + 1], c = coef_[k + 2];
        amax = std::max(amax, r * r);
        bmax = std::max(bmax, poly2_max(b, c, r * r));
        r = poly_max(a, b, c, r);
        if (!(r <= 8.0) || !(bmax <= 1024.0))
            throw std::invalid_argument("newton_schulz: step " + std::to_string(k / 3) +
                                        " of these coefficients lets singular values grow past 8");
        ymax = std::max(ymax, r);
    }
    x_exp_ = scale_exp(ymax);
    a_exp_ = scale_exp(amax);
    b_exp_ = scale_exp(std::max(bmax, 1e-3));

    size_t at = 0;
    for (const NsShape& s : shapes) {
        if (s.rows <= 0 || s.cols <= 0 || s.batch <= 0 || s.ld < s.cols || s.offset < 0 || s.stride < 0 ||
            s.out_offset < 0)
            throw std::invalid_argument("newton_schulz: bad matrix");
        Matrix q;
        q.s = s;
        q.m = std::min(s.rows, s.cols);
        q.n = std::max(s.rows, s.cols);
        if (q.n > (1 << 24)) throw std::invalid_argument("newton_schulz: dimension over 2^24");
        q.mp = round_up(q.m, kPad);
        q.np = round_up(q.n, kPad);
        q.ws_stride = (long long)((ns_matrix_bytes(q.mp, q.np) + 255) & ~(size_t)255);
        q.ws = (long long)at;
        at += (size_t)q.ws_stride * s.batch;
        mats_.push_back(q);
    }
    for (const Matrix& q : mats_) at += (size_t)q.s.batch * kMaxPartials * sizeof(double);
    ws_bytes_ = at;
}

void NewtonSchulzPlan::check_workspace(const void* ws, size_t ws_bytes) const {
    if (ws_bytes < ws_bytes_ || ((uintptr_t)ws & 255) || (!ws && ws_bytes_))
        throw std::invalid_argument("newton_schulz: workspace too small or not 256-byte aligned");
}

// Up to kMaxProblems matrices of a plan and the table of the launch being made.
struct NewtonSchulzPlan::Launch {
    NsTable tab;
    long long blocks = 0;
    // `tiles(problem)`: blocks per matrix
    template <typename F>
    void count(const F& tiles) {
        blocks = 0;
        for (int i = 0; i < tab.count; ++i) {
            tab.p[i].tiles = (int)tiles(tab.p[i]);
            tab.first[i] = (int)blocks;
            blocks += (long long)tiles(tab.p[i]) * tab.p[i].batch;
            if (blocks > 0x7fffffffLL) throw std::invalid_argument("newton_schulz: too many blocks");
        }
        tab.first[tab.count] = (int)blocks;
    }
};

namespace {

template <int T, bool WIDE, typename OUT>
void launch_phase(int phase, const NsTable& tab, unsigned blocks, char* ws, const NsStep& s,
                  const NsResult& r, hipStream_t stream) {
    if (phase == GRAM)
        hipLaunchKernelGGL((ns_product_kernel<T, WIDE, GRAM, float>), dim3(blocks), dim3(256), 0, stream, tab, ws, s, r);
    else if (phase == POLY)
        hipLaunchKernelGGL((ns_product_kernel<T, WIDE, POLY, float>), dim3(blocks), dim3(256), 0, stream, tab, ws, s, r);
    else
        hipLaunchKernelGGL((ns_product_kernel<T, WIDE, APPLY, OUT>), dim3(blocks), dim3(256), 0, stream, tab, ws, s, r);
}
template <int T>
void launch_tile(bool wide, NsType type, int phase, const NsTable& tab, unsigned blocks, char* ws,
                 const NsStep& s, const NsResult& r, hipStream_t stream) {
    auto go = [&](auto w, auto out) {
        launch_phase<T, decltype(w)::value, decltype(out)>(phase, tab, blocks, ws, s, r, stream);
    };
    auto pick = [&](auto w) {
        if (type == NS_BF16) go(w, bf16_t{});
        else if (type == NS_F16) go(w, f16_t{});
        else go(w, 0.f);
    };
    if (wide) pick(std::true_type{});
    else pick(std::false_type{});
}

}  // namespace

template <typename Prepare, typename Finish>
void NewtonSchulzPlan::chain(void* ws_any, hipStream_t stream, const Prepare& prepare,
                             const Finish& finish) const {
    char* ws = (char*)ws_any;
    size_t mat_bytes = 0;
    for (const Matrix& q : mats_) mat_bytes = std::max(mat_bytes, (size_t)(q.ws + q.ws_stride * q.s.batch));
    double* partials = (double*)(ws + mat_bytes);
    for (size_t lo = 0; lo < mats_.size(); lo += kMaxProblems) {
        Launch l;
        NsTable& tab = l.tab;
        tab.count = (int)std::min((size_t)kMaxProblems, mats_.size() - lo);
        long long part = 0;
        for (size_t i = 0; i < lo; ++i) part += (long long)mats_[i].s.batch * kMaxPartials;
        for (int i = 0; i < tab.count; ++i) {
            const Matrix& q = mats_[lo + i];
            NsProblem& p = tab.p[i];
            p.rows = q.s.rows; p.cols = q.s.cols; p.m = q.m; p.n = q.n; p.mp = q.mp; p.np = q.np;
            p.batch = q.s.batch;
            p.trans = q.s.rows > q.s.cols;
            p.src = q.s.offset; p.ld = q.s.ld; p.stride = q.s.stride;
            p.out = q.s.out_offset; p.out_ld = q.s.out_ld; p.out_stride = q.s.out_stride;
            p.ws = q.ws; p.ws_stride = q.ws_stride;
            const long long tiles = (long long)((p.rows + 63) / 64) * ((p.cols + 255) / 256);
            p.parts = (int)std::min<long long>(tiles, kMaxPartials);
            p.part = (int)part;
            p.lr = q.s.lr;
            part += (long long)p.batch * kMaxPartials;
            if (part > 0x7fffffffLL) throw std::invalid_argument("newton_schulz: too many matrices");
        }
        l.count([](const NsProblem& p) { return (long long)p.parts; });
        prepare(0, tab, (unsigned)l.blocks, partials, 0.f);
        l.count([](const NsProblem& p) { return (long long)(p.mp / 64) * (p.np / 64); });
        prepare(1, tab, (unsigned)l.blocks, partials, std::ldexp(1.f, x_exp_));

        NsStep s;
        s.sx = std::ldexp(1.f, x_exp_);
        s.sa = std::ldexp(1.f, a_exp_);
        s.sb = std::ldexp(1.f, b_exp_);
        const int steps = (int)coef_.size() / 3;
        for (int k = 0; k < steps; ++k) {
            s.a = coef_[3 * k]; s.b = coef_[3 * k + 1]; s.c = coef_[3 * k + 2];
            s.buffer = k & 1;
            s.last = k == steps - 1;
            for (int phase : {(int)GRAM, (int)POLY, (int)APPLY}) {
                auto tiles_of = [&](int T) {
                    return [T, phase](const NsProblem& p) {
                        const long long tm = (p.mp + T - 1) / T, tn = (p.np + T - 1) / T;
                        return phase == APPLY ? tm * tn : tm * (tm + 1) / 2;
                    };
                };
                s.inv = std::ldexp(1.f, phase == GRAM ? -2 * x_exp_ : phase == POLY ? -2 * a_exp_ : -x_exp_ - b_exp_);
                l.count(tiles_of(128));
                const bool big = l.blocks >= 256;
                if (!big) l.count(tiles_of(64));
                finish(big, phase, tab, (unsigned)l.blocks, s);
            }
        }
    }
}

void NewtonSchulzPlan::orthogonalize(const void* x, void* out, NsType type, void* ws, size_t ws_bytes,
                                     hipStream_t stream) const {
    if (mats_.empty()) return;
    check_workspace(ws, ws_bytes);
    if (!x || !out) throw std::invalid_argument("newton_schulz: null matrix");
    auto prepare = [&](int pass, const NsTable& tab, unsigned blocks, double* partials, float scale) {
        auto go = [&](auto elem) {
            typedef decltype(elem) T;
            if (pass == 0)
                hipLaunchKernelGGL((ns_norm_kernel<T, false>), dim3(blocks), dim3(256), 0, stream, tab,
                                   (const T*)x, NsUpdate{}, partials);
            else
                hipLaunchKernelGGL((ns_load_kernel<T, false>), dim3(blocks), dim3(256), 0, stream, tab,
                                   (const T*)x, NsUpdate{}, partials, (char*)ws, eps_, scale);
        };
        if (type == NS_BF16) go(bf16_t{});
        else if (type == NS_F16) go(f16_t{});
        else go(0.f);
    };
    NsResult r{};
    r.out = out;
    chain(ws, stream, prepare, [&](bool big, int phase, const NsTable& tab, unsigned blocks, const NsStep& s) {
        if (big) launch_tile<128>(wide_, type, phase, tab, blocks, (char*)ws, s, r, stream);
        else launch_tile<64>(wide_, type, phase, tab, blocks, (char*)ws, s, r, stream);
    });
}

void NewtonSchulzPlan::muon(float* p, const float* g, float* m, const MuonArgs& a, void* ws,
                            size_t ws_bytes, hipStream_t stream) const {
    if (!p || !g || !m) throw std::invalid_argument("muon: null buffer");
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
        hipLaunchKernelGGL(ns_segments_kernel, dim3(bx, (unsigned)segs.count), dim3(256), 0, stream, segs,
                           p, g, m, a.sgd_lr, a.sgd_momentum, a.sgd_weight_decay, a.grad_scale);
    }
    if (mats_.empty()) return;
    NsUpdate u{g, m, a.momentum, a.grad_scale, a.nesterov ? 1 : 0};
    auto prepare = [&](int pass, const NsTable& tab, unsigned blocks, double* partials, float scale) {
        if (pass == 0)
            hipLaunchKernelGGL((ns_norm_kernel<float, true>), dim3(blocks), dim3(256), 0, stream, tab,
                               (const float*)nullptr, u, partials);
        else
            hipLaunchKernelGGL((ns_load_kernel<float, true>), dim3(blocks), dim3(256), 0, stream, tab,
                               (const float*)nullptr, u, partials, (char*)ws, eps_, scale);
    };
    NsResult r{};
    r.p = p;
    r.lr = a.lr;
    r.decay = 1.f - a.lr * a.weight_decay;
    chain(ws, stream, prepare, [&](bool big, int phase, const NsTable& tab, unsigned blocks, const NsStep& s) {
        if (big) launch_tile<128>(wide_, NS_F32, phase, tab, blocks, (char*)ws, s, r, stream);
        else launch_tile<64>(wide_, NS_F32, phase, tab, blocks, (char*)ws, s, r, stream);
    });
}

}  // namespace dml
