// Orthogonalising an update by Newton-Schulz products, and the momentum step around it.
//
//     X <- U / (|U|_F + eps), laid with its shorter side m first (m x n)
//     A = X X^T,  S = b A + c A A,  X <- a X + S X          a few times, with (a, b, c) of each step
// The polynomial a s + b s^3 + c s^5 acts on every singular value s of X and drives it towards 1. Where X is long, two steps go over it at once, on m x m matrices
// alone: with S of the first, T = a A + S A, A' = a T + S T is the next step's X X^T, S' its polynomial, and X <- Q X with
// Q = (a' + S') (a + S) = a a' + (a' S + a S' + S' S). Every m x m product is symmetric: half its tiles are computed.
// The first pair applies a a' X + (...) X, which keeps small singular values exact; later ones, whose Q is near 1, all of Q: a a' = 12 would cancel.
//
// Precision: fp32, on fp16 matrix instructions. A number v of X, A or S (spectral norm known to the host to stay below 2^15 / 2^e for the given
// coefficients) is kept as two fp16 planes of v 2^e: hi = fp16(v 2^e) and lo = fp16(v 2^e - hi) - 22 bits of a number near the matrix's scale; where lo is subnormal, 2^-25
// of v 2^e, so that rows 1e-5 below the others keep some 15 bits of theirs, 1e-7 below 9 - and a product of two such numbers is
// hi hi + hi lo + lo hi, accumulated in fp32: three MFMAs where fp16 has one, at a sixteenth of the time of an fp32 one. The term that is left out
// and the two roundings are 2^-22 of a product each, of random sign: the error of fp32 operands (the steps amplify what is lost on the small
// singular values up to a^5 = 480 times: one fp16 plane leaves 2e-3 of the result's norm, two leave what fp32 does, 2e-6).
// The common exponent e makes every scale of the chain 2^-e. Where eps outweighs the norm, X is too small for planes of that scale: with x0 = -log2 of
// |U| / (|U| + eps), no singular value of X before step k is above 2^(lg_k - x0), lg_k from the largest factors of the steps before, and X's planes - of all
// matrices - are 2^floor(x0 - lg_k) larger, if that is more than one (ns_extra). A and S, small against a, need no more.
//
// All matrices of a call ("units") go through each product in one launch: the shared core's matrices are small, and launches are what they cost.
//
// Bound: the matrix cores of large matrices, at the rate that power leaves them - a product of 4096 x 4096 in 355 us, 1.16 PFLOP/s of fp16 operations (three a
// product), pipes busy 64 % of the time at 1.63 GHz; torch's fp16 product reaches 1.33 PFLOP/s - and launch after launch of small ones: 8 us for each of the
// default core's 15 products, whose operations take 1. Whole calls, five steps: 4096 x 4096 bf16 3.9 ms, 8192 x 1024 fp32 446 us, twelve 777 x 1301 fp16 870 us,
// the default core's 24 matrices 141 us, one block of width 2048 (a momentum step over 4 matrices, 200 MB of weights) 4.2 ms, one 155 x 64 33 us.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <utility>
#include <vector>

#include "../../include/v1t_amd.h"
#include "common.h"

namespace {

constexpr int NS_BK = 32;            // K step of the products; planes are padded to it with zeros both ways
constexpr int NS_PART = 4096;        // least number of elements per partial sum of squares; at most 1024 partial sums a unit
constexpr int NS_TILE_PREP = 64;     // the first planes are written in 64 x 64 tiles
constexpr int NS_CHUNK = 24;         // units per table launch (kernel arguments: below 4 KB)
constexpr int NS_MAX_STEPS = 32, NS_MAX_UNITS = 1 << 16;

struct NsUnit {
    const void* in;   // the update, or the gradient
    void* out;        // the result, or nullptr: w is updated
    float *mom, *w;
    long long rs, cs;                // element strides of `in`; out, mom and w are row-major without gaps
    long long base;                  // byte offset in the workspace: X twice, then the m x m matrices (ns_x, ns_square_at)
    int rows, cols, n, mp, np;       // n: the longer side; mp, np: X's sides, in whole K steps
    int part, part0, nparts, prep0;  // elements per partial sum; first workgroup of this unit in the launches of each kind
    int first[3];                    // first tile in the products' launches: gram, poly, apply / last
    int group0[3], group[3];         // first tile and tiles of the run of units of this size
    float lr, decay, l1;             // w <- decay w - lr O;  gradient + l1 sign(w)
    __host__ __device__ int m() const { return rows < cols ? rows : cols; }
    __host__ __device__ bool trans() const { return rows > cols; }  // X is the update's transpose
    float x0;                        // -log2 of the norm of the first X; written by ns_prep_kernel
};

__host__ __device__ inline long long ns_align(long long x) { return (x + 255) / 256 * 256; }
__host__ __device__ inline long long ns_x(const NsUnit& u, int which) { return u.base + which * ns_align(4ll * u.mp * u.np); }
__host__ __device__ inline long long ns_square_at(const NsUnit& u, int which) { return ns_x(u, 2) + which * ns_align(4ll * u.mp * u.mp); }

// by what power of two X's planes are larger than the common scale
__host__ __device__ inline int ns_extra(float x0, float lg) {
    const float e = floorf(x0 - lg);
    return e > 0.f ? (int)(e < 100.f ? e : 100.f) : 0;  // (x0 is infinite for a matrix of zeros, NaN beside one)
}

struct NsChunk {
    NsUnit u[NS_CHUNK];
};
static_assert(sizeof(NsChunk) + 4 * (4 * NS_MAX_STEPS + 1) + 64 <= 4096, "kernel arguments");

// What a workgroup finds its unit by: per launch (0 .. 2 the products', 3 the partial sums', 4 the first planes') and unit its first workgroup, and the run of units of
// its size. Apart from the units, so that a wave reads 64 of them at once from few lines
typedef int ns_head __attribute__((ext_vector_type(4)));  // first, the run's first, the run's tiles, -

struct NsTable {
    const NsUnit* units;
    const ns_head* heads;  // [5][n]
    int n;
};

__global__ void ns_table_kernel(NsChunk c, int n, int at, int all, NsUnit* units, ns_head* heads) {
    // 4-byte words, one per lane: the argument is read as an array
    const uint32_t* src = (const uint32_t*)&c;
    for (int i = threadIdx.x; i < n * (int)(sizeof(NsUnit) / 4); i += blockDim.x) ((uint32_t*)(units + at))[i] = src[i];
    for (int i = threadIdx.x; i < 5 * n; i += blockDim.x) {
        const int k = i / n, e = i % n;
        const NsUnit& u = c.u[e];
        heads[(size_t)k * all + at + e] = k < 3 ? ns_head{u.first[k], u.group0[k], u.group[k], 0} : ns_head{k == 3 ? u.part0 : u.prep0, 0, 0, 0};
    }
}

// the unit whose range of workgroups `block` falls into - the last one that begins at or before it - and its head
template <int W>
DEVFN int ns_find(const NsTable& t, int block, ns_head& head) {
    const int lane = threadIdx.x & 63;
    const ns_head* h = t.heads + (size_t)W * t.n;
    int found = -1, i = 0;
    ns_head mine{};
    for (;; i += 64) {
        mine = i + lane < t.n ? h[i + lane] : ns_head{0x7fffffff, 0, 0, 0};
        const int k = __popcll(__ballot(mine[0] <= block));
        found += k;
        if (k < 64 || i + 64 >= t.n) break;
    }
    found = __builtin_amdgcn_readfirstlane(found);
    if (found < i) {  // the last one of the 64 before
        head = h[found];
        return found;
    }
#pragma unroll
    for (int e = 0; e < 3; ++e) head[e] = __builtin_amdgcn_readlane(mine[e], found - i);
    return found;
}

struct NsMomentum {
    float mu;
    int nesterov;
};

DEVFN float ns_sign(float x) { return (float)((x > 0.f) - (x < 0.f)); }

// sum over the workgroup of NT, in a fixed order
template <int NT = 256>
DEVFN double ns_block_sum(double v) {
    __shared__ double s[NT / 64];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) v += s[w];
    return v;
}

struct NsNorm {  // 64 bits: a norm may lie outside fp32's range where its elements do not
    float x0;
    double mul;  // the first planes are the update times this
    DEVFN NsNorm(double squares, float eps, float scale) {
        const double norm = sqrt(squares), by = 1.0 / (norm + (double)eps);
        x0 = -log2f((float)(norm * by));
        mul = ldexp((double)scale, ns_extra(x0, 0.f)) * by;
    }
};

// N elements of the update: gradient with its L1 term, momentum (MOM), then U. The loads of a batch stand together: each of a tensor that is written, too, would
// wait for the store before it
template <typename T, bool MOM, int N>
struct NsBatch {
    float g[N], m[N];
    DEVFN void load(const NsUnit& u, const long long (&src)[N], const long long (&at)[N], const bool (&on)[N]) {
        float w[N];
#pragma unroll
        for (int e = 0; e < N; ++e) g[e] = on[e] ? (float)((const T*)u.in)[src[e]] : 0.f;
        if constexpr (MOM) {
#pragma unroll
            for (int e = 0; e < N; ++e) m[e] = on[e] ? u.mom[at[e]] : 0.f;
            if (u.l1 != 0.f) {
#pragma unroll
                for (int e = 0; e < N; ++e) w[e] = on[e] ? u.w[at[e]] : 0.f;
#pragma unroll
                for (int e = 0; e < N; ++e) g[e] += u.l1 * ns_sign(w[e]);
            }
        }
    }
    // N / 4 runs of 4 neighbours: all in, of a tensor whose rows have unit stride (src: in the update, at: in the momentum)
    DEVFN void load_runs(const NsUnit& u, const long long (&src)[N / 4], const long long (&at)[N / 4]) {
        typedef T t4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
        typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
        t4 a[N / 4];
        f4 b[N / 4], w[N / 4];
#pragma unroll
        for (int r = 0; r < N / 4; ++r) a[r] = *(const t4*)((const T*)u.in + src[r]);
        if constexpr (MOM) {
#pragma unroll
            for (int r = 0; r < N / 4; ++r) b[r] = *(const f4*)(u.mom + at[r]);
            if (u.l1 != 0.f) {
#pragma unroll
                for (int r = 0; r < N / 4; ++r) w[r] = *(const f4*)(u.w + at[r]);
            }
        }
#pragma unroll
        for (int r = 0; r < N / 4; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                g[4 * r + e] = (float)a[r][e];
                if constexpr (MOM) {
                    m[4 * r + e] = b[r][e];
                    if (u.l1 != 0.f) g[4 * r + e] += u.l1 * ns_sign(w[r][e]);
                }
            }
    }
    DEVFN void next_momentum(const NsMomentum& mo) {
#pragma unroll
        for (int e = 0; e < N; ++e) m[e] = mo.mu * m[e] + g[e];
    }
    DEVFN float update(const NsMomentum& mo, int e) const { return !MOM ? g[e] : mo.nesterov ? g[e] + mo.mu * m[e] : m[e]; }
};

// partial sums of squares, in 64 bits (their range is that of the inputs squared); MOM: momentum <- mu momentum + gradient on the way
template <typename T, bool MOM>
__global__ __launch_bounds__(256) void ns_norm_kernel(NsTable tab, NsMomentum mo, double* parts) {
    constexpr int N = 16;
    ns_head head;
    const NsUnit& u = tab.units[ns_find<3>(tab, blockIdx.x, head)];
    const long long all = (long long)u.rows * u.cols, i0 = (long long)(blockIdx.x - u.part0) * u.part;
    const int len = (int)min((long long)u.part, all - i0);
    const bool flat = u.cs == 1 && u.rs == u.cols;
    double sum = 0.0;
    NsBatch<T, MOM, N> b;
    auto squares = [&] {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const double v = (double)b.update(mo, e);
            sum += v * v;
        }
    };
    int k0 = 0;
    if (flat)
        for (; k0 + 256 * N <= len; k0 += 256 * N) {
            long long at[N / 4];
#pragma unroll
            for (int r = 0; r < N / 4; ++r) at[r] = i0 + k0 + 1024 * r + 4 * (int)threadIdx.x;
            b.load_runs(u, at, at);
            if constexpr (MOM) {
                b.next_momentum(mo);
                typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll
                for (int r = 0; r < N / 4; ++r) *(f4*)(u.mom + at[r]) = f4{b.m[4 * r], b.m[4 * r + 1], b.m[4 * r + 2], b.m[4 * r + 3]};
            }
            squares();
        }
    for (; k0 < len; k0 += 256 * N) {
        long long src[N], at[N];
        bool on[N];
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const int k = k0 + 256 * e + (int)threadIdx.x;
            on[e] = k < len;
            at[e] = src[e] = i0 + k;
            if (!flat) {
                const long long r = at[e] / u.cols;
                src[e] = r * u.rs + (at[e] - r * u.cols) * u.cs;
            }
        }
        b.load(u, src, at, on);
        if constexpr (MOM) {
            b.next_momentum(mo);
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (on[e]) u.mom[at[e]] = b.m[e];
        }
        squares();
    }
    sum = ns_block_sum(sum);
    if (threadIdx.x == 0) parts[blockIdx.x] = sum;
}

// A matrix in the workspace, rows x ld (multiples of 32): 32 numbers of a row lie as 64 fp16, their 32 hi in front of their 32 lo, so that the 32 numbers of a row that a K step
// reads are one line of 128 B. Where number (i, j)'s hi lies; its lo is 32 behind
DEVFN size_t ns_at(int i, int j, int ld) { return (size_t)i * (2 * ld) + (j >> 5) * 64 + (j & 31); }
constexpr int NS_LO = 32;

DEVFN void ns_split(float v, f16_t& hi, f16_t& lo) {
    hi = (f16_t)v;
    lo = (f16_t)(v - (float)hi);
}

// the first planes: 64 x 64 tiles of X, read along the update's rows and turned through LDS where X is its transpose. MOM && zero: the gradient is
// cleared behind its last reader
template <typename T, bool MOM>
__global__ __launch_bounds__(256) void ns_prep_kernel(NsTable tab, NsMomentum mo, const double* parts, char* ws, float eps, float scale, int zero) {
    ns_head head;
    const NsUnit& u = tab.units[ns_find<4>(tab, blockIdx.x, head)];
    __shared__ float s[NS_TILE_PREP][NS_TILE_PREP + 1];
    const int tj = (u.np + NS_TILE_PREP - 1) / NS_TILE_PREP, t = blockIdx.x - u.prep0;
    const int i0 = t / tj * NS_TILE_PREP, j0 = t % tj * NS_TILE_PREP;  // in X
    const int r0 = u.trans() ? j0 : i0, c0 = u.trans() ? i0 : j0;            // in the update
    constexpr int N = 16;  // all of a thread's; loaded before the norm is added up
    NsBatch<T, MOM, N> b;
    const bool whole = u.cs == 1 && r0 + NS_TILE_PREP <= u.rows && c0 + NS_TILE_PREP <= u.cols;  // a whole tile, along its rows: runs of 4
    const int tr = threadIdx.x / 16, tc = 4 * (threadIdx.x % 16);
    long long src[N];
    bool on[N];
    if (whole) {
        long long runs[N / 4], at[N / 4];
#pragma unroll
        for (int e = 0; e < N / 4; ++e) {
            runs[e] = src[4 * e] = (long long)(r0 + tr + 16 * e) * u.rs + c0 + tc;
            at[e] = (long long)(r0 + tr + 16 * e) * u.cols + c0 + tc;
        }
        b.load_runs(u, runs, at);
    } else {
        long long at[N];
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const int k = 256 * e + (int)threadIdx.x, r = r0 + k / NS_TILE_PREP, c = c0 + k % NS_TILE_PREP;
            on[e] = r < u.rows && c < u.cols;
            src[e] = (long long)r * u.rs + (long long)c * u.cs;
            at[e] = (long long)r * u.cols + c;
        }
        b.load(u, src, at, on);
    }
    double sum = 0.0;
    for (int i = threadIdx.x; i < u.nparts; i += 256) sum += parts[u.part0 + i];
    sum = ns_block_sum(sum);
    const NsNorm norm(sum, eps, scale);
    const double mul = norm.mul;
    if (t == 0 && threadIdx.x == 0) const_cast<NsUnit&>(u).x0 = norm.x0;  // for the launches behind this one
    if (whole) {
        if constexpr (MOM) {
            typedef T t4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
            if (zero) {
#pragma unroll
                for (int e = 0; e < N / 4; ++e) *(t4*)((T*)u.in + src[4 * e]) = t4{};
            }
        }
#pragma unroll
        for (int e = 0; e < N; ++e) s[tr + 16 * (e / 4)][tc + e % 4] = (float)((double)b.update(mo, e) * mul);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const int k = 256 * e + (int)threadIdx.x;
            if constexpr (MOM) {
                if (zero && on[e]) ((T*)u.in)[src[e]] = (T)0.f;
            }
            s[k / NS_TILE_PREP][k % NS_TILE_PREP] = on[e] ? (float)((double)b.update(mo, e) * mul) : 0.f;
        }
    }
    __syncthreads();
    f16_t* const X = (f16_t*)(ws + ns_x(u, 0));
    for (int k = threadIdx.x; k < NS_TILE_PREP * NS_TILE_PREP / 8; k += 256) {
        const int i = k / (NS_TILE_PREP / 8), j = 8 * (k % (NS_TILE_PREP / 8));
        if (i0 + i >= u.mp || j0 + j >= u.np) continue;  // np is a multiple of 32: groups of 8 are whole
        f16x8 h, l;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            f16_t a, b;
            ns_split(u.trans() ? s[j + e][i] : s[i][j + e], a, b);
            h[e] = a;
            l[e] = b;
        }
        f16_t* to = X + ns_at(i0 + i, j0 + j, u.np);
        *(f16x8*)to = h;
        *(f16x8*)(to + NS_LO) = l;
    }
}

// ---- the products -------------------------------------------------------------------------
// C[i][j] = sum_k P[i][k] Q[j][k]: a workgroup of 4 waves computes a 64 TW x 64 TW tile, wave (wi, wj) a quarter of it, in K steps of 32. The tile's rows of P
// and Q go to LDS by LDS-DMA into a ring of NST stages. In the accumulators i is on the lanes and j in the registers, four in a row.
enum NsKind { NS_GRAM = 0, NS_SQUARE = 1, NS_APPLY = 2, NS_LAST = 3 };  // A = X X^T; sq[out] = sq[p] sq[q] + ..; X = sq[p] X + ..; the same, the result
struct NsStep {
    float alpha, beta, beta2, diagonal;  // C <- alpha (P Q^T) + beta D + beta2 D2 + diagonal 1, on the scaled planes
    int p, q, d, d2, out;                // which m x m matrices
    int from;            // which of the two X planes is read
    float inv;           // 2^-e
    float lg, lg_next;   // bounds of X, read and written (ns_extra)
    int whole, split;    // tiles [0, whole) are computed by a workgroup each, the others in `split` pieces of their K steps
    float* slab;         // the pieces' sums
};

constexpr int ns_launch(int kind) { return kind == NS_GRAM ? 0 : kind == NS_SQUARE ? 1 : 2; }

// The tile of a run that its workgroup number `local` computes: workgroups b, b + 8, .. share an XCD and its L2, and get neighbouring tiles. A run is all units of
// one size: over a whole launch one XCD would get the units with the longest K, over one unit an XCD would read a part of every unit
DEVFN int ns_deal(int local, int first, int count) {
    const int d = first & 7, v = local + d, x = v & 7, end = count + d;
    const int base = (end >> 3) * x + min(end & 7, x) - min(d, x);  // tiles of the XCDs before this one
    const int lead = x >= d ? x : x + 8;
    return base + ((v - lead) >> 3);
}
typedef f16_t f16x4 __attribute__((ext_vector_type(4)));

// Stages of the ring: two where two or more workgroups share a CU and cover each other's waits (the default core's products back on X: 8.7 us, with four 10.8); four for the 64
// tile of symmetric products, whose launches have few of them (1024 x 1024: 14.3 us, with two 20.2); three for the 192 tile, alone on its CU
template <int TW, bool SYM>
struct NsTile {
    static constexpr int B = 64 * TW, PL = 2 * B * NS_BK, SIDE = 32 * TW;  // PL: elements of an operand's stage, hi and lo
    static constexpr int PIECES = PL * 2 / 1024 / 4;      // LDS-DMA instructions per wave and operand
    static constexpr int NST = TW == 3 ? 3 : TW == 1 && SYM ? 4 : 2;
    static constexpr int LDS = NST * 2 * PL;              // elements; the epilogue's fp32 tile fits
    static_assert(4 * SIDE * SIDE * 4 <= LDS * 2, "epilogue");
};

// where a tile lies and what it reads and writes
struct NsWhere {
    int bi, bj, i0, j0;
    const f16_t *D, *D2;
    f16_t* C;
    int ldd, cols;
};
template <int TW, int KIND>
DEVFN NsWhere ns_where(const NsUnit& u, char* ws, const NsStep& st, int t) {  // t: the unit's tile
    constexpr bool SYM = KIND == NS_GRAM || KIND == NS_SQUARE;
    constexpr int B = 64 * TW;
    NsWhere w;
    // tiles in blocks of 8 x 8, so that those that run together on an XCD share rows of P and Q in its L2
    if constexpr (SYM) {  // bi <= bj: for each 8 columns the rows above their diagonal block, row by row, then the block's own triangle
        int g = (int)((sqrtf(8.f * t + 1.f) - 1.f) * (0.5f / 8));
        while (4 * (g + 1) * (8 * (g + 1) + 1) <= t) ++g;
        while (4 * g * (8 * g + 1) > t) --g;
        const int width = min(8, (u.mp + B - 1) / B - 8 * g), r = t - 4 * g * (8 * g + 1);
        if (r < 8 * g * width) {
            w.bi = r / width;
            w.bj = 8 * g + r % width;
        } else {
            const int q = r - 8 * g * width;
            int c = 0;
            while ((c + 1) * (c + 2) / 2 <= q) ++c;
            w.bi = 8 * g + q - c * (c + 1) / 2;
            w.bj = 8 * g + c;
        }
    } else {
        const int ni = (u.mp + B - 1) / B, nj = (u.np + B - 1) / B, g = t / (8 * nj), r = t - g * 8 * nj, height = min(8, ni - 8 * g);
        w.bi = 8 * g + r % height;
        w.bj = r / height;
    }
    w.i0 = w.bi * B;
    w.j0 = w.bj * B;
    w.D = KIND == NS_SQUARE ? (const f16_t*)(ws + ns_square_at(u, st.d)) : (const f16_t*)(ws + ns_x(u, st.from));
    w.D2 = (const f16_t*)(ws + ns_square_at(u, st.d2));
    w.ldd = KIND == NS_SQUARE ? u.mp : u.np;
    w.C = (f16_t*)(ws + (KIND == NS_GRAM ? ns_square_at(u, 0) : KIND == NS_SQUARE ? ns_square_at(u, st.out) : ns_x(u, st.from ^ 1)));
    w.cols = SYM ? u.mp : u.np;
    return w;
}

// Between a lane's writes to its wave's LDS and another lane's reads of them. The hardware keeps a wave's LDS operations in order; the fences, which cost no instruction, keep
// the compiler to it: the barrier alone orders no memory, and to one lane the other's address need not alias its own
DEVFN void ns_wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Accumulators -> alpha acc + beta D -> planes (both triangles of a symmetric product), or the result. Each wave turns its part over in its own LDS, so that
// planes are read and written 16 B a lane along their rows - also the mirrored tile's - and the result along its own rows, whichever way the matrix lies.
// LDS image [SIDE][SIDE] fp32, 16-B chunks of a row swizzled by the row: writes by lanes of one column and reads along rows both spread over the banks.
template <int TW, int KIND, typename T>
DEVFN void ns_epilogue(const NsUnit& u, const NsWhere& w, const NsStep& st, f32x16 (&acc)[TW][TW], float* img, int wi, int wj, int lane) {
    constexpr bool SYM = KIND == NS_GRAM || KIND == NS_SQUARE;
    constexpr int SIDE = 32 * TW;
    auto chunk = [&](int i, int c) { return i * SIDE + 4 * (TW == 2 ? c ^ (i & 15) : c ^ (i >> 1 & 7)); };
    const int r = lane & 31, h = lane >> 5, extra = KIND == NS_SQUARE ? 0 : ns_extra(u.x0, st.lg);
    const float grown = KIND == NS_APPLY ? ldexpf(1.f, ns_extra(u.x0, st.lg_next) - extra) : KIND == NS_GRAM ? ldexpf(1.f, -2 * extra) : 1.f;
    const float alpha = st.alpha * grown, beta = st.beta * grown, inv = KIND == NS_LAST ? ldexpf(st.inv, -extra) : 0.f;
    const int iw = w.i0 + SIDE * wi, jw = w.j0 + SIDE * wj;
    const bool mirror = SYM && w.bi != w.bj;  // the lower triangle
    // what is added to the product, loaded before the image is written: one after the other, each would wait behind the stores of the one before (8192 x 1024 455 against
    // 446 us). The 192 tile's registers are full: there the batches are single (4096 x 4096's A A 236 us, in nines 255)
    constexpr int LOOPS = SIDE * SIDE / 512, N = TW == 3 ? 1 : LOOPS;
    f16x8 dh[N], dl[N], eh[N], el[N];
    auto load = [&](int k0) {
        if constexpr (KIND != NS_GRAM) {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int k = k0 + 64 * n + lane, i = iw + k / (SIDE / 8), j = jw + 8 * (k % (SIDE / 8));
                dh[n] = dl[n] = eh[n] = el[n] = f16x8{};
                if (i >= u.mp || j >= w.cols) continue;
                if (beta != 0.f) {
                    const f16_t* d = w.D + ns_at(i, j, w.ldd);
                    dh[n] = *(const f16x8*)d;
                    dl[n] = *(const f16x8*)(d + NS_LO);
                }
                if (KIND == NS_SQUARE && st.beta2 != 0.f) {
                    const f16_t* d = w.D2 + ns_at(i, j, w.ldd);
                    eh[n] = *(const f16x8*)d;
                    el[n] = *(const f16x8*)(d + NS_LO);
                }
            }
        }
    };
    if constexpr (N > 1) load(0);
#pragma unroll
    for (int ti = 0; ti < TW; ++ti)
#pragma unroll
        for (int tj = 0; tj < TW; ++tj)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x16& a = acc[ti][tj];
                *(f32x4*)(img + chunk(32 * ti + r, 8 * tj + 2 * q + h)) =
                    f32x4{alpha * a[4 * q], alpha * a[4 * q + 1], alpha * a[4 * q + 2], alpha * a[4 * q + 3]};
            }
    ns_wave_sync();
#pragma unroll 1
    for (int l = 0; l < LOOPS; l += N) {
        if constexpr (N == 1) load(64 * l);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int k = 64 * (l + n) + lane, il = k / (SIDE / 8), jl = 8 * (k % (SIDE / 8)), i = iw + il, j = jw + jl;
            if (i >= u.mp || j >= w.cols) continue;  // both are multiples of 32: groups of 8 are whole
            f32x4 v0 = *(const f32x4*)(img + chunk(il, jl / 4)), v1 = *(const f32x4*)(img + chunk(il, jl / 4 + 1));
            if constexpr (KIND != NS_GRAM) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v0[e] += beta * ((float)dh[n][e] + (float)dl[n][e]);
                    v1[e] += beta * ((float)dh[n][4 + e] + (float)dl[n][4 + e]);
                }
            }
            if constexpr (KIND == NS_SQUARE) {
                if (st.beta2 != 0.f) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        v0[e] += st.beta2 * ((float)eh[n][e] + (float)el[n][e]);
                        v1[e] += st.beta2 * ((float)eh[n][4 + e] + (float)el[n][4 + e]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (i == j + e && i < u.m()) v0[e] += st.diagonal;
                    if (i == j + 4 + e && i < u.m()) v1[e] += st.diagonal;
                }
            }
            if constexpr (KIND != NS_LAST) {
                f16x8 ch, cl;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    f16_t a, b;
                    ns_split(e < 4 ? v0[e] : v1[e - 4], a, b);
                    ch[e] = a;
                    cl[e] = b;
                }
                f16_t* to = w.C + ns_at(i, j, w.cols);
                *(f16x8*)to = ch;
                *(f16x8*)(to + NS_LO) = cl;
            }
            if (KIND == NS_LAST || (KIND == NS_SQUARE && mirror)) {
                *(f32x4*)(img + chunk(il, jl / 4)) = v0;
                *(f32x4*)(img + chunk(il, jl / 4 + 1)) = v1;
            }
        }
    }
    ns_wave_sync();
    auto at = [&](int il, int jl) { return img[chunk(il, jl / 4) + (jl & 3)]; };
    if constexpr (SYM) {
        if (!mirror) return;
        for (int k = lane; k < SIDE * SIDE / 8; k += 64) {
            const int jl = k / (SIDE / 8), il = 8 * (k % (SIDE / 8)), i = iw + il, j = jw + jl;
            if (i >= u.mp || j >= w.cols) continue;
            f16x8 ch, cl;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                f16_t a, b;
                ns_split(at(il + e, jl), a, b);
                ch[e] = a;
                cl[e] = b;
            }
            f16_t* to = w.C + ns_at(j, i, w.cols);
            *(f16x8*)to = ch;
            *(f16x8*)(to + NS_LO) = cl;
        }
    } else if constexpr (KIND == NS_LAST) {
        constexpr int N = 16;
        const bool trans = u.trans();
        const int row0 = trans ? jw : iw, col0 = trans ? iw : jw;
        if (row0 + SIDE <= u.rows && col0 + SIDE <= u.cols) {  // all of it: runs of 4
            typedef T t4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
            typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
            constexpr int R = 4;
            for (int k0 = 4 * lane; k0 < SIDE * SIDE; k0 += 256 * R) {
                long long x[R];
                f32x4 o[R];
                f4 wt[R];
#pragma unroll
                for (int q = 0; q < R; ++q) {
                    const int a = (k0 + 256 * q) / SIDE, b = (k0 + 256 * q) % SIDE;
                    x[q] = (long long)(row0 + a) * u.cols + col0 + b;
                    if (!u.out) wt[q] = *(const f4*)(u.w + x[q]);
                    if (trans) o[q] = f32x4{at(b, a), at(b + 1, a), at(b + 2, a), at(b + 3, a)};
                    else o[q] = *(const f32x4*)(img + chunk(a, b / 4));
                }
#pragma unroll
                for (int q = 0; q < R; ++q) {
                    t4 r;
                    f4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float y = o[q][e] * inv;
                        r[e] = (T)y;
                        if (!u.out) v[e] = u.decay * wt[q][e] - u.lr * y;
                    }
                    if (u.out) *(t4*)((T*)u.out + x[q]) = r;
                    else *(f4*)(u.w + x[q]) = v;
                }
            }
            return;
        }
        for (int k0 = lane; k0 < SIDE * SIDE; k0 += 64 * N) {  // a batch's loads of the weights stand together
            long long x[N];
            float o[N], wt[N];
            bool on[N];
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int a = (k0 + 64 * e) / SIDE, b = (k0 + 64 * e) % SIDE;  // b runs along the result's rows
                const int row = row0 + a, col = col0 + b;
                on[e] = row < u.rows && col < u.cols;
                x[e] = (long long)row * u.cols + col;
                o[e] = (trans ? at(b, a) : at(a, b)) * inv;
            }
            if (u.out) {
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (on[e]) ((T*)u.out)[x[e]] = (T)o[e];
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) wt[e] = on[e] ? u.w[x[e]] : 0.f;
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (on[e]) u.w[x[e]] = u.decay * wt[e] - u.lr * o[e];
            }
        }
    }
}

template <int TW, int KIND, typename T>
__global__ __launch_bounds__(256, TW == 3 ? 1 : 2) void ns_gemm_kernel(NsTable tab, char* ws, NsStep st) {
    constexpr bool SYM = KIND == NS_GRAM || KIND == NS_SQUARE, TR = !SYM;  // TR: Q is stored [k][j]
    using Tile = NsTile<TW, SYM>;
    constexpr int B = Tile::B, PL = Tile::PL, PIECES = Tile::PIECES, NST = Tile::NST;
    __shared__ __attribute__((aligned(16))) f16_t lds[Tile::LDS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wi = wave >> 1, wj = wave & 1;
    constexpr int W = ns_launch(KIND);
    const int b = blockIdx.x, over = b - st.whole;
    const bool piece = SYM && over >= 0;  // workgroup-uniform
    // the pieces K range by K range, an XCD's workgroups one behind the other: they read the same part of the rows
    int number = b, range = 0;
    if (piece) {
        const int pieces = (int)gridDim.x - st.whole, rest = pieces / st.split, at = ns_deal(over, st.whole, pieces);
        range = at / rest;
        number = st.whole + at - range * rest;
    }
    ns_head head;
    int unit = ns_find<W>(tab, number, head);
    if (!piece) {
        number = head[1] + ns_deal(b - head[1], head[1], SYM ? min(head[2], st.whole - head[1]) : head[2]);
        unit = ns_find<W>(tab, number, head);
    }
    const NsUnit& u = tab.units[unit];
    const NsWhere w = ns_where<TW, KIND>(u, ws, st, number - head[0]);
    const int steps = (KIND == NS_GRAM ? u.np : u.mp) / NS_BK, each = piece ? (steps + st.split - 1) / st.split : steps;
    const int t0 = range * each, nk = max(0, min(each, steps - t0));  // this workgroup's K steps
    const f16_t* X = (const f16_t*)(ws + ns_x(u, st.from));
    const f16_t* P = KIND == NS_GRAM ? X : (const f16_t*)(ws + ns_square_at(u, st.p));
    const f16_t* Q = KIND == NS_SQUARE ? (const f16_t*)(ws + ns_square_at(u, st.q)) : X;
    const int ldp = KIND == NS_GRAM ? u.np : u.mp, ldq = KIND == NS_SQUARE ? u.mp : u.np;

    // A 1-KB piece fills 64 16-B chunks of a stage in order; which 16 B of the tile's row a chunk holds is swizzled, so that the fragment reads below spread over all
    // 64 banks. Rows [.][32 hi, 32 lo]: eight chunks a row, chunk c at c ^ (row / 2 % 8). Q as [k][j]: the row's 64-B granules (32 hi or lo) g at g ^ (k % 4). A lane's
    // byte offset from the tile's first row is loop-invariant; pieces 1 .. 3 of a group of four go by the instruction's offset, which moves the LDS and the global
    // address alike: the lane offset carries BIAS - 1024 (p % 4), the base BIAS less.
    constexpr int BIAS = TileDma<32, 32>::BIAS;
    unsigned po[PIECES], qo[PIECES];
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int c = 64 * (wave * PIECES + p) + lane, row = c / 8, at = BIAS - 1024 * (p & 3) + 16 * ((c & 7) ^ (row >> 1 & 7));
        po[p] = (unsigned)min(row, u.mp - 1 - w.i0) * (unsigned)(4 * ldp) + at;
        if constexpr (TR) {
            const int k = c / (B / 4), g = (c % (B / 4) / 4) ^ (k & 3);  // B / 4 chunks a row; granules past the matrix' columns re-read its last block
            qo[p] = (unsigned)k * (unsigned)(4 * ldq) + 64 * min(g, (u.np - w.j0) / 16 - 2 + (g & 1)) + 16 * (c & 3) + BIAS - 1024 * (p & 3);
        } else {
            qo[p] = (unsigned)min(row, u.mp - 1 - w.j0) * (unsigned)(4 * ldq) + at;
        }
    }
    const char* pb = (const char*)(P + (size_t)w.i0 * (2 * ldp)) - BIAS;
    const char* qb = (const char*)(TR ? Q + 2 * w.j0 : Q + (size_t)w.j0 * (2 * ldq)) - BIAS;
    const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(const __attribute__((address_space(3))) void*)lds);
    auto uniform = [](const char* p) {
        const unsigned long long b = (unsigned long long)(uintptr_t)p;
        const unsigned hi = (unsigned)__builtin_amdgcn_readfirstlane((int)(b >> 32)), lo = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)b);
        return (const char*)(uintptr_t)(((unsigned long long)hi << 32) | lo);
    };
    auto issue = [&](int t, int buf) {
        const size_t pk = (size_t)(t0 + t) * (4 * NS_BK), qk = TR ? (size_t)(t0 + t) * NS_BK * (4 * ldq) : pk;
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const char* base = uniform(side ? qb + qk : pb + pk);
            const unsigned* o = side ? qo : po;
#pragma unroll
            for (int p = 0; p < PIECES; p += 4) {
                constexpr int LAST = PIECES % 4 ? PIECES % 4 : 4;
                const unsigned m0 = lds0 + 2u * (unsigned)((buf * 2 + side) * PL) + 1024u * (unsigned)(wave * PIECES + p);
                auto at = [&](int x) { return o[p + x < PIECES ? p + x : PIECES - 1]; };
                if (p + 4 <= PIECES) TileDma<32, 32>::template group<4>(base, m0, at(0), at(1), at(2), at(3));
                else TileDma<32, 32>::template group<LAST>(base, m0, at(0), at(1), at(2), at(3));
            }
        }
    };

    const int r = lane & 31, h = lane >> 5;
    auto row_frag = [&](const f16_t* img, int row0, int s, int lo) -> bf16x8 {  // rows row0 + (lane & 31), k = 16 s + 8 h ..
        return *(const bf16x8*)(img + (row0 + r) * (2 * NS_BK) + 8 * ((4 * lo + 2 * s + h) ^ (r >> 1 & 7)));
    };
    const int tg = lane >> 4, tq = lane >> 2 & 3, tp = lane & 3;
    auto col_frag = [&](const f16_t* img, int col0, int s, int lo) -> bf16x8 {  // columns col0 + (lane & 31), the same k
        const int k = 16 * s + 8 * (tg >> 1) + tq, g = (col0 / 16 + lo) ^ tq;
        const bf16_t* a = (const bf16_t*)img + k * (2 * B) + 32 * g + 16 * (tg & 1) + 4 * tp;
        const bf16x4 x = lds_tr_read(a), y = lds_tr_read(a + 4 * (2 * B));
        return bf16x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
    };

    f32x16 acc[TW][TW];
#pragma unroll
    for (int i = 0; i < TW; ++i)
#pragma unroll
        for (int j = 0; j < TW; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    // a stage's fragments: [K half][plane][32-block]
    struct Frags {
        bf16x8 ph[TW], pl[TW], qh[TW], ql[TW];
    };
    auto read = [&](Frags& f, int buf, int s) {
        const f16_t *p = lds + buf * 2 * PL, *q = p + PL;
        auto other = [&](int i, int lo) { return TR ? col_frag(q, 32 * (TW * wj + i), s, lo) : row_frag(q, 32 * (TW * wj + i), s, lo); };
#pragma unroll
        for (int i = 0; i < TW; ++i) {
            f.ph[i] = row_frag(p, 32 * (TW * wi + i), s, 0);
            f.ql[i] = other(i, 1);
        }
#pragma unroll
        for (int i = 0; i < TW; ++i) {
            f.qh[i] = other(i, 0);
            f.pl[i] = row_frag(p, 32 * (TW * wi + i), s, 1);
        }
    };
    auto multiply = [&](const Frags& f) {
#pragma unroll
        for (int x = 0; x < 3; ++x)
#pragma unroll
            for (int i = 0; i < TW; ++i)
#pragma unroll
                for (int j = 0; j < TW; ++j) acc[i][j] = mfma32h(x == 0 ? f.ql[j] : f.qh[j], x == 2 ? f.pl[i] : f.ph[i], acc[i][j]);
    };
    // every wave issues 2 PIECES operations per stage: "all but the newest stages have landed" is one counted wait
    constexpr int READS = TR ? 6 * TW : 4 * TW, MF = 3 * TW * TW;
    // the next fragments' reads go out between the products of the last
    auto interleave = [] {
#pragma unroll
        for (int x = 0; x < (READS < MF ? READS : MF); ++x) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, READS > MF ? 2 : 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, MF, 0);
    };
#pragma unroll
    for (int t = 0; t < NST - 1; ++t)
        if (t < nk) issue(t, t);
    int buf = 0;
    if constexpr (TW < 3) {
        for (int t = 0; t < nk; ++t) {
            if (t + NST - 1 <= nk) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * PIECES * (NST - 2)) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();  // stage t is there for all; the stage before it has been read by all
            Frags f0, f1;
            read(f0, buf, 0);
            if (t + NST - 1 < nk) issue(t + NST - 1, buf == 0 ? NST - 1 : buf - 1);
            read(f1, buf, 1);
            multiply(f0);
            multiply(f1);
            interleave();
            buf = buf + 1 == NST ? 0 : buf + 1;
        }
    } else if (nk > 0) {
        // one wave a SIMD: nothing else covers a wait, so fragments are read across the barrier, too. In the middle of stage t, when its second half has been read,
        // stage t + 1 is waited for and its first half read between the products of t's second
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        Frags f0, f1;
        read(f0, 0, 0);
        for (int t = 0; t < nk; ++t) {
            const int next = buf + 1 == NST ? 0 : buf + 1;
            if (t + 2 < nk) issue(t + 2, next + 1 == NST ? 0 : next + 1);  // the buffer of stage t - 1: read by all before the barrier below, an iteration ago
            read(f1, buf, 1);
            multiply(f0);
            interleave();
            if (t + 2 < nk) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * PIECES) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (t + 1 < nk) read(f0, next, 0);
            multiply(f1);
            interleave();
            buf = next;
        }
    }
    if (piece) {  // its sums in the accumulators' order; ns_join_kernel adds the pieces up
        float* to = st.slab + ((size_t)((number - st.whole) * st.split + range) * 4 + wave) * (TW * TW * 1024) + 4 * lane;
#pragma unroll
        for (int i = 0; i < TW; ++i)
#pragma unroll
            for (int j = 0; j < TW; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) *(f32x4*)(to + ((i * TW + j) * 4 + q) * 256) = f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        return;
    }
    __syncthreads();
    ns_epilogue<TW, KIND, T>(u, w, st, acc, (float*)lds + wave * (32 * TW) * (32 * TW), wi, wj, lane);
}

// The pieces of the split tiles, added up in their order, and the epilogue: one wave per 32 x 32 of a tile (one per quarter of a 128 tile took 12 us for 36 tiles of 7 pieces)
template <int TW, int KIND>
__global__ __launch_bounds__(64) void ns_join_kernel(NsTable tab, char* ws, NsStep st) {
    constexpr int W = ns_launch(KIND), BLOCKS = 4 * TW * TW;
    __shared__ __attribute__((aligned(16))) float lds[32 * 32];
    const int lane = threadIdx.x, tile = blockIdx.x / BLOCKS, block = blockIdx.x % BLOCKS, wave = block / (TW * TW), ij = block % (TW * TW);
    ns_head head;
    const NsUnit& u = tab.units[ns_find<W>(tab, st.whole + tile, head)];
    NsWhere w = ns_where<TW, KIND>(u, ws, st, st.whole + tile - head[0]);
    w.i0 += 32 * (TW * (wave >> 1) + ij / TW);
    w.j0 += 32 * (TW * (wave & 1) + ij % TW);
    f32x16 acc[1][1];
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[0][0][e] = 0.f;
    const float* from = st.slab + ((size_t)tile * st.split * 4 + wave) * (TW * TW * 1024) + ij * 1024 + 4 * lane;
#pragma unroll 4
    for (int p = 0; p < st.split; ++p, from += 4 * TW * TW * 1024) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x4 v = *(const f32x4*)(from + q * 256);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[0][0][4 * q + e] += v[e];
        }
    }
    ns_epilogue<1, KIND, float>(u, w, st, acc, lds, 0, 0, lane);
}

// ---- small matrices -----------------------------------------------------------------------
// A matrix whose planes fit a CU's LDS goes through all its steps in one workgroup: what the products above cost there is their launches (155 x 64:
// 18 launches, 105 us; this 33: 15 products one behind the other, each a few dependent MFMAs and a barrier). X, A and S lie in LDS as two planes each, rows 16 B longer than their numbers, so that neighbouring rows start in other
// banks. The waves share the 32 x 32 tiles of A, S and X; a single tile of A
// is computed in quarters of K by four of them.
constexpr int NS_LDS = 150 * 1024, NS_PAD = 8, NS_SCRATCH = 4 * 32 * 32 * 4;
constexpr int ns_small_bytes(int mp, int np) { return 4 * mp * (np + NS_PAD) + 8 * mp * (mp + NS_PAD) + (mp == 32 ? NS_SCRATCH : 0); }
bool ns_small(int rows, int cols) {
    const int m = std::min(rows, cols), n = std::max(rows, cols);
    return m <= 96 && n <= 2048 && ns_small_bytes(round_up(m, 32), round_up(n, 32)) <= NS_LDS;
}

constexpr int ns_small_threads(int t32) { return t32 == 3 ? 512 : 1024; }

struct NsCoefficients {
    float c[3 * NS_MAX_STEPS], lg[NS_MAX_STEPS + 1];
};

template <int T32, typename T, bool MOM>
__global__ __launch_bounds__(ns_small_threads(T32)) void ns_small_kernel(NsChunk units, NsMomentum mo, NsCoefficients co, int steps, float eps, float scale, int zero) {
    constexpr int MP = 32 * T32, LDA = MP + NS_PAD, NT = ns_small_threads(T32), WAVES = NT / 64;
    __shared__ __attribute__((aligned(16))) char lds[NS_LDS];
    const NsUnit& u = units.u[blockIdx.x];
    const int LDX = u.np + NS_PAD, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, h = lane >> 5;
    f16_t* const X = (f16_t*)lds;             // hi, lo: [MP][LDX]
    f16_t* const A = X + 2 * MP * LDX;        // hi, lo: [MP][LDA]
    f16_t* const S = A + 2 * MP * LDA;
    float* const scratch = (float*)(S + 2 * MP * LDA);
    const int xlo = MP * LDX, alo = MP * LDA;
    const float inv = 1.f / scale;            // a power of two
    const int all = u.rows * u.cols;

    auto row_of = [&](int k) { return u.cols == 1 ? k : (int)__umulhi((unsigned)k, (unsigned)u.part); };  // part: 2^32 / cols, rounded up
    // the norm (and the momentum), then the planes
    constexpr int N = 8;
    auto batch = [&](int k0, NsBatch<T, MOM, N>& b, long long (&src)[N], long long (&at)[N], bool (&on)[N]) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const int k = k0 + NT * e + (int)threadIdx.x, row = row_of(k);
            on[e] = k < all;
            at[e] = k;
            src[e] = (long long)row * u.rs + (long long)(k - row * u.cols) * u.cs;
        }
        b.load(u, src, at, on);
    };
    double sum = 0.0;
    for (int k0 = 0; k0 < all; k0 += NT * N) {
        NsBatch<T, MOM, N> b;
        long long src[N], at[N];
        bool on[N];
        batch(k0, b, src, at, on);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            if constexpr (MOM) {
                b.m[e] = mo.mu * b.m[e] + b.g[e];
                if (on[e]) u.mom[at[e]] = b.m[e];
            }
            const double v = (double)b.update(mo, e);
            sum += v * v;
        }
    }
    sum = ns_block_sum<NT>(sum);
    const NsNorm norm(sum, eps, scale);
    const double mul = norm.mul;
    const float x0 = norm.x0;
    for (int k = threadIdx.x; k < 2 * MP * LDX / 8; k += NT) *(f16x8*)(X + 8 * k) = f16x8{};
    __syncthreads();
    for (int k0 = 0; k0 < all; k0 += NT * N) {  // the momentum was written by this thread
        NsBatch<T, MOM, N> b;
        long long src[N], at[N];
        bool on[N];
        batch(k0, b, src, at, on);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            if (!on[e]) continue;
            if constexpr (MOM) {
                if (zero) ((T*)u.in)[src[e]] = (T)0.f;
            }
            const int row = row_of((int)at[e]), col = (int)at[e] - row * u.cols, x = u.trans() ? col * LDX + row : row * LDX + col;
            ns_split((float)((double)b.update(mo, e) * mul), X[x], X[xlo + x]);
        }
    }
    __syncthreads();

    auto row_frag = [&](const f16_t* img, int ld, int row0, int k) -> bf16x8 { return *(const bf16x8*)(img + (row0 + r) * ld + k + 8 * h); };
    auto zeros = [](f32x16& a) {
#pragma unroll
        for (int e = 0; e < 16; ++e) a[e] = 0.f;
    };
    // 4 of a row in two planes
    auto get = [&](const f16_t* img, int lo, int x, int e) { return (float)img[x + e] + (float)img[lo + x + e]; };
    auto put = [&](f16_t* img, int lo, int x, const f32x4& v) {
        f16x4 a, b;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f16_t p, q;
            ns_split(v[e], p, q);
            a[e] = p;
            b[e] = q;
        }
        *(f16x4*)(img + x) = a;
        *(f16x4*)(img + lo + x) = b;
    };
    // tile (ti, tj) of P P^T over k in [k0, k1): i on the lanes, j in the registers
    auto product = [&](const f16_t* P, int ld, int lo, int ti, int tj, int k0, int k1) {
        f32x16 acc;
        zeros(acc);
#pragma unroll 4
        for (int k = k0; k < k1; k += 16) {
            const bf16x8 ph = row_frag(P, ld, 32 * ti, k), pl = row_frag(P + lo, ld, 32 * ti, k);
            const bf16x8 qh = row_frag(P, ld, 32 * tj, k), ql = row_frag(P + lo, ld, 32 * tj, k);
            acc = mfma32h(ql, ph, acc);
            acc = mfma32h(qh, pl, acc);
            acc = mfma32h(qh, ph, acc);
        }
        return acc;
    };
    for (int step = 0; step < steps; ++step) {
        const float a = co.c[3 * step], b = co.c[3 * step + 1], c = co.c[3 * step + 2];
        const int extra = ns_extra(x0, co.lg[step]);
        const float gram = ldexpf(inv, -2 * extra), grown = ldexpf(1.f, ns_extra(x0, co.lg[step + 1]) - extra);
        if constexpr (T32 == 1) {
            const int quarter = (u.np / 16 + 3) / 4 * 16;
            if (wave < 4) {
                const f32x16 acc = product(X, LDX, xlo, 0, 0, min(u.np, wave * quarter), min(u.np, (wave + 1) * quarter));
#pragma unroll
                for (int e = 0; e < 16; ++e) scratch[(wave * 16 + e) * 64 + lane] = acc[e];
            }
            __syncthreads();
            if (wave == 0) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    f32x4 v{};
#pragma unroll
                    for (int w = 0; w < 4; ++w)
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] += gram * scratch[(w * 16 + 4 * q + e) * 64 + lane];
                    put(A, alo, r * LDA + 8 * q + 4 * h, v);
                }
            }
        } else {
            for (int t = wave; t < T32 * T32; t += WAVES) {
                const f32x16 acc = product(X, LDX, xlo, t / T32, t % T32, 0, u.np);
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    put(A, alo, (32 * (t / T32) + r) * LDA + 32 * (t % T32) + 8 * q + 4 * h,
                        f32x4{gram * acc[4 * q], gram * acc[4 * q + 1], gram * acc[4 * q + 2], gram * acc[4 * q + 3]});
            }
        }
        __syncthreads();
        for (int t = wave; t < T32 * T32; t += WAVES) {
            const f32x16 acc = product(A, LDA, alo, t / T32, t % T32, 0, MP);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int x = (32 * (t / T32) + r) * LDA + 32 * (t % T32) + 8 * q + 4 * h;
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = c * inv * acc[4 * q + e] + b * get(A, alo, x, e);
                put(S, alo, x, v);
            }
        }
        __syncthreads();
        // tile (i, j) of X: all its tiles are computed before the first is written
        constexpr int MOST = T32 == 3 ? 3 : 2;  // tiles a wave, at the widest X that fits
        const int tiles = T32 * (u.np / 32);
        f32x16 acc[MOST];
#pragma unroll
        for (int n = 0; n < MOST; ++n) {
            const int t = wave + WAVES * n, i = t % T32, j0 = 32 * (t / T32);
            zeros(acc[n]);
            if (t < tiles)
#pragma unroll
                for (int k = 0; k < MP; k += 16) {
                    const bf16x8 qh = lds_tr_frag_nat((const bf16_t*)X, LDX, k, j0, lane), ql = lds_tr_frag_nat((const bf16_t*)(X + xlo), LDX, k, j0, lane);
                    const bf16x8 ph = row_frag(S, LDA, 32 * i, k), pl = row_frag(S + alo, LDA, 32 * i, k);
                    acc[n] = mfma32h(ql, ph, acc[n]);
                    acc[n] = mfma32h(qh, pl, acc[n]);
                    acc[n] = mfma32h(qh, ph, acc[n]);
                }
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < MOST; ++n) {
            const int t = wave + WAVES * n, i = t % T32, j0 = 32 * (t / T32);
            if (t < tiles)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int x = (32 * i + r) * LDX + j0 + 8 * q + 4 * h;
                    f32x4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = (grown * inv) * acc[n][4 * q + e] + (grown * a) * get(X, xlo, x, e);
                    put(X, xlo, x, v);
                }
        }
        __syncthreads();
    }
    const float back = ldexpf(inv, -ns_extra(x0, co.lg[steps]));
    for (int k0 = threadIdx.x; k0 < all; k0 += NT * N) {
        float wt[N];
        if (!u.out) {
#pragma unroll
            for (int e = 0; e < N; ++e) wt[e] = k0 + NT * e < all ? u.w[k0 + NT * e] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const int k = k0 + NT * e;
            if (k >= all) continue;
            const int row = row_of(k), col = k - row * u.cols, x = u.trans() ? col * LDX + row : row * LDX + col;
            const float o = get(X, xlo, x, 0) * back;
            if (u.out) ((T*)u.out)[k] = (T)o;
            else u.w[k] = u.decay * wt[e] - u.lr * o;
        }
    }
}

// no steps: the normalised update itself
template <typename T>
__global__ __launch_bounds__(256) void ns_copy_kernel(NsTable tab, const char* ws, float inv) {
    ns_head head;
    const NsUnit& u = tab.units[ns_find<4>(tab, blockIdx.x, head)];
    const int tj = (u.np + NS_TILE_PREP - 1) / NS_TILE_PREP, t = blockIdx.x - u.prep0;
    const int i0 = t / tj * NS_TILE_PREP, j0 = t % tj * NS_TILE_PREP;
    const f16_t* X = (const f16_t*)(ws + ns_x(u, 0));
    for (int k = threadIdx.x; k < NS_TILE_PREP * NS_TILE_PREP; k += 256) {
        const int i = i0 + k / NS_TILE_PREP, j = j0 + k % NS_TILE_PREP;
        if (i >= u.m() || j >= u.n) continue;
        const long long at = u.trans() ? (long long)j * u.cols + i : (long long)i * u.cols + j;
        const f16_t* from = X + ns_at(i, j, u.np);
        const float o = ((float)from[0] + (float)from[NS_LO]) * ldexpf(inv, -ns_extra(u.x0, 0.f));
        if (u.out) ((T*)u.out)[at] = (T)o;
        else u.w[at] = u.decay * u.w[at] - u.lr * o;
    }
}

// ---- host ---------------------------------------------------------------------------------
// A product's launch: tiles of 64 tw, the first `whole` computed whole, the others in `split` pieces
struct NsPlan {
    int tw = 1, tiles = 0, whole = 0, split = 1;
    double us = 0.0;
    int grid() const { return whole + (tiles - whole) * split; }
    int joined() const { return tiles - whole; }
    long long slab() const { return split > 1 ? (long long)(tiles - whole) * split * 16384ll * tw * tw : 0; }
};
struct NsLayout {
    long long table = 0, heads = 0, parts = 0, slab = 0, bytes = 0;
    int nparts = 0, nprep = 0;
    bool pairs = false;  // two steps at once
    NsPlan gram, poly, full;
};
// elements per partial sum, and how many sums
std::pair<int, int> ns_parts(long long elements) {
    const long long part = std::max<long long>(NS_PART, (elements + 1023) / 1024);
    return {(int)part, (int)((elements + part - 1) / part)};
}

// Tile (64, 128 or 192) and split of a product with t[.] tiles of each size whose K steps sum to k[.], at the least estimated time. A CU holds two workgroups of
// the smaller tiles, one of the largest. Measured, us per K step and round: 64 0.25 alone on its CU, 0.55 where a few CUs hold two and 0.85 where all do (power); 128 0.9,
// 1.25 and 1.6; 192 1.6 (so 128 does twice the work of 64 in a time, where there is enough of it; 192 does 1.13 times that of 128 where it fills the chip once,
// 2.25 times where 128 would leave one a CU); epilogues 1.5, 5 and 9; the launch that joins pieces 4, and their sums at 5 TB/s. Only tiles of the last, part-filled round
// are split, in pieces of at least 4 steps: all of them, or those beyond one a CU, whose pieces then run beside the whole ones (two of 2000 x 2000, 272
// tiles of 128: 1195 us a call, 1292 unsplit; twelve 777 x 1301, 336 tiles: 928 and 915, and the estimate leaves them whole).
// 8192 x 1024's Gram matrix, 36 tiles of 128 in seven pieces each, takes 35 us and 7 to join them; as 136 whole tiles of 64 it took 107.
// Where it is off: launches of less than a round. A product of two 1024 x 1024 is estimated 9.5 us and takes 14 (every XCD's L2 takes the operands in anew), the default core's
// A A 2.8 and 6.2, its Gram matrices 6.2 and 9.6; a product of 4096 x 4096 with X 420 and 360. What is compared - tiles and splits of one product - is off alike.
NsPlan ns_plan(const long long (&t)[3], const long long (&k)[3], bool may_split) {
    constexpr int CUS = 256;
    constexpr double FULL[3] = {0.85, 1.6, 1.6}, SOME[3] = {0.55, 1.25, 1.6}, ALONE[3] = {0.25, 0.9, 1.6}, TAIL[3] = {1.5, 5.0, 9.0};
    NsPlan best;
    double least = 1e30;
    for (int tw = 1; tw <= 3; ++tw) {
        const int slots = tw == 3 ? CUS : 2 * CUS;
        const long long tiles = t[tw - 1];
        const double steps = (double)k[tw - 1] / (double)tiles;
        auto step = [&](long long w) { return w <= CUS ? ALONE[tw - 1] : SOME[tw - 1] + (FULL[tw - 1] - SOME[tw - 1]) * (double)(w - CUS) / CUS; };
        auto round = [&](double k, long long w) { return w == 0 ? 0.0 : TAIL[tw - 1] + k * step(w); };
        for (int split = 1; split <= (may_split ? 16 : 1); ++split)
            for (int beside = 0; beside < (split > 1 && tw < 3 ? 2 : 1); ++beside) {  // pieces alone behind whole rounds, or beside one whole tile a CU
                const long long whole = split == 1 ? tiles : beside ? tiles / CUS * CUS : tiles / slots * slots, rest = tiles - whole, pieces = rest * split;
                if (beside && whole % slots != CUS) continue;
                if (split > 1 && (rest == 0 || pieces > (beside ? CUS : slots) || steps < 4 * split)) continue;
                double us = (double)(whole / slots) * round(steps, slots) + round(steps, beside ? 0 : whole % slots);
                if (beside) us += 4.0 + round(steps / split, CUS + pieces) + (steps - steps / split) * step(CUS);
                else if (split > 1) us += round(steps / split, pieces);
                if (split > 1) us += 4.0 + (double)pieces * tw * tw * 16384.0 * 2.0 / 5e6;
                if (us < least) {
                    least = us;
                    best.us = us; best.tw = tw; best.tiles = (int)tiles; best.whole = (int)whole; best.split = split;
                }
            }
    }
    return best;
}

// Places every unit's planes. `shape(i, rows, cols)`; `put` receives the filled units in the order of the table.
template <typename Shape, typename Put>
int ns_layout(int n, Shape shape, Put put, NsLayout& l) {
    if (n > NS_MAX_UNITS) return V1T_ERR_UNSUPPORTED;
    long long nparts = 0, prep = 0;
    long long gt[3] = {}, gk[3] = {}, pk[3] = {}, ft[3] = {}, fk[3] = {};  // tiles and K steps: 64, 128, 192
    std::vector<int> order(n);
    std::vector<std::pair<int, int>> size(n);
    for (int i = 0; i < n; ++i) {
        int rows, cols;
        shape(i, rows, cols);
        if (rows < 1 || cols < 1) return V1T_ERR_ARG;
        const long long m = std::min(rows, cols), nn = std::max(rows, cols);
        if (m > 32768 || nn > (1 << 22) || m * nn > (1ll << 31)) return V1T_ERR_UNSUPPORTED;
        size[i] = {(int)nn, (int)m};
        order[i] = i;
        for (int k = 0; k < 3; ++k) {
            const long long B = 64 * (k + 1), mp = round_up((int)m, NS_BK), np = round_up((int)nn, NS_BK), a = (mp + B - 1) / B, b = (np + B - 1) / B;
            gt[k] += a * (a + 1) / 2; gk[k] += a * (a + 1) / 2 * (np / NS_BK); pk[k] += a * (a + 1) / 2 * (mp / NS_BK);
            ft[k] += a * b; fk[k] += a * b * (mp / NS_BK);
        }
        nparts += ns_parts(m * nn).second;
        prep += (m / NS_TILE_PREP + 1) * (nn / NS_TILE_PREP + 1);
    }
    if (std::max(std::max(gt[0], ft[0]), std::max(nparts, prep)) >= (1 << 24)) return V1T_ERR_UNSUPPORTED;  // a launch has less than 2^32 threads
    if (n == 0) return V1T_OK;
    // the tiles with the longest K first: what is left for the last round is short
    std::sort(order.begin(), order.end(), [&](int a, int b) { return size[a] != size[b] ? size[a] > size[b] : a < b; });
    l.gram = ns_plan(gt, gk, true);
    l.poly = ns_plan(gt, pk, true);
    l.full = ns_plan(ft, fk, false);
    // two steps: gram, poly, full each twice, or gram, five m x m products, full; 3 us a launch. 8192 x 1024, four steps: 350 us in pairs, 420 one by one; 4096 x 4096's products are
    // all of one size, and it stays step by step. One plan serves all matrices of a call
    l.pairs = l.gram.us + 5 * l.poly.us + l.full.us + 21.0 < 0.9 * (2 * (l.gram.us + l.poly.us + l.full.us) + 18.0);
    l.table = 0;
    l.heads = ns_align((long long)n * (long long)sizeof(NsUnit));
    l.parts = ns_align(l.heads + 5ll * n * (long long)sizeof(ns_head));
    l.slab = ns_align(l.parts + 8 * nparts);
    long long at = ns_align(l.slab + std::max(l.gram.slab(), l.poly.slab()));
    int part = 0, first = 0, next[3] = {}, group0[3] = {}, group[3] = {};
    for (int k = 0; k < n; ++k) {
        NsUnit u{};
        shape(order[k], u.rows, u.cols);
        u.n = std::max(u.rows, u.cols);
        u.mp = round_up(std::min(u.rows, u.cols), NS_BK); u.np = round_up(u.n, NS_BK);
        u.base = at;
        at = ns_square_at(u, l.pairs ? 4 : 2);
        const auto ps = ns_parts((long long)u.rows * u.cols);
        u.part = ps.first; u.nparts = ps.second; u.part0 = part; u.prep0 = first;
        part += u.nparts;
        first += ((u.mp + NS_TILE_PREP - 1) / NS_TILE_PREP) * ((u.np + NS_TILE_PREP - 1) / NS_TILE_PREP);
        auto tiles = [&](int kind) {
            const NsPlan& p = kind == 0 ? l.gram : kind == 1 ? l.poly : l.full;
            const int a = (u.mp + 64 * p.tw - 1) / (64 * p.tw), b = (u.np + 64 * p.tw - 1) / (64 * p.tw);
            return kind < 2 ? a * (a + 1) / 2 : a * b;
        };
        if (k == 0 || size[order[k]] != size[order[k - 1]]) {
            int same = 1;
            while (k + same < n && size[order[k + same]] == size[order[k]]) ++same;
            for (int kind = 0; kind < 3; ++kind) {
                group0[kind] = next[kind];
                group[kind] = same * tiles(kind);
            }
        }
        for (int kind = 0; kind < 3; ++kind) {
            u.first[kind] = next[kind];
            u.group0[kind] = group0[kind];
            u.group[kind] = group[kind];
            next[kind] += tiles(kind);
        }
        put(k, order[k], u);
    }
    l.nparts = part; l.nprep = first;
    l.bytes = at;
    return V1T_OK;
}

// The exponent of the planes' common scale: 2^15 over the largest number of any plane. A step maps a singular value s in [0, top] to a s + b s^3 + c s^5;
// X, A = X X^T, S and, where steps are taken in pairs, T, the next A, S' and Q are bounded by their spectral norms. lg: before each step (and behind the last),
// the logarithm of the product of the largest factors a + b s^2 + c s^4 so far. The maxima are sampled, 0.1 % of a
// singular value and 1 % of the rest are added for what lies between the samples and for rounding.
struct NsScale {
    int exponent = 0;
    float lg[NS_MAX_STEPS + 1] = {};
};
bool ns_scale_of(const float* coefficients, int steps, bool pairs, NsScale& scale) {
    double top = 1.001, most = top, lg = 0.0;
    for (int k = 0; k < steps; ++k) {
        const float* f = coefficients + 3 * k;
        for (int e = 0; e < 3; ++e)
            if (!std::isfinite(f[e])) return false;
        const bool pair = pairs && k + 1 < steps;
        double next = 0.0, factor = std::ldexp(1.0, -20);
        scale.lg[k] = (float)lg;
        for (int i = 0; i <= 4096; ++i) {
            const double s = top * i / 4096.0, t = s * s, poly = t * (f[1] + t * f[2]);
            double by = f[0] + poly;
            most = std::max({most, t, std::fabs(poly)});
            if (pair) {
                const double a1 = f[3], t1 = t * by * by, poly1 = t1 * (f[4] + t1 * f[5]);
                most = std::max({most, std::fabs(t * by), t1, std::fabs(poly1), std::fabs((a1 + poly1) * by), std::fabs((a1 + poly1) * by - a1 * f[0])});
                by *= a1 + poly1;
            }
            next = std::max(next, std::fabs(s * by));
            factor = std::max(factor, std::fabs(by));
        }
        if (pair) scale.lg[++k] = (float)lg;  // not asked for
        lg += std::log2(1.01 * factor);
        top = 1.001 * next;
        most = std::max(most, top);
        if (!(most < 128.0)) return false;
    }
    scale.lg[steps] = (float)lg;
    scale.exponent = (int)std::floor(std::log2(32768.0 / (1.01 * most)));
    return true;
}

// the same, remembered for the coefficients of the calling thread's last calls (the samples cost more than the launches); nullptr: refused
const NsScale* ns_scale(const float* coefficients, int steps, bool pairs) {
    struct Known {
        float c[3 * NS_MAX_STEPS];
        int steps = -1;
        bool ok = false;
        NsScale scale;
    };
    static thread_local Known known[2];
    Known& k = known[pairs];
    if (k.steps != steps || (steps > 0 && std::memcmp(k.c, coefficients, sizeof(float) * 3 * steps) != 0)) {
        k.steps = -1;
        k.ok = ns_scale_of(coefficients, steps, pairs, k.scale);
        if (steps > 0) std::memcpy(k.c, coefficients, sizeof(float) * 3 * steps);
        k.steps = steps;
    }
    return k.ok ? &k.scale : nullptr;
}

template <int KIND, typename T>
int ns_gemm(const NsLayout& l, const NsTable& table, char* ws, NsStep st, hipStream_t s) {
    const NsPlan& p = KIND == NS_GRAM ? l.gram : KIND == NS_SQUARE ? l.poly : l.full;
    st.whole = p.whole; st.split = p.split; st.slab = (float*)(ws + l.slab);
    if (p.tw == 3) hipLaunchKernelGGL((ns_gemm_kernel<3, KIND, T>), dim3(p.grid()), dim3(256), 0, s, table, ws, st);
    else if (p.tw == 2) hipLaunchKernelGGL((ns_gemm_kernel<2, KIND, T>), dim3(p.grid()), dim3(256), 0, s, table, ws, st);
    else hipLaunchKernelGGL((ns_gemm_kernel<1, KIND, T>), dim3(p.grid()), dim3(256), 0, s, table, ws, st);
    if constexpr (KIND == NS_GRAM || KIND == NS_SQUARE)
        if (p.joined()) {
            if (p.tw == 3) hipLaunchKernelGGL((ns_join_kernel<3, KIND>), dim3(36 * p.joined()), dim3(64), 0, s, table, ws, st);
            else if (p.tw == 2) hipLaunchKernelGGL((ns_join_kernel<2, KIND>), dim3(16 * p.joined()), dim3(64), 0, s, table, ws, st);
            else hipLaunchKernelGGL((ns_join_kernel<1, KIND>), dim3(4 * p.joined()), dim3(64), 0, s, table, ws, st);
        }
    return hipGetLastError() == hipSuccess ? V1T_OK : V1T_ERR_LAUNCH;
}

#define NS_TRY(x) do { const int rc_ = (x); if (rc_ != V1T_OK) return rc_; } while (0)

NsStep ns_square(int out, int p, int q, float alpha, int d, float beta, int d2 = 0, float beta2 = 0.f, float diagonal = 0.f) {
    NsStep st{};
    st.alpha = alpha; st.p = p; st.q = q; st.d = d; st.beta = beta; st.d2 = d2; st.beta2 = beta2; st.diagonal = diagonal; st.out = out;
    return st;
}

template <typename T>
int ns_steps(const NsLayout& l, const NsTable& table, char* ws, int steps, const float* co, bool pairs, const NsScale& scale, hipStream_t s) {
    enum { A = 0, S = 1, U = 2, S1 = 3 };  // the m x m matrices; U holds T, then Q
    const float inv = std::ldexp(1.f, -scale.exponent);
    int from = 0;
    for (int k = 0; k < steps; ++k) {
        const float a = co[3 * k], b = co[3 * k + 1], c = co[3 * k + 2];
        NsStep st{};
        st.alpha = inv; st.from = from; st.inv = inv; st.lg = scale.lg[k];
        NS_TRY((ns_gemm<NS_GRAM, float>(l, table, ws, st, s)));
        NS_TRY((ns_gemm<NS_SQUARE, float>(l, table, ws, ns_square(S, A, A, c * inv, A, b), s)));
        st.p = S; st.beta = a;
        if (pairs && k + 1 < steps) {
            const float a1 = co[3 * k + 3], b1 = co[3 * k + 4], c1 = co[3 * k + 5];
            NS_TRY((ns_gemm<NS_SQUARE, float>(l, table, ws, ns_square(U, S, A, inv, A, a), s)));
            NS_TRY((ns_gemm<NS_SQUARE, float>(l, table, ws, ns_square(A, S, U, inv, U, a), s)));
            NS_TRY((ns_gemm<NS_SQUARE, float>(l, table, ws, ns_square(S1, A, A, c1 * inv, A, b1), s)));
            NS_TRY((ns_gemm<NS_SQUARE, float>(l, table, ws, ns_square(U, S1, S, inv, S, a1, S1, a, k == 0 ? 0.f : std::ldexp(a * a1, scale.exponent)), s)));
            st.p = U; st.beta = k == 0 ? a * a1 : 0.f;
            ++k;
        }
        st.lg_next = scale.lg[k + 1];
        if (k + 1 < steps) NS_TRY((ns_gemm<NS_APPLY, float>(l, table, ws, st, s)));
        else NS_TRY((ns_gemm<NS_LAST, T>(l, table, ws, st, s)));
        from ^= 1;
    }
    return V1T_OK;
}

template <typename T, bool MOM>
int ns_run(const NsLayout& l, int n, char* ws, const NsMomentum& mo, float eps, int zero, int steps, const float* co, hipStream_t s) {
    const NsScale* paired = l.pairs ? ns_scale(co, steps, true) : nullptr;  // coefficients whose pairs would leave the planes' range go step by step
    const NsScale* scale = paired ? paired : ns_scale(co, steps, false);
    if (!scale) return V1T_ERR_ARG;
    const bool pairs = paired != nullptr;
    const int exponent = scale->exponent;
    const NsTable table{(const NsUnit*)(ws + l.table), (const ns_head*)(ws + l.heads), n};
    double* parts = (double*)(ws + l.parts);
    hipLaunchKernelGGL((ns_norm_kernel<T, MOM>), dim3(l.nparts), dim3(256), 0, s, table, mo, parts);
    hipLaunchKernelGGL((ns_prep_kernel<T, MOM>), dim3(l.nprep), dim3(256), 0, s, table, mo, parts, ws, eps, std::ldexp(1.f, exponent), zero);
    if (hipGetLastError() != hipSuccess) return V1T_ERR_LAUNCH;
    if (steps == 0) {
        hipLaunchKernelGGL((ns_copy_kernel<T>), dim3(l.nprep), dim3(256), 0, s, table, ws, std::ldexp(1.f, -exponent));
        return hipGetLastError() == hipSuccess ? V1T_OK : V1T_ERR_LAUNCH;
    }
    return ns_steps<T>(l, table, ws, steps, co, pairs, *scale, s);
}

// the matrices that go through the products, by their numbers
template <typename Shape>
std::vector<int> ns_large(int n, Shape shape) {
    std::vector<int> large;
    for (int i = 0; i < n; ++i) {
        int rows, cols;
        shape(i, rows, cols);
        if (rows < 1 || cols < 1 || !ns_small(rows, cols)) large.push_back(i);
    }
    return large;
}
template <typename Shape>
int ns_layout_large(const std::vector<int>& large, Shape shape, NsLayout& l) {
    l.bytes = 256;
    return ns_layout((int)large.size(), [&](int i, int& r, int& c) { shape(large[i], r, c); }, [](int, int, NsUnit&) {}, l);
}

template <int T32, typename T, bool MOM>
int ns_launch_small(const NsChunk& c, int k, const NsMomentum& mo, const NsCoefficients& co, int steps, float eps, int exponent, int zero, hipStream_t s) {
    hipLaunchKernelGGL((ns_small_kernel<T32, T, MOM>), dim3(k), dim3(ns_small_threads(T32)), 0, s, c, mo, co, steps, eps, std::ldexp(1.f, exponent), zero);
    return hipGetLastError() == hipSuccess ? V1T_OK : V1T_ERR_LAUNCH;
}

// All of a call: checks, then the small matrices (by their sides: the kernel's tiles), then the table and the products of the large ones
template <typename T, bool MOM, typename Shape, typename Fill>
int ns_call(int n, Shape shape, Fill fill, const NsMomentum& mo, float eps, int zero, int steps, const float* co, void* workspace, long long ws_bytes,
            hipStream_t s) try {
    if (n > NS_MAX_UNITS) return V1T_ERR_UNSUPPORTED;
    const std::vector<int> large = ns_large(n, shape);
    NsLayout l;
    NS_TRY(ns_layout_large(large, shape, l));
    if (!workspace || ws_bytes < l.bytes) return V1T_ERR_WORKSPACE;
    if ((uintptr_t)workspace & 15) return V1T_ERR_ARG;
    const NsScale* scale = ns_scale(co, steps, false);
    if (!scale) return V1T_ERR_ARG;
    const int exponent = scale->exponent;
    NsCoefficients cs{};
    for (int i = 0; i < 3 * steps; ++i) cs.c[i] = co[i];
    for (int i = 0; i <= steps; ++i) cs.lg[i] = scale->lg[i];
    NsChunk c;
    for (int t32 = 1; t32 <= 3; ++t32) {
        int k = 0;
        for (int i = 0; i <= n; ++i) {
            NsUnit u{};
            bool mine = false;
            if (i < n) {
                shape(i, u.rows, u.cols);
                u.n = std::max(u.rows, u.cols);
                u.mp = round_up(std::min(u.rows, u.cols), 32); u.np = round_up(u.n, 32);
                mine = u.mp == 32 * t32 && ns_small(u.rows, u.cols);
            }
            if (mine) {
                u.part = (int)(u.cols == 1 ? 0 : ((1ull << 32) + u.cols - 1) / u.cols);  // exact: below 2^18 numbers, a rest below 2^11
                fill(i, u);
                c.u[k++] = u;
            }
            if (k == NS_CHUNK || (i == n && k > 0)) {
                NS_TRY(t32 == 1 ? (ns_launch_small<1, T, MOM>(c, k, mo, cs, steps, eps, exponent, zero, s))
                     : t32 == 2 ? (ns_launch_small<2, T, MOM>(c, k, mo, cs, steps, eps, exponent, zero, s))
                                : (ns_launch_small<3, T, MOM>(c, k, mo, cs, steps, eps, exponent, zero, s)));
                k = 0;
            }
        }
    }
    if (large.empty()) return V1T_OK;
    NsUnit* table = (NsUnit*)((char*)workspace + l.table);
    const int m = (int)large.size();
    int rc = V1T_OK;
    NsLayout again;
    ns_layout(m, [&](int i, int& r, int& cl) { shape(large[i], r, cl); }, [&](int i, int from, NsUnit& u) {
        fill(large[from], u);
        c.u[i % NS_CHUNK] = u;
        if (i % NS_CHUNK == NS_CHUNK - 1 || i == m - 1) {
            const int k = i % NS_CHUNK + 1;
            hipLaunchKernelGGL(ns_table_kernel, dim3(1), dim3(256), 0, s, c, k, i - k + 1, m, table, (ns_head*)((char*)workspace + l.heads));
            if (hipGetLastError() != hipSuccess) rc = V1T_ERR_LAUNCH;
        }
    }, again);
    if (rc != V1T_OK) return rc;
    return ns_run<T, MOM>(l, m, (char*)workspace, mo, eps, zero, steps, co, s);
} catch (...) {
    return V1T_ERR_WORKSPACE;  // (the host's own tables: nothing leaves a C entry but a code)
}

}  // namespace

extern "C" long long v1t_orthogonalize_ws_bytes(const int* rows, const int* cols, int n) {
    if (n < 0 || (n > 0 && (!rows || !cols))) return V1T_ERR_ARG;
    if (n > NS_MAX_UNITS) return V1T_ERR_UNSUPPORTED;
    try {
        auto shape = [&](int i, int& r, int& c) { r = rows[i]; c = cols[i]; };
        NsLayout l;
        const int rc = ns_layout_large(ns_large(n, shape), shape, l);
        return rc == V1T_OK ? l.bytes : rc;
    } catch (...) {
        return V1T_ERR_WORKSPACE;
    }
}

extern "C" int v1t_orthogonalize(const v1t_matrix* units, int n, int dtype, int steps, const float* coefficients, float eps, void* workspace, long long ws_bytes,
                                 void* stream) {
    if (n < 0 || (n > 0 && !units) || dtype < 0 || dtype > 2 || steps < 0 || steps > NS_MAX_STEPS || (steps > 0 && !coefficients) || !(eps >= 0.f)) return V1T_ERR_ARG;
    if (!ns_scale(coefficients, steps, false)) return V1T_ERR_ARG;
    for (int i = 0; i < n; ++i)
        if (!units[i].in || !units[i].out) return V1T_ERR_ARG;
    if (n == 0) return V1T_OK;
    auto shape = [&](int i, int& r, int& c) { r = units[i].rows; c = units[i].cols; };
    auto fill = [&](int i, NsUnit& u) { u.in = units[i].in; u.out = units[i].out; u.rs = units[i].row_stride; u.cs = units[i].col_stride; };
    const NsMomentum mo{0.f, 0};
    hipStream_t s = (hipStream_t)stream;
    if (dtype == 0) return ns_call<bf16_t, false>(n, shape, fill, mo, eps, 0, steps, coefficients, workspace, ws_bytes, s);
    if (dtype == 1) return ns_call<f16_t, false>(n, shape, fill, mo, eps, 0, steps, coefficients, workspace, ws_bytes, s);
    return ns_call<float, false>(n, shape, fill, mo, eps, 0, steps, coefficients, workspace, ws_bytes, s);
}

extern "C" int v1t_muon_step(const v1t_muon_range* units, int n, float momentum, int nesterov, int steps, const float* coefficients, float eps, int zero_grad,
                             void* workspace, long long ws_bytes, void* stream) {
    if (n < 0 || (n > 0 && !units) || steps < 0 || steps > NS_MAX_STEPS || (steps > 0 && !coefficients) || !(eps >= 0.f) || !std::isfinite(momentum)) return V1T_ERR_ARG;
    if (!ns_scale(coefficients, steps, false)) return V1T_ERR_ARG;
    for (int i = 0; i < n; ++i)
        if (!units[i].p || !units[i].g || !units[i].m) return V1T_ERR_ARG;
    if (n == 0) return V1T_OK;
    auto shape = [&](int i, int& r, int& c) { r = units[i].rows; c = units[i].cols; };
    auto fill = [&](int i, NsUnit& u) {
        u.in = units[i].g; u.rs = units[i].cols; u.cs = 1; u.mom = units[i].m; u.w = units[i].p;
        u.lr = units[i].lr; u.decay = units[i].decay; u.l1 = units[i].l1;
    };
    return ns_call<float, true>(n, shape, fill, NsMomentum{momentum, nesterov}, eps, zero_grad, steps, coefficients, workspace, ws_bytes, (hipStream_t)stream);
}
