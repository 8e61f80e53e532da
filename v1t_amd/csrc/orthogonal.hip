// Orthogonalising an update by Newton-Schulz products, and the momentum step around it.
//
//     X <- U / (|U|_F + eps), laid with its shorter side m first (m x n)
//     A = X X^T,  S = b A + c A A,  X <- a X + S X          a few times, with (a, b, c) of each step
// The polynomial a s + b s^3 + c s^5 acts on every singular value s of X and drives it towards 1.
//
// Precision: fp32, on fp16 matrix instructions. A number v of X, A or S (spectral norm known to the host to stay below 2^15 / 2^e for the given
// coefficients) is kept as two fp16 planes of v 2^e: hi = fp16(v 2^e) and lo = fp16(v 2^e - hi), 22 bits of it, and a product of two such numbers is
// hi hi + hi lo + lo hi, accumulated in fp32: three MFMAs where fp16 has one, at a sixteenth of the time of an fp32 one. The term that is left out
// and the two roundings are 2^-22 of a product each, of random sign: the error of fp32 operands (the steps amplify what is lost on the small
// singular values up to a^5 = 480 times: one fp16 plane leaves 2e-3 of the result's norm, two leave what fp32 does, 2e-6).
// The common exponent e makes every scale of the chain 2^-e.
//
// All matrices of a call ("units") go through each product in one launch: the shared core's matrices are small, and launches are what they cost.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <utility>

#include "../../include/v1t_amd.h"
#include "common.h"

namespace {

constexpr int NS_BK = 32;            // K step of the products; planes are padded to it with zeros both ways
constexpr int NS_PART = 4096;        // least number of elements per partial sum of squares; at most 1024 partial sums a unit
constexpr int NS_TILE_PREP = 64;     // the first planes are written in 64 x 64 tiles
constexpr int NS_CHUNK = 16;         // units per table launch (kernel arguments)
constexpr int NS_MAX_STEPS = 32;

struct NsUnit {
    const void* in;   // the update, or the gradient
    void* out;        // the result, or nullptr: w is updated
    float *mom, *w;
    long long rs, cs;                // element strides of `in`; out, mom and w are row-major without gaps
    long long x[2], a, s;            // byte offsets of the planes in the workspace (hi, and lo behind it)
    int rows, cols, m, n, mp, np, trans;
    int part, part0, nparts, prep0, sym0, full0;  // first workgroup of this unit in the launches of each kind
    float lr, decay, l1;             // w <- decay w - lr O;  gradient + l1 sign(w)
};

struct NsChunk {
    NsUnit u[NS_CHUNK];
};

__global__ void ns_table_kernel(NsChunk c, int n, NsUnit* to) {
    // 4-byte words, one per lane: the argument is read as an array
    const uint32_t* src = (const uint32_t*)&c;
    for (int i = threadIdx.x; i < n * (int)(sizeof(NsUnit) / 4); i += blockDim.x) ((uint32_t*)to)[i] = src[i];
}

// the unit whose range of workgroups `block` falls into: the last one that begins at or before it
DEVFN const NsUnit& ns_find(const NsUnit* u, int n, int block, int NsUnit::*first) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (u[mid].*first <= block) lo = mid;
        else hi = mid - 1;
    }
    return u[lo];
}

struct NsMomentum {
    float mu;
    int nesterov;
};

DEVFN float ns_sign(float x) { return (float)((x > 0.f) - (x < 0.f)); }

// sum over the workgroup of 256, in a fixed order
DEVFN double ns_block_sum(double v) {
    __shared__ double s[256];
    s[threadIdx.x] = v;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) s[threadIdx.x] += s[threadIdx.x + o];
        __syncthreads();
    }
    return s[0];
}

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
    DEVFN float update(const NsMomentum& mo, int e) const { return !MOM ? g[e] : mo.nesterov ? g[e] + mo.mu * m[e] : m[e]; }
};

// partial sums of squares, in 64 bits (their range is that of the inputs squared); MOM: momentum <- mu momentum + gradient on the way
template <typename T, bool MOM>
__global__ __launch_bounds__(256) void ns_norm_kernel(const NsUnit* units, int n, NsMomentum mo, double* parts) {
    constexpr int N = 8;
    const NsUnit& u = ns_find(units, n, blockIdx.x, &NsUnit::part0);
    const long long all = (long long)u.rows * u.cols, i0 = (long long)(blockIdx.x - u.part0) * u.part;
    const int len = (int)min((long long)u.part, all - i0);
    const bool flat = u.cs == 1 && u.rs == u.cols;
    double sum = 0.0;
    for (int k0 = 0; k0 < len; k0 += 256 * N) {
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
        NsBatch<T, MOM, N> b;
        b.load(u, src, at, on);
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
    sum = ns_block_sum(sum);
    if (threadIdx.x == 0) parts[blockIdx.x] = sum;
}

DEVFN void ns_split(float v, f16_t& hi, f16_t& lo) {
    hi = (f16_t)v;
    lo = (f16_t)(v - (float)hi);
}

// the first planes: 64 x 64 tiles of X, read along the update's rows and turned through LDS where X is its transpose. MOM && zero: the gradient is
// cleared behind its last reader
template <typename T, bool MOM>
__global__ __launch_bounds__(256) void ns_prep_kernel(const NsUnit* units, int n, NsMomentum mo, const double* parts, char* ws, float eps, float scale, int zero) {
    const NsUnit& u = ns_find(units, n, blockIdx.x, &NsUnit::prep0);
    __shared__ float s[NS_TILE_PREP][NS_TILE_PREP + 1];
    double sum = 0.0;
    for (int i = threadIdx.x; i < u.nparts; i += 256) sum += parts[u.part0 + i];
    sum = ns_block_sum(sum);
    const double mul = (double)scale / (sqrt(sum) + (double)eps);  // 64 bits: a norm may lie outside fp32's range where its elements do not
    const int tj = (u.np + NS_TILE_PREP - 1) / NS_TILE_PREP, t = blockIdx.x - u.prep0;
    const int i0 = t / tj * NS_TILE_PREP, j0 = t % tj * NS_TILE_PREP;  // in X
    const int r0 = u.trans ? j0 : i0, c0 = u.trans ? i0 : j0;            // in the update
    constexpr int N = 8;
#pragma unroll
    for (int k0 = 0; k0 < NS_TILE_PREP * NS_TILE_PREP; k0 += 256 * N) {
        long long src[N], at[N];
        bool on[N];
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const int k = k0 + 256 * e + (int)threadIdx.x, r = r0 + k / NS_TILE_PREP, c = c0 + k % NS_TILE_PREP;
            on[e] = r < u.rows && c < u.cols;
            src[e] = (long long)r * u.rs + (long long)c * u.cs;
            at[e] = (long long)r * u.cols + c;
        }
        NsBatch<T, MOM, N> b;
        b.load(u, src, at, on);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const int k = k0 + 256 * e + (int)threadIdx.x;
            if constexpr (MOM) {
                if (zero && on[e]) ((T*)u.in)[src[e]] = (T)0.f;
            }
            s[k / NS_TILE_PREP][k % NS_TILE_PREP] = on[e] ? (float)((double)b.update(mo, e) * mul) : 0.f;
        }
    }
    __syncthreads();
    f16_t* hi = (f16_t*)(ws + u.x[0]);
    f16_t* lo = hi + (size_t)u.mp * u.np;
    for (int k = threadIdx.x; k < NS_TILE_PREP * NS_TILE_PREP / 8; k += 256) {
        const int i = k / (NS_TILE_PREP / 8), j = 8 * (k % (NS_TILE_PREP / 8));
        if (i0 + i >= u.mp || j0 + j >= u.np) continue;  // np is a multiple of 32: groups of 8 are whole
        f16x8 h, l;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            f16_t a, b;
            ns_split(u.trans ? s[j + e][i] : s[i][j + e], a, b);
            h[e] = a;
            l[e] = b;
        }
        *(f16x8*)(hi + (size_t)(i0 + i) * u.np + j0 + j) = h;
        *(f16x8*)(lo + (size_t)(i0 + i) * u.np + j0 + j) = l;
    }
}

// ---- the products -------------------------------------------------------------------------
// C[i][j] = sum_k P[i][k] Q[j][k]: a workgroup of 4 waves computes a 64 TW x 64 TW tile, wave (wi, wj) a quarter of it, in K steps of 32. The tile's rows of P
// and Q go to LDS by LDS-DMA into a ring of NST stages. In the accumulators i is on the lanes and j in the registers, four in a row.
enum NsKind { NS_GRAM = 0, NS_POLY = 1, NS_APPLY = 2, NS_LAST = 3 };
struct NsStep {
    float alpha, beta;   // C <- alpha (P Q^T) + beta D, on the scaled planes
    int from;            // which of the two X planes is read
    float inv;           // 2^-e
};
typedef f16_t f16x4 __attribute__((ext_vector_type(4)));

template <int TW>
struct NsTile {
    static constexpr int B = 64 * TW, PL = B * NS_BK, SIDE = 32 * TW;
    static constexpr int PIECES = PL * 2 / 1024 / 4;      // LDS-DMA instructions per wave and plane: one per 64 rows
    static constexpr int NST = TW == 1 ? 4 : TW == 2 ? 2 : 3;
    static constexpr int LDS = NST * 4 * PL;              // elements; the epilogue's fp32 tile fits
    static_assert(4 * SIDE * SIDE * 4 <= LDS * 2, "epilogue");
};

// where a tile lies and what it reads and writes
struct NsWhere {
    int bi, bj, i0, j0;
    const f16_t *D, *Dl;
    f16_t *C, *Cl;
    int ldd, cols;
};
template <int TW, int KIND>
DEVFN NsWhere ns_where(const NsUnit& u, char* ws, const NsStep& st, int block) {
    constexpr bool SYM = KIND == NS_GRAM || KIND == NS_POLY;
    constexpr int B = NsTile<TW>::B;
    NsWhere w;
    if constexpr (SYM) {  // tile number -> (bi <= bj) of the upper triangle, columns of tiles one after another
        const int t = block - u.sym0;
        w.bj = (int)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
        while ((w.bj + 1) * (w.bj + 2) / 2 <= t) ++w.bj;
        while (w.bj * (w.bj + 1) / 2 > t) --w.bj;
        w.bi = t - w.bj * (w.bj + 1) / 2;
    } else {
        const int t = block - u.full0, ni = (u.mp + B - 1) / B;
        w.bi = t % ni;
        w.bj = t / ni;
    }
    w.i0 = w.bi * B;
    w.j0 = w.bj * B;
    const size_t xlo = (size_t)u.mp * u.np, alo = (size_t)u.mp * u.mp;
    w.D = KIND == NS_POLY ? (const f16_t*)(ws + u.a) : (const f16_t*)(ws + u.x[st.from]);
    w.Dl = w.D + (KIND == NS_POLY ? alo : xlo);
    w.ldd = KIND == NS_POLY ? u.mp : u.np;
    w.C = (f16_t*)(ws + (KIND == NS_GRAM ? u.a : KIND == NS_POLY ? u.s : u.x[st.from ^ 1]));
    w.Cl = w.C + (SYM ? alo : xlo);
    w.cols = SYM ? u.mp : u.np;
    return w;
}

// Accumulators -> alpha acc + beta D -> planes (both triangles of a symmetric product), or the result. Each wave turns its part over in its own LDS, so that
// planes are read and written 16 B a lane along their rows - also the mirrored tile's - and the result along its own rows, whichever way the matrix lies.
// LDS image [SIDE][SIDE] fp32, 16-B chunks of a row swizzled by the row: writes by lanes of one column and reads along rows both spread over the banks.
template <int TW, int KIND, typename T>
DEVFN void ns_epilogue(const NsUnit& u, const NsWhere& w, const NsStep& st, f32x16 (&acc)[TW][TW], float* img, int wi, int wj, int lane) {
    constexpr bool SYM = KIND == NS_GRAM || KIND == NS_POLY;
    constexpr int SIDE = 32 * TW;
    auto chunk = [&](int i, int c) { return i * SIDE + 4 * (TW == 2 ? c ^ (i & 15) : c ^ (i >> 1 & 7)); };
    const int r = lane & 31, h = lane >> 5;
#pragma unroll
    for (int ti = 0; ti < TW; ++ti)
#pragma unroll
        for (int tj = 0; tj < TW; ++tj)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x16& a = acc[ti][tj];
                *(f32x4*)(img + chunk(32 * ti + r, 8 * tj + 2 * q + h)) =
                    f32x4{st.alpha * a[4 * q], st.alpha * a[4 * q + 1], st.alpha * a[4 * q + 2], st.alpha * a[4 * q + 3]};
            }
    __builtin_amdgcn_wave_barrier();
    const int iw = w.i0 + SIDE * wi, jw = w.j0 + SIDE * wj;
    const bool mirror = SYM && w.bi != w.bj;  // the lower triangle
    for (int k = lane; k < SIDE * SIDE / 8; k += 64) {
        const int il = k / (SIDE / 8), jl = 8 * (k % (SIDE / 8)), i = iw + il, j = jw + jl;
        if (i >= u.mp || j >= w.cols) continue;  // both are multiples of 32: groups of 8 are whole
        f32x4 v0 = *(const f32x4*)(img + chunk(il, jl / 4)), v1 = *(const f32x4*)(img + chunk(il, jl / 4 + 1));
        if constexpr (KIND != NS_GRAM) {
            const f16x8 dh = *(const f16x8*)(w.D + (size_t)i * w.ldd + j), dl = *(const f16x8*)(w.Dl + (size_t)i * w.ldd + j);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v0[e] += st.beta * ((float)dh[e] + (float)dl[e]);
                v1[e] += st.beta * ((float)dh[4 + e] + (float)dl[4 + e]);
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
            *(f16x8*)(w.C + (size_t)i * w.cols + j) = ch;
            *(f16x8*)(w.Cl + (size_t)i * w.cols + j) = cl;
        }
        if (KIND == NS_LAST || (KIND == NS_POLY && mirror)) {
            *(f32x4*)(img + chunk(il, jl / 4)) = v0;
            *(f32x4*)(img + chunk(il, jl / 4 + 1)) = v1;
        }
    }
    __builtin_amdgcn_wave_barrier();
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
            *(f16x8*)(w.C + (size_t)j * w.cols + i) = ch;
            *(f16x8*)(w.Cl + (size_t)j * w.cols + i) = cl;
        }
    } else if constexpr (KIND == NS_LAST) {
        constexpr int N = 8;
        for (int k0 = lane; k0 < SIDE * SIDE; k0 += 64 * N) {  // a batch's loads of the weights stand together
            long long x[N];
            float o[N], wt[N];
            bool on[N];
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int a = (k0 + 64 * e) / SIDE, b = (k0 + 64 * e) % SIDE;  // b runs along the result's rows
                const int row = (u.trans ? jw : iw) + a, col = (u.trans ? iw : jw) + b;
                on[e] = row < u.rows && col < u.cols;
                x[e] = (long long)row * u.cols + col;
                o[e] = (u.trans ? at(b, a) : at(a, b)) * st.inv;
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
__global__ __launch_bounds__(256, TW == 3 ? 1 : 2) void ns_gemm_kernel(const NsUnit* units, int n, char* ws, NsStep st) {
    constexpr bool SYM = KIND == NS_GRAM || KIND == NS_POLY, TR = !SYM;  // TR: Q is stored [k][j]
    using Tile = NsTile<TW>;
    constexpr int B = Tile::B, PL = Tile::PL, PIECES = Tile::PIECES, NST = Tile::NST;
    __shared__ __attribute__((aligned(16))) f16_t lds[Tile::LDS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wi = wave >> 1, wj = wave & 1;
    const int block = xcd_remap(blockIdx.x, gridDim.x);
    const NsUnit& u = ns_find(units, n, block, SYM ? &NsUnit::sym0 : &NsUnit::full0);
    const NsWhere w = ns_where<TW, KIND>(u, ws, st, block);
    const int K = KIND == NS_GRAM ? u.np : u.mp, nk = K / NS_BK;
    const f16_t* X = (const f16_t*)(ws + u.x[st.from]);
    const f16_t* A = (const f16_t*)(ws + u.a);
    const f16_t* P = KIND == NS_GRAM ? X : KIND == NS_POLY ? A : (const f16_t*)(ws + u.s);
    const f16_t* Q = KIND == NS_POLY ? A : X;
    const size_t xlo = (size_t)u.mp * u.np, alo = (size_t)u.mp * u.mp;
    const int ldp = KIND == NS_GRAM ? u.np : u.mp, ldq = KIND == NS_POLY ? u.mp : u.np;
    const size_t plo = KIND == NS_GRAM ? xlo : alo, qlo = KIND == NS_POLY ? alo : xlo;

    // A 1-KB piece fills 64 16-B chunks of a plane in order; which 16 B of the tile's row a chunk holds is swizzled, so that the fragment reads below spread over
    // all banks. Rows [.][32]: four chunks a row, chunk c at c ^ (row / 4 % 4). Q as [k][j], B / 8 chunks a row: c ^ 4 (k % 4) - B = 64, where two rows fill
    // the 64 banks: c ^ 4 (k / 2 % 2). A lane's byte offset from the tile's first row is loop-invariant; piece p of a wave goes by the instruction's offset, which
    // moves the LDS and the global address alike: the lane offset carries 1024 p less, the base 2048 less.
    unsigned po[PIECES], qo[PIECES];
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int c = 64 * (wave * PIECES + p) + lane;
        po[p] = (unsigned)min(c / 4, u.mp - 1 - w.i0) * (unsigned)(2 * ldp) + 16 * ((c & 3) ^ (c >> 4 & 3)) + 2048 - 1024 * p;
        if constexpr (TR) {
            const int k = c / (B / 8), cc = (c % (B / 8)) ^ (B == 64 ? (k >> 1 & 1) << 2 : (k & 3) << 2);
            qo[p] = (unsigned)k * (unsigned)(2 * ldq) + 2 * min(8 * cc, u.np - 8 - w.j0) + 2048 - 1024 * p;
        } else {
            qo[p] = (unsigned)min(c / 4, u.mp - 1 - w.j0) * (unsigned)(2 * ldq) + 16 * ((c & 3) ^ (c >> 4 & 3)) + 2048 - 1024 * p;
        }
    }
    const char* pb = (const char*)(P + (size_t)w.i0 * ldp) - 2048;
    const char* qb = (const char*)(TR ? Q + w.j0 : Q + (size_t)w.j0 * ldq) - 2048;
    const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(const __attribute__((address_space(3))) void*)lds);
    auto uniform = [](const char* p) {
        const unsigned long long b = (unsigned long long)(uintptr_t)p;
        const unsigned hi = (unsigned)__builtin_amdgcn_readfirstlane((int)(b >> 32)), lo = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)b);
        return (const char*)(uintptr_t)(((unsigned long long)hi << 32) | lo);
    };
    auto issue = [&](int t, int buf) {
        const size_t pk = (size_t)t * (2 * NS_BK), qk = TR ? (size_t)t * (2 * NS_BK) * ldq : (size_t)t * (2 * NS_BK);
#pragma unroll
        for (int plane = 0; plane < 4; ++plane) {
            const char* base = uniform(plane == 0 ? pb + pk : plane == 1 ? pb + pk + 2 * plo : plane == 2 ? qb + qk : qb + qk + 2 * qlo);
            const unsigned m0 = lds0 + 2u * (unsigned)((buf * 4 + plane) * PL) + 1024u * (unsigned)(wave * PIECES);
            const unsigned* o = plane < 2 ? po : qo;
            TileDma<32, 32>::template group<PIECES>(base, m0, o[0], o[PIECES > 1 ? 1 : 0], o[PIECES > 2 ? 2 : 0], 0);
        }
    };

    const int r = lane & 31, h = lane >> 5;
    auto row_frag = [&](const f16_t* img, int row0, int s) -> bf16x8 {  // rows row0 + (lane & 31), k = 16 s + 8 h ..
        return *(const bf16x8*)(img + (row0 + r) * NS_BK + 8 * ((2 * s + h) ^ (r >> 2 & 3)));
    };
    const int tg = lane >> 4, tq = lane >> 2 & 3, tp = lane & 3;
    auto col_frag = [&](const f16_t* img, int col0, int s) -> bf16x8 {  // columns col0 + (lane & 31), the same k
        const int k = 16 * s + 8 * (tg >> 1) + tq;
        const int c = (col0 / 8 + 2 * (tg & 1) + (tp >> 1)) ^ (B == 64 ? (tq >> 1) << 2 : tq << 2);
        const bf16_t* a = (const bf16_t*)img + k * B + 8 * c + 4 * (tp & 1);
        const bf16x4 x = lds_tr_read(a), y = lds_tr_read(a + 4 * B);
        return bf16x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
    };

    f32x16 acc[TW][TW];
#pragma unroll
    for (int i = 0; i < TW; ++i)
#pragma unroll
        for (int j = 0; j < TW; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    auto compute = [&](int buf) {
        const f16_t* img = lds + buf * 4 * PL;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            bf16x8 ph[TW], pl[TW], qh[TW], ql[TW];
#pragma unroll
            for (int i = 0; i < TW; ++i) {
                ph[i] = row_frag(img, 32 * (TW * wi + i), s);
                pl[i] = row_frag(img + PL, 32 * (TW * wi + i), s);
                if constexpr (TR) {
                    qh[i] = col_frag(img + 2 * PL, 32 * (TW * wj + i), s);
                    ql[i] = col_frag(img + 3 * PL, 32 * (TW * wj + i), s);
                } else {
                    qh[i] = row_frag(img + 2 * PL, 32 * (TW * wj + i), s);
                    ql[i] = row_frag(img + 3 * PL, 32 * (TW * wj + i), s);
                }
            }
#pragma unroll
            for (int x = 0; x < 3; ++x)
#pragma unroll
                for (int i = 0; i < TW; ++i)
#pragma unroll
                    for (int j = 0; j < TW; ++j) acc[i][j] = mfma32h(x == 0 ? ql[j] : qh[j], x == 1 ? pl[i] : ph[i], acc[i][j]);
        }
    };
    // every wave issues 4 PIECES operations per stage: "all but the newest NST - 2 stages have landed" is one counted wait
#pragma unroll
    for (int t = 0; t < NST - 1; ++t)
        if (t < nk) issue(t, t);
    int buf = 0;
    for (int t = 0; t < nk; ++t) {
        if (t + NST - 1 <= nk) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(4 * PIECES * (NST - 2)) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();  // stage t is there for all; the stage before it has been read by all
        if (t + NST - 1 < nk) issue(t + NST - 1, buf == 0 ? NST - 1 : buf - 1);
        compute(buf);
        buf = buf + 1 == NST ? 0 : buf + 1;
    }
    __syncthreads();
    ns_epilogue<TW, KIND, T>(u, w, st, acc, (float*)lds + wave * (32 * TW) * (32 * TW), wi, wj, lane);
}

// no steps: the normalised update itself
template <typename T>
__global__ __launch_bounds__(256) void ns_copy_kernel(const NsUnit* units, int n, const char* ws, float inv) {
    const NsUnit& u = ns_find(units, n, blockIdx.x, &NsUnit::prep0);
    const int tj = (u.np + NS_TILE_PREP - 1) / NS_TILE_PREP, t = blockIdx.x - u.prep0;
    const int i0 = t / tj * NS_TILE_PREP, j0 = t % tj * NS_TILE_PREP;
    const f16_t* hi = (const f16_t*)(ws + u.x[0]);
    const f16_t* lo = hi + (size_t)u.mp * u.np;
    for (int k = threadIdx.x; k < NS_TILE_PREP * NS_TILE_PREP; k += 256) {
        const int i = i0 + k / NS_TILE_PREP, j = j0 + k % NS_TILE_PREP;
        if (i >= u.m || j >= u.n) continue;
        const long long at = u.trans ? (long long)j * u.cols + i : (long long)i * u.cols + j;
        const float o = ((float)hi[(size_t)i * u.np + j] + (float)lo[(size_t)i * u.np + j]) * inv;
        if (u.out) ((T*)u.out)[at] = (T)o;
        else u.w[at] = u.decay * u.w[at] - u.lr * o;
    }
}

// ---- host ---------------------------------------------------------------------------------
struct NsLayout {
    long long table = 0, parts = 0, bytes = 0;
    int nparts = 0, nprep = 0, nsym = 0, nfull = 0, tile = 128;
    long long sym128 = 0, full128 = 0;
};
// elements per partial sum, and how many sums
std::pair<int, int> ns_parts(long long elements) {
    const long long part = std::max<long long>(NS_PART, (elements + 1023) / 1024);
    return {(int)part, (int)((elements + part - 1) / part)};
}
long long ns_align(long long x) { return (x + 255) / 256 * 256; }

// Places every unit's planes. `shape(i, rows, cols)`; `put` (or null) receives the filled units in order.
template <typename Shape, typename Put>
int ns_layout(int n, Shape shape, Put put, NsLayout& l) {
    long long nparts = 0;
    long long sym = 0, full = 0;
    for (int i = 0; i < n; ++i) {
        int rows, cols;
        shape(i, rows, cols);
        if (rows < 1 || cols < 1) return V1T_ERR_ARG;
        const long long m = std::min(rows, cols), nn = std::max(rows, cols);
        if (m > 32768 || nn > (1 << 22) || m * nn > (1ll << 31)) return V1T_ERR_UNSUPPORTED;
        const long long a = (m + 127) / 128, b = (nn + 127) / 128;
        sym += a * (a + 1) / 2;
        full += a * b;
        nparts += ns_parts(m * nn).second;
    }
    l.sym128 = sym; l.full128 = full;
    l.tile = sym >= 256 ? 128 : 64;
    l.table = 0;
    l.parts = ns_align((long long)n * (long long)sizeof(NsUnit));
    long long at = ns_align(l.parts + 8 * nparts);
    long long part = 0, prep = 0, s0 = 0, f0 = 0;
    for (int i = 0; i < n; ++i) {
        NsUnit u{};
        shape(i, u.rows, u.cols);
        u.trans = u.rows > u.cols;
        u.m = std::min(u.rows, u.cols); u.n = std::max(u.rows, u.cols);
        u.mp = round_up(u.m, NS_BK); u.np = round_up(u.n, NS_BK);
        const long long xb = ns_align(4ll * u.mp * u.np), ab = ns_align(4ll * u.mp * u.mp);
        u.x[0] = at; u.x[1] = at + xb; u.a = at + 2 * xb; u.s = u.a + ab;
        at = u.s + ab;
        const long long ti = (u.mp + l.tile - 1) / l.tile, tj = (u.np + l.tile - 1) / l.tile;
        const long long pi = (u.mp + NS_TILE_PREP - 1) / NS_TILE_PREP, pj = (u.np + NS_TILE_PREP - 1) / NS_TILE_PREP;
        u.part = ns_parts((long long)u.rows * u.cols).first; u.part0 = (int)part; u.nparts = ns_parts((long long)u.rows * u.cols).second;
        u.prep0 = (int)prep; u.sym0 = (int)s0; u.full0 = (int)f0;
        part += u.nparts; prep += pi * pj; s0 += ti * (ti + 1) / 2; f0 += ti * tj;
        if (std::max(std::max(part, prep), std::max(s0, f0)) > 0x7fffffffll) return V1T_ERR_UNSUPPORTED;
        put(i, u);
    }
    l.nparts = (int)part; l.nprep = (int)prep; l.nsym = (int)s0; l.nfull = (int)f0;
    l.bytes = at;
    return V1T_OK;
}

// The exponent of the planes' common scale: 2^15 over the largest number of any plane. A step maps a singular value s in [0, top] to a s + b s^3 + c s^5;
// X, A = X X^T and S are bounded by their spectral norms. The maxima are sampled, 0.1 % is added for what lies between the samples and for rounding.
bool ns_exponent(const float* coefficients, int steps, int* exponent) {
    double top = 1.001, most = top;
    for (int k = 0; k < steps; ++k) {
        const double a = coefficients[3 * k], b = coefficients[3 * k + 1], c = coefficients[3 * k + 2];
        if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return false;
        double next = 0.0;
        most = std::max(most, top * top);
        for (int i = 0; i <= 4096; ++i) {
            const double s = top * i / 4096.0, t = s * s;
            next = std::max(next, std::fabs(s * (a + t * (b + t * c))));
            most = std::max(most, std::fabs(t * (b + t * c)));
        }
        top = 1.001 * next;
        most = std::max(most, top);
        if (!(most < 128.0)) return false;
    }
    *exponent = (int)std::floor(std::log2(32768.0 / (1.01 * most)));
    return true;
}

template <int TW, int KIND, typename T>
int ns_gemm(const NsLayout& l, const NsUnit* table, int n, char* ws, const NsStep& st, hipStream_t s) {
    const int grid = KIND == NS_GRAM || KIND == NS_POLY ? l.nsym : l.nfull;
    hipLaunchKernelGGL((ns_gemm_kernel<TW, KIND, T>), dim3(grid), dim3(256), 0, s, table, n, ws, st);
    return hipGetLastError() == hipSuccess ? V1T_OK : V1T_ERR_LAUNCH;
}

#define NS_TRY(x) do { const int rc_ = (x); if (rc_ != V1T_OK) return rc_; } while (0)

template <int TW, typename T>
int ns_steps(const NsLayout& l, const NsUnit* table, int n, char* ws, int steps, const float* co, int exponent, hipStream_t s) {
    const float inv = std::ldexp(1.f, -exponent);
    for (int k = 0; k < steps; ++k) {
        const float a = co[3 * k], b = co[3 * k + 1], c = co[3 * k + 2];
        NS_TRY((ns_gemm<TW, NS_GRAM, float>(l, table, n, ws, NsStep{inv, 0.f, k & 1, inv}, s)));
        NS_TRY((ns_gemm<TW, NS_POLY, float>(l, table, n, ws, NsStep{c * inv, b, k & 1, inv}, s)));
        const NsStep last{inv, a, k & 1, inv};
        if (k + 1 < steps) NS_TRY((ns_gemm<TW, NS_APPLY, float>(l, table, n, ws, last, s)));
        else NS_TRY((ns_gemm<TW, NS_LAST, T>(l, table, n, ws, last, s)));
    }
    return V1T_OK;
}

template <typename T, bool MOM>
int ns_run(const NsLayout& l, int n, char* ws, const NsMomentum& mo, float eps, int zero, int steps, const float* co, int exponent, hipStream_t s) {
    const NsUnit* table = (const NsUnit*)(ws + l.table);
    double* parts = (double*)(ws + l.parts);
    hipLaunchKernelGGL((ns_norm_kernel<T, MOM>), dim3(l.nparts), dim3(256), 0, s, table, n, mo, parts);
    hipLaunchKernelGGL((ns_prep_kernel<T, MOM>), dim3(l.nprep), dim3(256), 0, s, table, n, mo, parts, ws, eps, std::ldexp(1.f, exponent), zero);
    if (hipGetLastError() != hipSuccess) return V1T_ERR_LAUNCH;
    if (steps == 0) {
        hipLaunchKernelGGL((ns_copy_kernel<T>), dim3(l.nprep), dim3(256), 0, s, table, n, ws, std::ldexp(1.f, -exponent));
        return hipGetLastError() == hipSuccess ? V1T_OK : V1T_ERR_LAUNCH;
    }
    return l.tile == 128 ? ns_steps<2, T>(l, table, n, ws, steps, co, exponent, s) : ns_steps<1, T>(l, table, n, ws, steps, co, exponent, s);
}

// lays out the units, checks the workspace, writes the table
template <typename Shape, typename Fill>
int ns_begin(int n, Shape shape, Fill fill, void* workspace, long long ws_bytes, NsLayout& l, hipStream_t s) {
    NS_TRY(ns_layout(n, shape, [](int, NsUnit&) {}, l));
    if (!workspace || ws_bytes < l.bytes) return V1T_ERR_WORKSPACE;
    if ((uintptr_t)workspace & 15) return V1T_ERR_ARG;
    NsChunk c;
    NsUnit* table = (NsUnit*)((char*)workspace + l.table);
    int rc = V1T_OK;
    NsLayout again;
    ns_layout(n, shape, [&](int i, NsUnit& u) {
        fill(i, u);
        c.u[i % NS_CHUNK] = u;
        if (i % NS_CHUNK == NS_CHUNK - 1 || i == n - 1) {
            const int k = i % NS_CHUNK + 1;
            hipLaunchKernelGGL(ns_table_kernel, dim3(1), dim3(256), 0, s, c, k, table + (i - k + 1));
            if (hipGetLastError() != hipSuccess) rc = V1T_ERR_LAUNCH;
        }
    }, again);
    return rc;
}

}  // namespace

extern "C" long long v1t_orthogonalize_ws_bytes(const int* rows, const int* cols, int n) {
    if (n < 0 || (n > 0 && (!rows || !cols))) return V1T_ERR_ARG;
    NsLayout l;
    const int rc = ns_layout(n, [&](int i, int& r, int& c) { r = rows[i]; c = cols[i]; }, [](int, NsUnit&) {}, l);
    return rc == V1T_OK ? l.bytes : rc;
}

extern "C" int v1t_orthogonalize(const v1t_matrix* units, int n, int dtype, int steps, const float* coefficients, float eps, void* workspace, long long ws_bytes,
                                 void* stream) {
    if (n < 0 || (n > 0 && !units) || dtype < 0 || dtype > 2 || steps < 0 || steps > NS_MAX_STEPS || (steps > 0 && !coefficients) || !(eps >= 0.f)) return V1T_ERR_ARG;
    int exponent = 0;
    if (!ns_exponent(coefficients, steps, &exponent)) return V1T_ERR_ARG;
    for (int i = 0; i < n; ++i)
        if (!units[i].in || !units[i].out) return V1T_ERR_ARG;
    if (n == 0) return V1T_OK;
    NsLayout l;
    hipStream_t s = (hipStream_t)stream;
    NS_TRY(ns_begin(n, [&](int i, int& r, int& c) { r = units[i].rows; c = units[i].cols; },
                    [&](int i, NsUnit& u) { u.in = units[i].in; u.out = units[i].out; u.rs = units[i].row_stride; u.cs = units[i].col_stride; },
                    workspace, ws_bytes, l, s));
    const NsMomentum mo{0.f, 0};
    char* ws = (char*)workspace;
    if (dtype == 0) return ns_run<bf16_t, false>(l, n, ws, mo, eps, 0, steps, coefficients, exponent, s);
    if (dtype == 1) return ns_run<f16_t, false>(l, n, ws, mo, eps, 0, steps, coefficients, exponent, s);
    return ns_run<float, false>(l, n, ws, mo, eps, 0, steps, coefficients, exponent, s);
}

extern "C" int v1t_muon_step(const v1t_muon_range* units, int n, float momentum, int nesterov, int steps, const float* coefficients, float eps, int zero_grad,
                             void* workspace, long long ws_bytes, void* stream) {
    if (n < 0 || (n > 0 && !units) || steps < 0 || steps > NS_MAX_STEPS || (steps > 0 && !coefficients) || !(eps >= 0.f) || !std::isfinite(momentum)) return V1T_ERR_ARG;
    int exponent = 0;
    if (!ns_exponent(coefficients, steps, &exponent)) return V1T_ERR_ARG;
    for (int i = 0; i < n; ++i)
        if (!units[i].p || !units[i].g || !units[i].m) return V1T_ERR_ARG;
    if (n == 0) return V1T_OK;
    NsLayout l;
    hipStream_t s = (hipStream_t)stream;
    NS_TRY(ns_begin(n, [&](int i, int& r, int& c) { r = units[i].rows; c = units[i].cols; },
                    [&](int i, NsUnit& u) {
                        u.in = units[i].g; u.rs = units[i].cols; u.cs = 1; u.mom = units[i].m; u.w = units[i].p;
                        u.lr = units[i].lr; u.decay = units[i].decay; u.l1 = units[i].l1;
                    },
                    workspace, ws_bytes, l, s));
    return ns_run<float, true>(l, n, (char*)workspace, NsMomentum{momentum, nesterov}, eps, zero_grad, steps, coefficients, exponent, s);
}
