// Rotary positions with several axes (a patch's row and column, a frame's time): token t of sequence b sits at p[b][t][a], pair j of a head's
// features belongs to axis axis[j] and turns by the angle p * rate[j]:
//     y0 = x0 cos - x1 sin,  y1 = x0 sin + x1 cos        (backward: the same with the angle negated - a rotation's transpose is its inverse)
// Features behind the 2 * pairs rotated ones pass through. One pass: every element is read once and written once.
//
// Bound: HBM (2 B of flops per byte). A workgroup owns a run of tokens. It writes their (cos, sin) to LDS once and applies them to every head
// of q and of k, and to every sequence of its batch chunk where the sequences share their positions: the angle (a 64-bit product, below)
// would otherwise cost as much as the memory traffic of the element it turns. A thread moves "slots" of 4 pairs, the unit at which one
// 16-byte access of 16-bit pairs is whole.
//
// Numerics: the angle is held as a number of turns in 64 bits, p * (rate / 2 pi), and reduced to [-1/2, 1/2] before it is rounded to 32: a
// 32-bit product is off by 0.03 rad at position 10^6. Products and sums of the rotation are fp32, rounded once to the tensor's type.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/v1t_amd.h"
#include "common.h"

namespace {

constexpr int ROT_MAX_PAIRS = 256;
constexpr int ROT_THREADS = 256;
constexpr int ROT_LDS_PAIRS = 2048;  // (token, pair) entries of the table in LDS: 16 KB

struct RotRates {  // kernel argument: a captured graph keeps it, no device memory behind it
    double turns[ROT_MAX_PAIRS];
    unsigned char axis[ROT_MAX_PAIRS];
};

struct RotArgs {
    const void* x[2];
    void* y[2];
    long long xb[2], xt[2], xh[2], yb[2], yt[2], yh[2];  // element strides of sequence, token, head
    int heads[2];
    const void* pos;
    long long pb, pt, pa;
    int B, T, D, pairs, halves, inverse;
    int nt, nb;          // tokens and sequences per workgroup
    int slots, tails;    // per head: slots of 4 pairs, and groups of 8 features behind the rotated ones
    unsigned items_mul, row_mul;  // divide an item's number by (slots + tails) * heads and by (slots + tails) (division_multiplier)
};

DEVFN int quotient(int x, int d, unsigned mul) { return mul ? (int)__umulhi((unsigned)x, mul) : x / d; }

template <typename T> DEVFN float to_f(T v) { return (float)v; }

// n elements from p in accesses of VB bytes (the launcher's guarantee: every run starts at a multiple of VB)
template <typename T, int N, int VB>
DEVFN void load_run(const T* p, float (&v)[N]) {
    constexpr int E = VB / (int)sizeof(T);
    typedef T vec __attribute__((ext_vector_type(E == 1 ? 2 : E)));
    if constexpr (E == 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = to_f(p[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; i += E) {
            const vec a = *reinterpret_cast<const vec*>(p + i);
#pragma unroll
            for (int j = 0; j < E; ++j) v[i + j] = to_f(a[j]);
        }
    }
}
template <typename T, int N, int VB>
DEVFN void store_run(T* p, const float (&v)[N]) {
    constexpr int E = VB / (int)sizeof(T);
    typedef T vec __attribute__((ext_vector_type(E == 1 ? 2 : E)));
    if constexpr (E == 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = (T)v[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; i += E) {
            vec a;
#pragma unroll
            for (int j = 0; j < E; ++j) a[j] = (T)v[i + j];
            *reinterpret_cast<vec*>(p + i) = a;
        }
    }
}

template <typename T, int VB, bool HALVES, typename P>
__global__ __launch_bounds__(ROT_THREADS) void rotary_kernel(RotArgs g, RotRates rates) {
    __shared__ __attribute__((aligned(16))) float s_cos[ROT_LDS_PAIRS], s_sin[ROT_LDS_PAIRS];
    const int t0 = blockIdx.x * g.nt, b0 = blockIdx.y * g.nb;
    const int nt = min(g.nt, g.T - t0), nb = min(g.nb, g.B - b0);
    const int row = g.slots + g.tails, per_token = row * (g.heads[0] + g.heads[1]);
    const int ldp = (g.pairs + 3) & ~3;
    const bool same_place = g.pb == 0;
    auto table = [&](int b) {
        const P* pos = (const P*)g.pos + (long long)b * g.pb;
        for (int i = threadIdx.x; i < nt * ldp; i += ROT_THREADS) {
            const int t = i / ldp, j = i - t * ldp;
            if (j < g.pairs) {
                const double turns = (double)pos[(long long)(t0 + t) * g.pt + rates.axis[j] * g.pa] * rates.turns[j];
                const float r = (float)(turns - rint(turns));
                float s, c;
                sincospif(2.f * r, &s, &c);
                s_cos[i] = c;
                s_sin[i] = g.inverse ? -s : s;
            }
        }
    };
    if (same_place) {
        table(0);
        __syncthreads();
    }
    for (int b = b0; b < b0 + nb; ++b) {
        if (!same_place) {
            __syncthreads();
            table(b);
            __syncthreads();
        }
        for (int i = threadIdx.x; i < nt * per_token; i += ROT_THREADS) {
            const int t = quotient(i, per_token, g.items_mul), r = i - t * per_token;
            const int hh = quotient(r, row, g.row_mul), v = r - hh * row;
            const int w = hh >= g.heads[0], h = w ? hh - g.heads[0] : hh;
            const T* x = (const T*)g.x[w] + (long long)b * g.xb[w] + (long long)(t0 + t) * g.xt[w] + (long long)h * g.xh[w];
            T* y = (T*)g.y[w] + (long long)b * g.yb[w] + (long long)(t0 + t) * g.yt[w] + (long long)h * g.yh[w];
            if (v < g.slots) {
                const int j = 4 * v;
                const f32x4 c = *(const f32x4*)&s_cos[t * ldp + j], s = *(const f32x4*)&s_sin[t * ldp + j];
                if (j + 4 <= g.pairs) {
                    if constexpr (HALVES) {
                        float a[4], d[4];
                        load_run<T, 4, VB>(x + j, a);
                        load_run<T, 4, VB>(x + g.pairs + j, d);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float p = a[e] * c[e] - d[e] * s[e], q = a[e] * s[e] + d[e] * c[e];
                            a[e] = p;
                            d[e] = q;
                        }
                        store_run<T, 4, VB>(y + j, a);
                        store_run<T, 4, VB>(y + g.pairs + j, d);
                    } else {
                        float a[8];
                        load_run<T, 8, VB>(x + 2 * j, a);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float p = a[2 * e] * c[e] - a[2 * e + 1] * s[e], q = a[2 * e] * s[e] + a[2 * e + 1] * c[e];
                            a[2 * e] = p;
                            a[2 * e + 1] = q;
                        }
                        store_run<T, 8, VB>(y + 2 * j, a);
                    }
                } else {  // the last slot of a number of pairs that 4 does not divide
                    for (int e = 0; j + e < g.pairs; ++e) {
                        const int i0 = HALVES ? j + e : 2 * (j + e), i1 = HALVES ? g.pairs + j + e : i0 + 1;
                        const float a = to_f(x[i0]), d = to_f(x[i1]);
                        y[i0] = (T)(a * c[e] - d * s[e]);
                        y[i1] = (T)(a * s[e] + d * c[e]);
                    }
                }
            } else {
                const int j = 2 * g.pairs + 8 * (v - g.slots);
                for (int e = j; e < min(j + 8, g.D); ++e) y[e] = x[e];
            }
        }
    }
}

// x / d = umulhi(x, mul) for 0 <= x < limit: mul = ceil(2^32 / d) is exact while x * (mul * d - 2^32) < 2^32; 0 where no 32-bit multiplier
// is (d = 1, very many heads): the kernel divides
unsigned division_multiplier(long long d, long long limit) {
    if (d < 2) return 0;
    const unsigned long long m = ((1ull << 32) + d - 1) / d, e = m * d - (1ull << 32);
    return e && (unsigned long long)limit > ((1ull << 32) - 1) / e ? 0 : (unsigned)m;
}

template <typename T, int VB, bool HALVES>
int launch_p(const RotArgs& a, const RotRates& r, int pos_type, dim3 grid, hipStream_t s) {
    if (pos_type == 0) hipLaunchKernelGGL((rotary_kernel<T, VB, HALVES, int>), grid, dim3(ROT_THREADS), 0, s, a, r);
    else if (pos_type == 1) hipLaunchKernelGGL((rotary_kernel<T, VB, HALVES, long long>), grid, dim3(ROT_THREADS), 0, s, a, r);
    else hipLaunchKernelGGL((rotary_kernel<T, VB, HALVES, float>), grid, dim3(ROT_THREADS), 0, s, a, r);
    return hipGetLastError() == hipSuccess ? V1T_OK : V1T_ERR_LAUNCH;
}
template <typename T, bool HALVES>
int launch_v(const RotArgs& a, const RotRates& r, int pos_type, int vb, dim3 grid, hipStream_t s) {
    if (!HALVES || sizeof(T) == 4)
        if (vb == 16) return launch_p<T, 16, HALVES>(a, r, pos_type, grid, s);
    if (vb >= 8) return launch_p<T, 8, HALVES>(a, r, pos_type, grid, s);
    if (sizeof(T) == 2 && vb >= 4) return launch_p<T, 4, HALVES>(a, r, pos_type, grid, s);
    return launch_p<T, (int)sizeof(T), HALVES>(a, r, pos_type, grid, s);
}
template <typename T>
int launch_t(const RotArgs& a, const RotRates& r, int pos_type, int vb, dim3 grid, hipStream_t s) {
    return a.halves ? launch_v<T, true>(a, r, pos_type, vb, grid, s) : launch_v<T, false>(a, r, pos_type, vb, grid, s);
}

}  // namespace

extern "C" int v1t_rotary(const v1t_rotary_operand* ops, int n_ops, int dtype, int B, int T, int D, const int* sections, int n_axes, double base, int shared,
                          int halves, int inverse, const void* positions, int position_type, long long pos_stride_b, long long pos_stride_t,
                          long long pos_stride_a, void* stream) {
    if (!ops || n_ops < 1 || n_ops > 2 || !sections || n_axes < 1 || n_axes > 4 || B < 0 || T < 0 || D < 1 || !positions) return V1T_ERR_ARG;
    if (dtype < 0 || dtype > 2 || position_type < 0 || position_type > 2 || !(base > 0.0) || !std::isfinite(base)) return V1T_ERR_ARG;
    long long pairs = 0;
    for (int a = 0; a < n_axes; ++a) {
        if (sections[a] < 0) return V1T_ERR_ARG;
        pairs += sections[a];
    }
    if (pairs < 1 || 2 * pairs > D) return V1T_ERR_ARG;
    if (pairs > ROT_MAX_PAIRS) return V1T_ERR_UNSUPPORTED;
    if (B == 0 || T == 0) return V1T_OK;
    RotArgs g{};
    RotRates r{};
    for (int a = 0, j = 0; a < n_axes; ++a)
        for (int i = 0; i < sections[a]; ++i, ++j) {
            const double part = shared ? (double)j / (double)pairs : (double)i / (double)sections[a];
            r.turns[j] = std::pow(base, -part) / 6.283185307179586476925286766559;
            r.axis[j] = (unsigned char)a;
        }
    const int es = dtype == 2 ? 4 : 2;
    int vb = 16;
    bool in_place = true;
    auto aligned = [&](long long bytes) {
        while (vb > es && (bytes & (vb - 1))) vb >>= 1;
    };
    for (int o = 0; o < n_ops; ++o) {
        const v1t_rotary_operand& p = ops[o];
        if (!p.x || !p.y || p.heads < 1) return V1T_ERR_ARG;
        g.x[o] = p.x; g.y[o] = p.y; g.heads[o] = p.heads;
        g.xb[o] = p.x_stride_b; g.xt[o] = p.x_stride_t; g.xh[o] = p.x_stride_h;
        g.yb[o] = p.y_stride_b; g.yt[o] = p.y_stride_t; g.yh[o] = p.y_stride_h;
        aligned((long long)(uintptr_t)p.x);
        aligned((long long)(uintptr_t)p.y);
        for (long long st : {p.x_stride_b, p.x_stride_t, p.x_stride_h, p.y_stride_b, p.y_stride_t, p.y_stride_h}) aligned(st * es);
        in_place = in_place && p.x == p.y && p.x_stride_b == p.y_stride_b && p.x_stride_t == p.y_stride_t && p.x_stride_h == p.y_stride_h;
    }
    if (halves) aligned(pairs * es);
    g.pos = positions; g.pb = B == 1 ? 0 : pos_stride_b; g.pt = pos_stride_t; g.pa = pos_stride_a;
    g.B = B; g.T = T; g.D = D; g.pairs = (int)pairs; g.halves = halves != 0; g.inverse = inverse != 0;
    g.slots = (int)((pairs + 3) / 4);
    g.tails = in_place ? 0 : (D - 2 * (int)pairs + 7) / 8;
    const long long row = g.slots + g.tails, heads = (long long)g.heads[0] + g.heads[1], per_token = row * heads;
    if (per_token > (1 << 20)) return V1T_ERR_UNSUPPORTED;
    // tokens per workgroup: enough items for its threads to have several each, as the table in LDS allows
    const int ldp = ((int)pairs + 3) & ~3;
    long long nt = std::max(1ll, std::min<long long>(ROT_LDS_PAIRS / ldp, 4 * ROT_THREADS / per_token));
    nt = std::min<long long>(nt, T);
    // sequences per workgroup: the table is computed once for all of them; at least 2048 workgroups (8 a CU) are kept
    const long long gx = (T + nt - 1) / nt;
    long long nb = g.pb == 0 ? std::max(1ll, std::min<long long>(16, gx * B / 2048)) : 1;
    nb = std::max(nb, ((long long)B + 65534) / 65535);
    g.nt = (int)nt; g.nb = (int)nb;
    g.items_mul = division_multiplier(per_token, nt * per_token);
    g.row_mul = division_multiplier(row, per_token);
    const dim3 grid((unsigned)gx, (unsigned)((B + nb - 1) / nb));
    hipStream_t st = (hipStream_t)stream;
    if (dtype == 0) return launch_t<bf16_t>(g, r, position_type, vb, grid, st);
    if (dtype == 1) return launch_t<f16_t>(g, r, position_type, vb, grid, st);
    return launch_t<float>(g, r, position_type, vb, grid, st);
}
