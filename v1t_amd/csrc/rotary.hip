// Rotary positions with several axes (a patch's row and column, a frame's time): token t of sequence b sits at p[b][t][a], pair j of a head's
// features belongs to axis axis[j] and turns by the angle p * rate[j]:
//     y0 = x0 cos - x1 sin,  y1 = x0 sin + x1 cos        (backward: the same with the angle negated - a rotation's transpose is its inverse)
// Features behind the 2 * pairs rotated ones pass through. One pass: every element is read once and written once.
//
// Bound: HBM (less than one operation a byte). A thread owns a "slot" of 4 pairs of one token - 16 B of 16-bit features - and with it 4 angles, whose cosines and
// sines stay in its registers while it walks over the heads of q and of k, and over the sequences of its batch chunk where these share their positions:
// the angle, a 64-bit product (below), costs as much as several slots' traffic, and the walk costs two address additions a slot. Four heads' loads
// stand together. Measured: q and k of 112 x 1654 tokens, 4 + 4 heads x 155 bf16 out of a padded projection into rows with room for 160 (919 MB) 192 us,
// 4.8 TB/s, where a copy of as much takes 176 us (an angle per slot: 348 us; without room, the last features one by one: 40 % more); one sequence of 39 672 tokens,
// 16 + 4 heads x 128 bf16 (406 MB) 84 us, 4.8 TB/s; one token of 8 streams 5 us of which nothing is traffic.
//
// Numerics: the angle is held as a number of turns in 64 bits, p * (rate / 2 pi), and reduced to [-1/2, 1/2] before it is rounded to 32: a
// 32-bit product is off by 0.03 rad at position 10^6. Cosine and sine are taken of the rounded angle: fp32 results err by 4.3e-8 of their norm, with those of
// 64 bits by 3.7e-8. Products and sums of the rotation are fp32, rounded once to the tensor's type.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/v1t_amd.h"
#include "common.h"

namespace {

constexpr int ROT_MAX_PAIRS = 256;
constexpr int ROT_THREADS = 256;

template <int P>
struct RotRates {  // kernel argument: a captured graph keeps it, no device memory behind it. P: 64 where they suffice - a launch copies all of it; 2.3 KB cost a
                   // small training pass of two launches 8 of 160 us. The default core's 2 x 38 pairs take the large one
    double turns[P];
    unsigned char axis[P];
};
using RotAllRates = RotRates<ROT_MAX_PAIRS>;

struct RotArgs {
    const void* x[2];
    void* y[2];
    long long xb[2], xt[2], xh[2], yb[2], yt[2], yh[2];  // element strides of sequence, token, head
    int heads[2];
    const void* pos;
    long long pb, pt, pa;
    int B, T, D, pairs, inverse;
    int slots, turned;   // slots of a token's head; the first `turned` of them turn, the others copy
    int nt;              // tokens per workgroup
    int nb, hc;          // sequences and heads (of q and k together) per workgroup
    int overlap;         // the last slot of a number of pairs that a slot's does not divide lies over the one before it (out of place: both write the same)
    int tail, tail_at;   // features behind the last slot that are copied
    unsigned pairs_mul;  // divides an entry's number by pairs
    unsigned tail_mul, per_mul;  // divide a copied feature's number by tail and by tail * heads (division_multiplier)
};

DEVFN int quotient(int x, int d, unsigned mul) { return mul ? (int)__umulhi((unsigned)x, mul) : x / d; }

// One rotation, the same operations wherever it stands: in place and out of place agree to the bit
DEVFN void rotate(float& p, float& q, float c, float s) {
    const float u = fmaf(p, c, -__fmul_rn(q, s)), v = fmaf(p, s, __fmul_rn(q, c));
    p = u;
    q = v;
}

// In memory a slot is one run of features, or ("halves") two. The vector types ask for an element's alignment only: the compiler's 16-byte accesses take any,
// and rows of odd lengths, or views, start anywhere
template <typename T, bool HALVES>
struct Slot {
    static constexpr int PAIRS = 4, RUN = HALVES ? 4 : 8;
    typedef T vec __attribute__((ext_vector_type(RUN), aligned(sizeof(T))));
    vec a, b;
    DEVFN void load(const T* x, int apart) {  // apart: from the first run to the second
        a = *(const vec*)x;
        if constexpr (HALVES) b = *(const vec*)(x + apart);
    }
    DEVFN void store(T* y, int apart) const {
        *(vec*)y = a;
        if constexpr (HALVES) *(vec*)(y + apart) = b;
    }
    DEVFN void up(int n) {  // feature e + n at e
#pragma unroll
        for (int step = 4; step > 0; step >>= 1)
            if (n & step)
#pragma unroll
                for (int e = 0; e + step < 8; ++e) {
                    const T x = !HALVES || e + step < 4 ? a[HALVES ? (e + step) & 3 : e + step] : b[(e + step) & 3];
                    if (!HALVES || e < 4) a[HALVES ? e & 3 : e] = x;
                    else b[e & 3] = x;
                }
    }
    DEVFN void turn(const float (&c)[PAIRS], const float (&s)[PAIRS]) {
#pragma unroll
        for (int e = 0; e < PAIRS; ++e) {
            float p = (float)(HALVES ? a[e] : a[2 * e]), q = (float)(HALVES ? b[e] : a[2 * e + 1]);
            rotate(p, q, c[e], s[e]);
            if constexpr (HALVES) {
                a[e] = (T)p;
                b[e] = (T)q;
            } else {
                a[2 * e] = (T)p;
                a[2 * e + 1] = (T)q;
            }
        }
    }
};

template <typename T, bool HALVES, typename P, int R>
__global__ __launch_bounds__(ROT_THREADS, 4) void rotary_kernel(RotArgs g, RotRates<R> rates) {
    const int t = threadIdx.x / g.slots, v = threadIdx.x - t * g.slots, t0 = blockIdx.x * g.nt;
    const bool mine = t < g.nt && t0 + t < g.T;
    using Part = Slot<T, HALVES>;
    constexpr int S = Part::PAIRS, N = 4;  // N heads' loads stand together
    const bool turns = v < g.turned;
    const int j = g.overlap ? min(S * v, g.pairs - S) : S * v, whole = turns ? min(S, g.pairs - j) : S;
    // the last of the copying slots may reach into y's room behind the features: it reads the row's last 8 and moves them up
    const int at = !turns ? 2 * g.pairs + 2 * S * (v - g.turned) : HALVES ? j : 2 * j, apart = turns ? g.pairs : Part::RUN;
    const int over = !turns ? max(0, at + 2 * S - g.D) : 0;
    const int h0 = blockIdx.z * g.hc, h1 = min(h0 + g.hc, g.heads[0] + g.heads[1]);
    // the cosines and sines of the workgroup's tokens, each computed once, then a thread's own in its registers
    __shared__ float s_cos[ROT_THREADS * S], s_sin[ROT_THREADS * S];
    float c[S], s[S];
    auto angles = [&](int b) {
        const P* pos = (const P*)g.pos + (long long)b * g.pb + (long long)t0 * g.pt;
        const int entries = min(g.nt, g.T - t0) * g.pairs;
        for (int i = threadIdx.x; i < entries; i += ROT_THREADS) {
            const int ti = quotient(i, g.pairs, g.pairs_mul), k = i - ti * g.pairs;
            const double turns = (double)pos[(long long)ti * g.pt + rates.axis[k] * g.pa] * rates.turns[k];
            float sine, cosine;
            sincospif(2.f * (float)(turns - rint(turns)), &sine, &cosine);
            s_cos[i] = cosine;
            s_sin[i] = g.inverse ? -sine : sine;
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < S; ++e) {
            const int i = t * g.pairs + min(j + e, g.pairs - 1);
            c[e] = mine && turns ? s_cos[i] : 1.f;
            s[e] = mine && turns ? s_sin[i] : 0.f;
        }
        __syncthreads();
    };
    // the features behind the last slot, one a thread, densely: in their slots' place they would leave most lanes of a wave waiting
    const int copies = g.tail > 0 ? min(g.nt, g.T - t0) * (h1 - h0) * g.tail : 0;
    auto copied = [&](int i, const T*& from, T*& to) {
        const int per = (h1 - h0) * g.tail, ti = g.hc == h1 - h0 ? quotient(i, per, g.per_mul) : i / per, r = i - ti * per;
        const int hh = quotient(r, g.tail, g.tail_mul), f = g.tail_at + r - hh * g.tail, w = h0 + hh >= g.heads[0], h = w ? h0 + hh - g.heads[0] : h0 + hh;
        from = (const T*)g.x[w] + (long long)(t0 + ti) * g.xt[w] + (long long)h * g.xh[w] + f;
        to = (T*)g.y[w] + (long long)(t0 + ti) * g.yt[w] + (long long)h * g.yh[w] + f;
        return w;
    };
    const int b0 = blockIdx.y * g.nb, b1 = min(b0 + g.nb, g.B);
    if (g.pb == 0) angles(0);
    for (int b = b0; b < b1; ++b) {
        if (g.pb != 0) {
            if (b > b0) __syncthreads();  // the last sequence's have been read by all: those in place read them here, not in registers
            angles(b);
        }
#pragma unroll 1
        for (int w = 0; w < 2; ++w) {
            if (!mine) break;
            const int first = w ? g.heads[0] : 0, lo = max(h0, first) - first, hi = min(h1 - first, g.heads[w]);
            const T* x = (const T*)g.x[w] + (long long)b * g.xb[w] + (long long)(t0 + t) * g.xt[w] + (long long)lo * g.xh[w] + at;
            T* y = (T*)g.y[w] + (long long)b * g.yb[w] + (long long)(t0 + t) * g.yt[w] + (long long)lo * g.yh[w] + at;
            if (whole == S) {
                int h = lo;
#pragma unroll 1
                for (; h + N <= hi; h += N) {
                    Part slot[N];
#pragma unroll
                    for (int n = 0; n < N; ++n) slot[n].load(x + n * g.xh[w] - over, apart);
#pragma unroll
                    for (int n = 0; n < N; ++n) {
                        if (turns) slot[n].turn(c, s);
                        else slot[n].up(over);
                        slot[n].store(y + n * g.yh[w], apart);
                    }
                    x += N * g.xh[w];
                    y += N * g.yh[w];
                }
#pragma unroll 1
                for (; h < hi; ++h, x += g.xh[w], y += g.yh[w]) {
                    Part slot;
                    slot.load(x - over, apart);
                    if (turns) slot.turn(c, s);
                    else slot.up(over);
                    slot.store(y, apart);
                }
            } else {  // in place, or fewer pairs than a slot in all
#pragma unroll 1
                for (int i = 0; i < (hi - lo) * whole; ++i) {
                    const int h = i / whole, e = i - h * whole, i0 = HALVES ? e : 2 * e, i1 = HALVES ? g.pairs + e : i0 + 1;
                    const T* xh = x + (long long)h * g.xh[w];
                    T* yh = y + (long long)h * g.yh[w];
                    float p = (float)xh[i0], q = (float)xh[i1];
                    rotate(p, q, s_cos[t * g.pairs + j + e], s_sin[t * g.pairs + j + e]);
                    yh[i0] = (T)p;
                    yh[i1] = (T)q;
                }
            }
        }
        for (int i = threadIdx.x; i < copies; i += ROT_THREADS) {
            const T* p;
            T* q;
            const int w = copied(i, p, q);
            q[(long long)b * g.yb[w]] = p[(long long)b * g.xb[w]];
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

template <typename T, bool HALVES, int R>
int launch_p(const RotArgs& a, const RotAllRates& all, int pos_type, dim3 grid, hipStream_t s) {
    RotRates<R> r;
    std::copy_n(all.turns, R, r.turns);
    std::copy_n(all.axis, R, r.axis);
    if (pos_type == 0) hipLaunchKernelGGL((rotary_kernel<T, HALVES, int, R>), grid, dim3(ROT_THREADS), 0, s, a, r);
    else if (pos_type == 1) hipLaunchKernelGGL((rotary_kernel<T, HALVES, long long, R>), grid, dim3(ROT_THREADS), 0, s, a, r);
    else hipLaunchKernelGGL((rotary_kernel<T, HALVES, float, R>), grid, dim3(ROT_THREADS), 0, s, a, r);
    return hipGetLastError() == hipSuccess ? V1T_OK : V1T_ERR_LAUNCH;
}
template <typename T, bool HALVES>
int launch_r(const RotArgs& a, const RotAllRates& r, int pos_type, dim3 grid, hipStream_t s) {
    return a.pairs <= 64 ? launch_p<T, HALVES, 64>(a, r, pos_type, grid, s) : launch_p<T, HALVES, ROT_MAX_PAIRS>(a, r, pos_type, grid, s);
}
template <typename T>
int launch_t(const RotArgs& a, const RotAllRates& r, int halves, int pos_type, dim3 grid, hipStream_t s) {
    return halves ? launch_r<T, true>(a, r, pos_type, grid, s) : launch_r<T, false>(a, r, pos_type, grid, s);
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
    RotArgs g{};
    RotAllRates r{};
    for (int a = 0, j = 0; a < n_axes; ++a)
        for (int i = 0; i < sections[a]; ++i, ++j) {
            const double part = shared ? (double)j / (double)pairs : (double)i / (double)sections[a];
            r.turns[j] = std::pow(base, -part) / 6.283185307179586476925286766559;
            r.axis[j] = (unsigned char)a;
        }
    bool in_place = true;
    long long heads = 0;
    int room = 1 << 30;
    for (int o = 0; o < n_ops; ++o) {
        const v1t_rotary_operand& p = ops[o];
        if (!p.x || !p.y || p.heads < 1) return V1T_ERR_ARG;
        g.x[o] = p.x; g.y[o] = p.y; g.heads[o] = p.heads;
        g.xb[o] = p.x_stride_b; g.xt[o] = p.x_stride_t; g.xh[o] = p.x_stride_h;
        g.yb[o] = p.y_stride_b; g.yt[o] = p.y_stride_t; g.yh[o] = p.y_stride_h;
        heads += p.heads;
        if (p.y_room < 0 || (p.y_room > 0 && p.y_room < D)) return V1T_ERR_ARG;
        room = std::min(room, p.y_room > 0 ? p.y_room : D);
        const bool same = p.x == p.y;
        if (o > 0 && same != in_place) return V1T_ERR_ARG;
        in_place = same;
        if (same && (p.x_stride_b != p.y_stride_b || p.x_stride_t != p.y_stride_t || p.x_stride_h != p.y_stride_h)) return V1T_ERR_ARG;
    }
    if (B == 0 || T == 0) return V1T_OK;
    g.pos = positions; g.pb = B == 1 ? 0 : pos_stride_b; g.pt = pos_stride_t; g.pa = pos_stride_a;
    g.B = B; g.T = T; g.D = D; g.pairs = (int)pairs; g.inverse = inverse != 0;
    constexpr int slot = 4;  // Slot::PAIRS
    g.turned = (int)((pairs + slot - 1) / slot);
    g.overlap = !in_place && pairs >= slot;
    const int rest = in_place ? 0 : D - 2 * (int)pairs;  // copied: by slots, and the remainder - if y's rows have no room for a whole one - by features
    const bool whole = room >= 2 * (int)pairs + (rest + 2 * slot - 1) / (2 * slot) * (2 * slot) && D >= 2 * slot;
    g.slots = std::min(g.turned + (whole ? rest + 2 * slot - 1 : rest) / (2 * slot), ROT_THREADS);
    g.tail_at = 2 * (int)pairs + 2 * slot * (g.slots - g.turned);
    g.tail = in_place ? 0 : std::max(0, D - g.tail_at);
    g.nt = std::max(1, std::min(ROT_THREADS / g.slots, T));
    g.pairs_mul = division_multiplier(pairs, g.nt * pairs);
    // A workgroup takes all heads and as many sequences as share their positions with it, while 2048 workgroups (8 a CU) are left; fewer tokens than that: the heads
    // are dealt out, down to the 4 whose loads stand together
    const long long gx = ((long long)T + g.nt - 1) / g.nt;
    if (gx >= (1 << 24)) return V1T_ERR_UNSUPPORTED;  // a launch has less than 2^32 threads
    long long nb = g.pb == 0 ? std::max(1ll, std::min<long long>(16, gx * B / 2048)) : 1;
    nb = std::max(nb, ((long long)B + 65534) / 65535);
    const long long gy = ((long long)B + nb - 1) / nb;
    long long hc = heads;
    while (hc > 4 && gx * gy * ((heads + hc - 1) / hc) < 2048) hc = (hc + 1) / 2;
    hc = std::max(hc, (heads + 65534) / 65535);
    if (heads > (1 << 24)) return V1T_ERR_UNSUPPORTED;
    g.nb = (int)nb; g.hc = (int)hc;
    if (g.tail > 0) {
        if ((long long)g.nt * hc * g.tail > (1ll << 30)) return V1T_ERR_UNSUPPORTED;
        g.tail_mul = division_multiplier(g.tail, hc * g.tail);
        g.per_mul = division_multiplier(hc * g.tail, g.nt * hc * g.tail);
    }
    const dim3 grid((unsigned)gx, (unsigned)gy, (unsigned)((heads + hc - 1) / hc));
    hipStream_t st = (hipStream_t)stream;
    if (dtype == 0) return launch_t<bf16_t>(g, r, halves, position_type, grid, st);
    if (dtype == 1) return launch_t<f16_t>(g, r, halves, position_type, grid, st);
    return launch_t<float>(g, r, halves, position_type, grid, st);
}
