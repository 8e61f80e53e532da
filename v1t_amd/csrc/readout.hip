// v1t_amd — Gaussian2d readout kernels (gfx950). Replaces, for one mouse,
//   F.grid_sample(z, grid, align_corners=True) -> * features -> sum(dim=1) -> + bias
// (reference gaussian2d.py:270-276) without materialising the (B,C,N) sampled tensor.
//
// Layout: the core's residual stream is read token-major as it lies in HBM ([b][cell][c], channel
// stride 1, so a bilinear tap is one contiguous C-float row); the feature weights are stored
// neuron-major [n][c] (row stride FS). One wave per neuron walks all images of the batch with
// lanes spanning channels: every load is a coalesced row, the feature row stays in registers, the
// channel sum is one wave reduction. HBM-bound; algorithmic bytes in DESIGN.md.
#include "readout.h"

#include <algorithm>

namespace {

struct Taps {
    int cell[4];
    float w[4];     // bilinear weight, 0 when the tap is outside the map (zeros padding)
    float ax, ay;
    bool in[4];
};

DEVFN Taps make_taps(float gx, float gy, int W, int H) {
    Taps t;
    const float px = (gx + 1.f) * 0.5f * (float)(W - 1);
    const float py = (gy + 1.f) * 0.5f * (float)(H - 1);
    const float fx = floorf(px), fy = floorf(py);
    const int x0 = (int)fx, y0 = (int)fy;
    t.ax = px - fx;
    t.ay = py - fy;
    const float wx[2] = {1.f - t.ax, t.ax}, wy[2] = {1.f - t.ay, t.ay};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int xi = x0 + (k & 1), yi = y0 + (k >> 1);
        t.in[k] = xi >= 0 && xi < W && yi >= 0 && yi < H;
        t.cell[k] = t.in[k] ? yi * W + xi : 0;
        t.w[k] = t.in[k] ? wx[k & 1] * wy[k >> 1] : 0.f;
    }
    return t;
}

template <int NE>
DEVFN void readout_fwd_body(const ReadoutArgs& a, int bx) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = bx * 4 + wave;
    if (n >= a.N) return;
    float f[NE];
#pragma unroll
    for (int i = 0; i < NE; ++i) {
        const int c = lane + 64 * i;
        f[i] = (c < a.C) ? a.feat[(size_t)n * a.FS + c] : 0.f;
    }
    const float bias = a.bias ? a.bias[n] : 0.f;
    for (int b = 0; b < a.B; ++b) {
        const float gx = a.grid[((size_t)b * a.N + n) * 2 + 0];
        const float gy = a.grid[((size_t)b * a.N + n) * 2 + 1];
        const Taps t = make_taps(gx, gy, a.W, a.H);
        const float* zb = a.z + (size_t)b * a.zsb;
        float acc = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float* zr = zb + (size_t)t.cell[k] * a.zsc;
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                const int c = lane + 64 * i;
                const float zv = (c < a.C) ? zr[c] : 0.f;
                acc += t.w[k] * f[i] * zv;
            }
        }
        acc = wave_sum(acc);
        if (lane == 0) a.out[(size_t)b * a.N + n] = acc + bias;
    }
}

template <int NE>
__global__ __launch_bounds__(256) void readout_fwd_kernel(ReadoutArgs a) { readout_fwd_body<NE>(a, blockIdx.x); }

// Backward: G = dL/du (B,N).  dbias[n] += sum_b G;  dfeat[n][c] += sum_b G * S[b][c]   (owned by the
// wave: plain +=);  dz[b][tap][c] += G * w_tap * F[n][c]  (fp32 atomics, 256-B contiguous runs);
// dgrid[b][n] = (dL/dgx, dL/dgy) through the bilinear weights.
template <int NE>
DEVFN void readout_bwd_body(const ReadoutArgs& a, int bx) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = bx * 4 + wave;
    if (n >= a.N) return;
    float f[NE], df[NE];
#pragma unroll
    for (int i = 0; i < NE; ++i) {
        const int c = lane + 64 * i;
        f[i] = (c < a.C) ? a.feat[(size_t)n * a.FS + c] : 0.f;
        df[i] = 0.f;
    }
    float gsum = 0.f;
    for (int b = 0; b < a.B; ++b) {
        const float gx = a.grid[((size_t)b * a.N + n) * 2 + 0];
        const float gy = a.grid[((size_t)b * a.N + n) * 2 + 1];
        const float G = a.gout[(size_t)b * a.N + n];
        gsum += G;
        const Taps t = make_taps(gx, gy, a.W, a.H);
        const float* zb = a.z + (size_t)b * a.zsb;
        float* dzb = a.dz ? a.dz + (size_t)b * a.dzsb : nullptr;
        float sx = 0.f, sy = 0.f;
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            const int c = lane + 64 * i;
            float zv[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) zv[k] = (c < a.C && t.in[k]) ? zb[(size_t)t.cell[k] * a.zsc + c] : 0.f;
            df[i] += G * (t.w[0] * zv[0] + t.w[1] * zv[1] + t.w[2] * zv[2] + t.w[3] * zv[3]);
            sx += f[i] * ((1.f - t.ay) * (zv[1] - zv[0]) + t.ay * (zv[3] - zv[2]));
            sy += f[i] * ((1.f - t.ax) * (zv[2] - zv[0]) + t.ax * (zv[3] - zv[1]));
            if (dzb && c < a.C) {  // no-scratch form only (launch_readout_bwd without ws)
                const float gf = G * f[i];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (t.in[k]) atomicAdd(&dzb[(size_t)t.cell[k] * a.dzsc + c], gf * t.w[k]);
            }
        }
        if (a.dgrid) {
            sx = wave_sum(sx);
            sy = wave_sum(sy);
            if (lane == 0) {
                a.dgrid[((size_t)b * a.N + n) * 2 + 0] = G * sx * 0.5f * (float)(a.W - 1);
                a.dgrid[((size_t)b * a.N + n) * 2 + 1] = G * sy * 0.5f * (float)(a.H - 1);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NE; ++i) {
        const int c = lane + 64 * i;
        if (a.dfeat && c < a.C) a.dfeat[(size_t)n * a.FS + c] += df[i];
    }
    if (a.dbias && lane == 0) a.dbias[n] += gsum;
}

template <int NE>
__global__ __launch_bounds__(256) void readout_bwd_kernel(ReadoutArgs a) { readout_bwd_body<NE>(a, blockIdx.x); }

// dz without float atomics (4 x C x N x B adds = 317 MB at N = 8000, B = 16: ~250 us at the chip-wide 1.3 TB/s atomic rate; LDS float
// atomics are slower still, ~1 lane per clock per CU - and the order of any of them changes the sums): invert the sampling. Everything is
// in a fixed order, so dz is the same bit for bit in every pass: the core's backward rounds it to bf16 next, where another last bit of a sum
// becomes another bf16 value, and that a row of every weight gradient behind it.
//   sort  : workgroup (slice s of the neurons, image b) sorts keys (cell, tap) by cell in LDS, in the order of the taps
//   merge : the image's slices into one list by cell, within a cell by neuron: (cell, tap id, bilinear weight); taps outside the map and the
//           list's padding carry the sentinel cell `cells` and come last
//   gather: a wave per 64 consecutive taps sums G[b][n] * w * F[n][:] (coalesced feature rows) while the cell stays the same. A run of equal
//           cells is all of its cell: added to dz. One that is cut between the waves of a workgroup is put together in LDS, one that is cut
//           between workgroups leaves a part in the scratch
//   join  : adds the parts of a run in order. Balanced for any distribution of the neurons over the map - including the freshly initialised
//           model, whose 8000 neurons all sit on a handful of cells
// 16 images, 8000 neurons: sort 17, merge 12, gather 31 and join 5 us where the neurons lie all over the map; 17, 9, 27 and 5 us where all lie in one cell (in an earlier form,
// whose runs met in atomics in any order, 18 us and 44, 18 and 33). The training step sorts and merges beside the core's forward.
constexpr int DZ_SLICES = 4;       // neuron slices per image at least (parallelism of the sort)
constexpr int DZ_SLICE = 2048;     // neurons per slice at most: 8192 keys in LDS
constexpr int DZ_MAX_CELLS = 4096; // LDS table capacity; larger maps use the atomic form
constexpr int DZ_TAP_BITS = 13;    // key = cell << 13 | tap of the slice
constexpr int DZ_GROUP = 256;      // taps per workgroup of the gather, 64 a wave
constexpr int DZ_PART = 256;       // floats of a part (C <= 256)
static_assert((4 * DZ_SLICE) >> DZ_TAP_BITS <= 1 && (unsigned long long)(DZ_MAX_CELLS + 1) << DZ_TAP_BITS < 0xffffffffu, "keys");
constexpr int DZ_DIGIT_BITS = 7, DZ_DIGITS = 1 << DZ_DIGIT_BITS;  // two passes over a cell's bits
static_assert(DZ_MAX_CELLS < DZ_DIGITS * DZ_DIGITS && DZ_DIGITS * 16 % 1024 == 0, "digits");
struct DzSort {
    unsigned* keys;   // [B][slices][4 * ns] sorted
    int* first;       // [B][slices][cells + 1] where a slice's cells begin
    unsigned* cell;   // [B][R]
    unsigned* id;     // tap id = 4 * (b * N + n) + k
    float* wt;
    float* part;      // [B * R / DZ_GROUP][2][DZ_PART]: a group's part of the run that began before it, of the run that goes on behind it
    int slices, ns, R;  // neurons per slice, taps per image (multiple of DZ_GROUP)
};

// One pass of a radix sort in LDS: n keys (a multiple of 1024) by 7 bits, equal ones in the order they came in. A wave owns n / 16 keys in a row, 64 at a time: the lanes of a
// digit find each other by ballots, their places in the wave's share are the digit's count so far and their number among themselves.
struct DzSortLds {
    unsigned key[2][4 * DZ_SLICE];
    int count[16][DZ_DIGITS + 1];  // [wave][digit]
    int sum[16];
};
DEVFN void dz_wave_sync() {  // between one lane's write to LDS and another's read, within a wave
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
// sum of v over the threads before this one of 1024; sum: LDS of 16
DEVFN int dz_exclusive_scan(int v, int* sum) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int inc = v;  // inclusive over the wave
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(inc, o);
        if (lane >= o) inc += x;
    }
    if (lane == 63) sum[wave] = inc;
    __syncthreads();
    int base = inc - v;
    for (int w = 0; w < wave; ++w) base += sum[w];
    return base;
}

DEVFN void dz_radix_pass(DzSortLds& L, int src, int n, int shift) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, own = n / 16;
    constexpr int GROUPS = 4 * DZ_SLICE / 1024;
    unsigned k[GROUPS];
    int at[GROUPS];
    for (int i = tid; i < 16 * (DZ_DIGITS + 1); i += 1024) (&L.count[0][0])[i] = 0;
    __syncthreads();
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        if (64 * g >= own) break;
        k[g] = L.key[src][wave * own + 64 * g + lane];
        const unsigned d = k[g] >> shift & (DZ_DIGITS - 1);
        unsigned long long same = ~0ull;
#pragma unroll
        for (int bit = 0; bit < DZ_DIGIT_BITS; ++bit) {
            const bool on = d >> bit & 1;
            const unsigned long long b = __ballot(on);
            same &= on ? b : ~b;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1)), before = L.count[wave][d];
        at[g] = before + rank;
        dz_wave_sync();
        if (rank == 0) L.count[wave][d] = before + __popcll(same);
        dz_wave_sync();
    }
    __syncthreads();
    // counts -> first places, digit by digit and wave by wave
    int v[DZ_DIGITS * 16 / 1024], tot = 0;
#pragma unroll
    for (int e = 0; e < DZ_DIGITS * 16 / 1024; ++e) {
        const int i = tid * (DZ_DIGITS * 16 / 1024) + e;
        v[e] = L.count[i & 15][i >> 4];
        tot += v[e];
    }
    int base = dz_exclusive_scan(tot, L.sum);
#pragma unroll
    for (int e = 0; e < DZ_DIGITS * 16 / 1024; ++e) {
        const int i = tid * (DZ_DIGITS * 16 / 1024) + e;
        L.count[i & 15][i >> 4] = base;
        base += v[e];
    }
    __syncthreads();
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        if (64 * g >= own) break;
        L.key[src ^ 1][L.count[wave][k[g] >> shift & (DZ_DIGITS - 1)] + at[g]] = k[g];
    }
    __syncthreads();
}

DEVFN void readout_sort_body(const ReadoutArgs& a, const DzSort& ix, int s, int b, DzSortLds& L) {
    const int tid = threadIdx.x;
    const int cells = a.H * a.W;
    const int n0 = min(a.N, s * ix.ns), cnt = min(a.N - n0, ix.ns), taps = 4 * cnt, n = (taps + 1023) / 1024 * 1024;
    for (int i = tid; i < n / 4; i += 1024) {
        u32x4 v = {~0u, ~0u, ~0u, ~0u};
        if (i < cnt) {
            const size_t g = 2 * ((size_t)b * a.N + n0 + i);
            const Taps t = make_taps(a.grid[g], a.grid[g + 1], a.W, a.H);
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = (unsigned)(t.in[q] ? t.cell[q] : cells) << DZ_TAP_BITS | (unsigned)(4 * i + q);
        }
        *(u32x4*)&L.key[0][4 * i] = v;
    }
    __syncthreads();
    dz_radix_pass(L, 0, n, DZ_TAP_BITS);
    dz_radix_pass(L, 1, n, DZ_TAP_BITS + DZ_DIGIT_BITS);
    const unsigned* key = L.key[0];
    const size_t reg = (size_t)b * ix.slices + s;
    for (int p = tid; p < taps; p += 1024) ix.keys[reg * (4 * ix.ns) + p] = key[p];
    for (int c = tid; c <= cells; c += 1024) {  // the first key at or above the cell's least
        int lo = 0, hi = taps;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (key[mid] < (unsigned)c << DZ_TAP_BITS) lo = mid + 1;
            else hi = mid;
        }
        ix.first[reg * (cells + 1) + c] = lo;
    }
}
__global__ __launch_bounds__(1024) void readout_sort_kernel(ReadoutArgs a, DzSort ix) {
    __shared__ __attribute__((aligned(16))) DzSortLds L;
    readout_sort_body(a, ix, blockIdx.x, blockIdx.y, L);
}

DEVFN void readout_merge_body(const ReadoutArgs& a, const DzSort& ix, int s, int b, int* to, int* wsum) {
    const int tid = threadIdx.x;
    const int cells = a.H * a.W;
    auto taps_of = [&](int x) { return 4 * max(0, min(a.N - x * ix.ns, ix.ns)); };
    // to[c]: what a tap of cell c adds to its place in the slice for its place in the image. Each thread owns a contiguous run of PER cells
    constexpr int MOST = (DZ_MAX_CELLS + 1 + 1023) / 1024;
    const int PER = (cells + 1 + 1023) / 1024;
    int run[MOST], mine[MOST], tot = 0;  // the image's taps of a cell; where this slice's begin behind them, less their place in the slice
#pragma unroll
    for (int e = 0; e < MOST; ++e) {
        const int c = tid * PER + e;
        run[e] = mine[e] = 0;
        if (e >= PER || c > cells) continue;
        for (int x = 0; x < ix.slices; ++x) {
            const int* first = ix.first + ((size_t)b * ix.slices + x) * (cells + 1);
            const int at = first[c], next = c < cells ? first[c + 1] : taps_of(x);
            if (x == s) mine[e] = run[e] - at;
            run[e] += next - at;
        }
        tot += run[e];
    }
    int base = dz_exclusive_scan(tot, wsum);
#pragma unroll
    for (int e = 0; e < MOST; ++e) {
        const int c = tid * PER + e;
        if (e < PER && c <= cells) {
            to[c] = base + mine[e];
            base += run[e];
        }
    }
    __syncthreads();
    const unsigned* keys = ix.keys + ((size_t)b * ix.slices + s) * (4 * ix.ns);
    const size_t reg = (size_t)b * ix.R, i0 = (size_t)b * a.N + (size_t)s * ix.ns;
    constexpr int MINE = 4 * DZ_SLICE / 1024;  // a thread's taps, all loads in flight together
    const int taps = taps_of(s);
    unsigned k[MINE];
    float gx[MINE], gy[MINE];
#pragma unroll
    for (int e = 0; e < MINE; ++e) k[e] = tid + 1024 * e < taps ? keys[tid + 1024 * e] : 0u;
#pragma unroll
    for (int e = 0; e < MINE; ++e) {
        const size_t i = i0 + ((k[e] & ((1u << DZ_TAP_BITS) - 1)) >> 2);
        const bool on = tid + 1024 * e < taps;
        gx[e] = on ? a.grid[2 * i] : 0.f;
        gy[e] = on ? a.grid[2 * i + 1] : 0.f;
    }
#pragma unroll
    for (int e = 0; e < MINE; ++e) {
        const int p = tid + 1024 * e;
        if (p >= taps) break;
        const unsigned c = k[e] >> DZ_TAP_BITS, tap = k[e] & ((1u << DZ_TAP_BITS) - 1);
        const Taps t = make_taps(gx[e], gy[e], a.W, a.H);
        const size_t at = reg + to[c] + p;
        ix.cell[at] = c;
        ix.id[at] = 4u * (unsigned)i0 + tap;
        ix.wt[at] = (tap & 2 ? (tap & 1 ? t.w[3] : t.w[2]) : (tap & 1 ? t.w[1] : t.w[0]));
    }
    if (s == 0)
        for (int p = 4 * a.N + tid; p < ix.R; p += 1024) ix.cell[reg + p] = (unsigned)cells;  // padding
}
__global__ __launch_bounds__(1024) void readout_merge_kernel(ReadoutArgs a, DzSort ix) {
    __shared__ int to[DZ_MAX_CELLS + 1];
    __shared__ int wsum[16];
    readout_merge_body(a, ix, blockIdx.x, blockIdx.y, to, wsum);
}

template <int NE>
DEVFN void readout_dz_gather_body(const ReadoutArgs& a, const DzSort& ix, int bx) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const unsigned groups = ix.R / DZ_GROUP, b = (unsigned)bx / groups, gi = (unsigned)bx % groups;
    const unsigned cells = a.H * a.W;
    __shared__ float s_cut[4][2][64 * NE];  // a wave's part of the run that began before its taps, and of the one that goes on behind them
    // lane j holds the wave's tap j
    const unsigned* cl = ix.cell + (size_t)bx * DZ_GROUP;
    const size_t me = (size_t)bx * DZ_GROUP + 64 * wave + lane;
    const unsigned key = ix.cell[me];
    auto cell_at = [&](int t) { return t < 0 && gi == 0 || t >= DZ_GROUP && gi + 1 == groups ? cells : cl[t]; };  // tap t of the group, the neighbouring groups' too
    const unsigned before = cell_at(64 * wave - 1), behind = cell_at(64 * wave + 64);
    const unsigned id = key < cells ? ix.id[me] : 0u;
    const float gw = key < cells ? ix.wt[me] * a.gout[id >> 2] : 0.f;
    const unsigned nn = (id >> 2) % (unsigned)a.N;
    float acc[NE];
#pragma unroll
    for (int j = 0; j < NE; ++j) acc[j] = 0.f;
    unsigned cur = __builtin_amdgcn_readfirstlane(key);
    bool head = cur == before;  // the current run began before this wave's taps
    auto add = [&](unsigned row) {  // the only addend of its pass: an atomic because nothing waits for it (a load to add to holds up the features')
        float* dzr = a.dz + (size_t)b * a.dzsb + (size_t)row * a.dzsc;
#pragma unroll
        for (int j = 0; j < NE; ++j)
            if (lane + 64 * j < a.C) atomicAdd(&dzr[lane + 64 * j], acc[j]);
    };
    auto flush = [&](unsigned row, bool cut) {  // cut: it goes on in the next wave's
        if (head || cut) {
#pragma unroll
            for (int j = 0; j < NE; ++j) s_cut[wave][head ? 0 : 1][lane + 64 * j] = acc[j];
        } else {
            add(row);
        }
#pragma unroll
        for (int j = 0; j < NE; ++j) acc[j] = 0.f;
        head = false;
    };
    constexpr int RIF = 8;  // feature rows in flight (4 -> 8 rows: 189 -> 178 us per step)
    for (int t0 = 0; t0 < 64; t0 += RIF) {
        unsigned kq[RIF], nq[RIF], gq[RIF];
        float f[RIF][NE];
#pragma unroll
        for (int u = 0; u < RIF; ++u) {
            kq[u] = __builtin_amdgcn_readlane(key, t0 + u);
            nq[u] = __builtin_amdgcn_readlane(nn, t0 + u);
            gq[u] = __builtin_amdgcn_readlane(__float_as_uint(gw), t0 + u);
        }
        if (kq[0] >= cells) break;  // sentinels and padding sort to the end of the image
#pragma unroll
        for (int u = 0; u < RIF; ++u)
#pragma unroll
            for (int j = 0; j < NE; ++j) {
                const int c = lane + 64 * j;
                f[u][j] = (c < a.C) ? a.feat[(size_t)nq[u] * a.FS + c] : 0.f;
            }
#pragma unroll
        for (int u = 0; u < RIF; ++u) {
            if (kq[u] >= cells) break;
            if (kq[u] != cur) {
                flush(cur, false);
                cur = kq[u];
            }
            const float g = __uint_as_float(gq[u]);
#pragma unroll
            for (int j = 0; j < NE; ++j) acc[j] += g * f[u][j];
        }
    }
    const unsigned first = __builtin_amdgcn_readfirstlane(key), last = __builtin_amdgcn_readlane(key, 63);
    if (cur < cells) flush(cur, last == cur && behind == cur);
    __syncthreads();
    // the cut runs, each by the wave that it begins in - one that began before the group by its first - in order
    const bool early = wave == 0 && first < cells && first == before;            // began before the group
    const bool starts = last < cells && last == behind && !(first == last && first == before);  // begins here and goes on
    auto whole_run = [&](unsigned row, int slot, bool began) {
        int w = wave;
#pragma unroll
        for (int j = 0; j < NE; ++j) acc[j] = s_cut[w][slot][lane + 64 * j];
        // wave w's part is followed by wave w + 1's while w's taps end and w + 1's begin with the run
        bool on = cell_at(64 * w + 63) == row && cell_at(64 * w + 64) == row;
        while (on && w < 3) {
            ++w;
#pragma unroll
            for (int j = 0; j < NE; ++j) acc[j] += s_cut[w][0][lane + 64 * j];
            on = cell_at(64 * w + 63) == row && cell_at(64 * w + 64) == row;
        }
        if (!began && !on) return add(row);
        float* to = ix.part + ((size_t)bx * 2 + (began ? 0 : 1)) * DZ_PART;
#pragma unroll
        for (int j = 0; j < NE; ++j) to[lane + 64 * j] = acc[j];
    };
    if (early) whole_run(first, 0, true);
    if (starts) whole_run(last, 1, false);
}
template <int NE>
__global__ __launch_bounds__(256) void readout_dz_gather_kernel(ReadoutArgs a, DzSort ix) { readout_dz_gather_body<NE>(a, ix, blockIdx.x); }

template <int NE>
DEVFN void readout_dz_join_body(const ReadoutArgs& a, const DzSort& ix, int bx) {
    const int lane = threadIdx.x & 63;
    const unsigned groups = ix.R / DZ_GROUP, group = __builtin_amdgcn_readfirstlane(bx * 4 + (int)(threadIdx.x >> 6));
    if (group >= (unsigned)a.B * groups) return;
    const unsigned cells = a.H * a.W, b = group / groups, gi = group % groups;
    const unsigned* cl = ix.cell + (size_t)group * DZ_GROUP;
    if (gi + 1 >= groups) return;
    const unsigned cur = cl[DZ_GROUP - 1], next = cl[DZ_GROUP], first = cl[0], before = gi > 0 ? cl[-1] : cells;
    if (cur >= cells || next != cur) return;         // no run is cut here
    if (first == cur && before == cur) return;       // it began in an earlier group
    // it goes on through groups gi + 1 .. gi + more: the cells are in order, so group x is the last one when group x + 1 begins with another
    unsigned more = 1;
    for (;; more += 64) {
        const unsigned x = gi + more + 1 + lane;
        const unsigned long long on = __ballot(x < groups && cl[(size_t)(x - gi) * DZ_GROUP] == cur);
        if (~on) {
            more += __builtin_ctzll(~on);
            break;
        }
    }
    const float* part = ix.part + (size_t)group * 2 * DZ_PART + lane;  // whole rows, so that nothing stands between the loads: what lies behind the channels is not used
    float acc[NE];
#pragma unroll
    for (int j = 0; j < NE; ++j) acc[j] = part[DZ_PART + 64 * j];
    constexpr unsigned IF = 8;  // parts in flight
    for (unsigned m = 1; m <= more; m += IF) {
        float v[IF][NE];
#pragma unroll
        for (unsigned u = 0; u < IF; ++u)
#pragma unroll
            for (int j = 0; j < NE; ++j) v[u][j] = part[(size_t)min(m + u, more) * 2 * DZ_PART + 64 * j];
#pragma unroll
        for (unsigned u = 0; u < IF; ++u)
#pragma unroll
            for (int j = 0; j < NE; ++j) acc[j] += m + u <= more ? v[u][j] : 0.f;
    }
    float* dzr = a.dz + (size_t)b * a.dzsb + (size_t)cur * a.dzsc;
#pragma unroll
    for (int j = 0; j < NE; ++j)
        if (lane + 64 * j < a.C) atomicAdd(&dzr[lane + 64 * j], acc[j]);  // as in the gather: calls that add to one dz at once lose nothing
}
template <int NE>
__global__ __launch_bounds__(256) void readout_dz_join_kernel(ReadoutArgs a, DzSort ix) { readout_dz_join_body<NE>(a, ix, blockIdx.x); }

// ---- the same kernels over SEVERAL units (mice) in one launch each: a training step runs the tails of all local mice as one launch
// per stage instead of one chain of small launches per mouse (v1t_tails_*). The unit table travels by value in the kernel arguments;
// a workgroup finds its unit from the prefix sums of the units' workgroup counts (wave-uniform scalar loads).
struct ReadoutMulti {
    ReadoutArgs a[TAILS_MAX_UNITS];
    DzSort ix[TAILS_MAX_UNITS];
    int start[TAILS_MAX_UNITS + 1];
    int n;
};
DEVFN int multi_unit(const int* start, int n, int bid, int& local) {
    int u = 0;
    while (u + 1 < n && bid >= start[u + 1]) ++u;
    local = bid - start[u];
    return u;
}
template <int NE>
__global__ __launch_bounds__(256) void readout_fwd_multi_kernel(ReadoutMulti m) {
    int bx;
    const int u = multi_unit(m.start, m.n, blockIdx.x, bx);
    readout_fwd_body<NE>(m.a[u], bx);
}
template <int NE>
__global__ __launch_bounds__(256) void readout_bwd_multi_kernel(ReadoutMulti m) {
    int bx;
    const int u = multi_unit(m.start, m.n, blockIdx.x, bx);
    readout_bwd_body<NE>(m.a[u], bx);
}
__global__ __launch_bounds__(1024) void readout_sort_multi_kernel(ReadoutMulti m) {
    __shared__ __attribute__((aligned(16))) DzSortLds L;
    int bx;
    const int u = multi_unit(m.start, m.n, blockIdx.x, bx);
    readout_sort_body(m.a[u], m.ix[u], bx % m.ix[u].slices, bx / m.ix[u].slices, L);
}
__global__ __launch_bounds__(1024) void readout_merge_multi_kernel(ReadoutMulti m) {
    __shared__ int to[DZ_MAX_CELLS + 1];
    __shared__ int wsum[16];
    int bx;
    const int u = multi_unit(m.start, m.n, blockIdx.x, bx);
    readout_merge_body(m.a[u], m.ix[u], bx % m.ix[u].slices, bx / m.ix[u].slices, to, wsum);
}
template <int NE>
__global__ __launch_bounds__(256) void readout_dz_gather_multi_kernel(ReadoutMulti m) {
    int bx;
    const int u = multi_unit(m.start, m.n, blockIdx.x, bx);
    readout_dz_gather_body<NE>(m.a[u], m.ix[u], bx);
}
template <int NE>
__global__ __launch_bounds__(256) void readout_dz_join_multi_kernel(ReadoutMulti m) {
    int bx;
    const int u = multi_unit(m.start, m.n, blockIdx.x, bx);
    readout_dz_join_body<NE>(m.a[u], m.ix[u], bx);
}

DzSort sort_plan(void* ws, int B, int H, int W, int N, size_t* bytes = nullptr) {
    DzSort d;
    d.slices = std::max(DZ_SLICES, (N + DZ_SLICE - 1) / DZ_SLICE);
    d.ns = (N + d.slices - 1) / d.slices;
    d.R = round_up(4 * N, DZ_GROUP);
    char* p = (char*)ws;
    auto take = [&](size_t words) {
        char* at = p;
        p += (words * 4 + 255) / 256 * 256;
        return at;
    };
    d.part = (float*)take((size_t)B * (d.R / DZ_GROUP) * 2 * DZ_PART);
    d.cell = (unsigned*)take((size_t)B * d.R);
    d.id = (unsigned*)take((size_t)B * d.R);
    d.wt = (float*)take((size_t)B * d.R);
    d.keys = (unsigned*)take((size_t)B * d.slices * 4 * d.ns);
    d.first = (int*)take((size_t)B * d.slices * ((size_t)H * W + 1));
    if (bytes) *bytes = (size_t)(p - (char*)ws);
    return d;
}

template <int NE>
int launch_t(const ReadoutArgs& a, bool bwd, void* ws, size_t ws_bytes, hipStream_t s, int parts = READOUT_BWD_ALL) {
    const dim3 grid((a.N + 3) / 4);
    if (!bwd) {
        hipLaunchKernelGGL(readout_fwd_kernel<NE>, grid, dim3(256), 0, s, a);
    } else if (ws && a.H * a.W <= DZ_MAX_CELLS && ws_bytes >= readout_bwd_ws_bytes(a.B, a.H, a.W, a.N) && (a.dz || parts != READOUT_BWD_ALL)) {
        // the kernels of the sorted form, individually selectable (the training step sorts the taps while the core is still
        // in its forward - the sort needs the sample positions only - and gathers dz before the parameter gradients, so that the
        // core's backward can start as early as possible)
        const DzSort ix = sort_plan(ws, a.B, a.H, a.W, a.N);
        if (parts & READOUT_BWD_SORT) {
            hipLaunchKernelGGL(readout_sort_kernel, dim3(ix.slices, a.B), dim3(1024), 0, s, a, ix);
            hipLaunchKernelGGL(readout_merge_kernel, dim3(ix.slices, a.B), dim3(1024), 0, s, a, ix);
        }
        if (parts & READOUT_BWD_PARAMS) {
            ReadoutArgs a2 = a;
            a2.dz = nullptr;
            hipLaunchKernelGGL(readout_bwd_kernel<NE>, grid, dim3(256), 0, s, a2);
        }
        if ((parts & READOUT_BWD_DZ) && a.dz) {
            const unsigned groups = (unsigned)a.B * (ix.R / DZ_GROUP);
            hipLaunchKernelGGL(readout_dz_gather_kernel<NE>, dim3(groups), dim3(256), 0, s, a, ix);
            hipLaunchKernelGGL(readout_dz_join_kernel<NE>, dim3((groups + 3) / 4), dim3(256), 0, s, a, ix);
        }
    } else if (parts != READOUT_BWD_ALL) {
        return V1T_ERR_WORKSPACE;  // the split form exists with the sorted workspace only
    } else {
        hipLaunchKernelGGL(readout_bwd_kernel<NE>, grid, dim3(256), 0, s, a);
    }
    return hipGetLastError() == hipSuccess ? V1T_OK : V1T_ERR_LAUNCH;
}

int dispatch(const ReadoutArgs& a, bool bwd, void* ws, size_t ws_bytes, hipStream_t s, int parts = READOUT_BWD_ALL) {
    if (a.C > 256 || a.N <= 0) return a.N <= 0 ? V1T_OK : V1T_ERR_UNSUPPORTED;
    switch ((a.C + 63) / 64) {
        case 1: return launch_t<1>(a, bwd, ws, ws_bytes, s, parts);
        case 2: return launch_t<2>(a, bwd, ws, ws_bytes, s, parts);
        case 3: return launch_t<3>(a, bwd, ws, ws_bytes, s, parts);
        default: return launch_t<4>(a, bwd, ws, ws_bytes, s, parts);
    }
}

template <int NE>
int launch_multi_t(ReadoutMulti& m, int stage, hipStream_t s) {
    auto deal = [&](auto blocks) {
        int tot = 0;
        for (int u = 0; u < m.n; ++u) {
            m.start[u] = tot;
            tot += blocks(m.a[u], m.ix[u]);
        }
        return m.start[m.n] = tot;
    };
    int tot = deal([&](const ReadoutArgs& a, const DzSort& ix) {
        return stage == TAILS_SORT ? ix.slices * a.B : stage == TAILS_DZ ? a.B * (ix.R / DZ_GROUP) : (a.N + 3) / 4;
    });
    if (tot == 0) return V1T_OK;
    switch (stage) {
        case TAILS_FWD: hipLaunchKernelGGL(readout_fwd_multi_kernel<NE>, dim3(tot), dim3(256), 0, s, m); break;
        case TAILS_PARAMS: hipLaunchKernelGGL(readout_bwd_multi_kernel<NE>, dim3(tot), dim3(256), 0, s, m); break;
        case TAILS_SORT:
            hipLaunchKernelGGL(readout_sort_multi_kernel, dim3(tot), dim3(1024), 0, s, m);
            hipLaunchKernelGGL(readout_merge_multi_kernel, dim3(tot), dim3(1024), 0, s, m);
            break;
        case TAILS_DZ:
            hipLaunchKernelGGL(readout_dz_gather_multi_kernel<NE>, dim3(tot), dim3(256), 0, s, m);
            tot = deal([](const ReadoutArgs& a, const DzSort& ix) { return (a.B * (ix.R / DZ_GROUP) + 3) / 4; });
            hipLaunchKernelGGL(readout_dz_join_multi_kernel<NE>, dim3(tot), dim3(256), 0, s, m);
            break;
        default: return V1T_ERR_ARG;
    }
    return hipGetLastError() == hipSuccess ? V1T_OK : V1T_ERR_LAUNCH;
}

}  // namespace

int launch_readout_multi(const ReadoutArgs* a, void* const* ws, const size_t* ws_bytes, int n, int stage, hipStream_t s) {
    if (n <= 0) return V1T_OK;
    if (n > TAILS_MAX_UNITS) return V1T_ERR_ARG;
    ReadoutMulti m{};
    m.n = n;
    for (int u = 0; u < n; ++u) {
        m.a[u] = a[u];
        if (a[u].C != a[0].C || a[u].C > 256 || a[u].N <= 0) return V1T_ERR_UNSUPPORTED;
        if (stage == TAILS_PARAMS) m.a[u].dz = nullptr;
        if (stage == TAILS_SORT || stage == TAILS_DZ) {
            if (!ws[u] || a[u].H * a[u].W > DZ_MAX_CELLS || ws_bytes[u] < readout_bwd_ws_bytes(a[u].B, a[u].H, a[u].W, a[u].N)) return V1T_ERR_WORKSPACE;
            m.ix[u] = sort_plan(ws[u], a[u].B, a[u].H, a[u].W, a[u].N);
        }
    }
    switch ((a[0].C + 63) / 64) {
        case 1: return launch_multi_t<1>(m, stage, s);
        case 2: return launch_multi_t<2>(m, stage, s);
        case 3: return launch_multi_t<3>(m, stage, s);
        default: return launch_multi_t<4>(m, stage, s);
    }
}

size_t readout_bwd_ws_bytes(int B, int H, int W, int N) {
    size_t bytes = 0;
    (void)sort_plan(nullptr, B, H, W, N, &bytes);
    return bytes;
}
int launch_readout_fwd(const ReadoutArgs& a, hipStream_t s) { return dispatch(a, false, nullptr, 0, s); }
int launch_readout_bwd(const ReadoutArgs& a, void* ws, size_t ws_bytes, hipStream_t s) { return dispatch(a, true, ws, ws_bytes, s); }
int launch_readout_bwd_parts(const ReadoutArgs& a, void* ws, size_t ws_bytes, int parts, hipStream_t s) { return dispatch(a, true, ws, ws_bytes, s, parts); }
