// Group norm over the rows of a channels-last matrix, fused with (+ residual) -> activation, forward and backward.
//
// x [n, c] holds the rows of `samples` samples (frames); sample s owns the positions offsets[s] .. offsets[s + 1], position p is row
// order[p] (or p).  With R_s the rows of sample s and C_g the channels of group g, over the |R_s| |C_g| values of each pair (s, g):
//   mu = mean x, v = mean (x - mu)^2, xhat = (x - mu) / sqrt(v + eps), z = w xhat + b (+ residual), y = act(z)
// and with gz = dy act'(z), gx = w gz:
//   db = sum gz, dw = sum gz xhat over all rows;   dx = (gx - mean gx - xhat mean(gx xhat)) / sqrt(v + eps);   dresidual = gz
//
// Ten to thirty flops per element: HBM bounds it.  A thread owns a chunk of one to four channels and walks down the rows, as in
// batchnorm.hip (eight 16-bit channels cost so many registers that half as many waves were resident); a workgroup owns a contiguous
// range of positions and takes the samples in it one after the other, so ragged samples, empty ones and shared workgroups need no
// padding and no atomics: the piece of sample s in workgroup k leaves its sums at index k + s (distinct, because later workgroups never
// see earlier samples).
// Sums are held in binary64: its adds run at the rate of binary32's here, and sum x^2 - (sum x)^2 / N keeps its digits.
#include "pvx_common.h"

namespace {

constexpr int kBlk = 512, kWaves = kBlk / 64;
constexpr int kResident = 4;             // waves of a SIMD that the registers leave room for
// Ranges of positions: all of them resident together, no second turn (with half / twice as many 117 301 x 64 bf16 takes 63 / 78 us
// instead of 65, 106 032 x 96 f16 forward 31 / 34 instead of 25, 520 013 x 128 binary32 453 / 445 instead of 410; chunks of four).
constexpr int kTargetBlocks = 256 * 4 * kResident / kWaves;
// Pieces x groups that the apply kernels add up for themselves rather than leave them to a launch between: the GPU's time is the same
// (117 301 x 64 bf16 forward and backward 65.1 us, 64.5 with that launch), the host's is shorter by two launches.
constexpr int kMergedSums = 8192;
// rows of a thread whose loads are on their way together
template <typename E, int V> constexpr int kAhead = sizeof(E) * V == 16 ? 2 : 4;
constexpr int kOneChunks = 4, kOneSamples = 512;        // the one-launch form: rows of a thread, and samples

template <typename E, int V> struct alignas(sizeof(E) * V) Pack { E e[V]; };

template <typename E, int V> __device__ __forceinline__ void load_pack(const E* p, float (&v)[V]) {
    const Pack<E, V> k = *reinterpret_cast<const Pack<E, V>*>(p);
#pragma unroll
    for (int j = 0; j < V; j++) v[j] = (float)k.e[j];
}

template <typename E, int V> __device__ __forceinline__ Pack<E, V> row_pack(const E* p, int row, int c, int chunk) {
    return *reinterpret_cast<const Pack<E, V>*>(p + (size_t)row * c + chunk * V);
}

template <typename E, int V> __device__ __forceinline__ void store_pack(E* p, const float (&v)[V]) {
    Pack<E, V> k;
#pragma unroll
    for (int j = 0; j < V; j++) k.e[j] = (E)v[j];
    *reinterpret_cast<Pack<E, V>*>(p) = k;
}

__device__ __forceinline__ float load_param(const void* p, int dtype, int i, float none) {
    if (!p) return none;
    if (dtype == PVX_F32) return reinterpret_cast<const float*>(p)[i];
    if (dtype == PVX_F16) return (float)reinterpret_cast<const _Float16*>(p)[i];
    return (float)reinterpret_cast<const __bf16*>(p)[i];
}

__device__ __forceinline__ void store_param(void* p, int dtype, int i, double v) {
    if (dtype == PVX_F32) reinterpret_cast<float*>(p)[i] = (float)v;
    else if (dtype == PVX_F16) reinterpret_cast<_Float16*>(p)[i] = (_Float16)(float)v;
    else reinterpret_cast<__bf16*>(p)[i] = (__bf16)(float)v;
}

// Phi(z), and e = exp(-z^2 / 2) on the way, by Abramowitz and Stegun 7.1.26: 1 - erf(x) = (a1 t + .. + a5 t^5) exp(-x^2) with
// t = 1 / (1 + p x), x = |z| / sqrt 2, within 1.5e-7 (the library's erff costs three times as much and two branches)
__device__ __forceinline__ float normal_cdf(float z, float& e) {
    e = __expf(-0.5f * z * z);
    const float t = __builtin_amdgcn_rcpf(1.f + 0.3275911f * 0.70710678f * fabsf(z));
    const float h = 0.5f * e * (t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f)))));
    return z < 0.f ? h : 1.f - h;
}

// (0 where e^-z overflows: 1 / inf)
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }

__device__ __forceinline__ float act_of(float z, int act) {
    if (act == PVX_ACT_RELU) return z < 0.f ? 0.f : z;       // keeps NaN
    if (act == PVX_ACT_SILU) return z * sigmoid(z);
    if (act == PVX_ACT_GELU) { float e; return z * normal_cdf(z, e); }
    return z;
}

__device__ __forceinline__ float slope_of(float z, int act) {
    if (act == PVX_ACT_RELU) return z <= 0.f ? 0.f : 1.f;     // a NaN lets the gradient through
    if (act == PVX_ACT_SILU) {
        const float p = sigmoid(z);
        return p * (1.f + z * (1.f - p));
    }
    if (act == PVX_ACT_GELU) { float e; const float p = normal_cdf(z, e); return p + z * 0.39894228f * e; }
    return 1.f;
}

// the rows: either offsets (device) or equal samples of n / samples rows
struct Rows {
    const int* offsets;
    const int* order;
    int n, samples, each;
    __device__ __forceinline__ int begin(int s) const {
        if (!offsets) return s * each;
        const int v = offsets[s];
        return v < 0 ? 0 : (v > n ? n : v);
    }
    // first sample that ends behind position p; every lane of the wave calls it.  Up to 64 samples in one load
    __device__ __forceinline__ int first(int p) const {
        if (!offsets) return p / each;
        if (samples <= 64) {
            const int lane = threadIdx.x & 63;
            return __popcll(__ballot(lane < samples && begin(min(lane, samples - 1) + 1) <= p));
        }
        int lo = 0, hi = samples;
        while (lo < hi) {
            const int mid = lo + ((hi - lo) >> 1);           // lo + hi passes 2^31 from 2^30 samples on
            if (begin(mid + 1) > p) hi = mid; else lo = mid + 1;
        }
        return lo;
    }
    // behind an empty sample s at position p: the one before the next that has p, so that a run of empty ones costs a search and not a step
    // each (700 rows in the first and last of 2^20 samples: forward 0.07 ms, 555 one by one)
    __device__ __forceinline__ int skip(int s, int p) const { return max(s, first(p) - 1); }
    // row at position p (kept inside the matrix, whatever `order` holds)
    __device__ __forceinline__ int row(int p) const { return order ? (int)min((unsigned)order[p], (unsigned)(n - 1)) : p; }
};

// which chunk of which row slot a thread owns: tiles of `tw` chunks along the row (blockIdx.y), `rpb` rows at a time
struct Place {
    int chunk, r_in, rpb, tw;
    bool on;
};

template <int V> __device__ __forceinline__ Place place(int c) {
    Place t;
    const int ch = c / V;
    t.tw = ch < kBlk ? ch : kBlk;
    t.rpb = kBlk / t.tw;
    t.r_in = threadIdx.x / t.tw;
    t.chunk = blockIdx.y * t.tw + threadIdx.x % t.tw;
    t.on = t.r_in < t.rpb && t.chunk < ch;
    return t;
}

// Sums two binary64 vectors of V channels over the row slots of the workgroup; the result is in slot 0's threads and, behind a
// barrier, at red[q][chunk][j] for everybody.  red: [2][kBlk][V + 1].  Chunk counts that divide a wave are folded by lane exchanges
// first (one barrier), others by halves in LDS.
template <int V> __device__ __forceinline__ void fold_rows(double (&s0)[V], double (&s1)[V], const Place& t, double* red) {
    double(*r0)[V + 1] = reinterpret_cast<double(*)[V + 1]>(red);
    double(*r1)[V + 1] = r0 + kBlk;
    __syncthreads();                     // the buffer's last readers are done
    if (t.tw <= 64 && (t.tw & (t.tw - 1)) == 0) {
        for (int off = t.tw; off < 64; off <<= 1) {
#pragma unroll
            for (int j = 0; j < V; j++) { s0[j] += __shfl_xor(s0[j], off); s1[j] += __shfl_xor(s1[j], off); }
        }
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        if (lane < t.tw) {
#pragma unroll
            for (int j = 0; j < V; j++) { r0[wave * t.tw + lane][j] = s0[j]; r1[wave * t.tw + lane][j] = s1[j]; }
        }
        __syncthreads();
        if ((int)threadIdx.x < t.tw) {
#pragma unroll
            for (int w = 1; w < kWaves; w++) {
#pragma unroll
                for (int j = 0; j < V; j++) { s0[j] += r0[w * t.tw + threadIdx.x][j]; s1[j] += r1[w * t.tw + threadIdx.x][j]; }
            }
#pragma unroll
            for (int j = 0; j < V; j++) { r0[threadIdx.x][j] = s0[j]; r1[threadIdx.x][j] = s1[j]; }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < V; j++) { r0[threadIdx.x][j] = s0[j]; r1[threadIdx.x][j] = s1[j]; }
    for (int w = t.rpb; w > 1;) {
        const int h = (w + 1) >> 1;
        __syncthreads();
        if (t.r_in < w - h) {
            const int o = threadIdx.x + h * t.tw;
#pragma unroll
            for (int j = 0; j < V; j++) { r0[threadIdx.x][j] += r0[o][j]; r1[threadIdx.x][j] += r1[o][j]; }
        }
        w = h;
    }
#pragma unroll
    for (int j = 0; j < V; j++) { s0[j] = r0[threadIdx.x][j]; s1[j] = r1[threadIdx.x][j]; }
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    return v;
}

// the groups' sums of what fold_rows left in red (whole rows in the workgroup: one tile), to per_group[group][2]
template <int V> __device__ __forceinline__ void group_sums(int c, int groups, double* red, double* per_group) {
    double(*r0)[V + 1] = reinterpret_cast<double(*)[V + 1]>(red);
    double(*r1)[V + 1] = r0 + kBlk;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, cpg = c / groups;
    __syncthreads();
    if (cpg <= 16) {                     // a thread for each sum
        for (int i = threadIdx.x; i < 2 * groups; i += kBlk) {
            double(*r)[V + 1] = i & 1 ? r1 : r0;
            double a = 0.0;
            for (int k = 0, cc = (i >> 1) * cpg; k < cpg; k++, cc++) a += r[cc / V][cc % V];
            per_group[i] = a;
        }
    } else {                             // a wave for each group
        for (int g = wave; g < groups; g += kWaves) {
            double a = 0.0, b = 0.0;
            for (int i = lane; i < cpg; i += 64) {
                const int cc = g * cpg + i;
                a += r0[cc / V][cc % V];
                b += r1[cc / V][cc % V];
            }
            a = wave_sum(a);
            b = wave_sum(b);
            if (lane == 0) { per_group[2 * g] = a; per_group[2 * g + 1] = b; }
        }
    }
    __syncthreads();
}

// sums of x and x^2 for each piece: partial[piece][units][2], a unit being a group where a workgroup sees whole rows, else a channel
template <typename E, int V>
__global__ __launch_bounds__(kBlk, kResident) void gn_sums_kernel(const E* __restrict__ x, Rows rows, int c, int groups, int units, int range,
                                                       double* __restrict__ partial) {
    __shared__ double red[2 * kBlk * (V + 1)];
    extern __shared__ double per_group[];                // [groups][2]
    const Place t = place<V>(c);
    const int p0 = blockIdx.x * range, p1 = p0 + min(rows.n - p0, range);
    for (int s = rows.first(p0); s < rows.samples; s++) {
        const int begin = rows.begin(s), lo = max(p0, begin), hi = min(p1, rows.begin(s + 1));
        if (begin >= p1) break;
        if (lo >= hi) { s = rows.skip(s, lo); continue; }
        double s0[V], s1[V];
#pragma unroll
        for (int j = 0; j < V; j++) { s0[j] = 0; s1[j] = 0; }
        if (t.on) {
            constexpr int U = 2 * kAhead<E, V>;
            for (int p = lo + t.r_in; p < hi; p += U * t.rpb) {
                Pack<E, V> v[U];
#pragma unroll
                for (int u = 0; u < U; u++) v[u] = row_pack<E, V>(x, rows.row(min(p + u * t.rpb, hi - 1)), c, t.chunk);
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const bool on = p + u * t.rpb < hi;          // past the end: the last row again, for nothing
#pragma unroll
                    for (int j = 0; j < V; j++) { const double d = on ? (float)v[u].e[j] : 0.f; s0[j] += d; s1[j] = fma(d, d, s1[j]); }
                }
            }
        }
        fold_rows<V>(s0, s1, t, red);
        double* out = partial + (size_t)(blockIdx.x + s) * 2 * units;
        if (units == groups) {
            group_sums<V>(c, groups, red, per_group);
            for (int i = threadIdx.x; i < 2 * groups; i += kBlk) out[i] = per_group[i];
        } else if (t.on && t.r_in == 0) {
#pragma unroll
            for (int j = 0; j < V; j++) { out[2 * (t.chunk * V + j)] = s0[j]; out[2 * (t.chunk * V + j) + 1] = s1[j]; }
        }
    }
}

// the sums of workgroup-wide `v` in every thread; red: kWaves doubles
__device__ __forceinline__ double block_sum(double v, double* red) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int w = 0; w < kWaves; w++) v += red[w];
    return v;
}

// mean and 1 / sqrt(variance + eps) of each (sample, group) from its pieces
__global__ __launch_bounds__(kBlk) void gn_finish_kernel(const double* __restrict__ partial, Rows rows, int c, int groups, int units, int range,
                                                          float eps, float* __restrict__ mean, float* __restrict__ rstd) {
    __shared__ double red[kWaves];
    const int cpg = c / groups, upg = units / groups;
    for (int pair = blockIdx.x; pair < rows.samples * groups; pair += gridDim.x) {
        const int s = pair / groups, g = pair % groups, lo = rows.begin(s), hi = rows.begin(s + 1);
        double a = 0.0, b = 0.0;
        if (hi > lo) {
            const int k0 = lo / range, pieces = (hi - 1) / range - k0 + 1;
            for (int i = threadIdx.x; i < pieces * upg; i += kBlk) {
                const double2 q = *reinterpret_cast<const double2*>(partial + ((size_t)(k0 + s + i / upg) * units + g * upg + i % upg) * 2);
                a += q.x;
                b += q.y;
            }
        }
        a = block_sum(a, red);
        b = block_sum(b, red);
        if (threadIdx.x != 0) continue;
        const double count = hi > lo ? (double)(hi - lo) * cpg : 1.0, mu = a / count;
        double var = b / count - mu * mu;
        if (var < 0.0) var = 0.0;
        mean[pair] = (float)mu;
        rstd[pair] = (float)(1.0 / sqrt(var + (double)eps));
    }
}

// a thread's channels of one sample
template <int V> struct Chan { float mu[V], rs[V], w[V], b[V]; };

template <int V>
__device__ __forceinline__ void load_chan(Chan<V>& k, int c0, int s, int groups, int cpg, const void* weight, const void* bias, int pd,
                                          const float* mean, const float* rstd) {
#pragma unroll
    for (int j = 0; j < V; j++) {
        const int i = s * groups + (c0 + j) / cpg;
        k.mu[j] = mean[i];
        k.rs[j] = rstd[i];
        k.w[j] = load_param(weight, pd, c0 + j, 1.f);
        k.b[j] = load_param(bias, pd, c0 + j, 0.f);
    }
}

// a sample's sums over its pieces, partial[piece][groups][2], to per_group[group][2]; every workgroup of the sample does this for itself
__device__ __forceinline__ void sample_sums(const double* partial, int first_piece, int pieces, int groups, double* per_group) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __syncthreads();                     // the last readers are done
    for (int g = wave; g < groups; g += kWaves) {
        double a = 0.0, b = 0.0;
        for (int i = lane; i < pieces; i += 64) {
            const double2 q = *reinterpret_cast<const double2*>(partial + ((size_t)(first_piece + i) * groups + g) * 2);
            a += q.x;
            b += q.y;
        }
        a = wave_sum(a);
        b = wave_sum(b);
        if (lane == 0) { per_group[2 * g] = a; per_group[2 * g + 1] = b; }
    }
    __syncthreads();
}

// y of a workgroup's positions, from the last to the first: what the pass before read last is still in the cache (the ranges' ends, of a
// tensor larger than it).  With `partial` the statistics are finished here (and kept by the workgroup that holds the sample's
// first row), while the first rows are on their way; without, gn_finish_kernel has left them.
template <typename E, int V, int ACT>
__global__ __launch_bounds__(kBlk, kResident) void gn_apply_kernel(const E* __restrict__ x, const E* __restrict__ residual, Rows rows, int c, int groups,
                                                         int range, const void* __restrict__ weight, const void* __restrict__ bias, int pd,
                                                         const double* __restrict__ partial, float eps, float* __restrict__ mean,
                                                         float* __restrict__ rstd, E* __restrict__ y) {
    extern __shared__ double per_group[];
    const Place t = place<V>(c);
    const int p0 = blockIdx.x * range, p1 = p0 + min(rows.n - p0, range), cpg = c / groups;
    const float zero[V] = {};
    float w[V], b[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        w[j] = t.on ? load_param(weight, pd, t.chunk * V + j, 1.f) : 0.f;
        b[j] = t.on ? load_param(bias, pd, t.chunk * V + j, 0.f) : 0.f;
    }
    int done = p0;                       // positions below it are written
    for (int s = rows.first(p0); s < rows.samples; s++) {
        const int begin = rows.begin(s), end = rows.begin(s + 1), lo = max(p0, begin), hi = min(p1, end);
        if (begin >= p1) break;
        if (lo >= hi) { s = rows.skip(s, lo); continue; }
        for (int p = done + t.r_in; p < lo && t.on; p += t.rpb) {       // positions of no sample
            const int row = rows.row(p);
            store_pack<E, V>(y + (size_t)row * c + t.chunk * V, zero);
        }
        done = hi;
        constexpr int U = kAhead<E, V>;
        Pack<E, V> xs[U], res[U];
        int row[U];
#define GN_ROWS(from)                                                                               \
        _Pragma("unroll") for (int u = 0; u < U; u++) {                                             \
            row[u] = rows.row(max(hi - 1 - ((from) - lo + u * t.rpb), lo));                         \
            xs[u] = row_pack<E, V>(x, row[u], c, t.chunk);                                          \
            if (residual) res[u] = row_pack<E, V>(residual, row[u], c, t.chunk);                    \
        }
        if (t.on) { GN_ROWS(lo + t.r_in) }
        if (partial) {
            const int k0 = begin / range;
            sample_sums(partial, k0 + s, (end - 1) / range - k0 + 1, groups, per_group);
            for (int g = threadIdx.x; g < groups; g += kBlk) {
                const double count = (double)(end - begin) * cpg, mu = per_group[2 * g] / count;
                double var = per_group[2 * g + 1] / count - mu * mu;
                if (var < 0.0) var = 0.0;
                const float m = (float)mu, r = (float)(1.0 / sqrt(var + (double)eps));
                per_group[2 * g] = m;
                per_group[2 * g + 1] = r;
                if (lo == begin) { mean[(size_t)s * groups + g] = m; rstd[(size_t)s * groups + g] = r; }
            }
            __syncthreads();
        }
        if (!t.on) continue;
        float mu[V], rs[V];
#pragma unroll
        for (int j = 0; j < V; j++) {
            const int g = (t.chunk * V + j) / cpg;
            mu[j] = partial ? (float)per_group[2 * g] : mean[(size_t)s * groups + g];
            rs[j] = partial ? (float)per_group[2 * g + 1] : rstd[(size_t)s * groups + g];
        }
        for (int p = lo + t.r_in; p < hi; p += U * t.rpb) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (p + u * t.rpb >= hi) break;
                float v[V];
#pragma unroll
                for (int j = 0; j < V; j++) {
                    float z = ((float)xs[u].e[j] - mu[j]) * rs[j] * w[j] + b[j];
                    if (residual) z += (float)res[u].e[j];
                    v[j] = act_of(z, ACT);
                }
                store_pack<E, V>(y + (size_t)row[u] * c + t.chunk * V, v);
            }
            if (p + U * t.rpb < hi) { GN_ROWS(p + U * t.rpb) }
        }
#undef GN_ROWS
    }
    for (int p = done + t.r_in; p < p1 && t.on; p += t.rpb) {
        const int row = rows.row(p);
        store_pack<E, V>(y + (size_t)row * c + t.chunk * V, zero);
    }
}

// backward, first pass: sums of gz and gz xhat for each piece and channel, partial[piece][c][2], and, where a workgroup sees whole
// rows, of w gz and w gz xhat for each piece and group, gpart[piece][groups][2]
template <typename E, int V, int ACT>
__global__ __launch_bounds__(kBlk, kResident) void gn_bwd_sums_kernel(const E* __restrict__ dy, const E* __restrict__ x, const E* __restrict__ residual,
                                                            Rows rows, int c, int groups, int range, const void* __restrict__ weight,
                                                            const void* __restrict__ bias, int pd, const float* __restrict__ mean,
                                                            const float* __restrict__ rstd, double* __restrict__ partial,
                                                            double* __restrict__ gpart) {
    __shared__ double red[2 * kBlk * (V + 1)];
    extern __shared__ double per_group[];
    const Place t = place<V>(c);
    const int p0 = blockIdx.x * range, p1 = p0 + min(rows.n - p0, range), cpg = c / groups;
    for (int s = rows.first(p0); s < rows.samples; s++) {
        const int begin = rows.begin(s), lo = max(p0, begin), hi = min(p1, rows.begin(s + 1));
        if (begin >= p1) break;
        if (lo >= hi) { s = rows.skip(s, lo); continue; }
        double s0[V], s1[V];
        Chan<V> k;
#pragma unroll
        for (int j = 0; j < V; j++) { s0[j] = 0; s1[j] = 0; k.w[j] = 0.f; }
        if (t.on) {
            load_chan<V>(k, t.chunk * V, s, groups, cpg, weight, bias, pd, mean, rstd);
            constexpr int U = 2;
            for (int p = lo + t.r_in; p < hi; p += U * t.rpb) {
                Pack<E, V> gs[U], xs[U], res[U];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int row = rows.row(min(p + u * t.rpb, hi - 1));
                    gs[u] = row_pack<E, V>(dy, row, c, t.chunk);
                    xs[u] = row_pack<E, V>(x, row, c, t.chunk);
                    if (residual) res[u] = row_pack<E, V>(residual, row, c, t.chunk);
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (p + u * t.rpb >= hi) break;
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        const float xh = ((float)xs[u].e[j] - k.mu[j]) * k.rs[j];
                        float z = xh * k.w[j] + k.b[j];
                        if (residual) z += (float)res[u].e[j];
                        const float gz = (float)gs[u].e[j] * slope_of(z, ACT);
                        s0[j] += (double)gz;
                        s1[j] = fma((double)gz, (double)xh, s1[j]);
                    }
                }
            }
        }
        fold_rows<V>(s0, s1, t, red);
        if (t.on && t.r_in == 0) {
            double* out = partial + ((size_t)(blockIdx.x + s) * c + t.chunk * V) * 2;
            double(*r0)[V + 1] = reinterpret_cast<double(*)[V + 1]>(red);
#pragma unroll
            for (int j = 0; j < V; j++) {
                out[2 * j] = s0[j];
                out[2 * j + 1] = s1[j];
                r0[threadIdx.x][j] = s0[j] * (double)k.w[j];
                r0[kBlk + threadIdx.x][j] = s1[j] * (double)k.w[j];
            }
        }
        if (gpart) {
            group_sums<V>(c, groups, red, per_group);
            double* out = gpart + (size_t)(blockIdx.x + s) * 2 * groups;
            for (int i = threadIdx.x; i < 2 * groups; i += kBlk) out[i] = per_group[i];
        }
    }
}

// db and dw of channel cc, summed over the pieces in a fixed order by the workgroup
__device__ __forceinline__ void channel_finish(const double* partial, const Rows& rows, int c, int range, int cc, int pd, void* dweight, void* dbias,
                                               double* red) {
    double a = 0.0, b = 0.0;
    // as many lanes a sample as it has pieces on average, so that the samples are not walked one after the other
    const int average = (rows.n - 1) / range / rows.samples + 2;
    int lanes = 1;
    while (lanes < average && lanes < kBlk) lanes <<= 1;
    for (int s = threadIdx.x / lanes; s < rows.samples; s += kBlk / lanes) {
        const int lo = rows.begin(s), hi = rows.begin(s + 1);
        if (hi <= lo) continue;
        const int k0 = lo / range, pieces = (hi - 1) / range - k0 + 1;
        for (int i = threadIdx.x & (lanes - 1); i < pieces; i += lanes) {
            const double2 q = *reinterpret_cast<const double2*>(partial + ((size_t)(k0 + s + i) * c + cc) * 2);
            a += q.x;
            b += q.y;
        }
    }
    a = block_sum(a, red);
    b = block_sum(b, red);
    if (threadIdx.x == 0) {
        if (dbias) store_param(dbias, pd, cc, a);
        if (dweight) store_param(dweight, pd, cc, b);
    }
}

// backward, finish: mean gx and mean(gx xhat) of each (sample, group), and behind them db and dw of each channel
__global__ __launch_bounds__(kBlk) void gn_bwd_finish_kernel(const double* __restrict__ partial, Rows rows, int c, int groups, int range,
                                                              const void* __restrict__ weight, int pd, float* __restrict__ m0,
                                                              float* __restrict__ m1, void* __restrict__ dweight, void* __restrict__ dbias) {
    __shared__ double red[kWaves];
    const int pairs = rows.samples * groups, cpg = c / groups;
    for (int pair = blockIdx.x; pair < pairs + c; pair += gridDim.x) {
        if (pair >= pairs) {
            channel_finish(partial, rows, c, range, pair - pairs, pd, dweight, dbias, red);
            continue;
        }
        const int s = pair / groups, g = pair % groups, lo = rows.begin(s), hi = rows.begin(s + 1);
        double a = 0.0, b = 0.0;
        if (hi > lo) {
            const int k0 = lo / range, pieces = (hi - 1) / range - k0 + 1;
            for (int i = threadIdx.x; i < pieces * cpg; i += kBlk) {
                const int cc = g * cpg + i % cpg;
                const double2 q = *reinterpret_cast<const double2*>(partial + ((size_t)(k0 + s + i / cpg) * c + cc) * 2);
                const double w = load_param(weight, pd, cc, 1.f);
                a += w * q.x;
                b += w * q.y;
            }
        }
        a = block_sum(a, red);
        b = block_sum(b, red);
        if (threadIdx.x == 0) {
            const double count = hi > lo ? (double)(hi - lo) * cpg : 1.0;
            m0[pair] = (float)(a / count);
            m1[pair] = (float)(b / count);
        }
    }
}

// dx (and dresidual) of a workgroup's positions.  With `gpart` the two means are finished here, and the workgroups behind the `blocks`
// first ones finish db and dw, a channel each; without, gn_bwd_finish_kernel has done both.
template <typename E, int V, int ACT>
__global__ __launch_bounds__(kBlk, kResident) void gn_bwd_apply_kernel(const E* __restrict__ dy, const E* __restrict__ x, const E* __restrict__ residual,
                                                             Rows rows, int c, int groups, int range, int blocks, const void* __restrict__ weight,
                                                             const void* __restrict__ bias, int pd, const float* __restrict__ mean,
                                                             const float* __restrict__ rstd, const double* __restrict__ partial,
                                                             const double* __restrict__ gpart, const float* __restrict__ m0,
                                                             const float* __restrict__ m1, E* __restrict__ dx, E* __restrict__ dres,
                                                             void* __restrict__ dweight, void* __restrict__ dbias) {
    __shared__ double red[kWaves];
    extern __shared__ double per_group[];
    if ((int)blockIdx.x >= blocks) {
        channel_finish(partial, rows, c, range, blockIdx.x - blocks, pd, dweight, dbias, red);
        return;
    }
    const Place t = place<V>(c);
    const int p0 = blockIdx.x * range, p1 = p0 + min(rows.n - p0, range), cpg = c / groups;
    const float zero[V] = {};
    int done = p0;
    for (int s = rows.first(p0); s < rows.samples; s++) {
        const int begin = rows.begin(s), end = rows.begin(s + 1), lo = max(p0, begin), hi = min(p1, end);
        if (begin >= p1) break;
        if (lo >= hi) { s = rows.skip(s, lo); continue; }
        for (int p = done + t.r_in; p < lo && t.on; p += t.rpb) {
            const int row = rows.row(p);
            const size_t off = (size_t)row * c + t.chunk * V;
            store_pack<E, V>(dx + off, zero);
            if (dres) store_pack<E, V>(dres + off, zero);
        }
        done = hi;
        constexpr int U = 2;
        Pack<E, V> gs[U], xs[U], res[U];
        int row[U];
#define GN_ROWS(from)                                                                               \
        _Pragma("unroll") for (int u = 0; u < U; u++) {                                             \
            row[u] = rows.row(max(hi - 1 - ((from) - lo + u * t.rpb), lo));                         \
            gs[u] = row_pack<E, V>(dy, row[u], c, t.chunk);                                         \
            xs[u] = row_pack<E, V>(x, row[u], c, t.chunk);                                          \
            if (residual) res[u] = row_pack<E, V>(residual, row[u], c, t.chunk);                    \
        }
        if (t.on) { GN_ROWS(lo + t.r_in) }
        if (gpart) {
            const int k0 = begin / range;
            sample_sums(gpart, k0 + s, (end - 1) / range - k0 + 1, groups, per_group);
        }
        if (!t.on) continue;
        Chan<V> k;
        load_chan<V>(k, t.chunk * V, s, groups, cpg, weight, bias, pd, mean, rstd);
        float a[V], b[V];
        const double count = (double)(end - begin) * cpg;
#pragma unroll
        for (int j = 0; j < V; j++) {
            const int g = (t.chunk * V + j) / cpg;
            a[j] = gpart ? (float)(per_group[2 * g] / count) : m0[(size_t)s * groups + g];
            b[j] = gpart ? (float)(per_group[2 * g + 1] / count) : m1[(size_t)s * groups + g];
        }
        for (int p = lo + t.r_in; p < hi; p += U * t.rpb) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (p + u * t.rpb >= hi) break;
                const size_t off = (size_t)row[u] * c + t.chunk * V;
                float g[V], o[V];
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float xh = ((float)xs[u].e[j] - k.mu[j]) * k.rs[j];
                    float z = xh * k.w[j] + k.b[j];
                    if (residual) z += (float)res[u].e[j];
                    g[j] = (float)gs[u].e[j] * slope_of(z, ACT);
                    o[j] = k.rs[j] * (g[j] * k.w[j] - a[j] - xh * b[j]);
                }
                store_pack<E, V>(dx + off, o);
                if (dres) store_pack<E, V>(dres + off, g);
            }
            if (p + U * t.rpb < hi) { GN_ROWS(p + U * t.rpb) }
        }
#undef GN_ROWS
    }
    for (int p = done + t.r_in; p < p1 && t.on; p += t.rpb) {
        const int row = rows.row(p);
        const size_t off = (size_t)row * c + t.chunk * V;
        store_pack<E, V>(dx + off, zero);
        if (dres) store_pack<E, V>(dres + off, zero);
    }
}

// One launch: a workgroup holds one sample's rows in registers (kOneChunks chunks a thread), so x is read once and nothing but the
// statistics goes through memory.  Taken where every sample is known to fit and all workgroups run at a time: latency is what such calls
// cost.  Against the form of several launches, forward / forward and backward: 128 rows x 64 binary32 8.2 / 16.5 us and 9.5 / 17.3, 256
// samples of 30 rows 7.4 / 18 and 14 / 28; but 1000 samples of 120 rows 19 / 60 and 20 / 47, and with sixteen rows a thread (eight
// backward) 510 rows 13 / 22 and 9.5 / 18.  blockIdx.x == samples: the positions of no sample.
template <typename E, int V>
__device__ __forceinline__ void zero_uncovered(const Place& t, const Rows& rows, int c, E* a, E* b) {
    if (!t.on) return;
    const int lo = rows.begin(0), hi = rows.begin(rows.samples);
    const float zero[V] = {};
    for (int p = t.r_in; p < rows.n; p += t.rpb) {
        if (p >= lo && p < hi) continue;
        const int row = rows.row(p);
        const size_t off = (size_t)row * c + t.chunk * V;
        store_pack<E, V>(a + off, zero);
        if (b) store_pack<E, V>(b + off, zero);
    }
}

template <typename E, int V>
__global__ __launch_bounds__(kBlk) void gn_one_kernel(const E* __restrict__ x, const E* __restrict__ residual, Rows rows, int c, int groups,
                                                       const void* __restrict__ weight, const void* __restrict__ bias, int pd, float eps,
                                                       int act, E* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
    __shared__ double red[2 * kBlk * (V + 1)];
    extern __shared__ double per_group[];                // [groups][2]
    const Place t = place<V>(c);
    constexpr int U = kOneChunks;
    const int cpg = c / groups, s = blockIdx.x;
    if (s == rows.samples) { zero_uncovered<E, V>(t, rows, c, y, (E*)nullptr); return; }
    float w[V], b[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        w[j] = t.on ? load_param(weight, pd, t.chunk * V + j, 1.f) : 0.f;
        b[j] = t.on ? load_param(bias, pd, t.chunk * V + j, 0.f) : 0.f;
    }
    const int lo = rows.begin(s), hi = min(rows.begin(s + 1), lo + U * t.rpb);
    float v[U][V];
    double s0[V], s1[V];
#pragma unroll
    for (int j = 0; j < V; j++) { s0[j] = 0; s1[j] = 0; }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int p = lo + t.r_in + u * t.rpb;
        const int row = t.on && p < hi ? rows.row(p) : -1;
#pragma unroll
        for (int j = 0; j < V; j++) v[u][j] = 0.f;
        if (row >= 0) load_pack<E, V>(x + (size_t)row * c + t.chunk * V, v[u]);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
#pragma unroll
        for (int j = 0; j < V; j++) { const double d = v[u][j]; s0[j] += d; s1[j] = fma(d, d, s1[j]); }
    }
    fold_rows<V>(s0, s1, t, red);
    group_sums<V>(c, groups, red, per_group);
    for (int g = threadIdx.x; g < groups; g += kBlk) {
        const double count = hi > lo ? (double)(hi - lo) * cpg : 1.0;
        const double mu = per_group[2 * g] / count;
        double var = per_group[2 * g + 1] / count - mu * mu;
        if (var < 0.0) var = 0.0;
        const double rs = 1.0 / sqrt(var + (double)eps);
        per_group[2 * g] = mu;
        per_group[2 * g + 1] = rs;
        mean[(size_t)s * groups + g] = (float)mu;
        rstd[(size_t)s * groups + g] = (float)rs;
    }
    __syncthreads();
    if (!t.on) return;
    float mu[V], rs[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        const int g = (t.chunk * V + j) / cpg;
        mu[j] = (float)per_group[2 * g];
        rs[j] = (float)per_group[2 * g + 1];
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int p = lo + t.r_in + u * t.rpb;
        const int row = p < hi ? rows.row(p) : -1;
        if (row < 0) continue;
        const size_t off = (size_t)row * c + t.chunk * V;
        float r[V];
        if (residual) load_pack<E, V>(residual + off, r);
#pragma unroll
        for (int j = 0; j < V; j++) {
            float z = (v[u][j] - mu[j]) * rs[j] * w[j] + b[j];
            if (residual) z += r[j];
            v[u][j] = act_of(z, act);
        }
        store_pack<E, V>(y + off, v[u]);
    }
}

// the backward of the same; a workgroup leaves its sample's share of db and dw in partial[sample][2][c]
template <typename E, int V>
__global__ __launch_bounds__(kBlk) void gn_bwd_one_kernel(const E* __restrict__ dy, const E* __restrict__ x, const E* __restrict__ residual,
                                                           Rows rows, int c, int groups, const void* __restrict__ weight,
                                                           const void* __restrict__ bias, int pd, const float* __restrict__ mean,
                                                           const float* __restrict__ rstd, int act, E* __restrict__ dx, E* __restrict__ dres,
                                                           void* __restrict__ dweight, void* __restrict__ dbias, double* __restrict__ partial) {
    __shared__ double red[2 * kBlk * (V + 1)];
    extern __shared__ double per_group[];
    const Place t = place<V>(c);
    constexpr int U = kOneChunks;
    const int cpg = c / groups, s = blockIdx.x;
    if (s == rows.samples) { zero_uncovered<E, V>(t, rows, c, dx, dres); return; }
    const int lo = rows.begin(s), hi = min(rows.begin(s + 1), lo + U * t.rpb);
    float xh[U][V], gz[U][V];
    Chan<V> k;
#pragma unroll
    for (int j = 0; j < V; j++) { k.mu[j] = 0.f; k.rs[j] = 0.f; k.w[j] = 0.f; k.b[j] = 0.f; }
    if (t.on) load_chan<V>(k, t.chunk * V, s, groups, cpg, weight, bias, pd, mean, rstd);
    double s0[V], s1[V];
#pragma unroll
    for (int j = 0; j < V; j++) { s0[j] = 0; s1[j] = 0; }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int p = lo + t.r_in + u * t.rpb;
        const int row = t.on && p < hi ? rows.row(p) : -1;
#pragma unroll
        for (int j = 0; j < V; j++) { xh[u][j] = 0.f; gz[u][j] = 0.f; }
        if (row < 0) continue;
        const size_t off = (size_t)row * c + t.chunk * V;
        float r[V];
        load_pack<E, V>(dy + off, gz[u]);
        load_pack<E, V>(x + off, xh[u]);
        if (residual) load_pack<E, V>(residual + off, r);
#pragma unroll
        for (int j = 0; j < V; j++) {
            xh[u][j] = (xh[u][j] - k.mu[j]) * k.rs[j];
            float z = xh[u][j] * k.w[j] + k.b[j];
            if (residual) z += r[j];
            gz[u][j] *= slope_of(z, act);
            s0[j] += (double)gz[u][j];
            s1[j] = fma((double)gz[u][j], (double)xh[u][j], s1[j]);
        }
    }
    fold_rows<V>(s0, s1, t, red);
    if (t.on && t.r_in == 0) {
        double(*r0)[V + 1] = reinterpret_cast<double(*)[V + 1]>(red);
#pragma unroll
        for (int j = 0; j < V; j++) {
            r0[threadIdx.x][j] = s0[j] * (double)k.w[j];     // the groups' sums take w gz
            r0[kBlk + threadIdx.x][j] = s1[j] * (double)k.w[j];
        }
    }
    group_sums<V>(c, groups, red, per_group);
    if (!t.on) return;
    const double count = hi > lo ? (double)(hi - lo) * cpg : 1.0;
    float a[V], b[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        const int g = (t.chunk * V + j) / cpg;
        a[j] = (float)(per_group[2 * g] / count);
        b[j] = (float)(per_group[2 * g + 1] / count);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int p = lo + t.r_in + u * t.rpb;
        const int row = p < hi ? rows.row(p) : -1;
        if (row < 0) continue;
        const size_t off = (size_t)row * c + t.chunk * V;
        float o[V];
#pragma unroll
        for (int j = 0; j < V; j++) o[j] = k.rs[j] * (gz[u][j] * k.w[j] - a[j] - xh[u][j] * b[j]);
        store_pack<E, V>(dx + off, o);
        if (dres) store_pack<E, V>(dres + off, gz[u]);
    }
    if (t.r_in == 0) {
        double* out = partial + (size_t)s * 2 * c + t.chunk * V;
#pragma unroll
        for (int j = 0; j < V; j++) {
            if (rows.samples == 1) {
                if (dbias) store_param(dbias, pd, t.chunk * V + j, s0[j]);
                if (dweight) store_param(dweight, pd, t.chunk * V + j, s1[j]);
            } else {
                out[j] = s0[j];
                out[c + j] = s1[j];
            }
        }
    }
}

// dw and db from the workgroups' sums: a wave for each channel, in a fixed order
__global__ __launch_bounds__(64) void gn_bwd_channels_kernel(const double* __restrict__ partial, int blocks, int c, int pd,
                                                             void* __restrict__ dweight, void* __restrict__ dbias) {
    const int cc = blockIdx.x;
    double a = 0.0, b = 0.0;
    for (int s = threadIdx.x; s < blocks; s += 64) {
        a += partial[(size_t)s * 2 * c + cc];
        b += partial[(size_t)s * 2 * c + c + cc];
    }
    a = wave_sum(a);
    b = wave_sum(b);
    if (threadIdx.x != 0) return;
    if (dbias) store_param(dbias, pd, cc, a);
    if (dweight) store_param(dweight, pd, cc, b);
}

struct Shape {
    int v, tw, rpb, tiles, range, blocks;
    bool merged;                         // the apply kernels finish the sums
};

// elements of a thread's chunk that c and the addresses allow: four, two or one
int chunk_of(int c, int dtype, std::initializer_list<const void*> ptrs) {
    const int es = dtype == PVX_F32 ? 4 : 2;
    uintptr_t low = 0;
    for (const void* p : ptrs) low |= (uintptr_t)p;
    for (int v = 4; v > 1; v /= 2)
        if (c % v == 0 && low % ((uintptr_t)v * es) == 0) return v;
    return 1;
}

Shape shape_of(int n, int c, int groups, int v) {
    Shape s;
    s.v = v;
    const int ch = c / v;
    s.tw = ch < kBlk ? ch : kBlk;
    s.rpb = kBlk / s.tw;
    s.tiles = PVX_CDIV(ch, s.tw);
    const long long r = PVX_CDIV((long long)n, (long long)kTargetBlocks);
    s.range = (int)(PVX_CDIV(r < 2LL * s.rpb ? 2LL * s.rpb : r, (long long)s.rpb) * s.rpb);
    s.blocks = (int)PVX_CDIV((long long)n, (long long)s.range);      // n + range may pass 2^31
    s.merged = s.tiles == 1 && (long long)s.blocks * groups <= kMergedSums;
    return s;
}

// Elements of a chunk in the forms of several launches.  Wide ones move more bytes an instruction, narrow ones have fewer sums to fold
// at a range's end and shorter ranges.  Forward and backward, four / two / one of them: 30 000 x 64 bf16 46 / 36 / 33 us, 60 000 x 64
// binary32 53 / 46 / 44, 117 301 x 64 bf16 56 / 50 / 52, 200 000 x 128 binary32 155 / 148 / 163, 400 000 x 128 bf16 157 / 169 / 235,
// 520 013 x 128 binary32 398 / 483 / 508.  A row stays within one workgroup where it can: its groups are summed there.
int narrowed(int v, int n, int c) {
    const long long elements = (long long)n * c;
    const int most = elements <= (1 << 22) ? 1 : (elements <= (1 << 25) ? 2 : 4);
    while (v > most && 2 * (c / v) <= kBlk) v /= 2;
    return v;
}

// workspace: one piece for each workgroup and one more for each sample that begins inside one (equal samples that fit the one-launch
// form whatever the alignment need one each), and the backward's two means per (sample, group)
size_t pieces_cap(int n, int c, int samples, bool ragged) {
    if (!ragged && c <= kBlk && samples <= kOneSamples && n / samples <= kOneChunks * (kBlk / c)) return samples;
    return (size_t)(n < kTargetBlocks ? n : kTargetBlocks) + samples;
}

struct Ws { double *partial, *gpart; float *m0, *m1; };

template <typename C> Ws carve(C& cv, int c, int samples, int groups, size_t pieces) {
    Ws w;
    w.partial = cv.template take<double>(pieces * 2 * c);
    w.gpart = cv.template take<double>(pieces * 2 * groups);
    w.m0 = cv.template take<float>((size_t)samples * groups);
    w.m1 = cv.template take<float>((size_t)samples * groups);
    return w;
}

// the shape, and in `one` whether a workgroup takes a whole sample
Shape shape_for(const Rows& rows, int c, int groups, int v, bool& one) {
    const Shape whole = shape_of(rows.n, c, groups, v);
    one = whole.tiles == 1 && groups <= 1024 && rows.samples <= kOneSamples
          && PVX_CDIV(rows.offsets ? rows.n : rows.each, whole.rpb) <= kOneChunks;
    return one ? whole : shape_of(rows.n, c, groups, narrowed(v, rows.n, c));
}

int check_args(int n, int c, int dtype, int samples, const int* offsets, int groups, int param_dtype, int act) {
    if (n < 0 || c <= 0 || samples <= 0 || groups <= 0 || c % groups != 0) return PVX_ERR_INVALID;
    if (dtype < PVX_F32 || dtype > PVX_BF16 || param_dtype < PVX_F32 || param_dtype > PVX_BF16) return PVX_ERR_INVALID;
    if (act < PVX_ACT_NONE || act > PVX_ACT_GELU) return PVX_ERR_INVALID;
    if (!offsets && n % samples != 0) return PVX_ERR_INVALID;
    // the finishing kernels walk (sample, group) and channel in steps of a grid; positions, pieces and piece x channel products by 32 bits
    if ((long long)samples * groups + c > 0x7fffffffLL - (1 << 16) || n > 0x7fffffff - (1 << 20) || c > (1 << 20)) return PVX_ERR_RANGE;
    return PVX_OK;
}

dim3 finish_grid(long long results) { return dim3((unsigned)(results < 65536 ? results : 65536)); }

#define GN_DISPATCH(E, v, CALL)                                                            \
    do {                                                                                   \
        if (v == 4) { CALL(E, 4); }                                                        \
        else if (v == 2) { CALL(E, 2); }                                                   \
        else { CALL(E, 1); }                                                               \
    } while (0)
#define GN_WITH_ACT(act, E, V, CALL)                                                       \
    do {                                                                                   \
        if (act == PVX_ACT_RELU) CALL(E, V, PVX_ACT_RELU);                                 \
        else if (act == PVX_ACT_SILU) CALL(E, V, PVX_ACT_SILU);                            \
        else if (act == PVX_ACT_GELU) CALL(E, V, PVX_ACT_GELU);                            \
        else CALL(E, V, PVX_ACT_NONE);                                                     \
    } while (0)

template <typename E>
int fwd_impl(const void* x, const Rows& rows, int c, int groups, const void* weight, const void* bias, int pd, float eps,
             const void* residual, int act, void* y, float* mean, float* rstd, const Ws& ws, const Shape& sh, bool is_one, hipStream_t st) {
    if (is_one) {
        const dim3 one(rows.samples + (rows.offsets ? 1 : 0));
        const size_t lds = sizeof(double) * 2 * groups;
#define GN_ONE(E, V) hipLaunchKernelGGL((gn_one_kernel<E, V>), one, dim3(kBlk), lds, st, (const E*)x, (const E*)residual, rows, c, groups, \
                                        weight, bias, pd, eps, act, (E*)y, mean, rstd)
        GN_DISPATCH(E, sh.v, GN_ONE);
        PVX_CHECK_LAUNCH();
        return PVX_OK;
    }
    const dim3 grid(sh.blocks, sh.tiles);
    const int units = sh.tiles == 1 ? groups : c;
    const size_t lds = sizeof(double) * 2 * (sh.tiles == 1 ? groups : 0);
#define GN_SUMS(E, V) hipLaunchKernelGGL((gn_sums_kernel<E, V>), grid, dim3(kBlk), lds, st, (const E*)x, rows, c, groups, units, sh.range, ws.partial)
    GN_DISPATCH(E, sh.v, GN_SUMS);
    PVX_CHECK_LAUNCH();
    if (!sh.merged) {
        hipLaunchKernelGGL(gn_finish_kernel, finish_grid((long long)rows.samples * groups), dim3(kBlk), 0, st, ws.partial, rows, c, groups, units, sh.range, eps, mean, rstd);
        PVX_CHECK_LAUNCH();
    }
#define GN_APPLY_ACT(E, V, A) hipLaunchKernelGGL((gn_apply_kernel<E, V, A>), grid, dim3(kBlk), sh.merged ? lds : 0, st, (const E*)x,         \
                                                 (const E*)residual, rows, c, groups, sh.range, weight, bias, pd,                            \
                                                 sh.merged ? ws.partial : (const double*)nullptr, eps, mean, rstd, (E*)y)
#define GN_APPLY(E, V) GN_WITH_ACT(act, E, V, GN_APPLY_ACT)
    GN_DISPATCH(E, sh.v, GN_APPLY);
    PVX_CHECK_LAUNCH();
    return PVX_OK;
}

template <typename E>
int bwd_impl(const void* dy, const void* x, const void* residual, const Rows& rows, int c, int groups, const void* weight, const void* bias,
             int pd, const float* mean, const float* rstd, int act, void* dx, void* dres, void* dweight, void* dbias, const Ws& ws,
             const Shape& sh, bool is_one, hipStream_t st) {
    if (is_one) {
        const dim3 one(rows.samples + (rows.offsets ? 1 : 0));
        const size_t lds = sizeof(double) * 2 * groups;
#define GN_BONE(E, V) hipLaunchKernelGGL((gn_bwd_one_kernel<E, V>), one, dim3(kBlk), lds, st, (const E*)dy, (const E*)x,                \
                                         (const E*)residual, rows, c, groups, weight, bias, pd, mean, rstd, act, (E*)dx, (E*)dres,     \
                                         dweight, dbias, ws.partial)
        GN_DISPATCH(E, sh.v, GN_BONE);
        PVX_CHECK_LAUNCH();
        if (rows.samples > 1 && (dweight || dbias)) {
            hipLaunchKernelGGL(gn_bwd_channels_kernel, dim3(c), dim3(64), 0, st, ws.partial, rows.samples, c, pd, dweight, dbias);
            PVX_CHECK_LAUNCH();
        }
        return PVX_OK;
    }
    const dim3 grid(sh.blocks, sh.tiles);
    const size_t lds = sh.merged ? sizeof(double) * 2 * groups : 0;
    double* gpart = sh.merged ? ws.gpart : nullptr;
#define GN_BSUMS_ACT(E, V, A) hipLaunchKernelGGL((gn_bwd_sums_kernel<E, V, A>), grid, dim3(kBlk), lds, st, (const E*)dy, (const E*)x,        \
                                                 (const E*)residual, rows, c, groups, sh.range, weight, bias, pd, mean, rstd, ws.partial, gpart)
#define GN_BSUMS(E, V) GN_WITH_ACT(act, E, V, GN_BSUMS_ACT)
    GN_DISPATCH(E, sh.v, GN_BSUMS);
    PVX_CHECK_LAUNCH();
    if (!sh.merged) {
        hipLaunchKernelGGL(gn_bwd_finish_kernel, finish_grid((long long)rows.samples * groups + c), dim3(kBlk), 0, st, ws.partial, rows, c, groups, sh.range, weight, pd,
                           ws.m0, ws.m1, dweight, dbias);
        PVX_CHECK_LAUNCH();
    }
    const dim3 last(sh.blocks + (sh.merged && (dweight || dbias) ? c : 0), sh.tiles);
#define GN_BAPPLY_ACT(E, V, A) hipLaunchKernelGGL((gn_bwd_apply_kernel<E, V, A>), last, dim3(kBlk), lds, st, (const E*)dy, (const E*)x,      \
                                                  (const E*)residual, rows, c, groups, sh.range, sh.blocks, weight, bias, pd, mean, rstd,   \
                                                  ws.partial, gpart, ws.m0, ws.m1, (E*)dx, (E*)dres, dweight, dbias)
#define GN_BAPPLY(E, V) GN_WITH_ACT(act, E, V, GN_BAPPLY_ACT)
    GN_DISPATCH(E, sh.v, GN_BAPPLY);
    PVX_CHECK_LAUNCH();
    return PVX_OK;
}

__global__ void gn_zero_params_kernel(void* dweight, void* dbias, int pd, int c) {
    const int i = blockIdx.x * kBlk + threadIdx.x;
    if (i >= c) return;
    if (dweight) store_param(dweight, pd, i, 0.0);
    if (dbias) store_param(dbias, pd, i, 0.0);
}

struct SizerShim {
    PvxSizer s;
    template <typename T> T* take(size_t k) { s.take<T>(k); return nullptr; }
};

}  // namespace

extern "C" size_t pvx_group_norm_act_workspace_bytes(int n, int c, int samples, int ragged, int groups) {
    if (n <= 0 || c <= 0 || samples <= 0 || groups <= 0) return 256;
    SizerShim shim;
    carve(shim, c, samples, groups, pieces_cap(n, c, samples, ragged != 0));
    return shim.s.total();
}

extern "C" int pvx_group_norm_act_fwd(const void* x, int n, int c, int dtype, int samples, const int* offsets, const int* order, int groups,
                                      const void* weight, const void* bias, int param_dtype, float eps, const void* residual, int act,
                                      void* y, float* save_mean, float* save_rstd, void* workspace, size_t workspace_bytes, void* stream) {
    const int bad = check_args(n, c, dtype, samples, offsets, groups, param_dtype, act);
    if (bad != PVX_OK) return bad;
    if (!(eps >= 0.f) || !save_mean || !save_rstd) return PVX_ERR_INVALID;
    if (n == 0) return PVX_OK;
    if (!x || !y) return PVX_ERR_INVALID;
    PvxCarver cv(workspace, workspace_bytes);
    const Ws ws = carve(cv, c, samples, groups, pieces_cap(n, c, samples, offsets != nullptr));
    if (!cv.ok()) return PVX_ERR_WORKSPACE;
    const Rows rows{offsets, order, n, samples, offsets ? 0 : n / samples};
    bool one;
    const Shape sh = shape_for(rows, c, groups, chunk_of(c, dtype, {x, residual, y}), one);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == PVX_F32) return fwd_impl<float>(x, rows, c, groups, weight, bias, param_dtype, eps, residual, act, y, save_mean, save_rstd, ws, sh, one, st);
    if (dtype == PVX_F16) return fwd_impl<_Float16>(x, rows, c, groups, weight, bias, param_dtype, eps, residual, act, y, save_mean, save_rstd, ws, sh, one, st);
    return fwd_impl<__bf16>(x, rows, c, groups, weight, bias, param_dtype, eps, residual, act, y, save_mean, save_rstd, ws, sh, one, st);
}

extern "C" int pvx_group_norm_act_bwd(const void* dy, const void* x, const void* residual, int n, int c, int dtype, int samples,
                                      const int* offsets, const int* order, int groups, const void* weight, const void* bias,
                                      int param_dtype, const float* save_mean, const float* save_rstd, int act, void* dx, void* dresidual,
                                      void* dweight, void* dbias, void* workspace, size_t workspace_bytes, void* stream) {
    const int bad = check_args(n, c, dtype, samples, offsets, groups, param_dtype, act);
    if (bad != PVX_OK) return bad;
    hipStream_t st = (hipStream_t)stream;
    if (n == 0) {
        if (!dweight && !dbias) return PVX_OK;
        hipLaunchKernelGGL(gn_zero_params_kernel, dim3(PVX_CDIV(c, kBlk)), dim3(kBlk), 0, st, dweight, dbias, param_dtype, c);
        PVX_CHECK_LAUNCH();
        return PVX_OK;
    }
    if (!dy || !x || !dx || !save_mean || !save_rstd) return PVX_ERR_INVALID;
    PvxCarver cv(workspace, workspace_bytes);
    const Ws ws = carve(cv, c, samples, groups, pieces_cap(n, c, samples, offsets != nullptr));
    if (!cv.ok()) return PVX_ERR_WORKSPACE;
    const Rows rows{offsets, order, n, samples, offsets ? 0 : n / samples};
    bool one;
    const Shape sh = shape_for(rows, c, groups, chunk_of(c, dtype, {dy, x, residual, dx, dresidual}), one);
    if (dtype == PVX_F32) return bwd_impl<float>(dy, x, residual, rows, c, groups, weight, bias, param_dtype, save_mean, save_rstd, act, dx, dresidual, dweight, dbias, ws, sh, one, st);
    if (dtype == PVX_F16) return bwd_impl<_Float16>(dy, x, residual, rows, c, groups, weight, bias, param_dtype, save_mean, save_rstd, act, dx, dresidual, dweight, dbias, ws, sh, one, st);
    return bwd_impl<__bf16>(dy, x, residual, rows, c, groups, weight, bias, param_dtype, save_mean, save_rstd, act, dx, dresidual, dweight, dbias, ws, sh, one, st);
}
