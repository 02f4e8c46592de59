// Group norm over the rows of a channels-last matrix, fused with (+ residual) -> activation, forward and backward.
//
// x [n, c] holds the rows of `samples` samples (frames); sample s owns the positions offsets[s] .. offsets[s + 1], position p is row
// order[p] (or p).  With R_s the rows of sample s and C_g the channels of group g, over the |R_s| |C_g| values of each pair (s, g):
//   mu = mean x, v = mean (x - mu)^2, xhat = (x - mu) / sqrt(v + eps), z = w xhat + b (+ residual), y = act(z)
// and with gz = dy act'(z), gx = w gz:
//   db = sum gz, dw = sum gz xhat over all rows;   dx = (gx - mean gx - xhat mean(gx xhat)) / sqrt(v + eps);   dresidual = gz
//
// Ten to thirty flops per element: HBM bounds it.  A thread owns one 16-byte chunk of channels (narrower where c or an address does not
// allow it) and walks down the rows, as in batchnorm.hip; a workgroup owns a contiguous range of positions and takes the samples in
// it one after the other, so ragged samples, empty ones and shared workgroups need no padding and no atomics: the piece of sample s in
// workgroup k leaves its sums at index k + s (distinct, because later workgroups never see earlier samples).
// Sums are held in binary64: its adds run at the rate of binary32's here, and sum x^2 - (sum x)^2 / N keeps its digits.
#include "pvx_common.h"

namespace {

constexpr int kBlk = 256;
constexpr int kTargetBlocks = 1024;      // ranges of positions: four workgroups for each CU
constexpr int kOneChunks = 16;           // chunks a thread of the one-launch form holds
constexpr int kOneBlocks = 2048;         // workgroups of that form: more samples than this are taken in turns

template <typename E, int V> struct alignas(sizeof(E) * V) Pack { E e[V]; };

template <typename E, int V> __device__ __forceinline__ void load_pack(const E* p, float (&v)[V]) {
    const Pack<E, V> k = *reinterpret_cast<const Pack<E, V>*>(p);
#pragma unroll
    for (int j = 0; j < V; j++) v[j] = (float)k.e[j];
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

constexpr float kSqrtHalf = 0.70710678118654752f, kInvSqrt2Pi = 0.39894228040143268f;

// `act` is the same for the whole launch: the branches are scalar
__device__ __forceinline__ float act_of(float z, int act) {
    if (act == PVX_ACT_RELU) return z < 0.f ? 0.f : z;       // keeps NaN
    if (act == PVX_ACT_SILU) return z / (1.f + __expf(-z));
    if (act == PVX_ACT_GELU) return 0.5f * z * (1.f + erff(z * kSqrtHalf));
    return z;
}

__device__ __forceinline__ float slope_of(float z, int act) {
    if (act == PVX_ACT_RELU) return z > 0.f ? 1.f : 0.f;
    if (act == PVX_ACT_SILU) {
        const float p = 1.f / (1.f + __expf(-z));
        return p * (1.f + z * (1.f - p));
    }
    if (act == PVX_ACT_GELU) return 0.5f * (1.f + erff(z * kSqrtHalf)) + z * kInvSqrt2Pi * __expf(-0.5f * z * z);
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
    // first sample that ends behind position p
    __device__ __forceinline__ int first(int p) const {
        if (!offsets) return p / each;
        int lo = 0, hi = samples;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (begin(mid + 1) > p) hi = mid; else lo = mid + 1;
        }
        return lo;
    }
    // row at position p, -1 if `order` does not hold one
    __device__ __forceinline__ int row(int p) const {
        if (!order) return p;
        const int r = order[p];
        return r >= 0 && r < n ? r : -1;
    }
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

// sums two binary64 vectors of V channels over the row slots of the workgroup; the result is in slot 0's threads.
// red: [2][kBlk][V + 1]
template <int V> __device__ __forceinline__ void fold_rows(double (&s0)[V], double (&s1)[V], const Place& t, double* red) {
    double(*r0)[V + 1] = reinterpret_cast<double(*)[V + 1]>(red);
    double(*r1)[V + 1] = r0 + kBlk;
    __syncthreads();                     // the buffer's last readers are done
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

// sums of x and x^2 for each piece and channel: partial[piece][2][c]
template <typename E, int V>
__global__ __launch_bounds__(kBlk) void gn_sums_kernel(const E* __restrict__ x, Rows rows, int c, int range, double* __restrict__ partial) {
    __shared__ double red[2 * kBlk * (V + 1)];
    const Place t = place<V>(c);
    const int p0 = blockIdx.x * range, p1 = min(rows.n, p0 + range);
    for (int s = rows.first(p0); s < rows.samples; s++) {
        const int lo = max(p0, rows.begin(s)), hi = min(p1, rows.begin(s + 1));
        if (rows.begin(s) >= p1) break;
        if (lo >= hi) continue;
        double s0[V], s1[V];
#pragma unroll
        for (int j = 0; j < V; j++) { s0[j] = 0; s1[j] = 0; }
        if (t.on) {
#pragma unroll 4
            for (int p = lo + t.r_in; p < hi; p += t.rpb) {
                const int row = rows.row(p);
                if (row < 0) continue;
                float v[V];
                load_pack<E, V>(x + (size_t)row * c + t.chunk * V, v);
#pragma unroll
                for (int j = 0; j < V; j++) { const double d = v[j]; s0[j] += d; s1[j] = fma(d, d, s1[j]); }
            }
        }
        fold_rows<V>(s0, s1, t, red);
        if (t.on && t.r_in == 0) {
            double* out = partial + (size_t)(blockIdx.x + s) * 2 * c + t.chunk * V;
#pragma unroll
            for (int j = 0; j < V; j++) { out[j] = s0[j]; out[c + j] = s1[j]; }
        }
    }
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    return v;
}

// the sums of workgroup-wide `v` in every thread; red: 4 doubles
__device__ __forceinline__ double block_sum(double v, double* red) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return red[0] + red[1] + red[2] + red[3];
}

// mean and 1 / sqrt(variance + eps) of each (sample, group) from its pieces
__global__ __launch_bounds__(kBlk) void gn_finish_kernel(const double* __restrict__ partial, Rows rows, int c, int groups, int range, float eps,
                                                          float* __restrict__ mean, float* __restrict__ rstd) {
    __shared__ double red[4];
    const int s = blockIdx.x / groups, g = blockIdx.x % groups, cpg = c / groups;
    const int lo = rows.begin(s), hi = rows.begin(s + 1);
    double a = 0.0, b = 0.0;
    if (hi > lo) {
        const int k0 = lo / range, pieces = (hi - 1) / range - k0 + 1;
        for (int i = threadIdx.x; i < pieces * cpg; i += kBlk) {
            const double* q = partial + (size_t)(k0 + s + i / cpg) * 2 * c + g * cpg + i % cpg;
            a += q[0];
            b += q[c];
        }
    }
    a = block_sum(a, red);
    b = block_sum(b, red);
    if (threadIdx.x != 0) return;
    const double count = hi > lo ? (double)(hi - lo) * cpg : 1.0;
    const double mu = a / count;
    double var = b / count - mu * mu;
    if (var < 0.0) var = 0.0;
    mean[blockIdx.x] = (float)mu;
    rstd[blockIdx.x] = (float)(1.0 / sqrt(var + (double)eps));
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

template <typename E, int V>
__global__ __launch_bounds__(kBlk) void gn_apply_kernel(const E* __restrict__ x, const E* __restrict__ residual, Rows rows, int c, int groups,
                                                         int range, const void* __restrict__ weight, const void* __restrict__ bias, int pd,
                                                         const float* __restrict__ mean, const float* __restrict__ rstd, int act,
                                                         E* __restrict__ y) {
    const Place t = place<V>(c);
    if (!t.on) return;
    const int p0 = blockIdx.x * range, p1 = min(rows.n, p0 + range), cpg = c / groups;
    int done = p0;                       // positions below it are written
    for (int s = rows.first(p0); s < rows.samples; s++) {
        const int lo = max(p0, rows.begin(s)), hi = min(p1, rows.begin(s + 1));
        if (rows.begin(s) >= p1) break;
        if (lo >= hi) continue;
        for (int p = done + t.r_in; p < lo; p += t.rpb) {       // positions of no sample
            const int row = rows.row(p);
            const float zero[V] = {};
            if (row >= 0) store_pack<E, V>(y + (size_t)row * c + t.chunk * V, zero);
        }
        Chan<V> k;
        load_chan<V>(k, t.chunk * V, s, groups, cpg, weight, bias, pd, mean, rstd);
#pragma unroll 4
        for (int p = lo + t.r_in; p < hi; p += t.rpb) {
            const int row = rows.row(p);
            if (row < 0) continue;
            const size_t off = (size_t)row * c + t.chunk * V;
            float v[V], r[V];
            load_pack<E, V>(x + off, v);
            if (residual) load_pack<E, V>(residual + off, r);
#pragma unroll
            for (int j = 0; j < V; j++) {
                float z = (v[j] - k.mu[j]) * k.rs[j] * k.w[j] + k.b[j];
                if (residual) z += r[j];
                v[j] = act_of(z, act);
            }
            store_pack<E, V>(y + off, v);
        }
        done = hi;
    }
    for (int p = done + t.r_in; p < p1; p += t.rpb) {
        const int row = rows.row(p);
        const float zero[V] = {};
        if (row >= 0) store_pack<E, V>(y + (size_t)row * c + t.chunk * V, zero);
    }
}

// backward, first pass: sums of gz and gz xhat for each piece and channel
template <typename E, int V>
__global__ __launch_bounds__(kBlk) void gn_bwd_sums_kernel(const E* __restrict__ dy, const E* __restrict__ x, const E* __restrict__ residual,
                                                            Rows rows, int c, int groups, int range, const void* __restrict__ weight,
                                                            const void* __restrict__ bias, int pd, const float* __restrict__ mean,
                                                            const float* __restrict__ rstd, int act, double* __restrict__ partial) {
    __shared__ double red[2 * kBlk * (V + 1)];
    const Place t = place<V>(c);
    const int p0 = blockIdx.x * range, p1 = min(rows.n, p0 + range), cpg = c / groups;
    for (int s = rows.first(p0); s < rows.samples; s++) {
        const int lo = max(p0, rows.begin(s)), hi = min(p1, rows.begin(s + 1));
        if (rows.begin(s) >= p1) break;
        if (lo >= hi) continue;
        double s0[V], s1[V];
#pragma unroll
        for (int j = 0; j < V; j++) { s0[j] = 0; s1[j] = 0; }
        if (t.on) {
            Chan<V> k;
            load_chan<V>(k, t.chunk * V, s, groups, cpg, weight, bias, pd, mean, rstd);
#pragma unroll 2
            for (int p = lo + t.r_in; p < hi; p += t.rpb) {
                const int row = rows.row(p);
                if (row < 0) continue;
                const size_t off = (size_t)row * c + t.chunk * V;
                float g[V], v[V], r[V];
                load_pack<E, V>(dy + off, g);
                load_pack<E, V>(x + off, v);
                if (residual) load_pack<E, V>(residual + off, r);
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float xh = (v[j] - k.mu[j]) * k.rs[j];
                    float z = xh * k.w[j] + k.b[j];
                    if (residual) z += r[j];
                    const float gz = g[j] * slope_of(z, act);
                    s0[j] += (double)gz;
                    s1[j] = fma((double)gz, (double)xh, s1[j]);
                }
            }
        }
        fold_rows<V>(s0, s1, t, red);
        if (t.on && t.r_in == 0) {
            double* out = partial + (size_t)(blockIdx.x + s) * 2 * c + t.chunk * V;
#pragma unroll
            for (int j = 0; j < V; j++) { out[j] = s0[j]; out[c + j] = s1[j]; }
        }
    }
}

// backward, finish: workgroups 0 .. samples * groups - 1 leave mean gx and mean(gx xhat) of their (sample, group); the c behind them
// leave db and dw of their channel, summed over the pieces in order
__global__ __launch_bounds__(kBlk) void gn_bwd_finish_kernel(const double* __restrict__ partial, Rows rows, int c, int groups, int range,
                                                              const void* __restrict__ weight, int pd, float* __restrict__ m0,
                                                              float* __restrict__ m1, void* __restrict__ dweight, void* __restrict__ dbias) {
    __shared__ double red[4];
    const int pairs = rows.samples * groups, cpg = c / groups;
    double a = 0.0, b = 0.0;
    if ((int)blockIdx.x < pairs) {
        const int s = blockIdx.x / groups, g = blockIdx.x % groups;
        const int lo = rows.begin(s), hi = rows.begin(s + 1);
        if (hi > lo) {
            const int k0 = lo / range, pieces = (hi - 1) / range - k0 + 1;
            for (int i = threadIdx.x; i < pieces * cpg; i += kBlk) {
                const int cc = g * cpg + i % cpg;
                const double* q = partial + (size_t)(k0 + s + i / cpg) * 2 * c + cc;
                const double w = load_param(weight, pd, cc, 1.f);
                a += w * q[0];
                b += w * q[c];
            }
        }
        a = block_sum(a, red);
        b = block_sum(b, red);
        if (threadIdx.x == 0) {
            const double count = hi > lo ? (double)(hi - lo) * cpg : 1.0;
            m0[blockIdx.x] = (float)(a / count);
            m1[blockIdx.x] = (float)(b / count);
        }
        return;
    }
    const int cc = blockIdx.x - pairs;
    // few samples: the threads stride over a sample's pieces; many: over the samples
    const bool many = rows.samples >= kBlk;
    for (int s = many ? threadIdx.x : 0; s < rows.samples; s += many ? kBlk : 1) {
        const int lo = rows.begin(s), hi = rows.begin(s + 1);
        if (hi <= lo) continue;
        const int k0 = lo / range, pieces = (hi - 1) / range - k0 + 1;
        for (int i = many ? 0 : threadIdx.x; i < pieces; i += many ? 1 : kBlk) {
            const double* q = partial + (size_t)(k0 + s + i) * 2 * c + cc;
            a += q[0];
            b += q[c];
        }
    }
    a = block_sum(a, red);
    b = block_sum(b, red);
    if (threadIdx.x == 0) {
        if (dbias) store_param(dbias, pd, cc, a);
        if (dweight) store_param(dweight, pd, cc, b);
    }
}

template <typename E, int V>
__global__ __launch_bounds__(kBlk) void gn_bwd_apply_kernel(const E* __restrict__ dy, const E* __restrict__ x, const E* __restrict__ residual,
                                                             Rows rows, int c, int groups, int range, const void* __restrict__ weight,
                                                             const void* __restrict__ bias, int pd, const float* __restrict__ mean,
                                                             const float* __restrict__ rstd, const float* __restrict__ m0,
                                                             const float* __restrict__ m1, int act, E* __restrict__ dx, E* __restrict__ dres) {
    const Place t = place<V>(c);
    if (!t.on) return;
    const int p0 = blockIdx.x * range, p1 = min(rows.n, p0 + range), cpg = c / groups;
    const float zero[V] = {};
    int done = p0;
    for (int s = rows.first(p0); s < rows.samples; s++) {
        const int lo = max(p0, rows.begin(s)), hi = min(p1, rows.begin(s + 1));
        if (rows.begin(s) >= p1) break;
        if (lo >= hi) continue;
        for (int p = done + t.r_in; p < lo; p += t.rpb) {
            const int row = rows.row(p);
            if (row < 0) continue;
            const size_t off = (size_t)row * c + t.chunk * V;
            store_pack<E, V>(dx + off, zero);
            if (dres) store_pack<E, V>(dres + off, zero);
        }
        Chan<V> k;
        load_chan<V>(k, t.chunk * V, s, groups, cpg, weight, bias, pd, mean, rstd);
        float a[V], b[V];
#pragma unroll
        for (int j = 0; j < V; j++) {
            const int i = s * groups + (t.chunk * V + j) / cpg;
            a[j] = m0[i];
            b[j] = m1[i];
        }
#pragma unroll 2
        for (int p = lo + t.r_in; p < hi; p += t.rpb) {
            const int row = rows.row(p);
            if (row < 0) continue;
            const size_t off = (size_t)row * c + t.chunk * V;
            float g[V], v[V], r[V], o[V];
            load_pack<E, V>(dy + off, g);
            load_pack<E, V>(x + off, v);
            if (residual) load_pack<E, V>(residual + off, r);
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float xh = (v[j] - k.mu[j]) * k.rs[j];
                float z = xh * k.w[j] + k.b[j];
                if (residual) z += r[j];
                g[j] *= slope_of(z, act);
                o[j] = k.rs[j] * (g[j] * k.w[j] - a[j] - xh * b[j]);
            }
            store_pack<E, V>(dx + off, o);
            if (dres) store_pack<E, V>(dres + off, g);
        }
        done = hi;
    }
    for (int p = done + t.r_in; p < p1; p += t.rpb) {
        const int row = rows.row(p);
        if (row < 0) continue;
        const size_t off = (size_t)row * c + t.chunk * V;
        store_pack<E, V>(dx + off, zero);
        if (dres) store_pack<E, V>(dres + off, zero);
    }
}

// One launch: a workgroup holds one sample's rows in registers (at most kOneChunks chunks a thread), so x is read once and nothing but
// the statistics goes through memory.  Taken where every sample is known to fit: latency is what such calls cost (three launches
// otherwise).  blockIdx.x == samples: the positions of no sample.
template <int V> __device__ __forceinline__ void group_sums(int c, int groups, double* red, double* per_group) {
    // slot 0's threads hold the channels' sums in red[0 / 1][chunk][j]; one wave takes a group at a time
    double(*r0)[V + 1] = reinterpret_cast<double(*)[V + 1]>(red);
    double(*r1)[V + 1] = r0 + kBlk;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, cpg = c / groups;
    __syncthreads();
    for (int g = wave; g < groups; g += kBlk / 64) {
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
    __syncthreads();
}

template <typename E, int V>
__device__ __forceinline__ void zero_uncovered(const Place& t, const Rows& rows, int c, E* a, E* b) {
    if (!t.on) return;
    const int lo = rows.begin(0), hi = rows.begin(rows.samples);
    const float zero[V] = {};
    for (int p = t.r_in; p < rows.n; p += t.rpb) {
        if (p >= lo && p < hi) continue;
        const int row = rows.row(p);
        if (row < 0) continue;
        const size_t off = (size_t)row * c + t.chunk * V;
        store_pack<E, V>(a + off, zero);
        if (b) store_pack<E, V>(b + off, zero);
    }
}

template <typename E, int V, int U>
__global__ __launch_bounds__(kBlk) void gn_one_kernel(const E* __restrict__ x, const E* __restrict__ residual, Rows rows, int c, int groups,
                                                       const void* __restrict__ weight, const void* __restrict__ bias, int pd, float eps,
                                                       int act, E* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
    __shared__ double red[2 * kBlk * (V + 1)];
    extern __shared__ double per_group[];                // [groups][2]
    const Place t = place<V>(c);
    const int cpg = c / groups, blocks = gridDim.x - (rows.offsets ? 1 : 0);
    if ((int)blockIdx.x == blocks) { zero_uncovered<E, V>(t, rows, c, y, (E*)nullptr); return; }
    for (int s = blockIdx.x; s < rows.samples; s += blocks) {
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
        if (!t.on) continue;
        float mu[V], rs[V], w[V], b[V];
#pragma unroll
        for (int j = 0; j < V; j++) {
            const int cc = t.chunk * V + j, g = cc / cpg;
            mu[j] = (float)per_group[2 * g];
            rs[j] = (float)per_group[2 * g + 1];
            w[j] = load_param(weight, pd, cc, 1.f);
            b[j] = load_param(bias, pd, cc, 0.f);
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
}

// the backward of the same; a workgroup adds dw and db up over its samples and leaves them in partial[workgroup][2][c]
template <typename E, int V, int U>
__global__ __launch_bounds__(kBlk) void gn_bwd_one_kernel(const E* __restrict__ dy, const E* __restrict__ x, const E* __restrict__ residual,
                                                           Rows rows, int c, int groups, const void* __restrict__ weight,
                                                           const void* __restrict__ bias, int pd, const float* __restrict__ mean,
                                                           const float* __restrict__ rstd, int act, E* __restrict__ dx, E* __restrict__ dres,
                                                           void* __restrict__ dweight, void* __restrict__ dbias, double* __restrict__ partial) {
    __shared__ double red[2 * kBlk * (V + 1)];
    extern __shared__ double per_group[];
    const Place t = place<V>(c);
    const int cpg = c / groups, blocks = gridDim.x - (rows.offsets ? 1 : 0);
    if ((int)blockIdx.x == blocks) { zero_uncovered<E, V>(t, rows, c, dx, dres); return; }
    double db[V], dw[V];
#pragma unroll
    for (int j = 0; j < V; j++) { db[j] = 0; dw[j] = 0; }
    for (int s = blockIdx.x; s < rows.samples; s += blocks) {
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
                db[j] += s0[j];
                dw[j] += s1[j];
                r0[threadIdx.x][j] = s0[j] * (double)k.w[j];     // the groups' sums take w gz
                r0[kBlk + threadIdx.x][j] = s1[j] * (double)k.w[j];
            }
        }
        group_sums<V>(c, groups, red, per_group);
        if (!t.on) continue;
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
    }
    if (t.on && t.r_in == 0) {
        double* out = partial + (size_t)blockIdx.x * 2 * c + t.chunk * V;
#pragma unroll
        for (int j = 0; j < V; j++) {
            if (blocks == 1) {
                if (dbias) store_param(dbias, pd, t.chunk * V + j, db[j]);
                if (dweight) store_param(dweight, pd, t.chunk * V + j, dw[j]);
            } else {
                out[j] = db[j];
                out[c + j] = dw[j];
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
    int v, ch, tw, rpb, tiles, range, blocks;
};

// elements of a thread's chunk: 16 bytes, or fewer where c or an address asks for it
int chunk_of(int c, int dtype, std::initializer_list<const void*> ptrs) {
    const int es = dtype == PVX_F32 ? 4 : 2;
    int v = 16 / es;
    uintptr_t low = 0;
    for (const void* p : ptrs) low |= (uintptr_t)p;
    while (v > 1 && (c % v != 0 || low % ((uintptr_t)v * es) != 0)) v >>= 1;
    return v;
}

int range_of(int n, int rpb) {
    long long r = PVX_CDIV((long long)n, (long long)kTargetBlocks);
    r = PVX_CDIV(r < 2LL * rpb ? 2LL * rpb : r, (long long)rpb) * rpb;
    return (int)r;
}

Shape shape_of(int n, int c, int v) {
    Shape s;
    s.v = v;
    s.ch = c / v;
    s.tw = s.ch < kBlk ? s.ch : kBlk;
    s.rpb = kBlk / s.tw;
    s.tiles = PVX_CDIV(s.ch, s.tw);
    s.range = range_of(n, s.rpb);
    s.blocks = PVX_CDIV(n, s.range);
    return s;
}

// workspace: one piece for each workgroup and one more for each sample that begins inside one (equal samples that fit the one-launch
// form whatever the alignment need its workgroups only), and the backward's two means per (sample, group)
size_t pieces_cap(int n, int c, int samples, bool ragged) {
    if (!ragged && c <= kBlk && n / samples <= kOneChunks * (kBlk / c)) return samples < kOneBlocks ? samples : kOneBlocks;
    return (size_t)(n < kTargetBlocks ? n : kTargetBlocks) + samples;
}

template <typename C> void carve(C& cv, int n, int c, int samples, int groups, size_t pieces, double** partial, float** m0, float** m1) {
    *partial = cv.template take<double>(pieces * 2 * c);
    *m0 = cv.template take<float>((size_t)samples * groups);
    *m1 = cv.template take<float>((size_t)samples * groups);
}

// chunks a thread holds when a workgroup takes a whole sample; 0: some sample may not fit
int one_chunks(const Rows& rows, const Shape& sh, int groups) {
    if (sh.tiles != 1 || groups > 1024) return 0;
    const int most = rows.offsets ? rows.n : rows.each, u = PVX_CDIV(most, sh.rpb);
    return u <= 4 ? 4 : (u <= kOneChunks ? kOneChunks : 0);
}

int check_args(int n, int c, int dtype, int samples, const int* offsets, int groups, int param_dtype, int act) {
    if (n < 0 || c <= 0 || samples <= 0 || groups <= 0 || c % groups != 0) return PVX_ERR_INVALID;
    if (dtype < PVX_F32 || dtype > PVX_BF16 || param_dtype < PVX_F32 || param_dtype > PVX_BF16) return PVX_ERR_INVALID;
    if (act < PVX_ACT_NONE || act > PVX_ACT_GELU) return PVX_ERR_INVALID;
    if (!offsets && n % samples != 0) return PVX_ERR_INVALID;
    // launches are indexed by (sample, group) and channel; positions, pieces and piece x channel products by 32 bits
    if ((long long)samples * groups + c > 0x7fffffffLL || n > 0x7fffffff - (1 << 20) || c > (1 << 20)) return PVX_ERR_RANGE;
    return PVX_OK;
}

#define GN_DISPATCH(E, v, CALL)                      \
    do {                                             \
        if (v == 8) { CALL(E, (16 / (int)sizeof(E))); } \
        else if (v == 4) { CALL(E, 4); }             \
        else if (v == 2) { CALL(E, 2); }             \
        else { CALL(E, 1); }                         \
    } while (0)

template <typename E>
int fwd_impl(const void* x, const Rows& rows, int c, int groups, const void* weight, const void* bias, int pd, float eps,
             const void* residual, int act, void* y, float* mean, float* rstd, double* partial, const Shape& sh, hipStream_t st) {
    if (const int u = one_chunks(rows, sh, groups)) {
        const int blocks = rows.samples < kOneBlocks ? rows.samples : kOneBlocks;
        const dim3 one(blocks + (rows.offsets ? 1 : 0));
        const size_t lds = sizeof(double) * 2 * groups;
#define GN_ONE(E, V)                                                                                                                        \
        if (u == 4) hipLaunchKernelGGL((gn_one_kernel<E, V, 4>), one, dim3(kBlk), lds, st, (const E*)x, (const E*)residual, rows, c, groups, \
                                       weight, bias, pd, eps, act, (E*)y, mean, rstd);                                                      \
        else hipLaunchKernelGGL((gn_one_kernel<E, V, kOneChunks>), one, dim3(kBlk), lds, st, (const E*)x, (const E*)residual, rows, c,       \
                                groups, weight, bias, pd, eps, act, (E*)y, mean, rstd)
        GN_DISPATCH(E, sh.v, GN_ONE);
        PVX_CHECK_LAUNCH();
        return PVX_OK;
    }
    const dim3 grid(sh.blocks, sh.tiles);
#define GN_SUMS(E, V) hipLaunchKernelGGL((gn_sums_kernel<E, V>), grid, dim3(kBlk), 0, st, (const E*)x, rows, c, sh.range, partial)
    GN_DISPATCH(E, sh.v, GN_SUMS);
    PVX_CHECK_LAUNCH();
    hipLaunchKernelGGL(gn_finish_kernel, dim3(rows.samples * groups), dim3(kBlk), 0, st, partial, rows, c, groups, sh.range, eps, mean, rstd);
    PVX_CHECK_LAUNCH();
#define GN_APPLY(E, V) hipLaunchKernelGGL((gn_apply_kernel<E, V>), grid, dim3(kBlk), 0, st, (const E*)x, (const E*)residual, rows, c, groups, \
                                          sh.range, weight, bias, pd, mean, rstd, act, (E*)y)
    GN_DISPATCH(E, sh.v, GN_APPLY);
    PVX_CHECK_LAUNCH();
    return PVX_OK;
}

template <typename E>
int bwd_impl(const void* dy, const void* x, const void* residual, const Rows& rows, int c, int groups, const void* weight, const void* bias,
             int pd, const float* mean, const float* rstd, int act, void* dx, void* dres, void* dweight, void* dbias, double* partial,
             float* m0, float* m1, const Shape& sh, hipStream_t st) {
    if (const int u = one_chunks(rows, sh, groups)) {
        const int blocks = rows.samples < kOneBlocks ? rows.samples : kOneBlocks;
        const dim3 one(blocks + (rows.offsets ? 1 : 0));
        const size_t lds = sizeof(double) * 2 * groups;
#define GN_BONE(E, V)                                                                                                                    \
        if (u == 4) hipLaunchKernelGGL((gn_bwd_one_kernel<E, V, 4>), one, dim3(kBlk), lds, st, (const E*)dy, (const E*)x,                \
                                       (const E*)residual, rows, c, groups, weight, bias, pd, mean, rstd, act, (E*)dx, (E*)dres, dweight, \
                                       dbias, partial);                                                                                  \
        else hipLaunchKernelGGL((gn_bwd_one_kernel<E, V, kOneChunks>), one, dim3(kBlk), lds, st, (const E*)dy, (const E*)x,               \
                                (const E*)residual, rows, c, groups, weight, bias, pd, mean, rstd, act, (E*)dx, (E*)dres, dweight, dbias, \
                                partial)
        GN_DISPATCH(E, sh.v, GN_BONE);
        PVX_CHECK_LAUNCH();
        if (blocks > 1 && (dweight || dbias)) {
            hipLaunchKernelGGL(gn_bwd_channels_kernel, dim3(c), dim3(64), 0, st, partial, blocks, c, pd, dweight, dbias);
            PVX_CHECK_LAUNCH();
        }
        return PVX_OK;
    }
    const dim3 grid(sh.blocks, sh.tiles);
#define GN_BSUMS(E, V) hipLaunchKernelGGL((gn_bwd_sums_kernel<E, V>), grid, dim3(kBlk), 0, st, (const E*)dy, (const E*)x, (const E*)residual, \
                                          rows, c, groups, sh.range, weight, bias, pd, mean, rstd, act, partial)
    GN_DISPATCH(E, sh.v, GN_BSUMS);
    PVX_CHECK_LAUNCH();
    hipLaunchKernelGGL(gn_bwd_finish_kernel, dim3(rows.samples * groups + c), dim3(kBlk), 0, st, partial, rows, c, groups, sh.range, weight, pd,
                       m0, m1, dweight, dbias);
    PVX_CHECK_LAUNCH();
#define GN_BAPPLY(E, V) hipLaunchKernelGGL((gn_bwd_apply_kernel<E, V>), grid, dim3(kBlk), 0, st, (const E*)dy, (const E*)x, (const E*)residual, \
                                           rows, c, groups, sh.range, weight, bias, pd, mean, rstd, m0, m1, act, (E*)dx, (E*)dres)
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
    double* p;
    float *a, *b;
    carve(shim, n, c, samples, groups, pieces_cap(n, c, samples, ragged != 0), &p, &a, &b);
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
    double* partial;
    float *m0, *m1;
    carve(cv, n, c, samples, groups, pieces_cap(n, c, samples, offsets != nullptr), &partial, &m0, &m1);
    if (!cv.ok()) return PVX_ERR_WORKSPACE;
    const Rows rows{offsets, order, n, samples, offsets ? 0 : n / samples};
    const Shape sh = shape_of(n, c, chunk_of(c, dtype, {x, residual, y}));
    hipStream_t st = (hipStream_t)stream;
    if (dtype == PVX_F32) return fwd_impl<float>(x, rows, c, groups, weight, bias, param_dtype, eps, residual, act, y, save_mean, save_rstd, partial, sh, st);
    if (dtype == PVX_F16) return fwd_impl<_Float16>(x, rows, c, groups, weight, bias, param_dtype, eps, residual, act, y, save_mean, save_rstd, partial, sh, st);
    return fwd_impl<__bf16>(x, rows, c, groups, weight, bias, param_dtype, eps, residual, act, y, save_mean, save_rstd, partial, sh, st);
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
    double* partial;
    float *m0, *m1;
    carve(cv, n, c, samples, groups, pieces_cap(n, c, samples, offsets != nullptr), &partial, &m0, &m1);
    if (!cv.ok()) return PVX_ERR_WORKSPACE;
    const Rows rows{offsets, order, n, samples, offsets ? 0 : n / samples};
    const Shape sh = shape_of(n, c, chunk_of(c, dtype, {dy, x, residual, dx, dresidual}));
    if (dtype == PVX_F32) return bwd_impl<float>(dy, x, residual, rows, c, groups, weight, bias, param_dtype, save_mean, save_rstd, act, dx, dresidual, dweight, dbias, partial, m0, m1, sh, st);
    if (dtype == PVX_F16) return bwd_impl<_Float16>(dy, x, residual, rows, c, groups, weight, bias, param_dtype, save_mean, save_rstd, act, dx, dresidual, dweight, dbias, partial, m0, m1, sh, st);
    return bwd_impl<__bf16>(dy, x, residual, rows, c, groups, weight, bias, param_dtype, save_mean, save_rstd, act, dx, dresidual, dweight, dbias, partial, m0, m1, sh, st);
}
