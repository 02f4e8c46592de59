// Rows of a table looked up by index, and the gradient of that by sorted index.
//
//   out[i] = scale T[index[i]]                      (rows of zeros where index[i] is outside [0, m))
//   dT[v]  = scale sum_{i : index[i] = v} dout[i]   (in ascending i; rows nobody looked up are zero)
//
// The gradient sorts the positions by index once (a stable counting sort by digits, below) and then every table row adds up its own
// run of the list: sums in binary32, no atomics, the same bits on every run, and every row of dT is written exactly once.  Both
// directions move bytes and nothing else: HBM bounds them, the launches at small sizes.
#include "pvx_common.h"

namespace {

constexpr int kBlk = 256;
constexpr int kTile = 2048;              // keys of a workgroup in a pass over many tiles
constexpr int kMaxBits = 11;             // digit of such a pass: 2^22 rows in two passes
constexpr int kOneBlk = 1024, kOneKeys = 8, kOneMax = kOneBlk * kOneKeys, kOneBits = 8;

template <typename I> __device__ __forceinline__ int key_of(I v, int m) { return v >= 0 && v < (I)m ? (int)v : m; }

// lanes of this wave whose digit equals the caller's (only lanes with `on`)
__device__ __forceinline__ unsigned long long same_digit(int digit, int bits, bool on) {
    unsigned long long mask = __ballot(on);
    for (int b = 0; b < bits; b++) {
        const unsigned long long set = __ballot((digit >> b) & 1);
        mask &= (digit >> b) & 1 ? set : ~set;
    }
    return mask;
}

// ---- one workgroup sorts everything: up to kOneMax keys, all passes in LDS -----------------------------------------------------
template <typename I>
__global__ __launch_bounds__(kOneBlk) void sort_one_kernel(const I* __restrict__ index, int n, int m, int total_bits, int* __restrict__ order,
                                                           int* __restrict__ keys_out, int* __restrict__ offsets) {
    constexpr int kWaves = kOneBlk / 64, kDigits = 1 << kOneBits;
    __shared__ int skey[kOneMax], sidx[kOneMax];
    __shared__ int cnt[kWaves][kDigits];
    __shared__ int wsum[kDigits / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int key[kOneKeys], idx[kOneKeys], at[kOneKeys];
#pragma unroll
    for (int r = 0; r < kOneKeys; r++) {
        const int i = (wave * kOneKeys + r) * 64 + lane;
        idx[r] = i;
        key[r] = i < n ? key_of<I>(index[i], m) : m;
    }
    for (int shift = 0; shift < total_bits; shift += kOneBits) {
        const int bits = total_bits - shift < kOneBits ? total_bits - shift : kOneBits;
        for (int i = threadIdx.x; i < kWaves * kDigits; i += kOneBlk) (&cnt[0][0])[i] = 0;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kOneKeys; r++) {
            const bool on = (wave * kOneKeys + r) * 64 + lane < n;
            const int d = (key[r] >> shift) & ((1 << bits) - 1);
            const unsigned long long mask = same_digit(d, bits, on);
            const int before = __popcll(mask & ((1ull << lane) - 1ull));
            if (on) at[r] = cnt[wave][d] + before;
            __builtin_amdgcn_wave_barrier();
            if (on && before == 0) cnt[wave][d] += __popcll(mask);
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
        // exclusive over (digit, wave): digit totals first
        int total = 0, incl = 0;
        if (threadIdx.x < kDigits) {
            for (int w = 0; w < kWaves; w++) { const int v = cnt[w][threadIdx.x]; cnt[w][threadIdx.x] = total; total += v; }
            incl = total;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) { const int v = __shfl_up(incl, off); if (lane >= off) incl += v; }
            if (lane == 63) wsum[wave] = incl;
        }
        __syncthreads();
        if (threadIdx.x < kDigits) {
            int base = incl - total;
            for (int w = 0; w < wave; w++) base += wsum[w];
            for (int w = 0; w < kWaves; w++) cnt[w][threadIdx.x] += base;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kOneKeys; r++) {
            if ((wave * kOneKeys + r) * 64 + lane < n) {
                const int to = cnt[wave][(key[r] >> shift) & ((1 << bits) - 1)] + at[r];
                skey[to] = key[r];
                sidx[to] = idx[r];
            }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kOneKeys; r++) {
            const int i = (wave * kOneKeys + r) * 64 + lane;
            if (i < n) { key[r] = skey[i]; idx[r] = sidx[i]; }
        }
        __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < kOneKeys; r++) {
        const int i = (wave * kOneKeys + r) * 64 + lane;
        if (i < n) { order[i] = idx[r]; keys_out[i] = key[r]; }
    }
    if (offsets) {                       // skey holds the sorted keys (total_bits >= 1: at least one pass ran)
        for (int v = threadIdx.x; v <= m; v += kOneBlk) {
            int lo = 0, hi = n;
            while (lo < hi) { const int mid = (lo + hi) >> 1; if (skey[mid] < v) lo = mid + 1; else hi = mid; }
            offsets[v] = lo;
        }
    }
}

// ---- many workgroups: per pass a histogram of each tile, a scan along the tiles of each digit, a stable scatter ------------------
// keys of the first pass come from `index`; those of the later ones from the pass before
template <typename I>
__global__ __launch_bounds__(kBlk) void sort_count_kernel(const I* __restrict__ index, int first, int n, int m, int shift, int bits, int tiles,
                                                          int* __restrict__ hist) {
    extern __shared__ int count[];
    const int digits = 1 << bits;
    for (int d = threadIdx.x; d < digits; d += kBlk) count[d] = 0;
    __syncthreads();
    const int base = blockIdx.x * kTile;
#pragma unroll
    for (int r = 0; r < kTile / kBlk; r++) {
        const int i = base + r * kBlk + threadIdx.x;
        if (i < n) {
            const I v = index[i];
            const int key = first ? key_of<I>(v, m) : (int)v;
            atomicAdd(&count[(key >> shift) & (digits - 1)], 1);
        }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += kBlk) hist[(size_t)d * tiles + blockIdx.x] = count[d];
}

// a wave for each digit: exclusive scan along its tiles, the digit's total behind them
__global__ __launch_bounds__(64) void sort_scan_kernel(int* __restrict__ hist, int tiles, int* __restrict__ totals) {
    int* row = hist + (size_t)blockIdx.x * tiles;
    int carry = 0;
    for (int base = 0; base < tiles; base += 64) {
        const int i = base + threadIdx.x;
        const int v = i < tiles ? row[i] : 0;
        int incl = v;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) { const int t = __shfl_up(incl, off); if ((int)threadIdx.x >= off) incl += t; }
        if (i < tiles) row[i] = carry + incl - v;
        carry += __shfl(incl, 63);
    }
    if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

template <typename I>
__global__ __launch_bounds__(kBlk) void sort_scatter_kernel(const I* __restrict__ index, const int* __restrict__ idx_in, int first, int n, int m,
                                                            int shift, int bits, int tiles, const int* __restrict__ hist,
                                                            const int* __restrict__ totals, int* __restrict__ keys_out,
                                                            int* __restrict__ idx_out) {
    constexpr int kWaves = kBlk / 64, kRounds = kTile / kBlk;
    extern __shared__ int cnt[];                             // [kWaves][digits], then kWaves sums
    const int digits = 1 << bits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int* wsum = cnt + kWaves * digits;
    for (int i = threadIdx.x; i < kWaves * digits; i += kBlk) cnt[i] = 0;
    __syncthreads();
    const int base = blockIdx.x * kTile + wave * (kTile / kWaves);
    int key[kRounds], at[kRounds], idx[kRounds];
#pragma unroll
    for (int r = 0; r < kRounds; r++) {
        const int i = base + r * 64 + lane;
        key[r] = m;
        idx[r] = i;
        if (i < n) {
            const I v = index[i];
            key[r] = first ? key_of<I>(v, m) : (int)v;
            if (!first) idx[r] = idx_in[i];
        }
    }
    int* mine = cnt + wave * digits;
#pragma unroll
    for (int r = 0; r < kRounds; r++) {
        const bool on = base + r * 64 + lane < n;
        const int d = (key[r] >> shift) & (digits - 1);
        const unsigned long long mask = same_digit(d, bits, on);
        const int before = __popcll(mask & ((1ull << lane) - 1ull));
        at[r] = on ? mine[d] + before : 0;
        __builtin_amdgcn_wave_barrier();
        if (on && before == 0) mine[d] += __popcll(mask);
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    // where this tile's keys of a digit begin: the digits before it (all tiles), the tiles before this one, the waves before
    const int per = digits / kBlk > 0 ? digits / kBlk : 1;
    const int d0 = threadIdx.x * per;
    int sum = 0;
    if (d0 < digits) for (int k = 0; k < per; k++) sum += totals[d0 + k];
    int incl = sum;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) { const int v = __shfl_up(incl, off); if (lane >= off) incl += v; }
    if (lane == 63) wsum[wave] = incl;
    __syncthreads();
    int begin = incl - sum;
    for (int w = 0; w < wave; w++) begin += wsum[w];
    if (d0 < digits) {
        for (int k = 0; k < per; k++) {
            int from = begin + hist[(size_t)(d0 + k) * tiles + blockIdx.x];
            begin += totals[d0 + k];
            for (int w = 0; w < kWaves; w++) { const int v = cnt[w * digits + d0 + k]; cnt[w * digits + d0 + k] = from; from += v; }
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; r++) {
        if (base + r * 64 + lane < n) {
            const int to = mine[(key[r] >> shift) & (digits - 1)] + at[r];
            keys_out[to] = key[r];
            idx_out[to] = idx[r];
        }
    }
}

// offsets[v] = first sorted position whose key is >= v, v = 0 .. m
__global__ __launch_bounds__(kBlk) void sort_offsets_kernel(const int* __restrict__ keys, int n, int m, int* __restrict__ offsets) {
    const long long v = (long long)blockIdx.x * kBlk + threadIdx.x;
    if (v > m) return;
    int lo = 0, hi = n;
    while (lo < hi) { const int mid = lo + ((hi - lo) >> 1); if (keys[mid] < v) lo = mid + 1; else hi = mid; }
    offsets[v] = lo;
}

__global__ __launch_bounds__(kBlk) void fill_int_kernel(int* __restrict__ p, long long n, int v) {
    const long long i = (long long)blockIdx.x * kBlk + threadIdx.x;
    if (i < n) p[i] = v;
}

// ---- rows ---------------------------------------------------------------------------------------------------------------------
template <typename E, int V> struct alignas(sizeof(E) * V) Pack { E e[V]; };

template <typename E, int V, typename I>
__global__ __launch_bounds__(kBlk) void lookup_kernel(const E* __restrict__ table, const I* __restrict__ index, long long chunks, int ch, int m,
                                                      float scale, E* __restrict__ out) {
    typedef Pack<E, V> P;
    for (long long i = (long long)blockIdx.x * kBlk + threadIdx.x; i < chunks; i += (long long)gridDim.x * kBlk) {
        const long long row = i / ch;
        const int k = (int)(i - row * ch);
        const I v = index[row];
        P p;
        if (v >= 0 && v < (I)m) {
            p = reinterpret_cast<const P*>(table)[(long long)v * ch + k];
            if (scale != 1.f) {
#pragma unroll
                for (int j = 0; j < V; j++) p.e[j] = (E)((float)p.e[j] * scale);
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; j++) p.e[j] = (E)0.f;
        }
        reinterpret_cast<P*>(out)[i] = p;
    }
}

// Long runs are added up in blocks of kFan positions (level 1), blocks of kFan such blocks (level 2) and once more (level 3), each only
// where a whole aligned block carries one key; a row then walks ends position by position and the middle by the largest blocks
// that fit: at most 2 * 3 * kFan + n / kFan^3 steps for a row, whatever share of the list it has.
constexpr int kFan = 32, kFanLog = 5, kLevels = 3;

template <typename E, int V>
__global__ __launch_bounds__(kBlk) void run_first_kernel(const E* __restrict__ dout, const int* __restrict__ order, const int* __restrict__ offsets,
                                                         const int* __restrict__ keys, int n, int m, int ch, int blocks,
                                                         float* __restrict__ part) {
    typedef Pack<E, V> P;
    const long long t = (long long)blockIdx.x * kBlk + threadIdx.x;
    const long long blk = t / ch;
    if (blk >= blocks) return;
    const int k = (int)(t - blk * ch), p0 = (int)blk * kFan;
    const int key = keys[p0];
    if (key >= m || keys[p0 + kFan - 1] != key) return;
    float acc[V];
#pragma unroll
    for (int j = 0; j < V; j++) acc[j] = 0.f;
#pragma unroll 8
    for (int i = 0; i < kFan; i++) {
        const int row = order[p0 + i];
        if ((unsigned)row >= (unsigned)n) continue;
        const P p = reinterpret_cast<const P*>(dout)[(long long)row * ch + k];
#pragma unroll
        for (int j = 0; j < V; j++) acc[j] += (float)p.e[j];
    }
    float* o = part + (blk * ch + k) * V;
#pragma unroll
    for (int j = 0; j < V; j++) o[j] = acc[j];
}

// a level's blocks from the level before; shift: log2 of the positions of a block of this level
__global__ __launch_bounds__(kBlk) void run_next_kernel(const float* __restrict__ in, const int* __restrict__ keys, int m, int width, int blocks,
                                                        int shift, float* __restrict__ part) {
    const long long t = (long long)blockIdx.x * kBlk + threadIdx.x;
    const long long blk = t / width;
    if (blk >= blocks) return;
    const int k = (int)(t - blk * width);
    const long long p0 = blk << shift;
    const int key = keys[p0];
    if (key >= m || keys[p0 + (1LL << shift) - 1] != key) return;
    float acc = 0.f;
#pragma unroll 8
    for (int i = 0; i < kFan; i++) acc += in[(blk * kFan + i) * width + k];
    part[blk * width + k] = acc;
}

struct Levels { const float* p[kLevels]; int n; };

template <typename E, int V>
__global__ __launch_bounds__(kBlk) void row_sum_kernel(const E* __restrict__ dout, const int* __restrict__ order, const int* __restrict__ offsets,
                                                       int n, int m, int ch, Levels lv, float scale, E* __restrict__ dtable) {
    typedef Pack<E, V> P;
    const long long total = (long long)m * ch;
    for (long long t = (long long)blockIdx.x * kBlk + threadIdx.x; t < total; t += (long long)gridDim.x * kBlk) {
        const int v = (int)(t / ch), k = (int)(t - (long long)v * ch);
        int p = offsets[v];
        const int end = min(offsets[v + 1], n);
        float acc[V];
#pragma unroll
        for (int j = 0; j < V; j++) acc[j] = 0.f;
        p = max(p, 0);
        while (p < end) {
            int level = 0;                   // the largest aligned block that fits
            while (level < lv.n && (p & ((kFan << (kFanLog * level)) - 1)) == 0 && p <= end - (kFan << (kFanLog * level))) level++;
            if (level > 0) {
                const int shift = kFanLog * level;
                const float* q = lv.p[level - 1] + ((long long)(p >> shift) * ch + k) * V;
#pragma unroll
                for (int j = 0; j < V; j++) acc[j] += q[j];
                p += 1 << shift;
                continue;
            }
            // positions up to the next place a block may begin
            const int stop = lv.n > 0 ? min(end, (p | (kFan - 1)) + 1) : end;
#pragma unroll 4
            for (; p < stop; p++) {
                const int row = order[p];
                if ((unsigned)row >= (unsigned)n) continue;
                const P q = reinterpret_cast<const P*>(dout)[(long long)row * ch + k];
#pragma unroll
                for (int j = 0; j < V; j++) acc[j] += (float)q.e[j];
            }
        }
        P o;
#pragma unroll
        for (int j = 0; j < V; j++) o.e[j] = (E)(acc[j] * scale);
        reinterpret_cast<P*>(dtable)[t] = o;
    }
}

int bits_of(int m) {                     // bits of the keys 0 .. m (m >= 1)
    int b = 1;
    while (b < 31 && (m >> b) != 0) b++;
    return b;
}

int tiles_of(int n) { return (int)PVX_CDIV((long long)n, (long long)kTile); }

struct SortWs { int *keys0, *keys1, *idx0, *hist, *totals; };

template <typename C> void carve_sort(C& cv, int n, SortWs* w) {
    const bool many = n > kOneMax;
    const size_t t = many ? (size_t)tiles_of(n) << kMaxBits : 0;
    w->keys0 = cv.template take<int>(many ? n : 0);
    w->keys1 = cv.template take<int>(many ? n : 0);
    w->idx0 = cv.template take<int>(many ? n : 0);
    w->hist = cv.template take<int>(t);
    w->totals = cv.template take<int>(many ? (size_t)1 << kMaxBits : 0);
}

template <typename I>
int sort_impl(const I* index, int n, int m, int* order, int* keys, int* offsets, const SortWs& w, hipStream_t st) {
    const int total_bits = bits_of(m);
    if (n <= kOneMax) {
        const bool inside = m <= 2 * kOneMax;          // few rows: the same workgroup writes their offsets
        hipLaunchKernelGGL((sort_one_kernel<I>), dim3(1), dim3(kOneBlk), 0, st, index, n, m, total_bits, order, keys, inside ? offsets : (int*)nullptr);
        PVX_CHECK_LAUNCH();
        if (inside) return PVX_OK;
    } else {
        const int passes = PVX_CDIV(total_bits, kMaxBits), tiles = tiles_of(n);
        int shift = 0;
        const int *kin = nullptr, *iin = nullptr;
        for (int p = 0; p < passes; p++) {
            const int bits = PVX_CDIV(total_bits - shift, passes - p), digits = 1 << bits;
            const bool last = p == passes - 1;
            // the last pass ends in the caller's arrays: the buffers alternate backwards from there
            int* kout = last ? keys : ((passes - p) % 2 == 0 ? w.keys0 : w.keys1);
            int* iout = (passes - 1 - p) % 2 == 0 ? order : w.idx0;
            const size_t lds = sizeof(int) * ((size_t)digits * (kBlk / 64) + kBlk / 64);
            if (p == 0) {
                hipLaunchKernelGGL((sort_count_kernel<I>), dim3(tiles), dim3(kBlk), sizeof(int) * digits, st, index, 1, n, m, shift, bits, tiles, w.hist);
                PVX_CHECK_LAUNCH();
                hipLaunchKernelGGL(sort_scan_kernel, dim3(digits), dim3(64), 0, st, w.hist, tiles, w.totals);
                PVX_CHECK_LAUNCH();
                hipLaunchKernelGGL((sort_scatter_kernel<I>), dim3(tiles), dim3(kBlk), lds, st, index, (const int*)nullptr, 1, n, m, shift, bits, tiles,
                                   w.hist, w.totals, kout, iout);
            } else {
                hipLaunchKernelGGL((sort_count_kernel<int>), dim3(tiles), dim3(kBlk), sizeof(int) * digits, st, kin, 0, n, m, shift, bits, tiles, w.hist);
                PVX_CHECK_LAUNCH();
                hipLaunchKernelGGL(sort_scan_kernel, dim3(digits), dim3(64), 0, st, w.hist, tiles, w.totals);
                PVX_CHECK_LAUNCH();
                hipLaunchKernelGGL((sort_scatter_kernel<int>), dim3(tiles), dim3(kBlk), lds, st, kin, iin, 0, n, m, shift, bits, tiles, w.hist, w.totals,
                                   kout, iout);
            }
            PVX_CHECK_LAUNCH();
            kin = kout;
            iin = iout;
            shift += bits;
        }
    }
    hipLaunchKernelGGL(sort_offsets_kernel, dim3((unsigned)PVX_CDIV((long long)m + 1, (long long)kBlk)), dim3(kBlk), 0, st, keys, n, m, offsets);
    PVX_CHECK_LAUNCH();
    return PVX_OK;
}

int vector_of(int width, int dtype, std::initializer_list<const void*> ptrs) {
    const int es = dtype == PVX_F32 ? 4 : 2;
    int v = 16 / es;
    uintptr_t low = 0;
    for (const void* p : ptrs) low |= (uintptr_t)p;
    while (v > 1 && (width % v != 0 || low % ((uintptr_t)v * es) != 0)) v >>= 1;
    return v;
}

template <typename C> Levels carve_levels(C& cv, int n, int width, float** out) {
    Levels lv;
    lv.n = 0;
    for (int l = 0; l < kLevels; l++) {
        const int blocks = n >> (kFanLog * (l + 1));
        out[l] = blocks >= 2 ? cv.template take<float>((size_t)blocks * width) : nullptr;
        lv.p[l] = out[l];
        if (blocks >= 2) lv.n = l + 1;
    }
    return lv;
}

template <typename E, int V>
int grad_impl(const E* dout, const int* order, const int* keys, const int* offsets, int n, int m, int width, float scale, E* dtable, float** part,
              const Levels& lv, hipStream_t st) {
    const int ch = width / V;
    for (int l = 0; l < lv.n; l++) {
        const int blocks = n >> (kFanLog * (l + 1));
        if (l == 0) {
            const long long work = (long long)blocks * ch;
            hipLaunchKernelGGL((run_first_kernel<E, V>), dim3((unsigned)PVX_CDIV(work, (long long)kBlk)), dim3(kBlk), 0, st, dout, order, offsets, keys, n, m,
                               ch, blocks, part[0]);
        } else {
            const long long work = (long long)blocks * width;
            hipLaunchKernelGGL(run_next_kernel, dim3((unsigned)PVX_CDIV(work, (long long)kBlk)), dim3(kBlk), 0, st, part[l - 1], keys, m, width, blocks,
                               kFanLog * (l + 1), part[l]);
        }
        PVX_CHECK_LAUNCH();
    }
    const long long work = PVX_CDIV((long long)m * ch, (long long)kBlk);
    hipLaunchKernelGGL((row_sum_kernel<E, V>), dim3((unsigned)(work > 65536 ? 65536 : work)), dim3(kBlk), 0, st, dout, order, offsets, n, m, ch, lv, scale,
                       dtable);
    PVX_CHECK_LAUNCH();
    return PVX_OK;
}

#define LK_DISPATCH(E, v, CALL)                        \
    do {                                               \
        if (v == 8) return CALL(E, (16 / (int)sizeof(E))); \
        if (v == 4) return CALL(E, 4);                 \
        if (v == 2) return CALL(E, 2);                 \
        return CALL(E, 1);                             \
    } while (0)

template <typename E>
int grad_dispatch(const void* dout, const int* order, const int* keys, const int* offsets, int n, int m, int width, float scale, void* dtable,
                  float** part, const Levels& lv, int v, hipStream_t st) {
#define LK_GRAD(E, V) grad_impl<E, V>((const E*)dout, order, keys, offsets, n, m, width, scale, (E*)dtable, part, lv, st)
    LK_DISPATCH(E, v, LK_GRAD);
}

template <typename E, int V>
int lookup_impl(const E* table, const void* index, int index64, int n, int m, int width, float scale, E* out, hipStream_t st) {
    const int ch = width / V;
    const long long chunks = (long long)n * ch, blocks = PVX_CDIV(chunks, (long long)kBlk);
    const dim3 grid((unsigned)(blocks > 65536 ? 65536 : blocks));
    if (index64) hipLaunchKernelGGL((lookup_kernel<E, V, long long>), grid, dim3(kBlk), 0, st, table, (const long long*)index, chunks, ch, m, scale, out);
    else hipLaunchKernelGGL((lookup_kernel<E, V, int>), grid, dim3(kBlk), 0, st, table, (const int*)index, chunks, ch, m, scale, out);
    PVX_CHECK_LAUNCH();
    return PVX_OK;
}

template <typename E>
int lookup_dispatch(const void* table, const void* index, int index64, int n, int m, int width, float scale, void* out, int v, hipStream_t st) {
#define LK_FWD(E, V) lookup_impl<E, V>((const E*)table, index, index64, n, m, width, scale, (E*)out, st)
    LK_DISPATCH(E, v, LK_FWD);
}

struct SizerShim {
    PvxSizer s;
    template <typename T> T* take(size_t k) { s.take<T>(k); return nullptr; }
};

constexpr int kMaxRows = 0x7fffffff - (1 << 20);     // positions and rows are 32-bit, and so are the sums that pass them by a tile

}  // namespace

extern "C" size_t pvx_sort_index_workspace_bytes(int n) {
    if (n <= 0) return 256;
    SizerShim shim;
    SortWs w;
    carve_sort(shim, n, &w);
    return shim.s.total();
}

extern "C" int pvx_sort_index(const void* index, int index64, int n, int m, int* order, int* keys, int* offsets, void* workspace,
                              size_t workspace_bytes, void* stream) {
    if (n < 0 || m <= 0 || !offsets || (n > 0 && (!index || !order || !keys))) return PVX_ERR_INVALID;
    if (n > kMaxRows || m > kMaxRows) return PVX_ERR_RANGE;
    hipStream_t st = (hipStream_t)stream;
    if (n == 0) {
        hipLaunchKernelGGL(fill_int_kernel, dim3((unsigned)PVX_CDIV((long long)m + 1, (long long)kBlk)), dim3(kBlk), 0, st, offsets, (long long)m + 1, 0);
        PVX_CHECK_LAUNCH();
        return PVX_OK;
    }
    PvxCarver cv(workspace, workspace_bytes);
    SortWs w;
    carve_sort(cv, n, &w);
    if (!cv.ok()) return PVX_ERR_WORKSPACE;
    if (index64) return sort_impl<long long>((const long long*)index, n, m, order, keys, offsets, w, st);
    return sort_impl<int>((const int*)index, n, m, order, keys, offsets, w, st);
}

extern "C" int pvx_lookup_rows(const void* table, int dtype, const void* index, int index64, int n, int m, int width, float scale, void* out,
                               void* stream) {
    if (n < 0 || m < 0 || width < 0 || dtype < PVX_F32 || dtype > PVX_BF16) return PVX_ERR_INVALID;
    if (n == 0 || width == 0) return PVX_OK;
    if (!index || !out || (m > 0 && !table)) return PVX_ERR_INVALID;
    if (n > kMaxRows || m > kMaxRows || width > (1 << 24)) return PVX_ERR_RANGE;
    const int v = vector_of(width, dtype, {table, out});
    hipStream_t st = (hipStream_t)stream;
    if (dtype == PVX_F32) return lookup_dispatch<float>(table, index, index64, n, m, width, scale, out, v, st);
    if (dtype == PVX_F16) return lookup_dispatch<_Float16>(table, index, index64, n, m, width, scale, out, v, st);
    return lookup_dispatch<__bf16>(table, index, index64, n, m, width, scale, out, v, st);
}

extern "C" size_t pvx_lookup_rows_grad_workspace_bytes(int n, int width) {
    if (n <= 0 || width <= 0) return 256;
    SizerShim shim;
    float* part[kLevels];
    carve_levels(shim, n, width, part);
    return shim.s.total() + 256;
}

extern "C" int pvx_lookup_rows_grad(const void* dout, int dtype, const int* order, const int* keys, const int* offsets, int n, int m, int width,
                                    float scale, void* dtable, void* workspace, size_t workspace_bytes, void* stream) {
    if (n < 0 || m < 0 || width < 0 || dtype < PVX_F32 || dtype > PVX_BF16) return PVX_ERR_INVALID;
    if (m == 0 || width == 0) return PVX_OK;
    if (!offsets || !dtable || (n > 0 && (!dout || !order || !keys))) return PVX_ERR_INVALID;
    if (n > kMaxRows || m > kMaxRows || width > (1 << 24)) return PVX_ERR_RANGE;
    PvxCarver cv(workspace, workspace_bytes);
    float* part[kLevels];
    const Levels lv = carve_levels(cv, n, width, part);
    if (!cv.ok()) return PVX_ERR_WORKSPACE;
    const int v = vector_of(width, dtype, {dout, dtable});
    hipStream_t st = (hipStream_t)stream;
    if (dtype == PVX_F32) return grad_dispatch<float>(dout, order, keys, offsets, n, m, width, scale, dtable, part, lv, v, st);
    if (dtype == PVX_F16) return grad_dispatch<_Float16>(dout, order, keys, offsets, n, m, width, scale, dtable, part, lv, v, st);
    return grad_dispatch<__bf16>(dout, order, keys, offsets, n, m, width, scale, dtable, part, lv, v, st);
}
