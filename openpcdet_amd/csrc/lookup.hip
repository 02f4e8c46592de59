// Rows of a table looked up by index, and the gradient of that by sorted index.
//
//   out[i] = scale T[index[i]]                      (rows of zeros where index[i] is outside [0, m))
//   dT[v]  = scale sum_{i : index[i] = v} dout[i]   (in ascending i; rows nobody looked up are zero)
//
// The gradient sorts the positions by index once (a stable counting sort by digits, below) and adds rows up in the order of the sorted
// list: sums in binary32, no atomics, the same bits on every run.  Both directions move bytes and nothing else: HBM bounds them, the
// launches at small sizes.
#include "pvx_common.h"

namespace {

constexpr int kBlk = 256;
constexpr int kMaxBits = 11;             // digit of a pass over many tiles: 2^22 rows in two passes
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

// Memory to set to zero by `blocks` workgroups.  The gradient's table rides behind the sort's first kernel, which leaves the chip idle,
// rather than in a launch of its own.
struct Clear {
    char* p;
    long long bytes;
    int blocks;
    __device__ __forceinline__ void part(int block, int threads) const {
        // whole 16-byte pieces between the ends; the allocation begins anywhere
        const long long head = min(bytes, (long long)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15)), pieces = (bytes - head) / 16;
        const long long i0 = (long long)block * threads + threadIdx.x, step = (long long)blocks * threads;
        uint4* q = reinterpret_cast<uint4*>(p + head);
        for (long long i = i0; i < pieces; i += step) q[i] = make_uint4(0, 0, 0, 0);
        for (long long i = i0; i < head; i += step) p[i] = 0;
        for (long long i = head + pieces * 16 + i0; i < bytes; i += step) p[i] = 0;
    }
};

// ---- one workgroup sorts everything: up to kOneMax keys, all passes in LDS -----------------------------------------------------
template <typename I>
__global__ __launch_bounds__(kOneBlk) void sort_one_kernel(const I* __restrict__ index, int n, int m, int total_bits, int* __restrict__ order,
                                                           int* __restrict__ keys_out, int* __restrict__ offsets, Clear clear) {
    if (blockIdx.x > 0) { clear.part(blockIdx.x - 1, kOneBlk); return; }
    constexpr int kWaves = kOneBlk / 64, kDigits = 1 << kOneBits;
    __shared__ int skey[kOneMax], sidx[kOneMax];
    __shared__ int cnt[kWaves][kDigits];
    __shared__ int wsum[kDigits / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int rounds = PVX_CDIV(n, kOneBlk), first = wave * rounds * 64 + lane;      // a wave's keys lie together, on all waves alike
    int key[kOneKeys], idx[kOneKeys], at[kOneKeys];
#pragma unroll
    for (int r = 0; r < kOneKeys; r++) {
        const int i = first + r * 64;
        if (r >= rounds) break;
        idx[r] = i;
        key[r] = i < n ? key_of<I>(index[i], m) : m;
    }
    for (int shift = 0; shift < total_bits; shift += kOneBits) {
        const int bits = total_bits - shift < kOneBits ? total_bits - shift : kOneBits;
        for (int i = threadIdx.x; i < kWaves * kDigits; i += kOneBlk) (&cnt[0][0])[i] = 0;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kOneKeys; r++) {
            if (r >= rounds) break;
            const bool on = first + r * 64 < n;
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
            if (r < rounds && first + r * 64 < n) {
                const int to = cnt[wave][(key[r] >> shift) & ((1 << bits) - 1)] + at[r];
                skey[to] = key[r];
                sidx[to] = idx[r];
            }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kOneKeys; r++) {
            const int i = first + r * 64;
            if (r < rounds && i < n) { key[r] = skey[i]; idx[r] = sidx[i]; }
        }
        __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < kOneKeys; r++) {
        const int i = first + r * 64;
        if (r < rounds && i < n) { order[i] = idx[r]; keys_out[i] = key[r]; }
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
// The first pass takes its keys from `index`; between passes key and position travel as one word, the last pass writes them apart.
template <typename I> struct From {      // the caller's index
    __device__ static __forceinline__ int key(const I* p, int i, int m) { return key_of<I>(p[i], m); }
    __device__ static __forceinline__ int2 both(const I* p, int i, int m) { return make_int2(key_of<I>(p[i], m), i); }
};
template <> struct From<int2> {
    __device__ static __forceinline__ int key(const int2* p, int i, int) { return p[i].x; }
    __device__ static __forceinline__ int2 both(const int2* p, int i, int) { return p[i]; }
};

// hist[tile * by_tile + digit * by_digit]
template <typename I, int R>
__global__ __launch_bounds__(kBlk) void sort_count_kernel(const I* __restrict__ in, int n, int m, int shift, int bits, int by_tile, int by_digit,
                                                          int* __restrict__ hist, int tiles, Clear clear) {
    extern __shared__ int count[];
    if ((int)blockIdx.x >= tiles) { clear.part(blockIdx.x - tiles, kBlk); return; }
    const int digits = 1 << bits;
    for (int d = threadIdx.x; d < digits; d += kBlk) count[d] = 0;
    __syncthreads();
    const int base = blockIdx.x * R * kBlk;
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int i = base + r * kBlk + threadIdx.x;
        if (i < n) atomicAdd(&count[(From<I>::key(in, i, m) >> shift) & (digits - 1)], 1);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += kBlk) hist[(size_t)blockIdx.x * by_tile + (size_t)d * by_digit] = count[d];
}

// many tiles: a wave for each digit, exclusive scan along its tiles, four at a time for each lane, the digit's total behind them
__global__ __launch_bounds__(64) void sort_scan_kernel(int* __restrict__ hist, int tiles, int* __restrict__ totals) {
    int* row = hist + (size_t)blockIdx.x * tiles;
    const int lane = threadIdx.x;
    int carry = 0;
    for (int base = 0; base < tiles; base += 256) {
        int v[4], sum = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int i = base + lane * 4 + e;
            v[e] = i < tiles ? row[i] : 0;
        }
#pragma unroll
        for (int e = 0; e < 4; e++) { const int t = v[e]; v[e] = sum; sum += t; }
        int incl = sum;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) { const int t = __shfl_up(incl, off); if (lane >= off) incl += t; }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int i = base + lane * 4 + e;
            if (i < tiles) row[i] = carry + incl - sum + v[e];
        }
        carry += __shfl(incl, 63);
    }
    if (lane == 0) totals[blockIdx.x] = carry;
}

// totals: what sort_scan_kernel left, or NULL: hist holds the tiles' own counts, [tile][digit], and this workgroup adds them up itself
template <typename I, int R, bool LAST>
__global__ __launch_bounds__(kBlk) void sort_scatter_kernel(const I* __restrict__ in, int n, int m, int shift, int bits, int tiles,
                                                            const int* __restrict__ hist, const int* __restrict__ totals, int2* __restrict__ out,
                                                            int* __restrict__ keys, int* __restrict__ order) {
    constexpr int kWaves = kBlk / 64;
    extern __shared__ int cnt[];                             // [kWaves][digits], then kWaves sums
    const int digits = 1 << bits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int* wsum = cnt + kWaves * digits;
    for (int i = threadIdx.x; i < kWaves * digits; i += kBlk) cnt[i] = 0;
    __syncthreads();
    const int base = (blockIdx.x * kWaves + wave) * R * 64;
    int2 item[R];
    int at[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const int i = base + r * 64 + lane;
        item[r] = i < n ? From<I>::both(in, i, m) : make_int2(m, 0);
    }
    int* mine = cnt + wave * digits;
#pragma unroll
    for (int r = 0; r < R; r++) {
        const bool on = base + r * 64 + lane < n;
        const int d = (item[r].x >> shift) & (digits - 1);
        const unsigned long long mask = same_digit(d, bits, on);
        const int before = __popcll(mask & ((1ull << lane) - 1ull));
        at[r] = on ? mine[d] + before : 0;
        __builtin_amdgcn_wave_barrier();
        if (on && before == 0) mine[d] += __popcll(mask);
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    // where this tile's keys of a digit begin: the digits before it (all tiles), the tiles before this one, the waves before.  A thread
    // takes the digits threadIdx.x * per ..
    constexpr int kPer = (1 << kMaxBits) / kBlk;
    const int per = digits / kBlk > 0 ? digits / kBlk : 1, d0 = threadIdx.x * per;
    int all[kPer], before[kPer], sum = 0;
#pragma unroll
    for (int k = 0; k < kPer; k++) {
        all[k] = before[k] = 0;
        if (k >= per || d0 + k >= digits) continue;
        if (totals) {
            all[k] = totals[d0 + k];
            before[k] = hist[(size_t)(d0 + k) * tiles + blockIdx.x];
        } else {
#pragma unroll 8
            for (int t = 0; t < tiles; t++) {
                const int v = hist[(size_t)t * digits + d0 + k];
                all[k] += v;
                before[k] += t < (int)blockIdx.x ? v : 0;
            }
        }
        sum += all[k];
    }
    int incl = sum;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) { const int v = __shfl_up(incl, off); if (lane >= off) incl += v; }
    if (lane == 63) wsum[wave] = incl;
    __syncthreads();
    int begin = incl - sum;
    for (int w = 0; w < wave; w++) begin += wsum[w];
#pragma unroll
    for (int k = 0; k < kPer; k++) {
        if (k >= per || d0 + k >= digits) continue;
        int from = begin + before[k];
        begin += all[k];
        for (int w = 0; w < kWaves; w++) { const int v = cnt[w * digits + d0 + k]; cnt[w * digits + d0 + k] = from; from += v; }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; r++) {
        if (base + r * 64 + lane < n) {
            const int to = mine[(item[r].x >> shift) & (digits - 1)] + at[r];
            if (LAST) { keys[to] = item[r].x; order[to] = item[r].y; }
            else out[to] = item[r];
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

// Which row and chunk a thread owns: whole rows side by side in a workgroup, so nothing is divided per element (a 64-bit division a
// thread was half of the lookup's time); rows wider than a workgroup are walked.
struct Lane {
    int slot, chunk, slots;              // row within the workgroup's, first chunk, rows of a workgroup (0: this thread has none)
    __device__ __forceinline__ explicit Lane(int ch) {
        const int tw = ch < kBlk ? ch : kBlk;
        slots = kBlk / tw;
        slot = threadIdx.x / tw;
        chunk = slot < slots ? threadIdx.x % tw : ch;
    }
    __device__ __forceinline__ long long first() const { return (long long)blockIdx.x * slots + slot; }
    __device__ __forceinline__ long long step() const { return (long long)gridDim.x * slots; }
};

template <typename E, int V, typename I>
__global__ __launch_bounds__(kBlk) void lookup_kernel(const E* __restrict__ table, const I* __restrict__ index, int n, int ch, int m, float scale,
                                                      E* __restrict__ out) {
    typedef Pack<E, V> P;
    constexpr int U = 4;                 // rows on their way together
    const Lane t(ch);
    for (int k = t.chunk; k < ch; k += kBlk) {
        for (long long i = t.first(); i < n; i += U * t.step()) {
            I v[U];
            P p[U];
#pragma unroll
            for (int u = 0; u < U; u++) v[u] = index[min(i + u * t.step(), (long long)n - 1)];
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (v[u] >= 0 && v[u] < (I)m) p[u] = reinterpret_cast<const P*>(table)[(long long)v[u] * ch + k];
                else {
#pragma unroll
                    for (int j = 0; j < V; j++) p[u].e[j] = (E)0.f;
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (i + u * t.step() >= n) break;
                if (scale != 1.f && v[u] >= 0 && v[u] < (I)m) {
#pragma unroll
                    for (int j = 0; j < V; j++) p[u].e[j] = (E)((float)p[u].e[j] * scale);
                }
                reinterpret_cast<P*>(out)[(i + u * t.step()) * ch + k] = p[u];
            }
        }
    }
}

// The gradient's sums.  `ch` lanes take a block of 2^fan positions of the sorted list and walk it, eight rows on their way at a time: they
// add rows up while the key stays, and where it changes the table's row is finished.  A run that crosses a border of the block
// leaves what the block holds of it: the run that comes in from the left (or is the whole block) as the block's head, the one that goes on
// to the right as its tail.  2^fan heads are added up where they carry one key, and so on by levels; then the block in which a crossing
// run begins joins its tail, whole blocks by the largest that fit, and the last head: at most 2^fan steps within a block and twice that
// many blocks on each level, and kWorth of the last, whatever share of the list the row has.  (A level is made where the one before has
// kWorth blocks: 2 us where no run is long, 240 000 keys 63 -> 64 us; 1 048 579 skewed keys 337 -> 264.)  All work is in proportion to
// the list, so the table is cleared beforehand; a walk through each row's run by its offsets instead took 1.7 times as long where the
// runs' lengths differ much.
constexpr int kLevels = 5, kWorth = 256;

template <typename E, int V> __device__ __forceinline__ void store_row(E* dtable, long long at, const float (&acc)[V], float scale) {
    Pack<E, V> o;
#pragma unroll
    for (int j = 0; j < V; j++) o.e[j] = (E)(acc[j] * scale);
    reinterpret_cast<Pack<E, V>*>(dtable)[at] = o;
}

template <typename E, int V>
__global__ __launch_bounds__(kBlk) void run_sum_kernel(const E* __restrict__ dout, const int* __restrict__ order, const int* __restrict__ keys, int n,
                                                       int m, int ch, int blocks, int fan, float scale, float* __restrict__ head, float* __restrict__ tail,
                                                       E* __restrict__ dtable) {
    constexpr int U = 8;
    const Lane t(ch);
    for (int k = t.chunk; k < ch; k += kBlk) {
        for (long long blk = t.first(); blk < blocks; blk += t.step()) {
            const int p0 = (int)blk << fan, p1 = min(p0 + (1 << fan), n);
            const int left = p0 > 0 ? keys[p0 - 1] : -1, right = p1 < n ? keys[p1] : -1;
            int key[U + 1], row[U], begin = p0;
            float acc[V];
#pragma unroll
            for (int j = 0; j < V; j++) acc[j] = 0.f;
#pragma unroll
            for (int u = 0; u < U; u++) {
                key[u] = keys[min(p0 + u, p1 - 1)];
                row[u] = order[min(p0 + u, p1 - 1)];
            }
            for (int p = p0; p < p1; p += U) {
                Pack<E, V> q[U];
                int next_key[U], next_row[U];
#pragma unroll
                for (int u = 0; u < U; u++) q[u] = reinterpret_cast<const Pack<E, V>*>(dout)[(long long)min((unsigned)row[u], (unsigned)(n - 1)) * ch + k];
#pragma unroll
                for (int u = 0; u < U; u++) {                // those of the next eight, behind the rows
                    next_key[u] = keys[min(p + U + u, p1 - 1)];
                    next_row[u] = order[min(p + U + u, p1 - 1)];
                }
                key[U] = next_key[0];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int at = p + u, v = key[u];
                    if (at >= p1) break;
#pragma unroll
                    for (int j = 0; j < V; j++) acc[j] += (float)q[u].e[j];
                    const bool last = at == p1 - 1;
                    if (!last && key[u + 1] == v) continue;
                    if ((unsigned)v < (unsigned)m) {
                        const bool from_left = begin == p0 && left == v, to_right = last && right == v;
                        if (!from_left && !to_right) {
                            store_row<E, V>(dtable, (long long)v * ch + k, acc, scale);
                        } else {
                            float* o = (begin == p0 ? head : tail) + (blk * ch + k) * V;
#pragma unroll
                            for (int j = 0; j < V; j++) o[j] = acc[j];
                        }
                    }
#pragma unroll
                    for (int j = 0; j < V; j++) acc[j] = 0.f;
                    begin = at + 1;
                }
#pragma unroll
                for (int u = 0; u < U; u++) { key[u] = next_key[u]; row[u] = next_row[u]; }
            }
        }
    }
}

// a level's whole blocks from the level before; shift: log2 of the positions of a block of this level
__global__ __launch_bounds__(kBlk) void run_next_kernel(const float* __restrict__ in, const int* __restrict__ keys, int m, int width, int blocks,
                                                        int fan, int shift, float* __restrict__ part) {
    const Lane t(width);
    for (int k = t.chunk; k < width; k += kBlk) {
        for (long long blk = t.first(); blk < blocks; blk += t.step()) {
            const long long p0 = blk << shift;
            const int key = keys[p0];
            if ((unsigned)key >= (unsigned)m || keys[p0 + (1LL << shift) - 1] != key) continue;
            float acc = 0.f;
#pragma unroll 16
            for (int i = 0; i < 1 << fan; i++) acc += in[((blk << fan) + i) * width + k];
            part[blk * width + k] = acc;
        }
    }
}

// first position in (p, end] whose key is not `key`; keys ascend and keys[p] == key
__device__ __forceinline__ int run_end(const int* keys, int p, int end, int key) {
    int step = 32;
    while (p < end - step && keys[p + step] == key) { p += step; step <<= 1; }
    int hi = p < end - step ? p + step : end;
    while (hi - p > 1) { const int mid = p + ((hi - p) >> 1); if (keys[mid] == key) p = mid; else hi = mid; }
    return hi;
}

struct Levels { const float *p[kLevels], *tail; int n; };

// the rows of runs that cross a border, each by the block it begins in
template <typename E, int V>
__global__ __launch_bounds__(kBlk) void run_join_kernel(const int* __restrict__ keys, int n, int m, int ch, int blocks, int fan, Levels lv, float scale,
                                                        E* __restrict__ dtable) {
    const Lane t(ch);
    for (int k = t.chunk; k < ch; k += kBlk) {
        for (long long blk = t.first(); blk < blocks - 1; blk += t.step()) {
            const int p0 = (int)blk << fan, v = keys[p0 + (1 << fan) - 1];
            if ((unsigned)v >= (unsigned)m || keys[p0 + (1 << fan)] != v) continue;
            const bool whole = keys[p0] == v;
            if (whole && p0 > 0 && keys[p0 - 1] == v) continue;                  // it began further left
            const float* q = (whole ? lv.p[0] : lv.tail) + (blk * ch + k) * V;
            float acc[V];
#pragma unroll
            for (int j = 0; j < V; j++) acc[j] = q[j];
            int p = p0 + (1 << fan);
            const int end = run_end(keys, p, n, v);
            while (p < end) {
                int level = 1;                       // the largest aligned block that fits
                while (level < lv.n && (p & ((1 << fan * (level + 1)) - 1)) == 0 && p <= end - (1 << fan * (level + 1))) level++;
                // the blocks of this level up to where a larger one may begin (the last, open one of level 1 is a head), eight at a time
                const int shift = fan * level, b0 = p >> shift, last = (int)(((long long)end + (1 << fan) - 1) >> fan);
                int b1 = level == 1 ? last : end >> shift;
                if (level < lv.n) b1 = min(b1, (b0 | ((1 << fan) - 1)) + 1);
                q = lv.p[level - 1] + k * V;
                for (int b = b0; b < b1; b += 8) {
                    float w[8][V];
#pragma unroll
                    for (int u = 0; u < 8; u++)
#pragma unroll
                        for (int j = 0; j < V; j++) w[u][j] = q[(long long)min(b + u, b1 - 1) * ch * V + j];
#pragma unroll
                    for (int u = 0; u < 8; u++)
                        if (b + u < b1) {
#pragma unroll
                            for (int j = 0; j < V; j++) acc[j] += w[u][j];
                        }
                }
                if (level == 1 && b1 == last) break;
                p = b1 << shift;
            }
            store_row<E, V>(dtable, (long long)v * ch + k, acc, scale);
        }
    }
}

__global__ __launch_bounds__(kBlk) void clear_kernel(Clear c) { c.part(blockIdx.x, kBlk); }

int bits_of(int m) {                     // bits of the keys 0 .. m (m >= 1)
    int b = 1;
    while (b < 31 && (m >> b) != 0) b++;
    return b;
}

// Keys of a thread in a pass: tiles of 1024 keys while they are few, so that the chip has work; of 2048 where their counts would weigh
// (lookup and gradient, four / eight: 240 000 keys 64 / 74 us, 1 048 579 keys 268 / 264).
int rounds_of(int n) { return n <= (1 << 19) ? 4 : 8; }
int tiles_of(int n) { return (int)PVX_CDIV((long long)n, (long long)rounds_of(n) * kBlk); }

struct SortWs { int2 *even, *odd; int *hist, *totals; };

template <typename C> void carve_sort(C& cv, int n, SortWs* w) {
    const bool many = n > kOneMax;
    w->even = cv.template take<int2>(many ? n : 0);
    w->odd = cv.template take<int2>(many ? n : 0);
    w->hist = cv.template take<int>(many ? (size_t)tiles_of(n) << kMaxBits : 0);
    w->totals = cv.template take<int>(many ? (size_t)1 << kMaxBits : 0);
}

// Counts that every scatter workgroup adds up itself rather than leave them to a launch between: the GPU's time is the same (49 us for
// 30 000 keys either way) and the host has two launches fewer; more counts cost time (240 000 keys 64 -> 80 us).
constexpr int kOwnScan = 1 << 14;

template <typename I>
int sort_pass(const I* in, int n, int m, int shift, int bits, bool last, const SortWs& w, int2* out, int* keys, int* order, const Clear& clear,
              hipStream_t st) {
    const int tiles = tiles_of(n), digits = 1 << bits;
    const bool own = (long long)tiles * digits <= kOwnScan;
    const size_t lds = sizeof(int) * ((size_t)digits * (kBlk / 64) + kBlk / 64);
    const int by_tile = own ? digits : 1, by_digit = own ? 1 : tiles;
    const int* totals = own ? nullptr : w.totals;
#define SORT_PASS(R)                                                                                                                             \
    do {                                                                                                                                         \
        hipLaunchKernelGGL((sort_count_kernel<I, R>), dim3(tiles + clear.blocks), dim3(kBlk), sizeof(int) * digits, st, in, n, m, shift, bits,   \
                           by_tile, by_digit, w.hist, tiles, clear);                                                                             \
        PVX_CHECK_LAUNCH();                                                                                                                      \
        if (!own) {                                                                                                                              \
            hipLaunchKernelGGL(sort_scan_kernel, dim3(digits), dim3(64), 0, st, w.hist, tiles, w.totals);                                        \
            PVX_CHECK_LAUNCH();                                                                                                                  \
        }                                                                                                                                        \
        if (last)                                                                                                                                \
            hipLaunchKernelGGL((sort_scatter_kernel<I, R, true>), dim3(tiles), dim3(kBlk), lds, st, in, n, m, shift, bits, tiles, w.hist, totals, \
                               out, keys, order);                                                                                                \
        else                                                                                                                                     \
            hipLaunchKernelGGL((sort_scatter_kernel<I, R, false>), dim3(tiles), dim3(kBlk), lds, st, in, n, m, shift, bits, tiles, w.hist,       \
                               totals, out, keys, order);                                                                                        \
        PVX_CHECK_LAUNCH();                                                                                                                      \
    } while (0)
    if (rounds_of(n) == 4) SORT_PASS(4);
    else SORT_PASS(8);
    return PVX_OK;
}

template <typename I>
int sort_impl(const I* index, int n, int m, int* order, int* keys, int* offsets, const SortWs& w, const Clear& clear, hipStream_t st) {
    const int total_bits = bits_of(m);
    if (n <= kOneMax) {
        const bool inside = offsets && m <= 2 * kOneMax;       // few rows: the same workgroup writes their offsets
        hipLaunchKernelGGL((sort_one_kernel<I>), dim3(1 + clear.blocks), dim3(kOneBlk), 0, st, index, n, m, total_bits, order, keys,
                           inside ? offsets : (int*)nullptr, clear);
        PVX_CHECK_LAUNCH();
        if (inside) return PVX_OK;
    } else {
        const int passes = PVX_CDIV(total_bits, kMaxBits);
        for (int p = 0, shift = 0; p < passes; p++) {
            const int bits = PVX_CDIV(total_bits - shift, passes - p);
            int2 *in = p % 2 ? w.even : w.odd, *out = p % 2 ? w.odd : w.even;
            const int rc = p == 0 ? sort_pass<I>(index, n, m, shift, bits, p == passes - 1, w, out, keys, order, clear, st)
                                  : sort_pass<int2>(in, n, m, shift, bits, p == passes - 1, w, out, keys, order, Clear{}, st);
            if (rc != PVX_OK) return rc;
            shift += bits;
        }
    }
    if (!offsets) return PVX_OK;
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

// log2 of a block's positions: shorter blocks where there are few, so that the chip has work.  Lookup and gradient with blocks chosen / of
// 64: 5000 x 64 29 / 38 us, 30 000 x 32 37 / 46, 240 000 x 32 58 / 64 (binary32), 100 000 x 64 bf16 50 / 61; with another threshold
// 500 000 x 64 117 (2^18) and 122 (2^19), 240 000 x 32 58 (2^18) and 63 (2^16); with blocks down to 8, 20 000 x 16 30 / 33.
int fan_of(int n, int width) {
    int fan = 6;
    while (fan > 4 && (long long)(n >> fan) * width < (1 << 18)) fan--;
    return fan;
}

// level 1 has a block for every begun 2^fan positions, the others for whole ones
int blocks_of(int n, int fan, int level) { return level == 0 ? PVX_CDIV(n, 1 << fan) : (int)((long long)n >> (fan * (level + 1))); }

template <typename C> Levels carve_levels(C& cv, int n, int width, float** out, float** tail) {
    const int fan = fan_of(n, width);
    Levels lv;
    lv.n = 0;
    for (int l = 0; l < kLevels; l++) {
        const bool worth = l == 0 ? n > 1 << fan : lv.n == l && blocks_of(n, fan, l - 1) >= kWorth;
        out[l] = worth ? cv.template take<float>((size_t)blocks_of(n, fan, l) * width) : nullptr;
        lv.p[l] = out[l];
        if (worth) lv.n = l + 1;
    }
    *tail = lv.n > 0 ? cv.template take<float>((size_t)blocks_of(n, fan, 0) * width) : nullptr;
    lv.tail = *tail;
    return lv;
}

// workgroups of `threads`, four pieces of 16 bytes a thread and no more than are resident several times
Clear clear_of(void* p, long long bytes, int threads) {
    const long long want = PVX_CDIV(bytes, 16LL * threads * 4), most = (1 << 20) / threads;
    return Clear{(char*)p, bytes, (int)(want > most ? most : want)};
}

// workgroups for `rows` rows of `ch` chunks, `each` of them a thread
dim3 grid_for(long long rows, int ch, int each) {
    const long long slots = kBlk / (ch < kBlk ? ch : kBlk), blocks = PVX_CDIV(rows, slots * each);
    return dim3((unsigned)(blocks < 1 ? 1 : (blocks > 65536 ? 65536 : blocks)));
}

template <typename E, int V>
int grad_impl(const E* dout, const int* order, const int* keys, int n, int m, int width, float scale, E* dtable, float** part, float* tail,
              const Levels& lv, hipStream_t st) {
    const int ch = width / V;
    const int fan = fan_of(n, width), blocks = blocks_of(n, fan, 0);
    hipLaunchKernelGGL((run_sum_kernel<E, V>), grid_for(blocks, ch, 1), dim3(kBlk), 0, st, dout, order, keys, n, m, ch, blocks, fan, scale,
                       part[0], tail, dtable);
    PVX_CHECK_LAUNCH();
    if (blocks == 1) return PVX_OK;
    for (int l = 1; l < lv.n; l++) {
        hipLaunchKernelGGL(run_next_kernel, grid_for(blocks_of(n, fan, l), width, 1), dim3(kBlk), 0, st, part[l - 1], keys, m, width,
                           blocks_of(n, fan, l), fan, fan * (l + 1), part[l]);
        PVX_CHECK_LAUNCH();
    }
    hipLaunchKernelGGL((run_join_kernel<E, V>), grid_for(blocks - 1, ch, 1), dim3(kBlk), 0, st, keys, n, m, ch, blocks, fan, lv, scale, dtable);
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
int grad_dispatch(const void* dout, const int* order, const int* keys, int n, int m, int width, float scale, void* dtable, float** part, float* tail, const Levels& lv, int v, hipStream_t st) {
#define LK_GRAD(E, V) grad_impl<E, V>((const E*)dout, order, keys, n, m, width, scale, (E*)dtable, part, tail, lv, st)
    LK_DISPATCH(E, v, LK_GRAD);
}

// A thread takes four rows where there are rows enough (four / one: 1000 x 64 binary32 5.9 / 4.6 us, 20 000 x 64 5.2 / 5.5, 60 000 x 32
// 5.4 / 6.1, 240 000 x 32 10 / 13, 1 048 579 x 128 bf16 80 / 107).
template <typename E, int V>
int lookup_impl(const E* table, const void* index, int index64, int n, int m, int width, float scale, E* out, hipStream_t st) {
    const int ch = width / V;
    const dim3 grid = grid_for(n, ch, n >= 16384 ? 4 : 1);
    if (index64) hipLaunchKernelGGL((lookup_kernel<E, V, long long>), grid, dim3(kBlk), 0, st, table, (const long long*)index, n, ch, m, scale, out);
    else hipLaunchKernelGGL((lookup_kernel<E, V, int>), grid, dim3(kBlk), 0, st, table, (const int*)index, n, ch, m, scale, out);
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
    return shim.s.total() + 256;
}

extern "C" int pvx_sort_index(const void* index, int index64, int n, int m, int* order, int* keys, int* offsets, void* workspace,
                              size_t workspace_bytes, void* stream) {
    if (n < 0 || m <= 0 || (n > 0 && (!index || !order || !keys))) return PVX_ERR_INVALID;
    if (n > kMaxRows || m > kMaxRows) return PVX_ERR_RANGE;
    hipStream_t st = (hipStream_t)stream;
    if (n == 0) {
        if (!offsets) return PVX_OK;
        hipLaunchKernelGGL(fill_int_kernel, dim3((unsigned)PVX_CDIV((long long)m + 1, (long long)kBlk)), dim3(kBlk), 0, st, offsets, (long long)m + 1, 0);
        PVX_CHECK_LAUNCH();
        return PVX_OK;
    }
    PvxCarver cv(workspace, workspace_bytes);
    SortWs w;
    carve_sort(cv, n, &w);
    if (!cv.ok()) return PVX_ERR_WORKSPACE;
    if (index64) return sort_impl<long long>((const long long*)index, n, m, order, keys, offsets, w, Clear{}, st);
    return sort_impl<int>((const int*)index, n, m, order, keys, offsets, w, Clear{}, st);
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

extern "C" size_t pvx_lookup_rows_grad_workspace_bytes(int n, int width, int sorted) {
    if (n <= 0 || width <= 0) return 256;
    SizerShim shim;
    float *part[kLevels], *tail;
    SortWs w;
    carve_levels(shim, n, width, part, &tail);
    if (!sorted) {
        shim.take<int>(n);
        shim.take<int>(n);
        carve_sort(shim, n, &w);
    }
    return shim.s.total() + 256;
}

extern "C" int pvx_lookup_rows_grad(const void* dout, int dtype, const void* index, int index64, const int* order, const int* keys, int n, int m,
                                    int width, float scale, void* dtable, void* workspace, size_t workspace_bytes, void* stream) {
    if (n < 0 || m < 0 || width < 0 || dtype < PVX_F32 || dtype > PVX_BF16) return PVX_ERR_INVALID;
    if (m == 0 || width == 0) return PVX_OK;
    if (!dtable || !order != !keys || (n > 0 && (!dout || (!order && !index)))) return PVX_ERR_INVALID;
    if (n > kMaxRows || m > kMaxRows || width > (1 << 24)) return PVX_ERR_RANGE;
    PvxCarver cv(workspace, workspace_bytes);
    float *part[kLevels], *tail;
    const Levels lv = carve_levels(cv, n, width, part, &tail);
    hipStream_t st = (hipStream_t)stream;
    const Clear clear = clear_of(dtable, (long long)m * width * (dtype == PVX_F32 ? 4 : 2), !order && n > 0 && n <= kOneMax ? kOneBlk : kBlk);
    if (!order && n > 0) {
        int *own = cv.take<int>(n), *own_keys = cv.take<int>(n);
        SortWs w;
        carve_sort(cv, n, &w);
        if (!cv.ok()) return PVX_ERR_WORKSPACE;
        const int rc = index64 ? sort_impl<long long>((const long long*)index, n, m, own, own_keys, nullptr, w, clear, st)
                               : sort_impl<int>((const int*)index, n, m, own, own_keys, nullptr, w, clear, st);
        if (rc != PVX_OK) return rc;
        order = own;
        keys = own_keys;
    } else {
        if (!cv.ok()) return PVX_ERR_WORKSPACE;
        hipLaunchKernelGGL(clear_kernel, dim3(clear.blocks), dim3(kBlk), 0, st, clear);
        PVX_CHECK_LAUNCH();
        if (n == 0) return PVX_OK;
    }
    const int v = vector_of(width, dtype, {dout, dtable});
    if (dtype == PVX_F32) return grad_dispatch<float>(dout, order, keys, n, m, width, scale, dtable, part, tail, lv, v, st);
    if (dtype == PVX_F16) return grad_dispatch<_Float16>(dout, order, keys, n, m, width, scale, dtable, part, tail, lv, v, st);
    return grad_dispatch<__bf16>(dout, order, keys, n, m, width, scale, dtable, part, tail, lv, v, st);
}
