// Newton-Schulz orthogonalisation of weight updates, many matrices in one call.
//
// For each matrix M (transposed if it has more rows than columns, so X is m x n with m <= n):
//   X = M / (|M|_F + eps);   steps times:  A = X X^T,  B = b A + c A A,  X <- a X + B X
// which applies the odd polynomial a s + b s^3 + c s^5 to every singular value.
//
// The products run on the bf16 matrix cores with the operands split into bf16 planes: x = x0 + x1 (+ x2), each plane the rounding of
// what the ones before it left.  binary32 matrices take three planes (24 bits) and the six products of total order <= 2, 16-bit
// ones two planes and three products (2^-17 relative, far under their own rounding), accumulated in binary32.  The binary32 matrix
// instruction would do one product at 1/16 of the bf16 rate; six at the full one are 2.7 times faster.  X is kept as planes, which
// is what the next product reads, and so are A and B; nothing is rounded to fewer bits than the planes hold.
//
// Every product is written as C[i][j] = sum_k L[i][k] R[j][k] with both operands contiguous in k: X X^T and A A (A is symmetric)
// are of that form, B X takes X^T, so the product that makes X leaves X^T beside it.  A and B are symmetric: only tiles on or below the
// diagonal are computed.  Buffers are padded with zeros to whole tiles, which the products reproduce.
#include "pvx_common.h"

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

constexpr int kBlk = 256, kBK = 32, kMaxMats = 64, kNormBlocks = 64, kNormChunk = 16384;

struct Mat {
    const void* in;
    void* out;
    long long base;                      // byte offset of this matrix's buffers in the workspace
    int m, n, mp, np;                    // m <= n; mp, np padded to tiles
    int tall, splits;                    // in / out are n x m; parts of the sum of X X^T
};

struct Table {
    Mat mat[kMaxMats];
    int first[kMaxMats + 1];             // first workgroup of each matrix
    int count;
};

// buffers of a matrix, in elements of bf16 from its base: X and X^T twice (read / written by turns), A, B, then the f32 parts of A and
// the f64 parts of the norm
template <int P> struct Buf {
    __bf16* base;
    size_t px, pa;                       // elements of a plane
    __device__ Buf(char* ws, const Mat& q) : base(reinterpret_cast<__bf16*>(ws + q.base)), px((size_t)q.mp * q.np), pa((size_t)q.mp * q.mp) {}
    __device__ __forceinline__ __bf16* x(int turn) const { return base + (size_t)turn * P * px; }
    __device__ __forceinline__ __bf16* xt(int turn) const { return base + (size_t)(2 + turn) * P * px; }
    __device__ __forceinline__ __bf16* a() const { return base + 4 * P * px; }
    __device__ __forceinline__ __bf16* b() const { return a() + P * pa; }
    __device__ __forceinline__ double* sums() const { return reinterpret_cast<double*>(b() + P * pa); }
    __device__ __forceinline__ float* part() const { return reinterpret_cast<float*>(sums() + kNormBlocks); }
};

__device__ __forceinline__ int matrix_of(const Table& t, int block) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= block) lo = mid; else hi = mid - 1;
    }
    return lo;
}

template <int P> __device__ __forceinline__ void split(float v, __bf16 (&s)[P]) {
#pragma unroll
    for (int p = 0; p < P; p++) {
        s[p] = (__bf16)v;
        v -= (float)s[p];
    }
}

// ---- |M|_F^2, in parts ---------------------------------------------------------------------------------------------------------
template <typename E>
__global__ __launch_bounds__(kBlk) void ns_norm_kernel(Table t, char* ws, int planes) {
    const int id = matrix_of(t, blockIdx.x), k = blockIdx.x - t.first[id], blocks = t.first[id + 1] - t.first[id];
    const Mat& q = t.mat[id];
    const size_t count = (size_t)q.m * q.n;
    const E* in = reinterpret_cast<const E*>(q.in);
    double s = 0.0;
    for (size_t i = (size_t)k * kBlk + threadIdx.x; i < count; i += (size_t)blocks * kBlk) {
        const double v = (double)(float)in[i];
        s = fma(v, v, s);
    }
    __shared__ double red[kBlk / 64];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double* sums = planes == 3 ? Buf<3>(ws, q).sums() : Buf<2>(ws, q).sums();
        sums[k] = red[0] + red[1] + red[2] + red[3];
        if (k == 0) for (int i = blocks; i < kNormBlocks; i++) sums[i] = 0.0;
    }
}

// ---- X and X^T as planes, 32 x 32 elements a workgroup ----------------------------------------------------------------------------
template <typename E, int P>
__global__ __launch_bounds__(kBlk) void ns_load_kernel(Table t, char* ws, float eps) {
    __shared__ float tile[32][33];
    __shared__ double scale;
    const int id = matrix_of(t, blockIdx.x);
    const Mat& q = t.mat[id];
    const Buf<P> buf(ws, q);
    if (threadIdx.x < 64) {
        double s = threadIdx.x < kNormBlocks ? buf.sums()[threadIdx.x] : 0.0;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
        if (threadIdx.x == 0) scale = 1.0 / (sqrt(s) + (double)eps);
    }
    const int local = blockIdx.x - t.first[id], tn = q.np / 32, i0 = (local / tn) * 32, j0 = (local % tn) * 32;
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const E* in = reinterpret_cast<const E*>(q.in);
    __syncthreads();
    for (int r = ty; r < 32; r += 8) {
        if (!q.tall) {
            const int i = i0 + r, j = j0 + tx;
            tile[r][tx] = i < q.m && j < q.n ? (float)((double)(float)in[(size_t)i * q.n + j] * scale) : 0.f;
        } else {
            const int j = j0 + r, i = i0 + tx;
            tile[tx][r] = i < q.m && j < q.n ? (float)((double)(float)in[(size_t)j * q.m + i] * scale) : 0.f;
        }
    }
    __syncthreads();
    for (int r = ty; r < 32; r += 8) {
        __bf16 s[P];
        split<P>(tile[r][tx], s);
#pragma unroll
        for (int p = 0; p < P; p++) buf.x(0)[p * buf.px + (size_t)(i0 + r) * q.np + j0 + tx] = s[p];
        split<P>(tile[tx][r], s);
#pragma unroll
        for (int p = 0; p < P; p++) buf.xt(0)[p * buf.px + (size_t)(j0 + r) * q.mp + i0 + tx] = s[p];
    }
}

// ---- the product ------------------------------------------------------------------------------------------------------------------
enum { kGram = 0, kPoly = 1, kApply = 2 };

// row and column of tile `l` of the lower triangle
__device__ __forceinline__ void triangle(int l, int& i, int& j) {
    i = (int)((sqrtf(8.f * (float)l + 1.f) - 1.f) * 0.5f);
    while ((i + 1) * (i + 2) / 2 <= l) i++;
    while (i * (i + 1) / 2 > l) i--;
    j = l - i * (i + 1) / 2;
}

// A workgroup of four waves computes a T x T tile, each wave (T / 2) x (T / 2) in 32 x 32 x 16 instructions.  k goes in steps of 32: the
// planes of the next step are on their way to registers while this one's are multiplied from LDS.  A row of a step is 64 bytes, four
// 16-byte pieces; the piece c of row r lies at c ^ (r / 4 mod 4), which spreads sixteen rows over all banks.
template <typename E, int P, int T, int MODE>
__global__ __launch_bounds__(kBlk) void ns_product_kernel(Table t, char* ws, int cur, int last, float fa, float fb, float fc) {
    constexpr int Q = T / 64, N = T / 64;                // staging rounds; 32 x 32 blocks of a wave along each side
    __shared__ u32x4 lds[2][P][T][4];
    const int id = matrix_of(t, blockIdx.x);
    const Mat& q = t.mat[id];
    const Buf<P> buf(ws, q);
    int local = blockIdx.x - t.first[id], ti, tj, k0 = 0, k1, part = 0;
    const __bf16 *L, *R;
    size_t pl, pr;
    int ld;
    if (MODE == kGram) {
        part = local % q.splits;
        local /= q.splits;
        triangle(local, ti, tj);
        const int steps = PVX_CDIV(q.n, kBK), per = PVX_CDIV(steps, q.splits);
        k0 = part * per * kBK;
        k1 = min(steps, (part + 1) * per) * kBK;
        L = R = buf.x(cur);
        pl = pr = buf.px;
        ld = q.np;
    } else if (MODE == kPoly) {
        triangle(local, ti, tj);
        k1 = PVX_CDIV(q.m, kBK) * kBK;
        L = R = buf.a();
        pl = pr = buf.pa;
        ld = q.mp;
    } else {
        const int tn = q.np / T;
        ti = local / tn;
        tj = local % tn;
        k1 = PVX_CDIV(q.m, kBK) * kBK;
        L = buf.b();
        R = buf.xt(cur);
        pl = buf.pa;
        pr = buf.px;
        ld = q.mp;
    }
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int srow = tid >> 2, sc = tid & 3;
    const __bf16* gl = L + (size_t)(ti * T + srow) * ld + sc * 8;
    const __bf16* gr = R + (size_t)(tj * T + srow) * ld + sc * 8;
    u32x4 nl[P][Q], nr[P][Q];
#define NS_FETCH(k)                                                                                                    \
    _Pragma("unroll") for (int p = 0; p < P; p++) _Pragma("unroll") for (int r = 0; r < Q; r++) {                      \
        nl[p][r] = *reinterpret_cast<const u32x4*>(gl + p * pl + (size_t)r * 64 * ld + (k));                           \
        nr[p][r] = *reinterpret_cast<const u32x4*>(gr + p * pr + (size_t)r * 64 * ld + (k));                           \
    }
    f32x16 acc[N][N];
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int j = 0; j < N; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][j][e] = 0.f;
    const int wi = (wave >> 1) * (T / 2), wj = (wave & 1) * (T / 2), fr = lane & 31, fh = lane >> 5;
    if (k0 < k1) { NS_FETCH(k0) }
    for (int k = k0; k < k1; k += kBK) {
        __syncthreads();
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int r = 0; r < Q; r++) {
                const int row = r * 64 + srow, at = sc ^ ((row >> 2) & 3);
                lds[0][p][row][at] = nl[p][r];
                lds[1][p][row][at] = nr[p][r];
            }
        __syncthreads();
        if (k + kBK < k1) { NS_FETCH(k + kBK) }
#pragma unroll
        for (int h = 0; h < kBK / 16; h++) {
            bf16x8 fl[P][N], fg[P][N];
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int rl = wi + i * 32 + fr, rr = wj + i * 32 + fr, c = h * 2 + fh;
#pragma unroll
                for (int p = 0; p < P; p++) {
                    fl[p][i] = __builtin_bit_cast(bf16x8, lds[0][p][rl][c ^ ((rl >> 2) & 3)]);
                    fg[p][i] = __builtin_bit_cast(bf16x8, lds[1][p][rr][c ^ ((rr >> 2) & 3)]);
                }
            }
#pragma unroll
            for (int o = P - 1; o >= 0; o--)             // smallest products first
#pragma unroll
                for (int p = 0; p <= o; p++)
#pragma unroll
                    for (int i = 0; i < N; i++)
#pragma unroll
                        for (int j = 0; j < N; j++)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fl[p][i], fg[o - p][j], acc[i][j], 0, 0, 0);
        }
    }
    // a lane holds column j = lane % 32 and rows 8 g + 4 (lane / 32) + 0 .. 3 of each 32 x 32 block
    if (MODE == kGram) {
        const int tiles = (q.mp / T) * (q.mp / T + 1) / 2;
        float* out = buf.part() + ((size_t)part * tiles + local) * T * T;
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int j = 0; j < N; j++)
#pragma unroll
                for (int e = 0; e < 16; e++)
                    out[(wi + i * 32 + 8 * (e >> 2) + 4 * fh + (e & 3)) * T + wj + j * 32 + fr] = acc[i][j][e];
        return;
    }
    const __bf16* old = MODE == kPoly ? buf.a() : buf.xt(cur);
    __bf16* direct = MODE == kPoly ? buf.b() : buf.x(cur ^ 1);
    __bf16* mirror = MODE == kPoly ? buf.b() : buf.xt(cur ^ 1);
    const int ldd = MODE == kPoly ? q.mp : q.np;
    E* out = reinterpret_cast<E*>(q.out);
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int j = 0; j < N; j++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const int row = ti * T + wi + i * 32 + 8 * g + 4 * fh, col = tj * T + wj + j * 32 + fr;
                const size_t at = (size_t)col * q.mp + row;      // the old value, read from the mirrored side: four rows at once
                float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int p = P - 1; p >= 0; p--) {
                    const bf16x4 o = *reinterpret_cast<const bf16x4*>(old + p * pr + at);
#pragma unroll
                    for (int e = 0; e < 4; e++) v[e] += (float)o[e];
                }
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = MODE == kPoly ? fb * v[e] + fc * acc[i][j][4 * g + e] : fa * v[e] + acc[i][j][4 * g + e];
                if (MODE == kApply && last) {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (row + e < q.m && col < q.n) out[q.tall ? (size_t)col * q.m + row + e : (size_t)(row + e) * q.n + col] = (E)v[e];
                    continue;
                }
                __bf16 s[4][P];
#pragma unroll
                for (int e = 0; e < 4; e++) split<P>(v[e], s[e]);
#pragma unroll
                for (int p = 0; p < P; p++) {
                    bf16x4 o;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        o[e] = s[e][p];
                        direct[p * pr + (size_t)(row + e) * ldd + col] = s[e][p];
                    }
                    if (MODE == kApply || ti != tj) *reinterpret_cast<bf16x4*>(mirror + p * pr + at) = o;
                }
            }
}

// A as planes, both triangles, from the parts of the sum in order; a workgroup takes a 32 x 32 block of a tile
template <int P, int T>
__global__ __launch_bounds__(kBlk) void ns_gather_kernel(Table t, char* ws) {
    __shared__ float tile[32][33];
    constexpr int kSub = (T / 32) * (T / 32);
    const int id = matrix_of(t, blockIdx.x);
    const Mat& q = t.mat[id];
    const Buf<P> buf(ws, q);
    const int local = blockIdx.x - t.first[id], l = local / kSub, si = (local % kSub) / (T / 32) * 32, sj = (local % kSub) % (T / 32) * 32;
    int ti, tj;
    triangle(l, ti, tj);
    const size_t tiles = (size_t)(q.mp / T) * (q.mp / T + 1) / 2;
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    for (int r = ty; r < 32; r += 8) {
        float v = 0.f;
        for (int s = 0; s < q.splits; s++) v += buf.part()[(s * tiles + l) * T * T + (si + r) * T + sj + tx];
        tile[r][tx] = v;
        __bf16 o[P];
        split<P>(v, o);
#pragma unroll
        for (int p = 0; p < P; p++) buf.a()[p * buf.pa + (size_t)(ti * T + si + r) * q.mp + tj * T + sj + tx] = o[p];
    }
    if (ti == tj) return;                                // the diagonal tile is whole already
    __syncthreads();
    for (int r = ty; r < 32; r += 8) {
        __bf16 o[P];
        split<P>(tile[tx][r], o);
#pragma unroll
        for (int p = 0; p < P; p++) buf.a()[p * buf.pa + (size_t)(tj * T + sj + r) * q.mp + ti * T + si + tx] = o[p];
    }
}

// steps == 0: the scaled matrix itself
template <typename E, int P>
__global__ __launch_bounds__(kBlk) void ns_store_kernel(Table t, char* ws) {
    const int id = matrix_of(t, blockIdx.x);
    const Mat& q = t.mat[id];
    const Buf<P> buf(ws, q);
    const size_t i = (size_t)(blockIdx.x - t.first[id]) * kBlk + threadIdx.x;
    if (i >= (size_t)q.m * q.n) return;
    const int w = q.tall ? q.m : q.n;
    const size_t r = i / w, c = i % w;
    float v = 0.f;
    for (int p = P - 1; p >= 0; p--) v += (float)(q.tall ? buf.xt(0)[p * buf.px + r * q.mp + c] : buf.x(0)[p * buf.px + r * q.np + c]);
    reinterpret_cast<E*>(q.out)[i] = (E)v;
}

int round_up(int v, int to) { return PVX_CDIV(v, to) * to; }

int planes_of(int dtype) { return dtype == PVX_F32 ? 3 : 2; }

// 128 x 128 tiles where the largest product has enough of them for the chip, 64 x 64 otherwise
int tile_of(const pvx_matrix* mats, int count) {
    long long tiles = 0;
    for (int i = 0; i < count; i++) tiles += (long long)PVX_CDIV(mats[i].rows, 128) * PVX_CDIV(mats[i].cols, 128);
    return tiles >= 256 ? 128 : 64;
}

constexpr int kPartWorkgroups = 512;

void fill(Table& t, const pvx_matrix* mats, int count, int tile, int planes, size_t* total) {
    t.count = count;
    size_t off = 0;
    long long tiles = 0;
    for (int i = 0; i < count; i++) {
        Mat& q = t.mat[i];
        q.in = mats[i].in;
        q.out = mats[i].out;
        q.tall = mats[i].rows > mats[i].cols;
        q.m = q.tall ? mats[i].cols : mats[i].rows;
        q.n = q.tall ? mats[i].rows : mats[i].cols;
        q.mp = round_up(q.m, tile);
        q.np = round_up(q.n, tile);
        tiles += (long long)(q.mp / tile) * (q.mp / tile + 1) / 2;
    }
    // the sum over n is cut where the batch has fewer tiles than fill the chip; a part keeps at least four steps
    const int want = (int)PVX_CDIV((long long)kPartWorkgroups, tiles < 1 ? 1 : tiles);
    for (int i = 0; i < count; i++) {
        Mat& q = t.mat[i];
        const int most = PVX_CDIV(PVX_CDIV(q.n, kBK), 4);
        q.splits = want < most ? want : most;
        q.base = (long long)off;
        const size_t px = (size_t)q.mp * q.np, pa = (size_t)q.mp * q.mp, lower = (size_t)(q.mp / tile) * (q.mp / tile + 1) / 2 * tile * tile;
        off += pvx_align_up((size_t)planes * 2 * (4 * px + 2 * pa) + sizeof(double) * kNormBlocks + sizeof(float) * lower * q.splits, 256);
    }
    *total = off;
}

template <typename F> int spread(Table& t, F blocks) {
    long long at = 0;
    for (int i = 0; i < t.count; i++) {
        t.first[i] = (int)at;
        at += blocks(t.mat[i]);
        if (at > 0x7fffffffLL) return -1;
    }
    t.first[t.count] = (int)at;
    return (int)at;
}

template <typename E, int P, int T>
int run(Table& t, char* ws, int steps, float a, float b, float c, float eps, hipStream_t st) {
    auto lower = [](const Mat& q) { return (long long)(q.mp / T) * (q.mp / T + 1) / 2; };
#define NS_LAUNCH(kernel, blocks_of, ...)                                                      \
    do {                                                                                       \
        const int blocks__ = spread(t, blocks_of);                                             \
        if (blocks__ < 0) return PVX_ERR_RANGE;                                                \
        hipLaunchKernelGGL(kernel, dim3(blocks__), dim3(kBlk), 0, st, t, ws, ##__VA_ARGS__);    \
        PVX_CHECK_LAUNCH();                                                                    \
    } while (0)
    auto norm_blocks = [](const Mat& q) {
        const long long k = PVX_CDIV((long long)q.m * q.n, (long long)kNormChunk);
        return k > kNormBlocks ? (long long)kNormBlocks : k;
    };
    NS_LAUNCH((ns_norm_kernel<E>), norm_blocks, P);
    NS_LAUNCH((ns_load_kernel<E, P>), ([](const Mat& q) { return (long long)(q.mp / 32) * (q.np / 32); }), eps);
    if (steps == 0) NS_LAUNCH((ns_store_kernel<E, P>), ([](const Mat& q) { return PVX_CDIV((long long)q.m * q.n, (long long)kBlk); }));
    for (int s = 0; s < steps; s++) {
        const int cur = s & 1, last = s == steps - 1;
        NS_LAUNCH((ns_product_kernel<E, P, T, kGram>), ([&](const Mat& q) { return lower(q) * q.splits; }), cur, last, a, b, c);
        NS_LAUNCH((ns_gather_kernel<P, T>), ([&](const Mat& q) { return lower(q) * (T / 32) * (T / 32); }));
        NS_LAUNCH((ns_product_kernel<E, P, T, kPoly>), lower, cur, last, a, b, c);
        NS_LAUNCH((ns_product_kernel<E, P, T, kApply>), ([](const Mat& q) { return (long long)(q.mp / T) * (q.np / T); }), cur, last, a, b, c);
    }
    return PVX_OK;
}

int check_args(const pvx_matrix* mats, int count, int dtype) {
    if (count < 0 || (count > 0 && !mats) || dtype < PVX_F32 || dtype > PVX_BF16) return PVX_ERR_INVALID;
    if (count > kMaxMats) return PVX_ERR_RANGE;
    for (int i = 0; i < count; i++) {
        if (mats[i].rows <= 0 || mats[i].cols <= 0) return PVX_ERR_INVALID;
        if (mats[i].rows > (1 << 20) || mats[i].cols > (1 << 20)) return PVX_ERR_RANGE;
    }
    return PVX_OK;
}

}  // namespace

extern "C" size_t pvx_orthogonalize_workspace_bytes(const pvx_matrix* mats, int count, int dtype) {
    if (check_args(mats, count, dtype) != PVX_OK || count == 0) return 256;
    Table t;
    size_t total;
    fill(t, mats, count, tile_of(mats, count), planes_of(dtype), &total);
    return total;
}

extern "C" int pvx_orthogonalize(const pvx_matrix* mats, int count, int dtype, int steps, float a, float b, float c, float eps, void* workspace,
                                 size_t workspace_bytes, void* stream) {
    const int bad = check_args(mats, count, dtype);
    if (bad != PVX_OK) return bad;
    if (steps < 0 || !(eps >= 0.f)) return PVX_ERR_INVALID;
    if (count == 0) return PVX_OK;
    for (int i = 0; i < count; i++)
        if (!mats[i].in || !mats[i].out) return PVX_ERR_INVALID;
    Table t;
    size_t total;
    const int tile = tile_of(mats, count);
    fill(t, mats, count, tile, planes_of(dtype), &total);
    if (!workspace || workspace_bytes < total || (reinterpret_cast<uintptr_t>(workspace) & 255)) return PVX_ERR_WORKSPACE;
    char* ws = reinterpret_cast<char*>(workspace);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == PVX_F32) return tile == 128 ? run<float, 3, 128>(t, ws, steps, a, b, c, eps, st) : run<float, 3, 64>(t, ws, steps, a, b, c, eps, st);
    if (dtype == PVX_F16) return tile == 128 ? run<_Float16, 2, 128>(t, ws, steps, a, b, c, eps, st) : run<_Float16, 2, 64>(t, ws, steps, a, b, c, eps, st);
    return tile == 128 ? run<__bf16, 2, 128>(t, ws, steps, a, b, c, eps, st) : run<__bf16, 2, 64>(t, ws, steps, a, b, c, eps, st);
}
