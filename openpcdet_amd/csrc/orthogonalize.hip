// Newton-Schulz orthogonalisation of weight updates, many matrices in one call.
//
// For each matrix M (transposed if it has more rows than columns, so X is m x n with m <= n):
//   X = M / (|M|_F + eps);   steps times:  A = X X^T,  B = a I + b A + c A A,  X <- B X
// which applies the odd polynomial a s + b s^3 + c s^5 to every singular value.
//
// The products run on the f16 matrix cores with each operand split in two: x = hi + lo, hi the rounding of x to 11 bits and lo that of
// the rest, 22 bits and more together, and three of the four products (lo lo is below 2^-24 of hi hi), accumulated in binary32.
// Against 64 bits this is as near as binary32 products are (1001 x 2003: 1.4e-6, binary32's 3.5e-6), at a third of the f16
// rate instead of a sixteenth of it, which is what the binary32 instruction has.  f16 has few exponents, so X, A and B are kept times
// powers of two of each matrix and step: the singular values start below |M| / (|M| + eps), the bound follows them through the
// polynomial, no entry is larger than the largest singular value, and 2^14 stands for the bound.  hi and lo share a word, so a
// matrix takes four bytes an element, as in binary32.
//
// A and B are symmetric: only tiles on or below the diagonal are computed, and both factors of A = X X^T and A A are read along k.
// B X reads X by rows of k: its fragments come out of LDS transposed (ds_read_b64_tr_b16).  Buffers are padded with zeros to whole
// tiles, which the products reproduce.
//
// Wide matrices are bound by the matrix cores: 2048 x 4096 takes 1167 to 1236 us (by card) for 926 Gflop in f16 (three products each),
// 750 to 794 Tflop/s, where the best library product of bf16 reaches 1054 (8192^3); they are busy half of the cycles, LDS 42 %.  Few or narrow ones are bound by their launches, five a step: a backbone's
// 21 layers take 172 us, of which the products are 23 a step.
#include "pvx_common.h"

#include <math.h>

namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;

constexpr int kBlk = 256, kBK = 32, kMaxMats = 64, kNormBlocks = 256, kNormChunk = 8192, kMaxSteps = 64;
// Rows up to which lo lo is added too.  There sums are short and a dropped 2^-24 is seen against binary32's own rounding; it costs 1 %
// (256 x 2304 147 us, 145 without).  Longer sums hide it, and it costs 14 % (2048 x 4096 1333 us, 1167 without).
constexpr int kWhole = 256;

struct Mat {
    const void* in;
    void* out;
    long long base;                      // byte offset of this matrix's buffers in the workspace
    int m, n, mp, np;                    // m <= n; mp, np padded to tiles
    int tall, parts, parts2;             // in / out are n x m; parts of the sums of X X^T and of A A
};

struct Table {
    Mat mat[kMaxMats];
    int first[kMaxMats + 1];             // first workgroup of each matrix
    int count;
};

// a step's factors: the polynomial's coefficients and the powers of two of what they multiply
struct Scales { float gram, poly0, poly1, poly2, apply, out; };

// buffers of a matrix: X twice (read and written by turns), A and B as words (hi, lo), the parts of the sums, those of the norm
struct Buf {
    unsigned* base;
    size_t px, pa;
    __device__ Buf(char* ws, const Mat& q) : base(reinterpret_cast<unsigned*>(ws + q.base)), px((size_t)q.mp * q.np), pa((size_t)q.mp * q.mp) {}
    __device__ __forceinline__ unsigned* x(int turn) const { return base + (size_t)turn * px; }
    __device__ __forceinline__ unsigned* a() const { return base + 2 * px; }
    __device__ __forceinline__ unsigned* b() const { return a() + pa; }
    __device__ __forceinline__ float* part() const { return reinterpret_cast<float*>(b() + pa); }
    __device__ __forceinline__ double* sums(const Mat& q, int tile) const {
        const size_t lower = (size_t)(q.mp / tile) * (q.mp / tile + 1) / 2 * tile * tile;
        return reinterpret_cast<double*>(part() + lower * max(q.parts, q.parts2));
    }
    __device__ __forceinline__ Scales* scales(const Mat& q, int tile) const { return reinterpret_cast<Scales*>(sums(q, tile) + kNormBlocks); }
};

// the matrix of a workgroup, in one load of the wave instead of a search's six
__device__ __forceinline__ int matrix_of(const Table& t, int block) {
    const int lane = threadIdx.x & 63;
    return __popcll(__ballot(lane < t.count && t.first[lane + 1] <= block));
}

__device__ __forceinline__ unsigned pack(float v) {
    f16x2 h;
    h[0] = (_Float16)v;
    h[1] = (_Float16)(v - (float)h[0]);
    return __builtin_bit_cast(unsigned, h);
}

__device__ __forceinline__ float value(unsigned w) {
    const f16x2 h = __builtin_bit_cast(f16x2, w);
    return (float)h[0] + (float)h[1];
}

// the hi halves and the lo halves of eight words
__device__ __forceinline__ void halves(u32x4 p, u32x4 q, u32x4& hi, u32x4& lo) {
    hi[0] = __builtin_amdgcn_perm(p[1], p[0], 0x05040100u);
    hi[1] = __builtin_amdgcn_perm(p[3], p[2], 0x05040100u);
    hi[2] = __builtin_amdgcn_perm(q[1], q[0], 0x05040100u);
    hi[3] = __builtin_amdgcn_perm(q[3], q[2], 0x05040100u);
    lo[0] = __builtin_amdgcn_perm(p[1], p[0], 0x07060302u);
    lo[1] = __builtin_amdgcn_perm(p[3], p[2], 0x07060302u);
    lo[2] = __builtin_amdgcn_perm(q[1], q[0], 0x07060302u);
    lo[3] = __builtin_amdgcn_perm(q[3], q[2], 0x07060302u);
}

// ---- |M|_F^2, in parts ---------------------------------------------------------------------------------------------------------
template <typename E>
__global__ __launch_bounds__(kBlk) void ns_norm_kernel(Table t, char* ws, int tile) {
    constexpr int V = 16 / (int)sizeof(E);
    struct alignas(16) Pack { E e[V]; };
    const int id = matrix_of(t, blockIdx.x), k = blockIdx.x - t.first[id], blocks = t.first[id + 1] - t.first[id];
    const Mat& q = t.mat[id];
    const size_t count = (size_t)q.m * q.n;
    const E* in = reinterpret_cast<const E*>(q.in);
    const size_t packs = (reinterpret_cast<uintptr_t>(in) & 15) == 0 ? count / V : 0;
    double s = 0.0;
#pragma unroll 4
    for (size_t i = (size_t)k * kBlk + threadIdx.x; i < packs; i += (size_t)blocks * kBlk) {
        const Pack p = reinterpret_cast<const Pack*>(in)[i];
#pragma unroll
        for (int j = 0; j < V; j++) { const double v = (double)(float)p.e[j]; s = fma(v, v, s); }
    }
    for (size_t i = packs * V + (size_t)k * kBlk + threadIdx.x; i < count; i += (size_t)blocks * kBlk) {
        const double v = (double)(float)in[i];
        s = fma(v, v, s);
    }
    __shared__ double red[kBlk / 64];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    double* sums = Buf(ws, q).sums(q, tile);
    if (threadIdx.x == 0) sums[k] = red[0] + red[1] + red[2] + red[3];
    if (k == 0 && (int)threadIdx.x >= blocks && threadIdx.x < kNormBlocks) sums[threadIdx.x] = 0.0;
}

// ---- the powers of two ----------------------------------------------------------------------------------------------------------
// What the singular values' bound r becomes in a step: the largest |f| on [0, r] of f(x) = x (a + b x^2 + c x^4), at its end or at a root
// of its derivative a + 3 b y + 5 c y^2, y = x^2.  The roots come from the host; binary32 will do: the exponents are bounds, with 1 %
// and more to spare a step.
struct Poly {
    float a, b, c;
    float x[2], f[2];                    // where |f| may have its extremes, and |f| there; 0 where there is none
    __device__ __forceinline__ float largest(float r) const {
        const float y = r * r;
        float most = fabsf(r * (a + y * (b + y * c)));
        if (x[0] < r) most = fmaxf(most, f[0]);
        if (x[1] < r) most = fmaxf(most, f[1]);
        return most;
    }
};

Poly poly_of(float a, float b, float c) {
    Poly p{a, b, c, {0.f, 0.f}, {0.f, 0.f}};
    double root[2] = {0.0, 0.0};
    if (c == 0.f) {
        if (b != 0.f) root[0] = -(double)a / (3.0 * b);
    } else {
        const double d = 9.0 * b * b - 20.0 * (double)a * c;
        if (d >= 0.0) { root[0] = (-3.0 * b + sqrt(d)) / (10.0 * c); root[1] = (-3.0 * b - sqrt(d)) / (10.0 * c); }
    }
    for (int i = 0; i < 2; i++) {
        if (!(root[i] > 0.0)) continue;
        const double x = sqrt(root[i]);
        p.x[i] = (float)x;
        p.f[i] = (float)fabs(x * (a + root[i] * (b + root[i] * c)));
    }
    return p;
}

// Whether the followed bound says enough about the values.  The largest singular value starts between 1 / 64 (4096 equal ones) and 1
// times the norm; [lo, r] is what a step makes of that range, r with the 1 % that the scales take.  f16 has 2^-39 of its bound as half
// its last step, so with r <= 128 lo an entry of A, kept against r^2, is off by at most 2^-25 of the square of the largest value: as
// binary32.  3 x - 2 x^3 shows what must not pass: the values stay below sqrt(2), at whose end the slope is -9, but 1 % more makes the
// bound 1.4, 1.6, 2.9, 39, 1e5, and everything is lost below f16's last step.  A norm near eps starts lower: 2^0, 2^-2, .. 2^-20.
// More than 4096 rows may start lower still, at 1 / sqrt(rows), down to 2^-10, beside a bound of 1.  What is accepted here has its slope a to
// within 1 % on [0, 1 / 64] (128 |f(1 / 64)| >= the largest |f| leaves |b| and |c| no more than some ten times |a|), so such a value goes
// through a I alone until it reaches the range that was followed; A's words matter beside a, not beside the value, and only X's own are
// nearer to f16's last step: off by up to 2^-28 of the largest value, at 2^20 rows, instead of 2^-32.
bool bound_holds(int steps, float a, float b, float c) {
    constexpr double kSpread = 128.0, kMost = 1e9;       // kMost: where above() ends
    const Poly p = poly_of(a, b, c);
    auto f = [&](double x) { return x * (a + x * x * (b + x * x * (double)c)); };
    for (int e = 0; e <= 20; e += 2) {
        double lo = ldexp(1.0 / 64.0, -e), r = ldexp(1.01, -e);
        for (int s = 0; s < steps; s++) {
            double at[4] = {lo, lo, lo, r};              // f is monotonic between these
            for (int i = 0; i < 2; i++)
                if (p.x[i] > lo && p.x[i] < r) at[1 + i] = p.x[i];
            if (at[1] > at[2]) { const double x = at[1]; at[1] = at[2]; at[2] = x; }
            double least = fabs(f(lo)), most = least;
            for (int i = 1; i < 4; i++) {
                const double v = f(at[i]);
                if (v * f(at[i - 1]) < 0.0) least = 0.0;
                least = fmin(least, fabs(v));
                most = fmax(most, fabs(v));
            }
            lo = least;
            r = 1.01 * most;
            if (r > kSpread * lo || r > kMost) return false;
        }
    }
    return true;
}

// the power of two above `most`, within what the scales can hold; 0 and NaN: anything will do
__device__ __forceinline__ int above(float most) {
    if (!(most > 1e-30f)) return most > 0.f ? -99 : 0;
    if (!(most < 1e9f)) return 30;
    return __builtin_amdgcn_frexp_expf(most);
}

__device__ __forceinline__ float two(int e) { return ldexpf(1.f, e); }

// X is kept times 2^(14 - above(its largest singular value)); at the start that is below nu = |M| / (|M| + eps)
__device__ __forceinline__ int start_above(float nu) { return above(1.01f * nu); }

__device__ void follow(float nu, int steps, const Poly& f, Scales* to) {
    float r = 1.01f * nu;                                // 1 % a step for what rounding adds
    int er = start_above(nu);
    for (int s = 0; s < steps; s++) {
        const int ea = 14 - 2 * er;                      // A <= 2^(2 er)
        const float y = r * r;
        const int eb = 14 - above(1.01f * (fabsf(f.a) + y * (fabsf(f.b) + y * fabsf(f.c))));
        r = 1.01f * f.largest(r);
        const int next = above(r);
        Scales k;
        k.gram = two(ea - 2 * (14 - er));
        k.poly0 = ldexpf(f.a, eb);
        k.poly1 = ldexpf(f.b, eb - ea);
        k.poly2 = ldexpf(f.c, eb - 2 * ea);
        k.apply = two(14 - next - eb - (14 - er));
        k.out = two(-eb - (14 - er));
        to[s] = k;
        er = next;
    }
}

// ---- X as words, 64 x 64 elements a workgroup -----------------------------------------------------------------------------------
template <typename E>
__global__ __launch_bounds__(kBlk) void ns_load_kernel(Table t, char* ws, int tile, float eps, int steps, Poly poly) {
    __shared__ float turn[64][65];
    __shared__ double part[kBlk / 64];
    const int id = matrix_of(t, blockIdx.x), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Mat& q = t.mat[id];
    const Buf buf(ws, q);
    static_assert(kNormBlocks == kBlk, "a thread for each part of the norm");
    double s = buf.sums(q, tile)[threadIdx.x];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
    if (lane == 0) part[wave] = s;
    __syncthreads();
    const double norm = sqrt(part[0] + part[1] + part[2] + part[3]);
    const float nu = (float)(norm / (norm + (double)eps));
    const double scale = ldexp(1.0 / (norm + (double)eps), 14 - start_above(nu));
    const int local = blockIdx.x - t.first[id], tn = q.np / 64, i0 = (local / tn) * 64, j0 = (local % tn) * 64;
    const E* in = reinterpret_cast<const E*>(q.in);
    unsigned* x = buf.x(0);
    if (local == 0 && threadIdx.x == kBlk - 1) {
        if (steps > 0) follow(nu, steps, poly, buf.scales(q, tile));
        else buf.scales(q, tile)[0].out = two(start_above(nu) - 14);
    }
    if (!q.tall) {                                       // sixteen lanes a row, four columns each
        const int j = j0 + 4 * (lane & 15);
        struct alignas(4 * sizeof(E)) Four { E e[4]; };
        const bool whole = q.n % 4 == 0 && reinterpret_cast<uintptr_t>(in) % sizeof(Four) == 0;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int i = i0 + 16 * r + 4 * wave + (lane >> 4);
            Four f;
            if (whole && i < q.m && j < q.n) f = *reinterpret_cast<const Four*>(in + (size_t)i * q.n + j);
            else {
#pragma unroll
                for (int e = 0; e < 4; e++) f.e[e] = i < q.m && j + e < q.n ? in[(size_t)i * q.n + j + e] : (E)0.f;
            }
            u32x4 o;
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = pack((float)((double)(float)f.e[e] * scale));
            *reinterpret_cast<u32x4*>(x + (size_t)i * q.np + j) = o;
        }
        return;
    }
#pragma unroll 4
    for (int r = wave; r < 64; r += 4) {
        const int j = j0 + r, i = i0 + lane;
        turn[lane][r] = i < q.m && j < q.n ? (float)((double)(float)in[(size_t)j * q.m + i] * scale) : 0.f;
    }
    __syncthreads();
#pragma unroll 4
    for (int r = wave; r < 64; r += 4) x[(size_t)(i0 + r) * q.np + j0 + lane] = pack(turn[r][lane]);
}

// ---- the products ---------------------------------------------------------------------------------------------------------------
enum { kGram = 0, kPoly = 1, kApply = 2 };

// row and column of tile `l` of the lower triangle
__device__ __forceinline__ void triangle(int l, int& i, int& j) {
    i = (int)((sqrtf(8.f * (float)l + 1.f) - 1.f) * 0.5f);
    while ((i + 1) * (i + 2) / 2 <= l) i++;
    while (i * (i + 1) / 2 > l) i--;
    j = l - i * (i + 1) / 2;
}

// A workgroup of four waves computes a T x T tile, each wave (T / 2) x (T / 2) in 32 x 32 x 16 instructions.  k goes in steps of 32: the
// words of the next step are on their way to registers while this one's halves are multiplied from LDS.  Along k a row of a step is 64
// bytes, four 16-byte pieces, and piece c of row r lies at c ^ (r / 4 mod 4), which spreads sixteen rows over all banks; across k
// (B X) a row of a step is T columns, 32 bytes apart from the next, so the four rows that a transposing read takes lie in different banks.
template <typename E, int T, int MODE>
__global__ __launch_bounds__(kBlk) void ns_product_kernel(Table t, char* ws, int step, int last) {
    constexpr int N = T / 64;                            // staging rounds; 32 x 32 blocks of a wave along each side
    constexpr int kRow = 2 * T + 32;                     // bytes of a row of k
    // LDS buffers: three workgroups on a CU with one of 128, four with two of 64 (one / two: 2048 x 4096 1167 / 1230 us, 512 x 2304 204 / 190)
    constexpr int kD = T == 128 ? 1 : 2;
    __shared__ u32x4 left[kD][2][T][4];
    __shared__ __attribute__((aligned(16))) char right[kD][2][MODE == kApply ? kBK * kRow : T * 64];
    const int id = matrix_of(t, blockIdx.x);
    const Mat& q = t.mat[id];
    const Buf buf(ws, q);
    const bool whole = q.m <= kWhole;
    int local = blockIdx.x - t.first[id], ti, tj, k0 = 0, k1, part = 0;
    const unsigned *L, *R;
    int ld, ldr;
    if (MODE == kApply) {
        const int tn = q.np / T;
        ti = local / tn;
        tj = local % tn;
        k1 = PVX_CDIV(q.m, kBK) * kBK;
        L = buf.b();
        R = buf.x(step & 1);
        ld = q.mp;
        ldr = q.np;
    } else {
        const int parts = MODE == kGram ? q.parts : q.parts2;
        part = local % parts;
        local /= parts;
        triangle(local, ti, tj);
        const int steps = PVX_CDIV(MODE == kGram ? q.n : q.m, kBK), per = PVX_CDIV(steps, parts);
        k0 = part * per * kBK;
        k1 = min(steps, (part + 1) * per) * kBK;
        L = R = MODE == kGram ? buf.x(step & 1) : buf.a();
        ld = ldr = MODE == kGram ? q.np : q.mp;
    }
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int srow = tid >> 2, spiece = tid & 3;
    const unsigned* gl = L + (size_t)(ti * T + srow) * ld + spiece * 8;
    // across k: 32 rows of T / 8 pieces
    const int arow = tid / (T / 8), apiece = tid % (T / 8);
    constexpr int kStride = kBlk / (T / 8);              // rows of k that one round of the workgroup stages
    const unsigned* gr = MODE == kApply ? R + (size_t)arow * ldr + tj * T + apiece * 8 : R + (size_t)(tj * T + srow) * ldr + spiece * 8;
    u32x4 nl[N][2], nr[N][2];
#define NS_FETCH(k)                                                                                                              \
    _Pragma("unroll") for (int r = 0; r < N; r++) {                                                                              \
        const u32x4* a__ = reinterpret_cast<const u32x4*>(gl + (size_t)r * 64 * ld + (k));                                       \
        const u32x4* b__ = reinterpret_cast<const u32x4*>(MODE == kApply ? gr + (size_t)((k) + r * kStride) * ldr                \
                                                                         : gr + (size_t)r * 64 * ldr + (k));                     \
        nl[r][0] = a__[0]; nl[r][1] = a__[1];                                                                                    \
        nr[r][0] = b__[0]; nr[r][1] = b__[1];                                                                                    \
    }
    f32x16 acc[N][N];
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int j = 0; j < N; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][j][e] = 0.f;
    const int wi = (wave >> 1) * (T / 2), wj = (wave & 1) * (T / 2), fr = lane & 31, fh = lane >> 5;
    // a transposing read: in each group of 16 lanes, lane 4 y + x names row y, columns 4 x .. 4 x + 3 of a block of 4 x 16, and lane c
    // receives column c of the four rows; groups 0 and 1 take columns 0 .. 31 of k = 0 .. 7, groups 2 and 3 those of k = 8 .. 15
    const int tr = (8 * fh + ((lane & 15) >> 2)) * kRow + (wj + 16 * ((lane >> 4) & 1) + 4 * (lane & 3)) * 2;
#define NS_STAGE(d)                                                                                                              \
    _Pragma("unroll") for (int r = 0; r < N; r++) {                                                                              \
        const int row = r * 64 + srow, at = spiece ^ ((row >> 2) & 3);                                                           \
        u32x4 hi, lo;                                                                                                            \
        halves(nl[r][0], nl[r][1], hi, lo);                                                                                      \
        left[d][0][row][at] = hi;                                                                                                \
        left[d][1][row][at] = lo;                                                                                                \
        halves(nr[r][0], nr[r][1], hi, lo);                                                                                      \
        const int to = MODE == kApply ? (arow + r * kStride) * kRow + apiece * 16 : row * 64 + at * 16;                          \
        *reinterpret_cast<u32x4*>(&right[d][0][to]) = hi;                                                                        \
        *reinterpret_cast<u32x4*>(&right[d][1][to]) = lo;                                                                        \
    }
    if (k0 < k1) { NS_FETCH(k0) }
    if (kD == 2 && k0 < k1) {
        NS_STAGE(0)
        if (k0 + kBK < k1) { NS_FETCH(k0 + kBK) }
    }
    int buf_at = 0;
    for (int k = k0; k < k1; k += kBK) {
        __syncthreads();
        if (kD == 1) {
            NS_STAGE(0)
            __syncthreads();
            if (k + kBK < k1) { NS_FETCH(k + kBK) }
        }
        const int d = kD == 2 ? buf_at : 0;
#pragma unroll
        for (int h = 0; h < kBK / 16; h++) {
            f16x8 fl[2][N], fg[2][N];
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int rl = wi + i * 32 + fr, rr = wj + i * 32 + fr, c = h * 2 + fh;
#pragma unroll
                for (int p = 0; p < 2; p++) {
                    fl[p][i] = __builtin_bit_cast(f16x8, left[d][p][rl][c ^ ((rl >> 2) & 3)]);
                    if (MODE == kApply) {
                        char* at = &right[d][p][tr + h * 16 * kRow + i * 64];
                        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)at);
                        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at + 4 * kRow));
                        fg[p][i] = __builtin_bit_cast(f16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
                    } else {
                        fg[p][i] = *reinterpret_cast<const f16x8*>(&right[d][p][rr * 64 + (c ^ ((rr >> 2) & 3)) * 16]);
                    }
                }
            }
            if (whole) {
#pragma unroll
                for (int i = 0; i < N; i++)
#pragma unroll
                    for (int j = 0; j < N; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fl[1][i], fg[1][j], acc[i][j], 0, 0, 0);
            }
#pragma unroll
            for (int o = 0; o < 3; o++)                  // lo hi, hi lo, hi hi: smallest first
#pragma unroll
                for (int i = 0; i < N; i++)
#pragma unroll
                    for (int j = 0; j < N; j++)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fl[o == 0 ? 1 : 0][i], fg[o == 1 ? 1 : 0][j], acc[i][j], 0, 0, 0);
        }
        if (kD == 2) {
            buf_at ^= 1;
            if (k + kBK < k1) {
                NS_STAGE(buf_at)
                if (k + 2 * kBK < k1) { NS_FETCH(k + 2 * kBK) }
            }
        }
    }
    // a lane holds column j = lane % 32 and rows 8 g + 4 (lane / 32) + 0 .. 3 of each 32 x 32 block
    const size_t tiles = (size_t)(q.mp / T) * (q.mp / T + 1) / 2;
    float* sum = buf.part() + ((size_t)part * tiles + local) * T * T;
    unsigned* x = buf.x((step & 1) ^ 1);
    E* out = reinterpret_cast<E*>(q.out);
    float scale = 1.f;
    if (MODE == kApply) {
        const Scales& k = buf.scales(q, T)[step];
        scale = last ? k.out : k.apply;
    }
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int j = 0; j < N; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int ri = wi + i * 32 + 8 * (e >> 2) + 4 * fh + (e & 3), cj = wj + j * 32 + fr;
                const float v = acc[i][j][e];
                if (MODE != kApply) {
                    sum[ri * T + cj] = v;
                } else if (last) {
                    const int row = ti * T + ri, col = tj * T + cj;
                    if (row < q.m && col < q.n) out[q.tall ? (size_t)col * q.m + row : (size_t)row * q.n + col] = (E)(v * scale);
                } else {
                    x[(size_t)(ti * T + ri) * q.np + tj * T + cj] = pack(v * scale);
                }
            }
}

// The parts of a sum of the lower tiles, in order, to words of the whole symmetric matrix: A, or B = a I + b A + c (the sum).  A
// workgroup takes a 32 x 32 block of a tile, a thread four columns of a row.
template <int T, int MODE>
__global__ __launch_bounds__(kBlk) void ns_gather_kernel(Table t, char* ws, int step) {
    __shared__ unsigned turn[32][33];
    constexpr int kSide = T / 32;
    const int id = matrix_of(t, blockIdx.x);
    const Mat& q = t.mat[id];
    const Buf buf(ws, q);
    const int local = blockIdx.x - t.first[id], l = local / (kSide * kSide), sub = local % (kSide * kSide);
    const int si = sub / kSide * 32, sj = sub % kSide * 32;
    int ti, tj;
    triangle(l, ti, tj);
    const size_t tiles = (size_t)(q.mp / T) * (q.mp / T + 1) / 2;
    const int r = threadIdx.x >> 3, c = (threadIdx.x & 7) * 4, parts = MODE == kGram ? q.parts : q.parts2;
    const int row = ti * T + si + r, col = tj * T + sj + c;
    const f32x4* in = reinterpret_cast<const f32x4*>(buf.part() + (size_t)l * T * T + (si + r) * T + sj + c);
    const size_t apart = tiles * T * T / 4;
    const Scales sc = buf.scales(q, T)[step];
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int s = 0; s < parts; s++) v += in[s * apart];
    if (MODE == kGram) {
        v *= sc.gram;
    } else {
        const u32x4 w = *reinterpret_cast<const u32x4*>(buf.a() + (size_t)row * q.mp + col);
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = sc.poly2 * v[e] + sc.poly1 * value(w[e]) + (row == col + e ? sc.poly0 : 0.f);
    }
    unsigned* to = MODE == kGram ? buf.a() : buf.b();
    u32x4 o;
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] = pack(v[e]);
    *reinterpret_cast<u32x4*>(to + (size_t)row * q.mp + col) = o;
    if (ti == tj) return;                                // a diagonal tile is whole already
#pragma unroll
    for (int e = 0; e < 4; e++) turn[c + e][r] = o[e];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] = turn[r][c + e];
    *reinterpret_cast<u32x4*>(to + (size_t)(tj * T + sj + r) * q.mp + ti * T + si + c) = o;
}

// steps == 0: the scaled matrix itself
template <typename E>
__global__ __launch_bounds__(kBlk) void ns_store_kernel(Table t, char* ws, int tile) {
    const int id = matrix_of(t, blockIdx.x);
    const Mat& q = t.mat[id];
    const Buf buf(ws, q);
    const size_t i = (size_t)(blockIdx.x - t.first[id]) * kBlk + threadIdx.x;
    if (i >= (size_t)q.m * q.n) return;
    const int w = q.tall ? q.m : q.n;
    const size_t r = i / w, c = i % w;
    reinterpret_cast<E*>(q.out)[i] = (E)(value(buf.x(0)[q.tall ? c * q.np + r : r * q.np + c]) * buf.scales(q, tile)[0].out);
}

// ---- small matrices: everything in one workgroup ------------------------------------------------------------------------------------
// X stays in LDS as binary32 and takes the binary32 matrix instruction (16 x 16 x 4): at 16 x 432 the products are nothing and the 27
// launches of the general form take 105 us, this one 17; 32 x 700 95 and 54, 24 such layers together 110 and 50.  Rows lie 4 words apart modulo 64, so 16 rows x 4 words touch every bank once.  The sum over
// k runs in any order, so a lane reads four consecutive k at once and gives one to each of four instructions.
constexpr int kSmallBlk = 1024, kSmallWaves = kSmallBlk / 64, kSmallWords = 32 * 772;
constexpr int small_width(int rows) { return (kSmallWords / rows - 4) / 64 * 64; }      // 1536 columns of 16 rows, 768 of 32

template <typename E, int MP>
__device__ __forceinline__ void small_body(const Mat& q, int steps, float ca, float cb, float cc, float eps, float* x, float* part, float* a, float* b,
                                           double* red) {
    constexpr int T = MP / 16, kTiles = T * (T + 1) / 2, kLdA = MP + 4;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lr = lane & 15, lq = lane >> 4;
    const int m = q.m, n = q.n, np = PVX_CDIV(n, 16) * 16, ld = PVX_CDIV(n, 64) * 64 + 4;
    const E* in = reinterpret_cast<const E*>(q.in);
    double s = 0.0;
    for (int i = tid; i < MP * np; i += kSmallBlk) {
        const int r = q.tall ? i % MP : i / np, c = q.tall ? i / MP : i % np;
        float v = 0.f;
        if (r < m && c < n) v = (float)in[q.tall ? (size_t)c * m + r : (size_t)r * n + c];
        x[r * ld + c] = v;
        s = fma((double)v, (double)v, s);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
    if (lane == 0) red[wave] = s;
    __syncthreads();
    s = 0.0;
#pragma unroll
    for (int w = 0; w < kSmallWaves; w++) s += red[w];
    const double scale = 1.0 / (sqrt(s) + (double)eps);
    for (int i = tid; i < MP * np; i += kSmallBlk) {
        const int r = q.tall ? i % MP : i / np, c = q.tall ? i / MP : i % np;
        x[r * ld + c] = (float)((double)x[r * ld + c] * scale);
    }
    for (int step = 0; step < steps; step++) {
        __syncthreads();
        f32x4 acc[kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; t++) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int k = wave * 16; k < np; k += kSmallWaves * 16) {
            f32x4 f[T];
#pragma unroll
            for (int i = 0; i < T; i++) f[i] = *reinterpret_cast<const f32x4*>(&x[(16 * i + lr) * ld + k + 4 * lq]);
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int i = 0; i < T; i++)
#pragma unroll
                    for (int j = 0; j <= i; j++)
                        acc[i * (i + 1) / 2 + j] = __builtin_amdgcn_mfma_f32_16x16x4f32(f[i][e], f[j][e], acc[i * (i + 1) / 2 + j], 0, 0, 0);
        }
        // a lane holds column lane % 16 and rows 4 (lane / 16) + 0 .. 3
#pragma unroll
        for (int t = 0; t < kTiles; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) part[((wave * kTiles + t) * 16 + 4 * lq + e) * 16 + lr] = acc[t][e];
        __syncthreads();
        for (int i = tid; i < kTiles * 256; i += kSmallBlk) {
            const int t = i >> 8, r = (i >> 4) & 15, c = i & 15, ti = t == 0 ? 0 : 1, tj = t == 2 ? 1 : 0;
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < kSmallWaves; w++) v += part[w * kTiles * 256 + i];
            a[(16 * ti + r) * kLdA + 16 * tj + c] = v;
            if (ti != tj) a[(16 * tj + c) * kLdA + 16 * ti + r] = v;
        }
        __syncthreads();
        for (int i = tid; i < MP * MP; i += kSmallBlk) {
            const int r = i / MP, c = i % MP;
            float v = 0.f;
#pragma unroll
            for (int k = 0; k < MP; k++) v = fmaf(a[r * kLdA + k], a[c * kLdA + k], v);
            b[r * kLdA + c] = fmaf(cc, v, cb * a[r * kLdA + c]);
        }
        __syncthreads();
        // X <- a X + B X by 16 columns, in place: a wave reads all of them before it writes
        for (int j = wave * 16; j < np; j += kSmallWaves * 16) {
            f32x4 o[T];
#pragma unroll
            for (int i = 0; i < T; i++) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < T; k++) {
                f32x4 f[T];
#pragma unroll
                for (int i = 0; i < T; i++) f[i] = *reinterpret_cast<const f32x4*>(&b[(16 * i + lr) * kLdA + 16 * k + 4 * lq]);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float g = x[(16 * k + 4 * lq + e) * ld + j + lr];
#pragma unroll
                    for (int i = 0; i < T; i++) o[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(f[i][e], g, o[i], 0, 0, 0);
                }
            }
#pragma unroll
            for (int i = 0; i < T; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float* to = &x[(16 * i + 4 * lq + e) * ld + j + lr];
                    *to = fmaf(ca, *to, o[i][e]);
                }
        }
    }
    __syncthreads();
    E* out = reinterpret_cast<E*>(q.out);
    for (int i = tid; i < m * n; i += kSmallBlk) {
        const int r = q.tall ? i % m : i / n, c = q.tall ? i / m : i % n;
        out[i] = (E)x[r * ld + c];
    }
}

template <typename E>
__global__ __launch_bounds__(kSmallBlk) void ns_small_kernel(Table t, int steps, float a, float b, float c, float eps) {
    __shared__ __attribute__((aligned(16))) float x[kSmallWords];
    __shared__ __attribute__((aligned(16))) float part[kSmallWaves * 3 * 256];
    __shared__ __attribute__((aligned(16))) float sa[32 * 36], sb[32 * 36];
    __shared__ double red[kSmallWaves];
    const Mat& q = t.mat[blockIdx.x];
    if (q.m <= 16) small_body<E, 16>(q, steps, a, b, c, eps, x, part, sa, sb, red);
    else small_body<E, 32>(q, steps, a, b, c, eps, x, part, sa, sb, red);
}

bool all_small(const pvx_matrix* mats, int count) {
    for (int i = 0; i < count; i++) {
        const int m = mats[i].rows < mats[i].cols ? mats[i].rows : mats[i].cols, n = mats[i].rows < mats[i].cols ? mats[i].cols : mats[i].rows;
        if (m > 32 || n > small_width(m <= 16 ? 16 : 32)) return false;
    }
    return true;
}

int round_up(int v, int to) { return PVX_CDIV(v, to) * to; }

// 128 x 128 tiles where the products of all matrices of the call together fill the chip with them (they read LDS half as often), 64 x 64
// otherwise (128 / 64: 2048 x 4096 1167 / 1422 us, 2048 x 2048 782 / 884, 1024 x 1024 342 / 257, 512 x 2304 245 / 190).  One tile for a
// call: lists of wide matrices gain (64 of 256 x 2304 1188 / 1462, 8 of 1024 x 1024 887 / 1047, 8 of 512 x 2304 541 / 633, 2 of 1536 x 2048
// 870 / 945), lists near the border stay within 6 % (16 of 256 x 2304 431 / 407, 5 of 1024 x 1024 668 / 656, 3 of 1024 x 2048 696 / 706), and
// many narrow ones, padded to 128 rows, lose (42 layers of 16 to 128 rows 333 / 265).
int tile_of(const pvx_matrix* mats, int count) {
    double tiles = 0.0;
    for (int i = 0; i < count; i++) tiles += (double)mats[i].rows * mats[i].cols / (128.0 * 128.0);
    return tiles >= 256.0 ? 128 : 64;
}

// Parts of a sum: `slots` workgroups run at a time on 256 CUs; the number of parts that leaves the fewest of them idle in the last turn, of
// those that fit one turn, a part keeping at least four steps of k (with one part: 256 x 2304 280 us instead of 147, 2048 x 4096 1414
// instead of 1167)
int parts_of(long long tiles, int k, int tile) {
    const int most = PVX_CDIV(PVX_CDIV(k, kBK), 4), slots = tile == 128 ? 3 : 6;
    int best = 1;
    double eff = 0.0;
    for (int p = 1; p <= most && tiles * p <= 256 * slots; p++) {
        const double turns = (double)tiles * p / 256.0, e = turns / (double)(long long)(turns + 0.999999);
        if (e > eff + 0.02) { eff = e; best = p; }
    }
    return best;
}

void fill(Table& t, const pvx_matrix* mats, int count, int tile, size_t* total) {
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
    for (int i = 0; i < count; i++) {
        Mat& q = t.mat[i];
        q.parts = parts_of(tiles, q.n, tile);
        q.parts2 = parts_of(tiles, q.m, tile);
        q.base = (long long)off;
        const size_t px = (size_t)q.mp * q.np, pa = (size_t)q.mp * q.mp, lower = (size_t)(q.mp / tile) * (q.mp / tile + 1) / 2 * tile * tile;
        const int parts = q.parts > q.parts2 ? q.parts : q.parts2;
        off += pvx_align_up(4 * (2 * px + 2 * pa + lower * parts) + sizeof(double) * kNormBlocks + sizeof(Scales) * kMaxSteps, 256);
    }
    *total = off;
}

template <typename F> int spread(Table& t, F blocks) {
    long long at = 0;
    for (int i = 0; i < t.count; i++) {
        t.first[i] = (int)at;
        at += blocks(t.mat[i]);
        if (at > 0xffffffLL) return -1;                  // workgroups x threads stay below 2^32
    }
    t.first[t.count] = (int)at;
    return (int)at;
}

template <typename E, int T>
int run(Table& t, char* ws, int steps, float a, float b, float c, float eps, hipStream_t st) {
    auto lower = [](const Mat& q) { return (long long)(q.mp / T) * (q.mp / T + 1) / 2; };
    auto blocks32 = [&](const Mat& q) { return lower(q) * (T / 32) * (T / 32); };
#define NS_LAUNCH(kernel, blocks_of, ...)                                                      \
    do {                                                                                       \
        const int blocks__ = spread(t, blocks_of);                                             \
        if (blocks__ < 0) return PVX_ERR_RANGE;                                                \
        hipLaunchKernelGGL(kernel, dim3(blocks__), dim3(kBlk), 0, st, t, ws, ##__VA_ARGS__);    \
        PVX_CHECK_LAUNCH();                                                                    \
    } while (0)
    NS_LAUNCH((ns_norm_kernel<E>), ([](const Mat& q) {
                  const long long k = PVX_CDIV((long long)q.m * q.n, (long long)kNormChunk);
                  return k > kNormBlocks ? (long long)kNormBlocks : k;
              }), T);
    NS_LAUNCH((ns_load_kernel<E>), ([](const Mat& q) { return (long long)(q.mp / 64) * (q.np / 64); }), T, eps, steps, poly_of(a, b, c));
    if (steps == 0) NS_LAUNCH((ns_store_kernel<E>), ([](const Mat& q) { return PVX_CDIV((long long)q.m * q.n, (long long)kBlk); }), T);
    for (int s = 0; s < steps; s++) {
        const int last = s == steps - 1;
        NS_LAUNCH((ns_product_kernel<E, T, kGram>), ([&](const Mat& q) { return lower(q) * q.parts; }), s, last);
        NS_LAUNCH((ns_gather_kernel<T, kGram>), blocks32, s);
        NS_LAUNCH((ns_product_kernel<E, T, kPoly>), ([&](const Mat& q) { return lower(q) * q.parts2; }), s, last);
        NS_LAUNCH((ns_gather_kernel<T, kPoly>), blocks32, s);
        NS_LAUNCH((ns_product_kernel<E, T, kApply>), ([](const Mat& q) { return (long long)(q.mp / T) * (q.np / T); }), s, last);
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
    if (check_args(mats, count, dtype) != PVX_OK || count == 0 || all_small(mats, count)) return 0;
    Table t;
    size_t total;
    fill(t, mats, count, tile_of(mats, count), &total);
    return total;
}

extern "C" int pvx_orthogonalize_holds(int steps, float a, float b, float c) {
    return steps >= 0 && steps <= kMaxSteps && bound_holds(steps, a, b, c);
}

extern "C" int pvx_orthogonalize(const pvx_matrix* mats, int count, int dtype, int steps, float a, float b, float c, float eps, void* workspace,
                                 size_t workspace_bytes, void* stream) {
    const int bad = check_args(mats, count, dtype);
    if (bad != PVX_OK) return bad;
    if (steps < 0 || !(eps >= 0.f)) return PVX_ERR_INVALID;
    if (steps > kMaxSteps || !bound_holds(steps, a, b, c)) return PVX_ERR_RANGE;
    if (count == 0) return PVX_OK;
    for (int i = 0; i < count; i++)
        if (!mats[i].in || !mats[i].out) return PVX_ERR_INVALID;
    Table t;
    size_t total;
    hipStream_t st = (hipStream_t)stream;
    const int tile = tile_of(mats, count);
    fill(t, mats, count, tile, &total);
    if (all_small(mats, count)) {
        if (dtype == PVX_F32) hipLaunchKernelGGL(ns_small_kernel<float>, dim3(count), dim3(kSmallBlk), 0, st, t, steps, a, b, c, eps);
        else if (dtype == PVX_F16) hipLaunchKernelGGL(ns_small_kernel<_Float16>, dim3(count), dim3(kSmallBlk), 0, st, t, steps, a, b, c, eps);
        else hipLaunchKernelGGL(ns_small_kernel<__bf16>, dim3(count), dim3(kSmallBlk), 0, st, t, steps, a, b, c, eps);
        PVX_CHECK_LAUNCH();
        return PVX_OK;
    }
    if (!workspace || workspace_bytes < total || (reinterpret_cast<uintptr_t>(workspace) & 255)) return PVX_ERR_WORKSPACE;
    char* ws = reinterpret_cast<char*>(workspace);
    if (dtype == PVX_F32) return tile == 128 ? run<float, 128>(t, ws, steps, a, b, c, eps, st) : run<float, 64>(t, ws, steps, a, b, c, eps, st);
    if (dtype == PVX_F16) return tile == 128 ? run<_Float16, 128>(t, ws, steps, a, b, c, eps, st) : run<_Float16, 64>(t, ws, steps, a, b, c, eps, st);
    return tile == 128 ? run<__bf16, 128>(t, ws, steps, a, b, c, eps, st) : run<__bf16, 64>(t, ws, steps, a, b, c, eps, st);
}
