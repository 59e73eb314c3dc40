// engram_ortho.cu -- orthogonalising an update by Newton-Schulz products, and the
// optimizer step that applies it.  Each matrix U of a stack is divided by its
// Frobenius norm and taken through steps of an odd polynomial,
//   X <- c0 X + (c1 G + c2 G G) X,   G = X X^T (the short side),
// which moves every singular value toward 1 and leaves the singular vectors.
//
// Short sides up to 64 (adapter factors): all steps act on the short side only.
// With G0 = U U^T / |U|^2, every iterate is X = P X0 with P a polynomial of G0, so
// U is read once for G0, the small matrices are iterated by one block, and U is
// read once more for P U.  That needs G0 and P far beyond fp32 (P cancels: it holds
// c0^steps, 485 for the default, along the weak directions and 1 / sigma along the
// strong ones), so this path sums in fp64 on the fp64 tensor cores
// (mma.sync m8n8k4).  It is one pass over U, and one more with the output.
//
// Longer sides: three tcgen05 products a step on planes of fp16.  A value is
// kept as y = 2^12 x = hi + lo, two fp16 (22 significant bits); a product is
// hi hi + hi lo + lo hi in fp32 accumulators in tensor memory.  22 bits of operands and sums that round toward zero
// leave results of noise 6e-5 off at 2560 x 2560 (plain fp32 4e-6): an update is a direction to step in, and 33 bits in
// three planes would take twice the products.  Every iterate has
// entries below 16 (checked for the coefficients on the host), so hi is far from
// fp16's limits, and lo's steps of 2^-24 are 2^-36 of x.  c0 is added to the
// diagonal of the polynomial, so X' is one product.  Results rounded to bf16 take
// one product of the hi planes, operands rounded to 2^-12; there X keeps its lo
// plane all the same and c0 X is added to the product from both, since an X rounded
// at each step drowns the weak directions (1.5e-2 off on updates whose noise is 1/50
// of their signal, against 2e-4 so; 1.8e-3 at most on any spectrum tried, beside
// 1.7e-3 of bf16 itself).  G and G G are symmetric: only tiles that reach the diagonal
// or lie above it are computed and stored twice.  The planes are read in the layout in which
// U was given: tall matrices use U^T U and X P, so nothing is transposed in memory;
// the descriptors take each operand along K or across it.
#include <algorithm>
#include <type_traits>

#include "engram_tensor.cuh"

using namespace engram;

namespace {

constexpr int kMaxSteps = 32;
constexpr int kSmallSide = 64;

struct Poly {
    double c[kMaxSteps][3];
    int steps;
};

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }

// Four elements from i on; vec: as one load (i a multiple of 4 from an aligned array), else `left` of them.
__device__ __forceinline__ float4 load4(const float* p, int64_t i, int left, bool vec) {
    if (vec) return *reinterpret_cast<const float4*>(p + i);
    return make_float4(p[i], left > 1 ? p[i + 1] : 0.f, left > 2 ? p[i + 2] : 0.f, left > 3 ? p[i + 3] : 0.f);
}
template <typename T>
__device__ __forceinline__ float4 load4(const T* p, int64_t i, int left, bool vec) {
    if (vec) {
        alignas(8) T v[4];
        *reinterpret_cast<uint2*>(v) = *reinterpret_cast<const uint2*>(p + i);
        return make_float4(to_f32(v[0]), to_f32(v[1]), to_f32(v[2]), to_f32(v[3]));
    }
    return make_float4(to_f32(p[i]), left > 1 ? to_f32(p[i + 1]) : 0.f, left > 2 ? to_f32(p[i + 2]) : 0.f,
                       left > 3 ? to_f32(p[i + 3]) : 0.f);
}
template <typename T>
__device__ __forceinline__ void store4(T* p, int64_t i, int left, bool vec, float4 v) {
    if (vec) {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(p + i) = v;
        } else {
            alignas(8) T o[4] = {from_f32<T>(v.x), from_f32<T>(v.y), from_f32<T>(v.z), from_f32<T>(v.w)};
            *reinterpret_cast<uint2*>(p + i) = *reinterpret_cast<const uint2*>(o);
        }
        return;
    }
    p[i] = from_f32<T>(v.x);
    if (left > 1) p[i + 1] = from_f32<T>(v.y);
    if (left > 2) p[i + 2] = from_f32<T>(v.z);
    if (left > 3) p[i + 3] = from_f32<T>(v.w);
}

// Where U comes from and where the result goes.  Plain: U = x, the result is out.
// Muon: m' = m + (1 - beta)(g - m), U = g + beta (m' - g) (Nesterov) or m'; the first
// pass writes m', the later one reads it; the result O gives p' = decay p - step O.
// fetch() only loads, so that the next elements are under way while others are worked
// on; the value follows from what it loaded.
template <typename T>
struct Plain {
    struct Raw {
        float4 x;
    };
    const T* x;
    T* out;
    bool aligned;  // both on four elements
    template <bool FIRST>
    __device__ __forceinline__ void fetch(Raw& r, int64_t i, int left, bool vec) const {
        r.x = load4(x, i, left, vec);
    }
    template <bool FIRST>
    __device__ __forceinline__ float4 value(const Raw& r, int64_t, int, bool) const {
        return r.x;
    }
    __device__ __forceinline__ void put(const Raw&, int64_t i, int left, bool vec, float4 o) const {
        store4(out, i, left, vec, o);
    }
    __device__ __forceinline__ void before(Raw&, int64_t, int, bool) const {}  // what put() needs
};
template <typename T>
struct MuonIo {
    struct Raw {
        float4 g, m, p;
    };
    const T* g;
    const float* m;
    float* m_out;
    const float* p;
    float* p_out;
    float beta, rest, decay, step;
    bool nesterov, aligned;
    __device__ __forceinline__ float update(float gv, float mv) const {
        return nesterov ? __fmaf_rn(beta, mv - gv, gv) : mv;
    }
    __device__ __forceinline__ float moved(float gv, float mv) const { return __fmaf_rn(rest, gv - mv, mv); }
    template <bool FIRST>
    __device__ __forceinline__ void fetch(Raw& r, int64_t i, int left, bool vec) const {
        r.g = load4(g, i, left, vec);
        r.m = load4(FIRST ? m : m_out, i, left, vec);
        if (!FIRST) r.p = load4(p, i, left, vec);
    }
    template <bool FIRST>
    __device__ __forceinline__ float4 value(const Raw& r, int64_t i, int left, bool vec) const {
        float4 n = r.m;
        if (FIRST) {
            n = make_float4(moved(r.g.x, r.m.x), moved(r.g.y, r.m.y), moved(r.g.z, r.m.z), moved(r.g.w, r.m.w));
            store4(m_out, i, left, vec, n);
        }
        return make_float4(update(r.g.x, n.x), update(r.g.y, n.y), update(r.g.z, n.z), update(r.g.w, n.w));
    }
    __device__ __forceinline__ void put(const Raw& r, int64_t i, int left, bool vec, float4 o) const {
        store4(p_out, i, left, vec,
               make_float4(__fmaf_rn(-step, o.x, decay * r.p.x), __fmaf_rn(-step, o.y, decay * r.p.y),
                           __fmaf_rn(-step, o.z, decay * r.p.z), __fmaf_rn(-step, o.w, decay * r.p.w)));
    }
    __device__ __forceinline__ void before(Raw& r, int64_t i, int left, bool vec) const { r.p = load4(p, i, left, vec); }
};

// ---- short sides up to 64 -------------------------------------------------------

__device__ __forceinline__ void dmma(double* d, double a, double b) {
    asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};"
                 : "+d"(d[0]), "+d"(d[1])
                 : "d"(a), "d"(b));
}

constexpr int kSmallThreads = 256;

// A tile of the m x L matrix in shared memory: KT columns of its long side, rows padded to 8 MB.  It lies as the
// matrix does, so both are copied four elements at a time: TALL (stored [L][m]) column by column, else row by row;
// the padding keeps the fragments' reads (8 rows x 4 columns) on unlike banks.
template <int MB, bool TALL>
struct SmallTile {
    static constexpr int RM = 8 * MB, KT = MB <= 2 ? 128 : 64;
    static constexpr int PITCH = TALL ? RM + 8 : KT + 4, SIZE = TALL ? KT * PITCH : RM * PITCH;
    static constexpr int N = RM * KT / 4 / kSmallThreads;  // pieces of four a thread copies
    static_assert(N >= 1 && RM * KT % (4 * kSmallThreads) == 0, "whole pieces a thread");
    static __device__ __forceinline__ int at(int i, int k) { return TALL ? k * PITCH + i : i * PITCH + k; }
    // Piece n of this thread: its first row and column, and its place in the matrix
    static __device__ __forceinline__ void piece(int n, int& i, int& k) {
        const int e = (int)threadIdx.x + n * kSmallThreads;
        if (TALL) i = e % (RM / 4) * 4, k = e / (RM / 4);
        else k = e % (KT / 4) * 4, i = e / (KT / 4);
    }
    static __device__ __forceinline__ int64_t place(int64_t base, int m, int64_t L, int64_t k0, int i, int k) {
        return TALL ? base + (k0 + k) * m + i : base + (int64_t)i * L + k0 + k;
    }
    // elements of the piece that exist
    static __device__ __forceinline__ int left(int m, int64_t cols, int i, int k) {
        if (i >= m || k >= cols) return 0;
        const int64_t n = TALL ? (int64_t)m - i : cols - k;
        return n < 4 ? (int)n : 4;
    }
};

template <bool FIRST, typename S, typename Io>
__device__ __forceinline__ void fetch_tile(const Io& io, typename Io::Raw (&raw)[S::N], int64_t base, int m, int64_t L,
                                           int64_t k0, int64_t k_end, bool vec) {
#pragma unroll
    for (int n = 0; n < S::N; n++) {
        int i, k;
        S::piece(n, i, k);
        const int left = S::left(m, k_end - k0, i, k);
        if (left) io.template fetch<FIRST>(raw[n], S::place(base, m, L, k0, i, k), left, vec && left == 4);
    }
}
template <bool FIRST, typename S, typename Io>
__device__ __forceinline__ void store_tile(const Io& io, const typename Io::Raw (&raw)[S::N], float* tile, int64_t base,
                                           int m, int64_t L, int64_t k0, int64_t k_end, bool vec) {
#pragma unroll
    for (int n = 0; n < S::N; n++) {
        int i, k;
        S::piece(n, i, k);
        const int left = S::left(m, k_end - k0, i, k);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (left) v = io.template value<FIRST>(raw[n], S::place(base, m, L, k0, i, k), left, vec && left == 4);
        if (left < 2) v.y = 0.f;
        if (left < 3) v.z = 0.f;
        if (left < 4) v.w = 0.f;
        *reinterpret_cast<float4*>(tile + S::at(i, k)) = v;
    }
}

// part[s, chunk] = U U^T over the chunk's columns, fp64, [8 MB][8 MB] (blocks of 8 on and above the
// diagonal).  Warp w sums columns 8 w .. 8 w + 7 (and 64 further) of each tile; the warps are added in
// their order.
template <int MB, bool TALL, typename Io>
__global__ void __launch_bounds__(kSmallThreads) k_small_gram(Io io, int m, int64_t L, int64_t chunk, bool vec,
                                                              double* __restrict__ part) {
    using S = SmallTile<MB, TALL>;
    constexpr int RM = 8 * MB, NT = MB * (MB + 1) / 2;
    // the tile, and after the last one the sums
    __shared__ __align__(16) double sum[RM * RM > S::SIZE / 2 ? RM * RM : S::SIZE / 2];
    float* tile = reinterpret_cast<float*>(sum);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    const int64_t base = (int64_t)blockIdx.y * m * L, k_begin = blockIdx.x * chunk;
    const int64_t k_end = k_begin + chunk < L ? k_begin + chunk : L;
    let_next_start();
    double acc[NT][2];
#pragma unroll
    for (int i = 0; i < NT; i++) acc[i][0] = acc[i][1] = 0.0;
    typename Io::Raw raw[S::N];
    fetch_tile<true, S>(io, raw, base, m, L, k_begin, k_end, vec);
    for (int64_t k0 = k_begin; k0 < k_end; k0 += S::KT) {
        __syncthreads();
        store_tile<true, S>(io, raw, tile, base, m, L, k0, k_end, vec);
        __syncthreads();
        if (k0 + S::KT < k_end) fetch_tile<true, S>(io, raw, base, m, L, k0 + S::KT, k_end, vec);
#pragma unroll
        for (int s = 0; s < S::KT / 32; s++) {
            double f[MB];
#pragma unroll
            for (int i = 0; i < MB; i++)
                f[i] = (double)tile[S::at(8 * i + g, 64 * (s >> 1) + 8 * warp + 4 * (s & 1) + q)];
            int at = 0;
#pragma unroll
            for (int i = 0; i < MB; i++)
#pragma unroll
                for (int j = i; j < MB; j++) dmma(acc[at++], f[i], f[j]);
        }
    }
    __syncthreads();
    for (int w = 0; w < kSmallThreads / 32; w++) {
        if (w == warp) {
            int at = 0;
#pragma unroll
            for (int i = 0; i < MB; i++)
#pragma unroll
                for (int j = i; j < MB; j++, at++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        double* d = sum + (8 * i + g) * RM + 8 * j + 2 * q + c;
                        *d = w ? *d + acc[at][c] : acc[at][c];
                    }
        }
        __syncthreads();
    }
    double* dst = part + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * RM * RM;
    for (int e = threadIdx.x; e < RM * RM; e += kSmallThreads)
        if (e % RM >= (e / RM & ~7)) dst[e] = sum[e];
}

// z = x y for symmetric matrices that commute (so z is symmetric): blocks of 8 on and above the
// diagonal, mirrored.  f(i, j, v) gives the stored value.
template <int MB, typename F>
__device__ __forceinline__ void small_product(const double* x, const double* y, double* z, F f) {
    constexpr int S = 8 * MB + 4, NT = MB * (MB + 1) / 2;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    for (int at = warp; at < NT; at += (int)blockDim.x / 32) {
        int i = 0, left = at;
        while (left >= MB - i) left -= MB - i, i++;
        const int j = i + left;
        double d[2][2] = {{0.0, 0.0}, {0.0, 0.0}};
#pragma unroll
        for (int s = 0; s < 2 * MB; s++)
            dmma(d[s & 1], x[(8 * i + g) * S + 4 * s + q], y[(8 * j + g) * S + 4 * s + q]);
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const int r = 8 * i + g, col = 8 * j + 2 * q + c;
            const double v = f(r, col, d[0][c] + d[1][c]);
            z[r * S + col] = v;
            if (i != j) z[col * S + r] = v;
        }
    }
    __syncthreads();
}

// The chunks' sums, in their order, into the first chunk's: an element a thread, where one block a matrix would wait
// for too many of them.
__global__ void __launch_bounds__(kSmallThreads) k_small_sum(double* part, int chunks, int size, int64_t total) {
    wait_for_previous();
    let_next_start();
    const int64_t i = blockIdx.x * (int64_t)kSmallThreads + threadIdx.x;
    if (i >= total) return;
    double* p = part + i / size * chunks * size + i % size;
    double v = 0.0;
#pragma unroll 16
    for (int c = 0; c < chunks; c++) v += p[(int64_t)c * size];
    *p = v;
}

// The steps on the small matrices: pmat[s] = P / max(|U|, eps).  A matrix has `stride` chunks, of which the first
// `chunks` are summed here.  Twenty products one after the other, on one block: 45 us of the 63 that a 64 x 2560 fp32
// matrix takes.  Sides over 16 have blocks enough for sixteen warps (eight: 74 us).
template <int MB>
constexpr int kPolyThreads = MB >= 4 ? 512 : 256;
template <int MB>
__global__ void __launch_bounds__(kPolyThreads<MB>) k_small_poly(const double* part, int chunks, int stride, int m,
                                                              Poly poly, double eps, double* __restrict__ pmat) {
    constexpr int RM = 8 * MB, S = RM + 4;
    extern __shared__ double sd[];
    double *A = sd, *B = A + RM * S, *P = B + RM * S, *Q = P + RM * S;
    __shared__ double inv_norm;
    const double* src = part + (int64_t)blockIdx.x * stride * RM * RM;
    wait_for_previous();
    let_next_start();
    for (int e = threadIdx.x; e < RM * RM; e += blockDim.x) {
        const int i = e / RM, j = e % RM;
        if (j < (i & ~7)) continue;
        double v = 0.0;
#pragma unroll 8
        for (int c = 0; c < chunks; c++) v += src[(int64_t)c * RM * RM + e];
        A[i * S + j] = v;
        if (j / 8 != i / 8) A[j * S + i] = v;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int i = 0; i < m; i++) t += A[i * S + i];
        const double norm = sqrt(t);
        inv_norm = 1.0 / (norm < eps ? eps : norm);  // a NaN stays one
    }
    __syncthreads();
    const double inv = inv_norm;
    for (int e = threadIdx.x; e < RM * RM; e += blockDim.x) {
        const int i = e / RM, j = e % RM;
        A[i * S + j] *= inv * inv;
        P[i * S + j] = i == j ? inv : 0.0;
    }
    __syncthreads();
    for (int s = 0; s < poly.steps; s++) {
        const double c0 = poly.c[s][0], c1 = poly.c[s][1], c2 = poly.c[s][2];
        // B = M = c0 + c1 A + c2 A A, then P <- M P and A <- M A M
        small_product<MB>(A, A, B, [&](int i, int j, double v) { return (i == j ? c0 : 0.0) + c1 * A[i * S + j] + c2 * v; });
        small_product<MB>(B, P, Q, [](int, int, double v) { return v; });
        double* t = P;
        P = Q, Q = t;
        if (s + 1 < poly.steps) {
            small_product<MB>(B, A, Q, [](int, int, double v) { return v; });
            small_product<MB>(B, Q, A, [](int, int, double v) { return v; });
        }
    }
    for (int e = threadIdx.x; e < RM * RM; e += blockDim.x)
        pmat[(int64_t)blockIdx.x * RM * RM + e] = P[(e / RM) * S + e % RM];
}

// The result P U, tile by tile.
template <int MB, bool TALL, typename Io>
__global__ void __launch_bounds__(kSmallThreads) k_small_apply(Io io, int m, int64_t L, int64_t chunk, bool vec,
                                                               const double* pmat) {
    using S = SmallTile<MB, TALL>;
    constexpr int RM = 8 * MB, SP = RM + 4;
    extern __shared__ double sd[];
    double* P = sd;
    float* tile = reinterpret_cast<float*>(P + RM * SP);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    const int64_t base = (int64_t)blockIdx.y * m * L, k_begin = blockIdx.x * chunk;
    const int64_t k_end = k_begin + chunk < L ? k_begin + chunk : L;
    typename Io::Raw raw[S::N];
    wait_for_previous();  // P, and what the first pass wrote
    let_next_start();
    fetch_tile<false, S>(io, raw, base, m, L, k_begin, k_end, vec);
    for (int e = threadIdx.x; e < RM * RM; e += kSmallThreads)
        P[(e / RM) * SP + e % RM] = pmat[(int64_t)blockIdx.y * RM * RM + e];
    for (int64_t k0 = k_begin; k0 < k_end; k0 += S::KT) {
        typename Io::Raw now[S::N];
#pragma unroll
        for (int n = 0; n < S::N; n++) now[n] = raw[n];
        __syncthreads();
        store_tile<false, S>(io, now, tile, base, m, L, k0, k_end, vec);
        __syncthreads();
        if (k0 + S::KT < k_end) fetch_tile<false, S>(io, raw, base, m, L, k0 + S::KT, k_end, vec);
#pragma unroll
        for (int part = 0; part < S::KT / 64; part++) {  // warp w: columns 8 w .. 8 w + 7, and 64 further
            double acc[MB][2];
#pragma unroll
            for (int i = 0; i < MB; i++) acc[i][0] = acc[i][1] = 0.0;
            const int k = 64 * part + 8 * warp;
#pragma unroll
            for (int s = 0; s < 2 * MB; s++) {
                const double b = (double)tile[S::at(4 * s + q, k + g)];
#pragma unroll
                for (int i = 0; i < MB; i++) dmma(acc[i], P[(8 * i + g) * SP + 4 * s + q], b);
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < MB; i++) {
                tile[S::at(8 * i + g, k + 2 * q)] = (float)acc[i][0];
                tile[S::at(8 * i + g, k + 2 * q + 1)] = (float)acc[i][1];
            }
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < S::N; n++) {
            int i, kk;
            S::piece(n, i, kk);
            const int left = S::left(m, k_end - k0, i, kk);
            if (left)
                io.put(now[n], S::place(base, m, L, k0, i, kk), left, vec && left == 4,
                       *reinterpret_cast<const float4*>(tile + S::at(i, kk)));
        }
    }
}

// ---- longer sides: planes ---------------------------------------------------------

constexpr float kPlaneScale = 4096.f;
constexpr int kNormThreads = 256;

// part[s, block] = the block's share of |U|^2, fp64 (updates of 1e-20 and of 1e20 alike).
template <typename Io>
__global__ void __launch_bounds__(kNormThreads) k_norm(Io io, int64_t size, bool vec, double* __restrict__ part) {
    __shared__ double warp_sum[kNormThreads / 32];
    let_next_start();
    const int64_t base = blockIdx.y * size, pieces = (size + 3) / 4, step = (int64_t)gridDim.x * kNormThreads;
    double v = 0.0;
    constexpr int N = 4;  // pieces under way a thread
    for (int64_t i0 = blockIdx.x * (int64_t)kNormThreads + threadIdx.x; i0 < pieces; i0 += N * step) {
        typename Io::Raw raw[N];
#pragma unroll
        for (int k = 0; k < N; k++) {
            const int64_t i = 4 * (i0 + k * step), left = size - i;
            if (left > 0) io.template fetch<true>(raw[k], base + i, (int)(left < 4 ? left : 4), vec);
        }
#pragma unroll
        for (int k = 0; k < N; k++) {
            const int64_t i = 4 * (i0 + k * step), left = size - i;
            if (left <= 0) continue;
            const float4 u = io.template value<true>(raw[k], base + i, (int)(left < 4 ? left : 4), vec);
            v += (double)u.x * u.x;
            if (left > 1) v += (double)u.y * u.y;
            if (left > 2) v += (double)u.z * u.z;
            if (left > 3) v += (double)u.w * u.w;
        }
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if ((threadIdx.x & 31) == 0) warp_sum[threadIdx.x >> 5] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kNormThreads / 32; w++) v += warp_sum[w];
        part[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = v;
    }
}

struct Planes {
    __half *hi, *lo;  // lo null: one product
    int64_t ld, stride;
};

__device__ __forceinline__ void put(const Planes& p, int64_t i, float y) {
    const __half h = __float2half_rn(y);
    p.hi[i] = h;
    if (p.lo) p.lo[i] = __float2half_rn(y - __half2float(h));
}

// planes = 2^12 U / max(|U|, eps); a warp takes 512 columns of a row at a time.
template <typename Io>
__global__ void __launch_bounds__(kNormThreads) k_planes(Io io, int64_t rows, int64_t cols, bool vec,
                                                         const double* part, int parts, double eps, Planes out) {
    __shared__ double total;
    wait_for_previous();
    let_next_start();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (warp == 0) {
        double v = 0.0;
        for (int i = lane; i < parts; i += 32) v += part[(int64_t)blockIdx.y * parts + i];
#pragma unroll
        for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
        if (lane == 0) total = v;
    }
    __syncthreads();
    const double norm = sqrt(total);
    const double inv = (double)kPlaneScale / (norm < eps ? eps : norm);
    const int64_t base = blockIdx.y * rows * cols;
    constexpr int N = 4;  // pieces of four under way a lane
    const int64_t per_row = (cols + N * 128 - 1) / (N * 128), units = rows * per_row;
    for (int64_t unit = blockIdx.x * (int64_t)(kNormThreads / 32) + warp; unit < units;
         unit += (int64_t)gridDim.x * (kNormThreads / 32)) {
        const int64_t r = unit / per_row, c0 = (unit - r * per_row) * (N * 128) + 4 * lane;
        {
            typename Io::Raw raw[N];
#pragma unroll
            for (int k = 0; k < N; k++) {
                const int64_t c = c0 + 128 * k, left = cols - c;
                if (left > 0) io.template fetch<false>(raw[k], base + r * cols + c, (int)(left < 4 ? left : 4), vec);
            }
#pragma unroll
            for (int k = 0; k < N; k++) {
                const int64_t c = c0 + 128 * k, left = cols - c;
                if (left <= 0) continue;
                const float4 u = io.template value<false>(raw[k], base + r * cols + c, (int)(left < 4 ? left : 4), vec);
                const float v[4] = {u.x, u.y, u.z, u.w};
                alignas(8) __half hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {  // the padding (to a multiple of 64) may be written
                    const float y = e < left ? (float)((double)v[e] * inv) : 0.f;
                    hi[e] = __float2half_rn(y);
                    lo[e] = __float2half_rn(y - __half2float(hi[e]));
                }
                const int64_t at = blockIdx.y * out.stride + r * out.ld + c;
                *reinterpret_cast<uint2*>(out.hi + at) = *reinterpret_cast<const uint2*>(hi);
                *reinterpret_cast<uint2*>(out.lo + at) = *reinterpret_cast<const uint2*>(lo);
            }
        }
    }
}

// ---- longer sides: the products -----------------------------------------------------

struct NoIo {
    struct Raw {};
};

enum Mode { GRAM, POLY, UPDATE, RESULT };

constexpr int BM = 128;
constexpr int kGemmThreads = 320, kEpilogueWarps = 8;
constexpr int kStageTotal = 192 * 1024;
// Longest sum that one accumulator takes, in products of three terms and of one (results of 8 bits).  An MMA cuts its
// 16 products to a grid of 2^-25 of the sum, toward zero, so what a sum of one sign loses grows with its length, by
// 2^-23 an MMA.  Without an end, 66 x 2^21 in fp32 was 2.0e-4 off and 1536 x 131072 2.9e-4, now 2.6e-5 and 1.4e-5
// (2.9e-6 and 1.5e-5 in plain fp32).  Ends at 2048: 1.3e-5 and 9e-6, but 1060 us where 2560 x 2560 takes 955.
constexpr int kChunk3 = 4096, kChunk1 = 16384;

// A tile is 128 x 256 on one block, or 256 x 256 on a pair (PAIR): a cluster of two blocks whose tensor cores
// work as one (cta_group::2).  Each block of a pair has half of A's rows and half of B's and reads the other half
// of B from its partner, so a slice is 32 KB a block where one block needs 48.  Small products take 128 x 64 on
// one block, and sums over a long K with few tiles are split over blocks.
// One K slice of the operands: 32 columns of four planes (A hi, B hi, A lo, B lo) or 64 of two.
template <int TERMS, bool PAIR, int BN>
struct Cfg {
    static constexpr int KS = TERMS == 3 ? 32 : 64, B_ROWS = PAIR ? BN / 2 : BN;
    static constexpr int A_BYTES = BM * KS * 2, B_BYTES = B_ROWS * KS * 2;
    static constexpr int STAGE_BYTES = (TERMS == 3 ? 2 : 1) * (A_BYTES + B_BYTES);
    static constexpr int STAGES = kStageTotal / STAGE_BYTES;
    static constexpr int SMEM = STAGES * STAGE_BYTES + kEpilogueWarps * 4096 + 1024 + 256;
    static constexpr int TILE_M = PAIR ? 2 * BM : BM;
    static constexpr int CHUNK = (TERMS == 3 ? kChunk3 : kChunk1) / KS;  // slices that one accumulator takes
};

struct Maps {
    CUtensorMap a_hi, a_lo, b_hi, b_lo;
};

template <typename Io>
struct Job {
    int M, N, K;       // D [M, N] = sum over K
    int tiles_m, tiles_n, tiles;  // tiles along M, along N, of a matrix
    int total;                    // tiles of the stack, times splits
    int splits;                   // blocks that share a tile's sum
    float* partial;               // [tile, split, 128, BN]: where they put theirs
    float4* carry;                // [block, 128 BN / 4]: a tile's sum so far, where it takes more than one accumulator
    Planes out;        // GRAM, POLY, UPDATE
    Planes g;          // POLY: the planes of G; UPDATE, RESULT of one term: those of X
    float c0, c1, c2;  // POLY
    Io io;             // RESULT
    bool vec;          // RESULT: rows of whole, aligned fours
};

// Shared-memory matrix descriptor.  Along K (rows of KS fp16, 64- or 128-byte swizzle): 8-row groups
// 8 KS 2 bytes apart.  Across K (blocks of 64 columns, each KS rows of 128 bytes, 128-byte swizzle):
// 8-row groups of K 1024 bytes apart, blocks KS 128 bytes apart.
template <bool MN, int KS>
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
    constexpr uint32_t lbo = MN ? KS * 128 : 16, sbo = MN ? 1024 : 8 * KS * 2;
    constexpr uint64_t swizzle = (MN || KS == 64) ? 2 : 4;
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(sbo >> 4) << 32) |
           ((uint64_t)1 << 46) | (swizzle << 61);
}

__device__ __forceinline__ void mbar_arrive_leader(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

template <bool A_MN, bool B_MN, bool PAIR, int BN>
__device__ __forceinline__ void umma_f16(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t accumulate) {
    // A and B fp16, D fp32, each operand along K or across it; M 128, or 256 over the pair
    constexpr uint32_t desc = (1u << 4) | ((A_MN ? 1u : 0u) << 15) | ((B_MN ? 1u : 0u) << 16) |
                              ((uint32_t)(BN >> 3) << 17) | ((uint32_t)((PAIR ? 256 : 128) >> 4) << 24);
    if constexpr (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
            "l"(da), "l"(db), "r"(desc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
            "l"(da), "l"(db), "r"(desc), "r"(accumulate)
            : "memory");
}
// Arrives at the barrier, of both blocks of a pair, once the MMAs issued so far are done.
template <bool PAIR>
__device__ __forceinline__ void commit(uint32_t bar) {
    if constexpr (PAIR)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
            "h"((uint16_t)3)
            : "memory");
    else
        umma_commit(bar);
}
// The same place in the shared memory of the pair's first block.
__device__ __forceinline__ uint32_t leaders(uint32_t addr) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// A tile of an operand; PAIR: onto a barrier of the pair's first block.
template <bool PAIR>
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    if constexpr (PAIR)
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, "
            "%4}], [%5];" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
            : "memory");
    else
        tma_load_3d(dst, map, x, y, z, bar);
}
template <bool MN, int KS, int ROWS, bool PAIR>
__device__ __forceinline__ void load_operand(uint32_t dst, const CUtensorMap* map, int row0, int k, int z, uint32_t bar) {
    if constexpr (MN) {
#pragma unroll
        for (int b = 0; b < ROWS / 64; b++) load_box<PAIR>(dst + b * KS * 128, map, row0 + 64 * b, k, z, bar);
    } else {
        load_box<PAIR>(dst, map, k, row0, z, bar);
    }
}

__device__ __forceinline__ void put8(const Planes& p, int64_t i, const float* v) {
    alignas(16) __half h[8], l[8];
#pragma unroll
    for (int k = 0; k < 8; k++) {
        h[k] = __float2half_rn(v[k]);
        l[k] = __float2half_rn(v[k] - __half2float(h[k]));
    }
    *reinterpret_cast<uint4*>(p.hi + i) = *reinterpret_cast<const uint4*>(h);
    if (p.lo) *reinterpret_cast<uint4*>(p.lo + i) = *reinterpret_cast<const uint4*>(l);
}

// Tile t of the stack.  Symmetric modes have those with an entry on or above the diagonal: of column block b
// the row blocks that begin above its last column.
template <bool SYM, int TILE_M, int BN, typename J>
__device__ __forceinline__ void tile_at(const J& job, int t, int& z, int& m0, int& n0) {
    z = t / job.tiles;
    int left = t - z * job.tiles;
    if constexpr (SYM) {
        int b = 0, rows = min((BN - 1) / TILE_M + 1, job.tiles_m);
        while (left >= rows) left -= rows, b++, rows = min((BN * (b + 1) - 1) / TILE_M + 1, job.tiles_m);
        m0 = left * TILE_M, n0 = b * BN;
    } else {
        m0 = left % job.tiles_m * TILE_M, n0 = left / job.tiles_m * BN;
    }
}

// What a lane needs from memory for its part of a 32 x 32 piece: fetched together, ahead of the accumulator (one by
// one, each waits for the one before: 11 us a tile).
template <int MODE, int TERMS, typename Io>
struct Before {
    static constexpr bool SYM = MODE == GRAM || MODE == POLY, PLANES = MODE == POLY || (TERMS == 1 && !SYM);
    static constexpr bool TWO = PLANES && (TERMS == 3 || !SYM);
    uint4 hi[PLANES ? 4 : 1], lo[TWO ? 4 : 1];
    typename Io::Raw raw[MODE == RESULT ? 8 : 1];
    __device__ __forceinline__ void fetch(const Job<Io>& job, int z, int r0, int c0, int lane) {
#pragma unroll
        for (int it = 0; it < 4; it++) {
            const int row = r0 + 8 * it + (lane >> 2), c = c0 + 8 * (lane & 3);
            if (row >= job.M || c >= job.N) continue;
            if constexpr (PLANES) {
                const int64_t at = (int64_t)z * job.g.stride + (int64_t)row * job.g.ld + c;
                hi[it] = *reinterpret_cast<const uint4*>(job.g.hi + at);
                if constexpr (TWO) lo[it] = *reinterpret_cast<const uint4*>(job.g.lo + at);
            }
            if constexpr (MODE == RESULT) {
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const int left = job.N - c - 4 * j;
                    if (left > 0)
                        job.io.before(raw[2 * it + j], ((int64_t)z * job.M + row) * job.N + c + 4 * j, left < 4 ? left : 4,
                                      job.vec && left >= 4);
                }
            }
        }
    }
    __device__ __forceinline__ void planes(int it, float* v) const {
        if constexpr (PLANES) {
            const __half* h = reinterpret_cast<const __half*>(&hi[it]);
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = __half2float(h[k]);
            if constexpr (TWO) {
                const __half* l = reinterpret_cast<const __half*>(&lo[it]);
#pragma unroll
                for (int k = 0; k < 8; k++) v[k] += __half2float(l[k]);
            }
        }
    }
};

// The mode's work on the 32 x 32 piece of products at (r0, c0), which lies in shared memory in rows of 128 bytes
// whose units of 16 are swapped by row: four lanes take 64 consecutive bytes of a row.
template <int MODE, int TERMS, typename Io>
__device__ __forceinline__ void finish_piece(const Job<Io>& job, uint8_t* tile, const Before<MODE, TERMS, Io>& before, int z,
                                             int r0, int c0, int lane) {
    constexpr bool SYM = MODE == GRAM || MODE == POLY;
#pragma unroll
    for (int it = 0; it < 4; it++) {
        const int lr = 8 * it + (lane >> 2), u = 2 * (lane & 3), row = r0 + lr, c = c0 + 4 * u;
        float* lo4 = reinterpret_cast<float*>(tile + lr * 128 + ((u ^ (lr & 7)) << 4));
        float* hi4 = reinterpret_cast<float*>(tile + lr * 128 + (((u + 1) ^ (lr & 7)) << 4));
        float v[8];
        *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(lo4);
        *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(hi4);
        const bool in = row < job.M && c < job.N;
        float other[8];
        before.planes(it, other);
        if constexpr (TERMS == 1 && !SYM) {  // c0 X, at the product's scale
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = fmaf(job.c0 * kPlaneScale, other[j], v[j]);
        }
        if constexpr (MODE == RESULT) {
            const int64_t at = ((int64_t)z * job.M + row) * job.N + c;
            constexpr float one = 1.f / (kPlaneScale * kPlaneScale);
#pragma unroll
            for (int j = 0; j < 8; j += 4) {
                const int left = job.N - c - j;
                if (in && left > 0)
                    job.io.put(before.raw[2 * it + j / 4], at + j, left < 4 ? left : 4, job.vec && left >= 4,
                               make_float4(v[j] * one, v[j + 1] * one, v[j + 2] * one, v[j + 3] * one));
            }
        } else {
            // products carry the square of the planes' scale; the rows' padding (to ld) may be written
            const int64_t at = (int64_t)z * job.out.stride + (int64_t)row * job.out.ld + c;
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] *= 1.f / kPlaneScale;
            if constexpr (MODE == POLY) {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    v[j] = fmaf(job.c2, v[j], job.c1 * other[j]) +
                           (TERMS == 3 && c + j == row ? job.c0 * kPlaneScale : 0.f);
            }
            if (in && (!SYM || c > row)) {
                put8(job.out, at, v);
            } else if (in && c + 7 >= row) {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (c + j >= row && c + j < job.N) put(job.out, at + j, v[j]);
            }
            if constexpr (SYM) {
                *reinterpret_cast<float4*>(lo4) = *reinterpret_cast<const float4*>(v);
                *reinterpret_cast<float4*>(hi4) = *reinterpret_cast<const float4*>(v + 4);
            }
        }
    }
    if constexpr (SYM) {  // the mirrored entries: row c0 + ., eight columns of it a lane
        __syncwarp();
#pragma unroll
        for (int it = 0; it < 4; it++) {
            const int lc = 8 * it + (lane >> 2), lr = 8 * (lane & 3), row = c0 + lc, c = r0 + lr;
            if (row >= job.N || c >= job.M || c >= row) continue;
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j++)
                v[j] = *reinterpret_cast<const float*>(tile + (lr + j) * 128 + (((lc >> 2) ^ j) << 4) + 4 * (lc & 3));
            const int64_t at = (int64_t)z * job.out.stride + (int64_t)row * job.out.ld + c;
            if (c + 7 < row && c + 7 < job.M) {
                put8(job.out, at, v);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (c + j < row && c + j < job.M) put(job.out, at + j, v[j]);
            }
        }
    }
}

// pieces x 32 columns of a warp's 32 rows of an accumulator, added to what stands in global memory (first: put there).
// A lane comes back to its own places, in order.
__device__ __forceinline__ void add_piece(uint32_t tmem, int pieces, bool first, float4* so_far) {
#pragma unroll 1
    for (int b = 0; b < pieces; b++) {
        uint32_t r[32];
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
            "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
              "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
              "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
              "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
            : "r"(tmem + 32 * b));
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int u = 0; u < 8; u++) {
            float4 v = make_float4(__uint_as_float(r[4 * u]), __uint_as_float(r[4 * u + 1]), __uint_as_float(r[4 * u + 2]),
                                   __uint_as_float(r[4 * u + 3]));
            float4* to = so_far + 256 * b + 32 * u;
            if (!first) {
                const float4 p = *to;
                v = make_float4(p.x + v.x, p.y + v.y, p.z + v.z, p.w + v.w);
            }
            *to = v;
        }
    }
}

// Tiles on persistent blocks, one an SM: warp 0 loads (TMA), one lane of warp 1 (of a pair's first block) issues the MMAs into
// two accumulators in turn, and warps 2 to 9 take each through the mode's epilogue (tensor-memory lanes 32
// (w % 4) .., half of the columns) while the next one is made: the epilogue, up to 8 us a tile beside 11 us
// of products, costs time only after a block's last tile.  A wait that gives up (never, in a correct run)
// makes the block's results from then on NaN.  LONG: sums that take more than one accumulator; all but a tile's last are
// added up in global memory, by the lanes that read them, while the next one is made.
template <int MODE, bool A_MN, bool B_MN, int TERMS, bool PAIR, int BN, bool LONG, typename Io>
__global__ void __launch_bounds__(kGemmThreads, 1) k_product(const __grid_constant__ Maps maps, const Job<Io> job) {
    using G = Cfg<TERMS, PAIR, BN>;
    constexpr int KS = G::KS, STAGES = G::STAGES;
    constexpr bool SPLIT = MODE == GRAM && BN == 64;  // may share tiles
    constexpr bool SYM = MODE == GRAM || MODE == POLY;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* turned = smem + STAGES * G::STAGE_BYTES;  // a 32 x 32 piece of each epilogue warp
    uint64_t* bars = reinterpret_cast<uint64_t*>(turned + kEpilogueWarps * 4096);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 4);
    const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + STAGES), acc_full = smem_u32(bars + 2 * STAGES);
    const uint32_t acc_empty = acc_full + 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int slices = (job.K + KS - 1) / KS;
    const int half = PAIR ? (int)(blockIdx.x & 1) : 0;  // of the pair: the cluster is two blocks along x
    const int first_tile = PAIR ? blockIdx.x >> 1 : blockIdx.x, tile_step = PAIR ? gridDim.x >> 1 : gridDim.x;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 1);
        }
        for (int a = 0; a < 2; a++) {
            mbar_init(acc_full + 8 * a, 1);
            mbar_init(acc_empty + 8 * a, (PAIR ? 2 : 1) * kEpilogueWarps);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if constexpr (PAIR) cluster_sync();  // both blocks are there, with their barriers
    if (warp == 1) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                         "r"((uint32_t)(2 * BN))
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                         "r"((uint32_t)(2 * BN))
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    if constexpr (PAIR) cluster_sync();
    else __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    wait_for_previous();
    let_next_start();

    if (warp == 0) {
        if (lane == 0) {
            int i = 0;
            bool ok = true;
            for (int t = first_tile; t < job.total && ok; t += tile_step) {
                int z, m0, n0;
                tile_at<SYM, G::TILE_M, BN>(job, SPLIT ? t / job.splits : t, z, m0, n0);
                m0 += half * BM, n0 += half * G::B_ROWS;
                const int part = SPLIT ? t % job.splits : 0, parts = SPLIT ? job.splits : 1;
                for (int k = slices * part / parts; k < slices * (part + 1) / parts; k++, i++) {
                    const int s = i % STAGES, round = i / STAGES;
                    if (round > 0) ok = mbar_wait(empty0 + 8 * s, (uint32_t)((round - 1) & 1), nullptr);
                    if (!ok) break;
                    const uint32_t bar = PAIR ? leaders(full0 + 8 * s) : full0 + 8 * s;
                    const uint32_t st = smem_u32(smem + s * G::STAGE_BYTES);
                    if (half == 0) mbar_expect_tx(full0 + 8 * s, (PAIR ? 2 : 1) * G::STAGE_BYTES);  // of both blocks
                    load_operand<A_MN, KS, BM, PAIR>(st, &maps.a_hi, m0, k * KS, z, bar);
                    load_operand<B_MN, KS, G::B_ROWS, PAIR>(st + G::A_BYTES, &maps.b_hi, n0, k * KS, z, bar);
                    if constexpr (TERMS == 3) {
                        load_operand<A_MN, KS, BM, PAIR>(st + G::A_BYTES + G::B_BYTES, &maps.a_lo, m0, k * KS, z, bar);
                        load_operand<B_MN, KS, G::B_ROWS, PAIR>(st + 2 * G::A_BYTES + G::B_BYTES, &maps.b_lo, n0, k * KS, z,
                                                                bar);
                    }
                }
            }
            // every load issued into this block's shared memory has landed before it ends (a pair's: both
            // blocks', before either passes the last barrier)
            if (half == 0)
                for (int k = i > STAGES ? i - STAGES : 0; k < i; k++)
                    mbar_wait(full0 + 8 * (k % STAGES), (uint32_t)((k / STAGES) & 1), nullptr);
        }
    } else if (warp == 1) {
        if (lane == 0 && half == 0) {
            int i = 0, made = 0;
            bool ok = true;
            for (int t = first_tile; t < job.total && ok; t += tile_step) {
                const int part = SPLIT ? t % job.splits : 0, parts = SPLIT ? job.splits : 1;
                const int begin = slices * part / parts, count = slices * (part + 1) / parts - begin;
                const int chunks = LONG ? (count + G::CHUNK - 1) / G::CHUNK : 1;
                for (int c = 0; c < chunks; c++, made++) {
                    const int acc = made & 1;
                    if (made >= 2) ok = ok && mbar_wait(acc_empty + 8 * acc, (uint32_t)((made / 2 - 1) & 1), nullptr);
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t d = tmem + acc * BN;
                    const int n0 = (int)((int64_t)count * c / chunks), n1 = (int)((int64_t)count * (c + 1) / chunks);
                    for (int n = n0; n < n1 && ok; n++, i++) {
                        const int s = i % STAGES;
                        ok = mbar_wait(full0 + 8 * s, (uint32_t)((i / STAGES) & 1), nullptr);
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint32_t a = smem_u32(smem + s * G::STAGE_BYTES), b = a + G::A_BYTES;
                        const uint32_t alo = b + G::B_BYTES, blo = alo + G::A_BYTES;
#pragma unroll
                        for (int k = 0; k < KS / 16; k++) {  // 16 of K: 32 bytes along it, 16 rows of 128 bytes across it
                            constexpr uint32_t sa = A_MN ? 2048 : 32, sb = B_MN ? 2048 : 32;
                            const uint64_t ah = operand_desc<A_MN, KS>(a + sa * k), bh = operand_desc<B_MN, KS>(b + sb * k);
                            const uint32_t first = (n > n0 || k > 0) ? 1u : 0u;
                            if constexpr (TERMS == 3) {  // the small terms first
                                umma_f16<A_MN, B_MN, PAIR, BN>(d, operand_desc<A_MN, KS>(alo + sa * k), bh, first);
                                umma_f16<A_MN, B_MN, PAIR, BN>(d, ah, operand_desc<B_MN, KS>(blo + sb * k), 1u);
                                umma_f16<A_MN, B_MN, PAIR, BN>(d, ah, bh, 1u);
                            } else {
                                umma_f16<A_MN, B_MN, PAIR, BN>(d, ah, bh, first);
                            }
                        }
                        commit<PAIR>(empty0 + 8 * s);
                    }
                    if (!ok) break;  // no accumulator any more: the epilogues' waits give up in their turn
                    commit<PAIR>(acc_full + 8 * acc);
                }
            }
        }
        __syncwarp();
    } else {
        const int w = warp & 3, part = (warp - 2) >> 2;
        int made = 0;
        bool ok = true;
        float4* so_far = job.carry + ((int64_t)blockIdx.x * kEpilogueWarps + warp - 2) * (BN * 4) + lane;
        for (int t = first_tile; t < job.total; t += tile_step, made++) {
        int z, m0, n0;
        tile_at<SYM, G::TILE_M, BN>(job, SPLIT ? t / job.splits : t, z, m0, n0);
        m0 += half * BM;
        const int share = SPLIT ? t % job.splits : 0, shares = SPLIT ? job.splits : 1;
        const int count = slices * (share + 1) / shares - slices * share / shares;
        const int chunks = LONG ? (count + G::CHUNK - 1) / G::CHUNK : 1;
        for (int c = 0; c + 1 < chunks; c++, made++) {  // all but the last accumulator of a long sum
            const int acc = made & 1;
            ok = ok && mbar_wait(acc_full + 8 * acc, (uint32_t)((made / 2) & 1), nullptr);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            add_piece(tmem + ((uint32_t)(32 * w) << 16) + (uint32_t)(acc * BN + part * (BN / 2)), BN / 64, c == 0, so_far);
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR) mbar_arrive_leader(leaders(acc_empty + 8 * acc));
                else mbar_arrive(acc_empty + 8 * acc);
            }
        }
        const int acc = made & 1;
        ok = ok && mbar_wait(acc_full + 8 * acc, (uint32_t)((made / 2) & 1), nullptr);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        uint8_t* tile = turned + (warp - 2) * 4096;
        for (int col = part * (BN / 2); col < (part + 1) * (BN / 2); col += 32) {
            const int r0 = m0 + 32 * w, c0 = n0 + col;
            Before<MODE, TERMS, Io> before;
            before.fetch(job, z, r0, c0, lane);
            uint32_t r[32];
            asm volatile(
                "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
                "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                  "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
                  "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
                  "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
                  "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                : "r"(tmem + ((uint32_t)(32 * w) << 16) + (uint32_t)(acc * BN + col)));
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            if (col + 32 == (part + 1) * (BN / 2)) {  // this warp's part of the accumulator has been read
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    if constexpr (PAIR) mbar_arrive_leader(leaders(acc_empty + 8 * acc));
                    else mbar_arrive(acc_empty + 8 * acc);
                }
            }
            if (r0 >= job.M || c0 >= job.N) continue;
            if constexpr (SYM)
                if (c0 + 31 < r0) continue;  // below the diagonal: its mirror image is computed
            // Through shared memory, so that four lanes take 64 consecutive bytes of a row: a lane has a row of
            // the accumulator, and 16 bytes of each of 32 rows a store are half a sector each, at a fifth of
            // the rate.
            __syncwarp();
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const uint32_t nan = 0x7fc00000u;
                *reinterpret_cast<uint4*>(tile + lane * 128 + ((u ^ (lane & 7)) << 4)) =
                    ok ? make_uint4(r[4 * u], r[4 * u + 1], r[4 * u + 2], r[4 * u + 3]) : make_uint4(nan, nan, nan, nan);
            }
            if (LONG && chunks > 1) {
#pragma unroll
                for (int u = 0; u < 8; u++) {
                    const float4 p = so_far[(col - part * (BN / 2)) * 8 + 32 * u];
                    float4* v = reinterpret_cast<float4*>(tile + lane * 128 + ((u ^ (lane & 7)) << 4));
                    *v = make_float4(v->x + p.x, v->y + p.y, v->z + p.z, v->w + p.w);
                }
            }
            __syncwarp();
            if (SPLIT && job.partial) {
                float* to = job.partial + ((int64_t)t * BM + 32 * w) * BN + col;
#pragma unroll
                for (int it = 0; it < 4; it++) {
                    const int lr = 8 * it + (lane >> 2), u = 2 * (lane & 3);
#pragma unroll
                    for (int j = 0; j < 2; j++)
                        *reinterpret_cast<uint4*>(to + lr * BN + 4 * (u + j)) =
                            *reinterpret_cast<const uint4*>(tile + lr * 128 + (((u + j) ^ (lr & 7)) << 4));
                }
            } else {
                finish_piece<MODE, TERMS, Io>(job, tile, before, z, r0, c0, lane);
            }
        }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    if constexpr (PAIR) cluster_sync();  // the partner reads this block's operands, and arrives at its barriers
    else __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if constexpr (PAIR)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)(2 * BN))
                         : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)(2 * BN))
                         : "memory");
    }
}

// The tiles that blocks shared: their sums, and the mode's work.  A block a 32 x 32 piece: warp w sums splits w, w + 8,
// .., and the warps are added in their order.
template <int TERMS, typename Io>
__global__ void __launch_bounds__(256) k_sum_tiles(const Job<Io> job) {
    constexpr int BN = 64;
    __shared__ __align__(128) float4 sums[8][8][32];
    __shared__ __align__(128) uint8_t tile[4096];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, piece = blockIdx.x & 7, t = blockIdx.x >> 3;
    int z, m0, n0;
    tile_at<true, BM, BN>(job, t, z, m0, n0);
    const int r0 = m0 + 32 * (piece & 3), c0 = n0 + 32 * (piece >> 2);
    wait_for_previous();
    let_next_start();
    if (r0 >= job.M || c0 >= job.N || c0 + 31 < r0) return;
    const float* from = job.partial + ((int64_t)t * job.splits * BM + 32 * (piece & 3)) * BN + 32 * (piece >> 2);
    const int u = 2 * (lane & 3);
    float4 v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = warp; k < job.splits; k += 8)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int lr = 8 * (i >> 1) + (lane >> 2);
            const float4 p = *reinterpret_cast<const float4*>(from + ((int64_t)k * BM + lr) * BN + 4 * (u + (i & 1)));
            v[i].x += p.x, v[i].y += p.y, v[i].z += p.z, v[i].w += p.w;
        }
#pragma unroll
    for (int i = 0; i < 8; i++) sums[warp][i][lane] = v[i];
    __syncthreads();
    if (warp != 0) return;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        float4 w = sums[0][i][lane];
        for (int k = 1; k < 8; k++) {
            const float4 p = sums[k][i][lane];
            w.x += p.x, w.y += p.y, w.z += p.z, w.w += p.w;
        }
        const int lr = 8 * (i >> 1) + (lane >> 2);
        *reinterpret_cast<float4*>(tile + lr * 128 + (((u + (i & 1)) ^ (lr & 7)) << 4)) = w;
    }
    __syncwarp();
    const Before<GRAM, TERMS, Io> before = {};
    finish_piece<GRAM, TERMS, Io>(job, tile, before, z, r0, c0, lane);
}

// ---- host ---------------------------------------------------------------------------


struct Shape {
    int64_t stack, rows, cols, side, length;  // side <= length
    bool tall;                                // stored [length, side]
};

// Chunks of the long side, in whole tiles, for about four blocks an SM.
int64_t small_chunk(const Shape& s) {
    const int64_t kt = s.side <= 16 ? 128 : 64, tiles = ceil_div(s.length, kt), per = ceil_div(4 * 148, s.stack);
    return ceil_div(tiles, per < tiles ? per : tiles) * kt;
}
int small_side(const Shape& s) { return s.side <= 8 ? 8 : s.side <= 16 ? 16 : s.side <= 32 ? 32 : 64; }

constexpr int kNormBlocks = 592;
int64_t norm_blocks(const Shape& s) {
    const int64_t want = ceil_div(s.rows * s.cols, 16 * kNormThreads), most = ceil_div(kNormBlocks, s.stack);
    return want < most ? want : most;
}

int64_t pad64(int64_t c) { return (c + 63) & ~int64_t(63); }

constexpr int kSplitTiles = 148;  // 128 x 64 tiles' sums that blocks share
constexpr int kMostBlocks = 148;  // of k_product: the workspace holds a tile's sum for each

struct Layout {
    int64_t part, pmat;                     // small
    int64_t partial, carry, x[2], g, b, bytes;  // planes: hi, then lo
    int64_t x_plane, s_plane;               // bytes of one plane
};

Layout layout_of(const Shape& s, int terms) {
    Layout l = {};
    int64_t at = 0;
    const auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += align256(bytes);
        return here;
    };
    if (s.side <= kSmallSide) {
        const int64_t rm = small_side(s), chunks = ceil_div(s.length, small_chunk(s));
        l.part = take(s.stack * chunks * rm * rm * 8);
        l.pmat = take(s.stack * rm * rm * 8);
    } else {
        l.part = take(s.stack * norm_blocks(s) * 8);
        l.partial = take(kSplitTiles * (int64_t)BM * 64 * 4);
        l.carry = take(s.length > (terms == 3 ? kChunk3 : kChunk1) ? kMostBlocks * (int64_t)BM * 256 * 4 : 0);
        l.x_plane = align256(s.stack * s.rows * pad64(s.cols) * 2);
        l.s_plane = align256(s.stack * s.side * pad64(s.side) * 2);
        const int planes = terms == 3 ? 2 : 1;
        for (int64_t* p : {&l.x[0], &l.x[1]}) *p = take(2 * l.x_plane);
        for (int64_t* p : {&l.g, &l.b}) *p = take(planes * l.s_plane);
    }
    l.bytes = at;
    return l;
}

// Elements of a matrix's chunks above which k_small_sum adds them.  In k_small_poly and in a launch of its own, fp32:
// 16 x 2560 (5120 elements) 11.4 and 12.4 us, 40 of 16 x 12800 (3840) 39 and 45, 8 x 12800 (6400) 12.9 and 12.7; 40 of
// 32 x 12800 (15360) 129 and 108, 64 x 2560 (163840) 99 and 74, 64 x 12800 (819200) 239 and 96.
constexpr int kSumElements = 8192;

template <int MB, bool TALL, typename Io>
int run_small(const Shape& s, const Layout& l, const Io& io, const Poly& poly, double eps, uint8_t* ws,
              cudaStream_t st) {
    using S = SmallTile<MB, TALL>;
    const int64_t chunk = small_chunk(s), chunks = ceil_div(s.length, chunk);
    double *part = (double*)(ws + l.part), *pmat = (double*)(ws + l.pmat);
    const dim3 grid((unsigned)chunks, (unsigned)s.stack);
    const bool vec = io.aligned && (TALL ? s.side : s.length) % 4 == 0;
    constexpr int RM = 8 * MB, SP = RM + 4;
    int e = start<k_small_gram<MB, TALL, Io>>(grid, kSmallThreads, 0, false, st, io, (int)s.side, s.length, chunk, vec,
                                              part);
    const bool sum = chunks * RM * RM > kSumElements;
    const int64_t total = s.stack * RM * RM;
    if (!e && sum)
        e = start<k_small_sum>(dim3((unsigned)ceil_div(total, kSmallThreads)), kSmallThreads, 0, true, st, part, (int)chunks,
                               RM * RM, total);
    if (!e)
        e = start<k_small_poly<MB>>(dim3((unsigned)s.stack), kPolyThreads<MB>, 4 * RM * SP * 8, true, st, part,
                                    sum ? 1 : (int)chunks, (int)chunks, (int)s.side, poly, eps, pmat);
    if (!e)
        e = start<k_small_apply<MB, TALL, Io>>(grid, kSmallThreads, RM * SP * 8 + S::SIZE * 4, true, st, io, (int)s.side,
                                               s.length, chunk, vec, pmat);
    return e;
}

// Map of one plane [stack, rows, ld] of which `cols` columns count, in boxes of bx columns and by rows.
bool plane_map(CUtensorMap* map, const __half* base, int64_t rows, int64_t cols, int64_t ld, int64_t stride,
               int64_t stack, int bx, int by) {
    const auto fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)stack};
    const cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)stride * 2};
    const cuuint32_t box[3] = {(cuuint32_t)bx, (cuuint32_t)by, 1}, step[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(base), dims, strides, box, step,
              CU_TENSOR_MAP_INTERLEAVE_NONE, bx == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Matrix {  // a plane pair and its extent
    Planes p;
    int64_t rows, cols;
};

// Pairs of blocks that the device runs at once (every k_product takes an SM a block).
int pairs_at_once(const void* kernel, int smem) {
    static int cached[64] = {0};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return 64;
    if (cached[dev] == 0) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(148);
        cfg.blockDim = dim3(kGemmThreads);
        cfg.dynamicSmemBytes = (size_t)smem;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim = {2, 1, 1};
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
            cudaGetLastError();
            n = 64;
        }
        cached[dev] = n;
    }
    return cached[dev];
}

// Tiles of TILE_M x BN of an M x N product (symmetric: those that reach the diagonal or lie above it).
int64_t count_tiles(bool sym, int64_t M, int64_t N, int tile_m, int bn) {
    const int64_t tm = ceil_div(M, tile_m), tn = ceil_div(N, bn);
    if (!sym) return tm * tn;
    int64_t n = 0;
    for (int64_t b = 0; b < tn; b++) n += std::min((bn * (b + 1) - 1) / tile_m + 1, tm);
    return n;
}

template <int MODE, bool A_MN, bool B_MN, int TERMS, bool PAIR, int BN, typename Io>
int run_tiles(const Matrix& a, const Matrix& b, int64_t stack, Job<Io> job, cudaStream_t st) {
    using G = Cfg<TERMS, PAIR, BN>;
    constexpr bool SYM = MODE == GRAM || MODE == POLY;
    Maps maps;
    memset(&maps, 0, sizeof(maps));
    const auto make = [&](CUtensorMap* map, const __half* plane, const Matrix& x, bool mn, int tile_rows) {
        return mn ? plane_map(map, plane, x.rows, x.cols, x.p.ld, x.p.stride, stack, 64, G::KS)
                  : plane_map(map, plane, x.rows, x.cols, x.p.ld, x.p.stride, stack, G::KS, tile_rows);
    };
    if (!make(&maps.a_hi, a.p.hi, a, A_MN, BM) || !make(&maps.b_hi, b.p.hi, b, B_MN, G::B_ROWS)) return ENGRAM_ERR_CUDA;
    if (TERMS == 3 && (!make(&maps.a_lo, a.p.lo, a, A_MN, BM) || !make(&maps.b_lo, b.p.lo, b, B_MN, G::B_ROWS)))
        return ENGRAM_ERR_CUDA;
    job.tiles_m = (int)ceil_div(job.M, G::TILE_M), job.tiles_n = (int)ceil_div(job.N, BN);
    const int64_t tiles = count_tiles(SYM, job.M, job.N, G::TILE_M, BN);
    if (tiles * stack > INT32_MAX) return ENGRAM_ERR_RANGE;
    job.tiles = (int)tiles;
    job.splits = 1;
    if (MODE == GRAM && BN == 64 && job.partial)
        job.splits = (int)std::max<int64_t>(1, std::min<int64_t>(kSplitTiles / (tiles * stack), ceil_div(job.K, 4 * G::KS)));
    if (job.splits == 1) job.partial = nullptr;
    job.total = (int)(tiles * stack * job.splits);
    // Where a sum is longer than an accumulator takes.  But for a Gram matrix the sums are as long as the short side,
    // and those of 4096 and more have tiles for pairs.
    constexpr bool MAY = PAIR || MODE == GRAM;
    const bool longer = ceil_div(ceil_div(job.K, G::KS), job.splits) > G::CHUNK;
    constexpr auto kernel = k_product<MODE, A_MN, B_MN, TERMS, PAIR, BN, false, Io>;
    constexpr auto kernel_longer = k_product<MODE, A_MN, B_MN, TERMS, PAIR, BN, MAY, Io>;
    if (longer && !MAY) return ENGRAM_ERR_RANGE;
    const int most = PAIR ? std::min(pairs_at_once((const void*)kernel, G::SMEM), kMostBlocks / 2)
                          : std::min(sm_count(), kMostBlocks);
    const int blocks = (PAIR ? 2 : 1) * std::min(job.total, most);
    const dim3 grid((unsigned)blocks);
    int e = longer ? start<kernel_longer, 0, PAIR ? 2 : 1>(grid, kGemmThreads, G::SMEM, true, st, maps, job)
                   : start<kernel, 0, PAIR ? 2 : 1>(grid, kGemmThreads, G::SMEM, true, st, maps, job);
    if constexpr (MODE == GRAM && BN == 64) {
        if (!e && job.partial)
            e = start<k_sum_tiles<TERMS, Io>>(dim3((unsigned)(8 * tiles * stack)), 256, 0, true, st, job);
    }
    return e;
}

// Which tiles: 256 x 256 on pairs of blocks where there are 50 or more of them, else 128 x 64 while every block gets
// at most one, else 128 x 256.  Pairs against 128 x 256, all steps: 10240 x 2560 in bf16 1124 against 1183 us, 2560 x
// 2560 in fp32 1041 against 1056; but 2048 x 2048 in bf16 362 against 350, 1024 x 1024 266 against 250.  128 x 64
// against 128 x 256: 1024 x 1024 in fp32 310 against 389, 256 x 256 147 against 218; but, at two a block, 1536 x 1536
// 619 against 514.
template <int MODE, bool A_MN, bool B_MN, int TERMS, typename Io>
int run_product(const Matrix& a, const Matrix& b, int64_t stack, const Job<Io>& job, cudaStream_t st) {
    constexpr bool SYM = MODE == GRAM || MODE == POLY;
    if (count_tiles(SYM, job.M, job.N, 256, 256) * stack >= 50)
        return run_tiles<MODE, A_MN, B_MN, TERMS, true, 256>(a, b, stack, job, st);
    if (count_tiles(SYM, job.M, job.N, 128, 64) * stack <= 148)
        return run_tiles<MODE, A_MN, B_MN, TERMS, false, 64>(a, b, stack, job, st);
    return run_tiles<MODE, A_MN, B_MN, TERMS, false, 256>(a, b, stack, job, st);
}

template <int TERMS, typename Io>
int run_planes(const Shape& s, const Layout& l, const Io& io, const Poly& poly, double eps, uint8_t* ws,
               cudaStream_t st) {
    double* part = (double*)(ws + l.part);
    const int64_t ldx = pad64(s.cols), lds = pad64(s.side);
    const auto planes = [&](int64_t at, int64_t plane, int64_t ld, int64_t rows, bool two) {
        return Planes{(__half*)(ws + at), two ? (__half*)(ws + at + plane) : nullptr, ld, rows * ld};
    };
    const Matrix x[2] = {{planes(l.x[0], l.x_plane, ldx, s.rows, true), s.rows, s.cols},
                         {planes(l.x[1], l.x_plane, ldx, s.rows, true), s.rows, s.cols}};
    const Matrix g = {planes(l.g, l.s_plane, lds, s.side, TERMS == 3), s.side, s.side};
    const Matrix b = {planes(l.b, l.s_plane, lds, s.side, TERMS == 3), s.side, s.side};
    const bool vec = io.aligned && s.cols % 4 == 0;
    const int nb = (int)norm_blocks(s);
    int e = start<k_norm<Io>>(dim3((unsigned)nb, (unsigned)s.stack), kNormThreads, 0, false, st, io, s.rows * s.cols,
                              io.aligned && s.rows * s.cols % 4 == 0, part);
    if (e) return e;
    const int64_t row_blocks = ceil_div(s.rows * ceil_div(s.cols, 512), kNormThreads / 32), most = ceil_div(8 * 148, s.stack);
    e = start<k_planes<Io>>(dim3((unsigned)(row_blocks < most ? row_blocks : most), (unsigned)s.stack), kNormThreads, 0,
                            true, st, io, s.rows, s.cols, vec, part, nb, eps, x[0].p);
    Job<NoIo> job = {};
    job.partial = (float*)(ws + l.partial);
    job.carry = (float4*)(ws + l.carry);
    for (int i = 0; i < poly.steps && !e; i++) {
        const Matrix &in = x[i & 1], &next = x[(i & 1) ^ 1];
        job.M = job.N = (int)s.side;
        job.K = (int)s.length;
        job.out = g.p;
        e = s.tall ? run_product<GRAM, true, true, TERMS>(in, in, s.stack, job, st)
                   : run_product<GRAM, false, false, TERMS>(in, in, s.stack, job, st);
        if (e) break;
        job.K = (int)s.side;
        job.out = b.p;
        job.g = g.p;
        job.c0 = (float)poly.c[i][0], job.c1 = (float)poly.c[i][1], job.c2 = (float)poly.c[i][2];
        e = run_product<POLY, false, false, TERMS>(g, g, s.stack, job, st);
        if (e) break;
        job.M = (int)s.rows;
        job.N = (int)s.cols;
        job.out = next.p;
        job.g = in.p;
        if (i + 1 < poly.steps) {
            e = s.tall ? run_product<UPDATE, false, false, TERMS>(in, b, s.stack, job, st)
                       : run_product<UPDATE, false, true, TERMS>(b, in, s.stack, job, st);
        } else {
            Job<Io> result = {};
            result.M = job.M, result.N = job.N, result.K = job.K;
            result.io = io;
            result.vec = vec;
            result.g = in.p, result.c0 = job.c0, result.carry = job.carry;
            e = s.tall ? run_product<RESULT, false, false, TERMS>(in, b, s.stack, result, st)
                       : run_product<RESULT, false, true, TERMS>(b, in, s.stack, result, st);
        }
    }
    return e;
}

template <int TERMS, typename Io>
int run(const Shape& s, const Layout& l, const Io& io, const Poly& poly, double eps, void* ws, void* stream) {
    uint8_t* w = (uint8_t*)ws;
    cudaStream_t st = (cudaStream_t)stream;
    const auto small = [&](auto mb) {
        constexpr int MB = decltype(mb)::value;
        return s.tall ? run_small<MB, true>(s, l, io, poly, eps, w, st) : run_small<MB, false>(s, l, io, poly, eps, w, st);
    };
    if (s.side <= 8) return small(std::integral_constant<int, 1>{});
    if (s.side <= 16) return small(std::integral_constant<int, 2>{});
    if (s.side <= 32) return small(std::integral_constant<int, 4>{});
    if (s.side <= kSmallSide) return small(std::integral_constant<int, 8>{});
    return run_planes<TERMS>(s, l, io, poly, eps, w, st);
}

int check_shape(int64_t stack, int64_t rows, int64_t cols, Shape* s) {
    if (stack < 0 || rows < 1 || cols < 1) return ENGRAM_ERR_ARG;
    if (stack > 65535 || rows > (1 << 24) || cols > (1 << 24) || (rows < cols ? rows : cols) > (1 << 15))
        return ENGRAM_ERR_RANGE;
    s->stack = stack, s->rows = rows, s->cols = cols;
    s->tall = rows > cols;
    s->side = s->tall ? cols : rows;
    s->length = s->tall ? rows : cols;
    return ENGRAM_OK;
}

// The iterates have to stay within what the planes hold: from singular values in [0, 1] on, each step's
// G, polynomial and result below 15.  `top` is the largest singular value that a step can meet, found on a
// grid over all that the step before can leave.  apart: c0 X is added beside the product (one term of longer
// sides), so the plane holds the polynomial without c0, which may be the larger one.
int check_poly(int32_t steps, const double* c, double eps, bool apart, Poly* poly) {
    if (steps < 1 || !c || !(eps > 0.0)) return ENGRAM_ERR_ARG;
    if (steps > kMaxSteps) return ENGRAM_ERR_RANGE;
    poly->steps = steps;
    constexpr int kPoints = 128;
    double top = 1.0;
    for (int i = 0; i < steps; i++) {
        const double c0 = c[3 * i], c1 = c[3 * i + 1], c2 = c[3 * i + 2];
        poly->c[i][0] = c0, poly->c[i][1] = c1, poly->c[i][2] = c2;
        double f_most = 0.0, x_most = 0.0;
        bool number = true;
        for (int p = 0; p <= kPoints; p++) {
            const double x = top * p / kPoints, g = x * x, rest = g * (c1 + g * c2), f = fabs(c0 + rest), y = x * f;
            const double held = apart && fabs(rest) > f ? fabs(rest) : f;
            number = number && held < 1e30;
            f_most = held > f_most ? held : f_most;
            x_most = y > x_most ? y : x_most;
        }
        if (!number || !(top * top < 15.0) || !(f_most < 15.0) || !(x_most < 3.8)) return ENGRAM_ERR_RANGE;
        top = x_most;
    }
    return ENGRAM_OK;
}

int terms_of(int32_t dtype) { return dtype == ENGRAM_DTYPE_BF16 ? 1 : 3; }


}  // namespace

int64_t engram::ortho_waits_given_up() { return read_given_up(g_waits_given_up); }

namespace {
__global__ void k_wait_for_nothing() {
    __shared__ uint64_t bar;
    mbar_init(smem_u32(&bar), 1);
    mbar_wait(smem_u32(&bar), 0, nullptr, 1000);
}
}  // namespace

extern "C" int64_t engram_waits_given_up(void) {
    if (cudaDeviceSynchronize() != cudaSuccess) return ENGRAM_ERR_CUDA;
    int64_t sum = 0;
    for (const int64_t v : {gemm_waits_given_up(), adapter_waits_given_up(), ortho_waits_given_up()}) {
        if (v < 0) return v;
        sum += v;
    }
    return sum;
}

extern "C" int engram_selftest_wait(void* stream) {
    k_wait_for_nothing<<<1, 1, 0, (cudaStream_t)stream>>>();
    count_launches(1);
    return cudaGetLastError() == cudaSuccess ? ENGRAM_OK : ENGRAM_ERR_CUDA;
}

extern "C" int64_t engram_orthogonalize_workspace_bytes(int32_t dtype, int64_t stack, int64_t rows, int64_t cols) {
    if (dtype < ENGRAM_DTYPE_F32 || dtype > ENGRAM_DTYPE_F16) return ENGRAM_ERR_FORMAT;
    Shape s;
    const int e = check_shape(stack, rows, cols, &s);
    if (e) return e;
    return stack ? layout_of(s, terms_of(dtype)).bytes : 0;
}

extern "C" int engram_orthogonalize(int32_t dtype, const void* x, int64_t stack, int64_t rows, int64_t cols,
                                    int32_t steps, const double* coefficients, double eps, void* out, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
    if (dtype < ENGRAM_DTYPE_F32 || dtype > ENGRAM_DTYPE_F16) return ENGRAM_ERR_FORMAT;
    Shape s;
    int e = check_shape(stack, rows, cols, &s);
    if (e) return e;
    Poly poly;
    e = check_poly(steps, coefficients, eps, terms_of(dtype) == 1 && s.side > kSmallSide, &poly);
    if (e) return e;
    if (stack == 0) return ENGRAM_OK;
    if (!x || !out || !aligned_to(x, dtype) || !aligned_to(out, dtype) || !workspace || !aligned16(workspace))
        return ENGRAM_ERR_ARG;
    const Layout l = layout_of(s, terms_of(dtype));
    if (workspace_bytes < l.bytes) return ENGRAM_ERR_WORKSPACE;
    const bool four = aligned16(x) && aligned16(out);
    switch (dtype) {
        case ENGRAM_DTYPE_F32:
            return run<3>(s, l, Plain<float>{(const float*)x, (float*)out, four}, poly, eps, workspace, stream);
        case ENGRAM_DTYPE_BF16:
            return run<1>(s, l, Plain<__nv_bfloat16>{(const __nv_bfloat16*)x, (__nv_bfloat16*)out, four}, poly,
                          eps, workspace, stream);
        default:
            return run<3>(s, l, Plain<__half>{(const __half*)x, (__half*)out, four}, poly, eps, workspace, stream);
    }
}

extern "C" int engram_muon_step(int32_t grad_dtype, const float* p, const void* grad, const float* m, float* p_out,
                                float* m_out, int64_t stack, int64_t rows, int64_t cols, double lr, double beta,
                                int32_t nesterov, double weight_decay, int32_t steps, const double* coefficients,
                                double eps, void* workspace, int64_t workspace_bytes, void* stream) {
    if (grad_dtype < ENGRAM_DTYPE_F32 || grad_dtype > ENGRAM_DTYPE_F16) return ENGRAM_ERR_FORMAT;
    Shape s;
    int e = check_shape(stack, rows, cols, &s);
    if (e) return e;
    Poly poly;
    e = check_poly(steps, coefficients, eps, false, &poly);
    if (e) return e;
    if (stack == 0) return ENGRAM_OK;
    if (!grad || !aligned_to(grad, grad_dtype) || !workspace || !aligned16(workspace)) return ENGRAM_ERR_ARG;
    for (const float* f : {p, m, (const float*)p_out, (const float*)m_out})
        if (!f || !aligned_to(f, ENGRAM_DTYPE_F32)) return ENGRAM_ERR_ARG;
    if (p_out == m_out || p == m_out || p_out == m || p == m || grad == p_out || grad == m_out) return ENGRAM_ERR_ARG;
    const Layout l = layout_of(s, 3);
    if (workspace_bytes < l.bytes) return ENGRAM_ERR_WORKSPACE;
    const double ratio = rows > cols ? sqrt((double)rows / (double)cols) : 1.0;
    const bool four = aligned16(p) && aligned16(grad) && aligned16(m) && aligned16(p_out) && aligned16(m_out);
    const auto io = [&](auto* g) {
        using T = std::remove_cv_t<std::remove_pointer_t<decltype(g)>>;
        return MuonIo<T>{g, m, m_out, p, p_out, (float)beta, (float)(1.0 - beta), (float)(1.0 - lr * weight_decay),
                         (float)(lr * ratio), nesterov != 0, four};
    };
    switch (grad_dtype) {
        case ENGRAM_DTYPE_F32: return run<3>(s, l, io((const float*)grad), poly, eps, workspace, stream);
        case ENGRAM_DTYPE_BF16: return run<3>(s, l, io((const __nv_bfloat16*)grad), poly, eps, workspace, stream);
        default: return run<3>(s, l, io((const __half*)grad), poly, eps, workspace, stream);
    }
}
