// engram_adapter.cu -- low-rank adapters of many requests beside a shared
// projection: out[t] = base[t] + s_i B_i (A_i x[t]) with i = index[t], A_i
// [rank, K] and B_i [N, rank], and the gradients of x, A and B.
//
// Positions are first grouped by adapter (k_plan), so that each tile of 16 or 32
// positions reads one adapter's factors.  Three products are then needed:
//   shrink  h[p, :] = s_i A_i x[t]          (sums over a width, rank columns out)
//   expand  out[t, :] = base[t, :] + B_i h[p, :]   (sums over the rank)
//   weight  G_i[f, :] = sum over i's positions of x[t, f] h[p, :]
// p is a position's place in the grouped order, t its row.  The backward uses the
// same three: dh = s_i B_i^T g (shrink over N), dx = A_i^T dh (expand), dA from
// (x, dh) and dB from (g, h).
//
// All three run on mma.sync m16n8k8 TF32 with fp32 accumulation, fragments loaded
// from global memory straight into registers.  The tensor work is small beside
// the bytes (2 rank flops an element of base and out), so the mma.sync rate is
// enough, and without a staging tile in shared memory nothing waits: a fragment's
// index inside a sum is arbitrary as long as both operands agree, so each lane
// takes 16 consecutive bytes of its row and the four lanes of a row 64.
//
// Arithmetic: an fp32 operand x is split as x = hi + lo, hi = x rounded to the 11
// significant bits of TF32, and a product is hi hi + hi lo + lo hi (the dropped
// term is 2^-24 of it); bf16 and fp16 values are exact in TF32 and need no split.
// h and dh, sums over a whole width, are kept in fp32 for every type.
#include "engram_common.cuh"

using namespace engram;

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kMaxAdapters = 16384;  // k_plan counts them in shared memory
constexpr int kMaxRank = 128;

// ---- the plan ----------------------------------------------------------------
// int32 arrays in the workspace.  off[i] = first place of adapter i in the grouped
// order, off[n] = first place of the positions without an adapter, off[n+1] = T;
// perm[p] = position; tile k covers places [start, start + rows) of one adapter.
struct Tile {
    int32_t adapter, start, rows, pad;
};
struct Plan {
    int32_t* off;    // [n + 2]
    int32_t* perm;   // [T]
    int32_t* tiles;  // [1]: number of tiles
    Tile* tile;      // [max tiles]
};

__device__ __forceinline__ int clamp_adapter(int32_t i, int n) { return (uint32_t)i < (uint32_t)n ? i : n; }

// Groups the positions by adapter, stable (so sums over an adapter's positions
// have one order).  Every block counts all indexes (they fit L1 and L2), and those
// before its own chunk, which gives the places of its chunk with no other block.
__global__ void __launch_bounds__(kPlanThreads) k_plan(const int32_t* __restrict__ index, int T, int n, int chunk,
                                                       int tile_rows, Plan plan) {
    extern __shared__ int32_t sm[];
    int32_t* cnt = sm;               // [n + 1], later the places' start
    int32_t* pre = cnt + n + 1;      // [n + 1]: positions of the adapter before the current ones
    int32_t* tile0 = pre + n + 1;    // [n + 2]: first tile of the adapter
    __shared__ int32_t warp_sum[2][32];
    __shared__ int32_t carry[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int c0 = blockIdx.x * chunk, c1 = min(T, c0 + chunk);
    for (int i = tid; i < 2 * (n + 1); i += kPlanThreads) sm[i] = 0;
    if (tid < 2) carry[tid] = 0;
    __syncthreads();
    for (int t0 = 0; t0 < T; t0 += kPlanThreads) {
        const int t = t0 + tid;
        const int a = t < T ? clamp_adapter(__ldg(index + t), n) : -1;
        const uint32_t same = __match_any_sync(0xffffffffu, a);
        const uint32_t before = __ballot_sync(0xffffffffu, t < c0) & same;
        if (a >= 0 && lane == __ffs(same) - 1) {
            atomicAdd(cnt + a, __popc(same));
            if (before) atomicAdd(pre + a, __popc(before));
        }
    }
    __syncthreads();
    // exclusive scans over the adapters: places, and tiles of tile_rows places
    for (int i0 = 0; i0 < n + 1; i0 += kPlanThreads) {
        const int i = i0 + tid;
        const int v0 = i <= n ? cnt[i] : 0, v1 = (v0 + tile_rows - 1) / tile_rows;
        int s0 = v0, s1 = v1;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int u0 = __shfl_up_sync(0xffffffffu, s0, d), u1 = __shfl_up_sync(0xffffffffu, s1, d);
            if (lane >= d) s0 += u0, s1 += u1;
        }
        if (lane == 31) warp_sum[0][warp] = s0, warp_sum[1][warp] = s1;
        __syncthreads();
        if (warp == 0) {
            int w0 = warp_sum[0][lane], w1 = warp_sum[1][lane];
            const int o0 = w0, o1 = w1;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int u0 = __shfl_up_sync(0xffffffffu, w0, d), u1 = __shfl_up_sync(0xffffffffu, w1, d);
                if (lane >= d) w0 += u0, w1 += u1;
            }
            warp_sum[0][lane] = w0 - o0 + carry[0];
            warp_sum[1][lane] = w1 - o1 + carry[1];
            __syncwarp();
            if (lane == 31) carry[0] += w0, carry[1] += w1;
        }
        __syncthreads();
        if (i <= n) {
            cnt[i] = warp_sum[0][warp] + s0 - v0;
            tile0[i] = warp_sum[1][warp] + s1 - v1;
        }
        __syncthreads();
    }
    const int n_tiles = carry[1];
    if (tid == 0) tile0[n + 1] = n_tiles;
    __syncthreads();
    if (blockIdx.x == 0) {
        for (int i = tid; i <= n; i += kPlanThreads) plan.off[i] = cnt[i];
        if (tid == 0) plan.off[n + 1] = T, *plan.tiles = n_tiles;
    }
    for (int k = blockIdx.x * kPlanThreads + tid; k < n_tiles; k += gridDim.x * kPlanThreads) {
        int lo = 0, hi = n + 1;  // the adapter with tile0[a] <= k < tile0[a + 1]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (tile0[mid] <= k) lo = mid; else hi = mid;
        }
        const int start = cnt[lo] + (k - tile0[lo]) * tile_rows;
        const int end = lo < n ? cnt[lo + 1] : T;
        plan.tile[k] = Tile{lo, start, min(tile_rows, end - start), 0};
    }
    for (int t0 = c0; t0 < c1; t0 += kPlanThreads) {
        const int t = t0 + tid;
        const int a = t < c1 ? clamp_adapter(__ldg(index + t), n) : -1;
        const uint32_t same = __match_any_sync(0xffffffffu, a);
        const int rank = __popc(same & ((1u << lane) - 1));
        int place = 0;
        for (int w = 0; w < kPlanThreads / 32; w++) {  // the warps in order: a stable grouping
            if (w == warp) {
                if (a >= 0) place = cnt[a] + pre[a] + rank;
                __syncwarp();
                if (a >= 0 && rank == 0) pre[a] += __popc(same);
            }
            __syncthreads();
        }
        if (a >= 0) plan.perm[place] = t;
    }
}

// ---- fragments -----------------------------------------------------------------

template <typename T> struct Io;
template <> struct Io<float> {
    static constexpr bool kSplit = true;
    static __device__ __forceinline__ float one(const float* p) { return __ldg(p); }
    static __device__ __forceinline__ float wide(float v) { return v; }
    static __device__ __forceinline__ float narrow(float v) { return v; }
};
template <> struct Io<__nv_bfloat16> {
    static constexpr bool kSplit = false;
    static __device__ __forceinline__ float one(const __nv_bfloat16* p) {
        return __uint_as_float((uint32_t)__ldg(reinterpret_cast<const unsigned short*>(p)) << 16);
    }
    static __device__ __forceinline__ float wide(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 narrow(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Io<__half> {
    static constexpr bool kSplit = false;
    static __device__ __forceinline__ float one(const __half* p) {
        return half_bits_to_float(__ldg(reinterpret_cast<const unsigned short*>(p)));
    }
    static __device__ __forceinline__ float wide(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half narrow(float v) { return __float2half_rn(v); }
};

__device__ __forceinline__ void widen2(uint32_t u, float* v, const __nv_bfloat16*) {
    v[0] = __uint_as_float(u << 16);
    v[1] = __uint_as_float(u & 0xffff0000u);
}
__device__ __forceinline__ void widen2(uint32_t u, float* v, const __half*) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
    v[0] = f.x;
    v[1] = f.y;
}

// C consecutive elements from p (a multiple of C elements past an aligned row when vec), of which
// `left` exist; the others are zero.
template <typename T, int C>
__device__ __forceinline__ void load_run(const T* __restrict__ p, int64_t left, bool vec, float* v) {
    if (vec) {
        if (left <= 0) {
#pragma unroll
            for (int i = 0; i < C; i++) v[i] = 0.f;
            return;
        }
        if constexpr (sizeof(T) == 4) {
            if constexpr (C == 1) {
                v[0] = __ldg(p);
            } else if constexpr (C == 2) {
                const float2 f = __ldg(reinterpret_cast<const float2*>(p));
                v[0] = f.x, v[1] = f.y;
            } else {
#pragma unroll
                for (int i = 0; i < C; i += 4) {
                    const float4 f = __ldg(reinterpret_cast<const float4*>(p + i));
                    v[i] = f.x, v[i + 1] = f.y, v[i + 2] = f.z, v[i + 3] = f.w;
                }
            }
        } else {
            if constexpr (C == 1) {
                v[0] = Io<T>::one(p);
            } else if constexpr (C == 2) {
                widen2(__ldg(reinterpret_cast<const uint32_t*>(p)), v, p);
            } else if constexpr (C == 4) {
                const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
                widen2(u.x, v, p);
                widen2(u.y, v + 2, p);
            } else {
#pragma unroll
                for (int i = 0; i < C; i += 8) {
                    const uint4 u = __ldg(reinterpret_cast<const uint4*>(p + i));
                    widen2(u.x, v + i, p);
                    widen2(u.y, v + i + 2, p);
                    widen2(u.z, v + i + 4, p);
                    widen2(u.w, v + i + 6, p);
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < C; i++) v[i] = i < left ? Io<T>::one(p + i) : 0.f;
    }
}

// 8 consecutive elements of a row of base, which may be the output itself: plain loads, not the
// read-only path.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int64_t left, bool vec, float* v) {
    if (vec && left >= 8) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
            const uint4 u = *reinterpret_cast<const uint4*>(p);
            widen2(u.x, v, p);
            widen2(u.y, v + 2, p);
            widen2(u.z, v + 4, p);
            widen2(u.w, v + 6, p);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = i < left ? Io<T>::wide(p[i]) : 0.f;
    }
}

// 8 consecutive elements of a row of the output.
template <typename T>
__device__ __forceinline__ void store8(T* p, int64_t left, bool vec, const float* v) {
    if (vec && left >= 8) {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            alignas(16) T h[8];
#pragma unroll
            for (int i = 0; i < 8; i++) h[i] = Io<T>::narrow(v[i]);
            *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < left) p[i] = Io<T>::narrow(v[i]);
    }
}

// TF32 head of x: rounded to 11 significant bits (to nearest, ties away).
__device__ __forceinline__ float tf32_head(float x) {
    return __uint_as_float((__float_as_uint(x) + 0x1000u) & 0xffffe000u);
}

__device__ __forceinline__ void mma_tf32(float* d, const float* a, float b0, float b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(__float_as_uint(a[0])), "r"(__float_as_uint(a[1])), "r"(__float_as_uint(a[2])),
          "r"(__float_as_uint(a[3])), "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
}

// An operand in TF32: its head, and its remainder where it has one.
template <bool SPLIT>
struct FragA {
    float hi[4], lo[SPLIT ? 4 : 1];
    __device__ __forceinline__ void set(int i, float x) {
        if constexpr (SPLIT) {
            hi[i] = tf32_head(x);
            lo[i] = x - hi[i];
        } else {
            hi[i] = x;
        }
    }
};
template <bool SPLIT>
struct FragB {
    float hi[2], lo[SPLIT ? 2 : 1];
    __device__ __forceinline__ void set(int i, float x) {
        if constexpr (SPLIT) {
            hi[i] = tf32_head(x);
            lo[i] = x - hi[i];
        } else {
            hi[i] = x;
        }
    }
};
// d += a b, the small terms first.
template <bool SA, bool SB>
__device__ __forceinline__ void mma_split(float* d, const FragA<SA>& a, const FragB<SB>& b) {
    if constexpr (SA) mma_tf32(d, a.lo, b.hi[0], b.hi[1]);
    if constexpr (SB) mma_tf32(d, a.hi, b.lo[0], b.lo[1]);
    mma_tf32(d, a.hi, b.hi[0], b.hi[1]);
}

// ---- shrink --------------------------------------------------------------------
// h[split, p, :] = scale_i * sum over this split's columns k of x[perm[p], k] W_i[:, k].
// TRANS = false: W_i = A_i [rank, K] (K consecutive); true: W_i = B_i [K, rank] (rank consecutive).
// One block per (tile, split); its 8 warps take the split's chunks in turn and are summed, in
// their order, through shared memory.  A lane holds rows g and g + 8 (g = lane / 4) and E
// consecutive columns, E of 16 bytes; the sums' step s uses its columns 2 s and 2 s + 1.
constexpr int kWarps = 8;

template <typename T, int RB, int MT, bool TRANS>
__global__ void __launch_bounds__(kWarps * 32) k_shrink(Plan plan, const T* __restrict__ x, int64_t ldx,
                                                        const T* __restrict__ w, const float* __restrict__ scale,
                                                        int n, int rank, int64_t K, int64_t k_split, int64_t T_rows,
                                                        bool vec, bool rvec, float* __restrict__ h) {
    constexpr int E = 16 / sizeof(T), CH = 4 * E, RP = 8 * RB, BM = 16 * MT;
    constexpr bool SP = Io<T>::kSplit;
    extern __shared__ float red[];  // [kWarps][BM][RP]
    if ((int)blockIdx.x >= __ldg(plan.tiles)) return;
    const Tile tile = plan.tile[blockIdx.x];
    if (tile.adapter >= n) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    const T* wi = w + (int64_t)tile.adapter * rank * K;
    const T* row[2 * MT];
#pragma unroll
    for (int m = 0; m < 2 * MT; m++) {
        const int p = 8 * m + g;
        row[m] = x + (int64_t)__ldg(plan.perm + tile.start + min(p, tile.rows - 1)) * ldx;
    }
    float acc[MT][RB][4];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int b = 0; b < RB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[m][b][i] = 0.f;
    const int64_t k_begin = blockIdx.y * k_split, k_end = min(K, k_begin + k_split);
#pragma unroll 2
    for (int64_t k0 = k_begin + warp * CH; k0 < k_end; k0 += kWarps * CH) {
        const int64_t k = k0 + E * q;
        float xv[2 * MT][E];
#pragma unroll
        for (int m = 0; m < 2 * MT; m++) load_run<T, E>(row[m] + k, k_end - k, vec, xv[m]);
        if constexpr (!TRANS) {
            float wv[RB][E];
#pragma unroll
            for (int b = 0; b < RB; b++) {
                const int r = 8 * b + g;
                load_run<T, E>(wi + (int64_t)r * K + k, r < rank ? k_end - k : 0, vec, wv[b]);
            }
#pragma unroll
            for (int s = 0; s < E / 2; s++) {
                FragA<SP> fa[MT];
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    fa[m].set(0, xv[2 * m][2 * s]);
                    fa[m].set(1, xv[2 * m + 1][2 * s]);
                    fa[m].set(2, xv[2 * m][2 * s + 1]);
                    fa[m].set(3, xv[2 * m + 1][2 * s + 1]);
                }
#pragma unroll
                for (int b = 0; b < RB; b++) {
                    FragB<SP> fb;
                    fb.set(0, wv[b][2 * s]);
                    fb.set(1, wv[b][2 * s + 1]);
#pragma unroll
                    for (int m = 0; m < MT; m++) mma_split<SP, SP>(acc[m][b], fa[m], fb);
                }
            }
        } else {
#pragma unroll
            for (int s = 0; s < E / 2; s++) {
                float wv[2][RB];  // columns k + 2 s, k + 2 s + 1; ranks RB g .. RB g + RB - 1
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const int64_t kk = k + 2 * s + j;
                    load_run<T, RB>(wi + kk * rank + RB * g, kk < k_end ? rank - RB * g : 0, rvec, wv[j]);
                }
                FragA<SP> fa[MT];
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    fa[m].set(0, xv[2 * m][2 * s]);
                    fa[m].set(1, xv[2 * m + 1][2 * s]);
                    fa[m].set(2, xv[2 * m][2 * s + 1]);
                    fa[m].set(3, xv[2 * m + 1][2 * s + 1]);
                }
#pragma unroll
                for (int b = 0; b < RB; b++) {
                    FragB<SP> fb;
                    fb.set(0, wv[0][b]);
                    fb.set(1, wv[1][b]);
#pragma unroll
                    for (int m = 0; m < MT; m++) mma_split<SP, SP>(acc[m][b], fa[m], fb);
                }
            }
        }
    }
    float* mine = red + warp * BM * RP;
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int b = 0; b < RB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int c = 2 * q + (i & 1), r = TRANS ? RB * c + b : 8 * b + c;
                mine[(16 * m + 8 * (i >> 1) + g) * RP + r] = acc[m][b][i];
            }
    __syncthreads();
    const float s = scale ? __ldg(scale + tile.adapter) : 1.f;
    float* dst = h + ((int64_t)blockIdx.y * T_rows + tile.start) * RP;
    for (int e = threadIdx.x; e < tile.rows * RP; e += kWarps * 32) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < kWarps; k++) v += red[k * BM * RP + e];
        dst[e] = s * v;
    }
}

// 4 consecutive ranks of a place of h, summed over the splits.
__device__ __forceinline__ void load_h(const float* __restrict__ h, int splits, int64_t stride, float* v) {
    float4 f = __ldg(reinterpret_cast<const float4*>(h));
    for (int k = 1; k < splits; k++) {
        const float4 u = __ldg(reinterpret_cast<const float4*>(h + k * stride));
        f.x += u.x, f.y += u.y, f.z += u.z, f.w += u.w;
    }
    v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
}

// ---- expand --------------------------------------------------------------------
// out[t, f] = base[t, f] + sum over ranks of h[p, r] W_i[f, r], t = perm[p]; positions without an
// adapter get base.  TRANS = false: W_i = B_i [F, rank]; true: W_i = A_i [rank, F].  base null: zeros.
// A warp keeps its tile's h fragments in registers and walks over 32 columns at a time; a lane ends
// up with 8 consecutive columns of rows g and g + 8, read and written as 16-byte pieces.
template <typename T, int RB, int MT, bool TRANS>
__global__ void __launch_bounds__(kWarps * 32) k_expand(Plan plan, const float* __restrict__ h, int splits,
                                                        const T* __restrict__ w, int n, int rank, int64_t F,
                                                        int64_t f_block, int64_t T_rows, const T* base,
                                                        int64_t ldb, T* out, int64_t ldo, bool vec, bool wvec) {
    constexpr int RP = 8 * RB, RC = RB / 2;  // RC chunks of 16 ranks
    constexpr bool SP = Io<T>::kSplit;
    if ((int)blockIdx.x >= __ldg(plan.tiles)) return;
    const Tile tile = plan.tile[blockIdx.x];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    const bool none = tile.adapter >= n;
    if (none && base == out) return;
    int64_t t[2 * MT];
    bool live[2 * MT];
#pragma unroll
    for (int m = 0; m < 2 * MT; m++) {
        live[m] = 8 * m + g < tile.rows;
        t[m] = __ldg(plan.perm + tile.start + min(8 * m + g, tile.rows - 1));
    }
    FragA<true> fa[MT][RB];
    if (!none) {
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int c = 0; c < RC; c++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int p = min(16 * m + 8 * u + g, tile.rows - 1);
                    float v[4];
                    load_h(h + ((int64_t)tile.start + p) * RP + 16 * c + 4 * q, splits, T_rows * RP, v);
                    fa[m][2 * c].set(u, v[0]);
                    fa[m][2 * c].set(2 + u, v[1]);
                    fa[m][2 * c + 1].set(u, v[2]);
                    fa[m][2 * c + 1].set(2 + u, v[3]);
                }
    }
    const T* wi = w + (none ? 0 : (int64_t)tile.adapter * rank * F);
    const int64_t f_begin = blockIdx.y * f_block, f_end = min(F, f_begin + f_block);
    for (int64_t f0 = f_begin + 32 * warp; f0 < f_end; f0 += 32 * kWarps) {
        const int64_t f = f0 + 8 * q, left = f_end - f;
        float acc[MT][4][4];
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int b = 0; b < 4; b++)
#pragma unroll
                for (int i = 0; i < 4; i++) acc[m][b][i] = 0.f;
        float bv[2 * MT][8];
#pragma unroll
        for (int m = 0; m < 2 * MT; m++) {
            if (base && live[m]) {
                load8<T>(base + t[m] * ldb + f, left, vec, bv[m]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) bv[m][i] = 0.f;
            }
        }
        if (!none) {
#pragma unroll
            for (int c = 0; c < RC; c++) {
                if constexpr (!TRANS) {  // block b, column 2 q + j of the product: feature f0 + 8 q + 2 b + j
                    float wv[4][4];
#pragma unroll
                    for (int b = 0; b < 4; b++) {
                        const int64_t fw = f0 + 8 * (g >> 1) + 2 * b + (g & 1);
                        const int r = 16 * c + 4 * q;
                        load_run<T, 4>(wi + fw * rank + r, fw < f_end ? rank - r : 0, wvec, wv[b]);
                    }
#pragma unroll
                    for (int b = 0; b < 4; b++)
#pragma unroll
                        for (int s = 0; s < 2; s++) {
                            FragB<SP> fb;
                            fb.set(0, wv[b][2 * s]);
                            fb.set(1, wv[b][2 * s + 1]);
#pragma unroll
                            for (int m = 0; m < MT; m++) mma_split<true, SP>(acc[m][b], fa[m][2 * c + s], fb);
                        }
                } else {  // block b, column 2 q + j: feature f0 + 8 q + 4 j + b
#pragma unroll
                    for (int s = 0; s < 2; s++) {
                        float wv[2][4];
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            const int r = 16 * c + 4 * q + 2 * s + j;
                            const int64_t fw = f0 + 4 * g;
                            load_run<T, 4>(wi + (int64_t)r * F + fw, r < rank ? f_end - fw : 0, wvec, wv[j]);
                        }
#pragma unroll
                        for (int b = 0; b < 4; b++) {
                            FragB<SP> fb;
                            fb.set(0, wv[0][b]);
                            fb.set(1, wv[1][b]);
#pragma unroll
                            for (int m = 0; m < MT; m++) mma_split<true, SP>(acc[m][b], fa[m][2 * c + s], fb);
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int m = 0; m < 2 * MT; m++) {
            if (!live[m]) continue;
            float v[8];
#pragma unroll
            for (int b = 0; b < 4; b++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const int e = TRANS ? 4 * j + b : 2 * b + j;
                    v[e] = bv[m][e] + acc[m >> 1][b][2 * (m & 1) + j];
                }
            store8<T>(out + t[m] * ldo + f, left, vec, v);
        }
    }
}

// ---- weight gradients ------------------------------------------------------------
// G_i = sum over adapter i's positions of x[t, f] h[p, r].  TRANS = false: G_i stored [rank, F] (dA,
// with h = dh); true: stored [F, rank] (dB, with x = the gradient of out).  One block per (32 columns,
// adapter); its warps take 8 positions each in turn and are summed, in their order, through shared
// memory.  An adapter without positions gets zeros.
template <typename T, int RB, bool TRANS>
__global__ void __launch_bounds__(kWarps * 32) k_weight(Plan plan, const T* __restrict__ x, int64_t ldx,
                                                        const float* __restrict__ h, int splits, int rank, int64_t F,
                                                        int64_t T_rows, bool vec, T* __restrict__ out) {
    constexpr int RP = 8 * RB, RM = RB / 2;  // RM blocks of 16 ranks; lane rows g, g + 8: ranks 2 RM g + ..
    constexpr bool SP = Io<T>::kSplit;
    extern __shared__ float red[];  // [kWarps][RP][32]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    const int a = blockIdx.y;
    const int p0 = __ldg(plan.off + a), p1 = __ldg(plan.off + a + 1);
    const int64_t f0 = (int64_t)blockIdx.x * 32;
    float acc[RM][4][4];
#pragma unroll
    for (int m = 0; m < RM; m++)
#pragma unroll
        for (int b = 0; b < 4; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[m][b][i] = 0.f;
#pragma unroll 2
    for (int p = p0 + 8 * warp; p < p1; p += 8 * kWarps) {
        float xv[2][4], hv[2][2 * RM];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int pp = p + q + 4 * j;
            const int64_t t = __ldg(plan.perm + min(pp, p1 - 1));
            load_run<T, 4>(x + t * ldx + f0 + 4 * g, pp < p1 ? F - (f0 + 4 * g) : 0, vec, xv[j]);
            const float* hp = h + (int64_t)min(pp, p1 - 1) * RP + 2 * RM * g;
#pragma unroll
            for (int r = 0; r < 2 * RM; r++) hv[j][r] = 0.f;
            if (pp < p1)
                for (int k = 0; k < splits; k++)
#pragma unroll
                    for (int r = 0; r < 2 * RM; r += 2) {
                        const float2 u = __ldg(reinterpret_cast<const float2*>(hp + (int64_t)k * T_rows * RP + r));
                        hv[j][r] += u.x;
                        hv[j][r + 1] += u.y;
                    }
        }
        FragB<SP> fb[4];
#pragma unroll
        for (int b = 0; b < 4; b++) {
            fb[b].set(0, xv[0][b]);
            fb[b].set(1, xv[1][b]);
        }
#pragma unroll
        for (int m = 0; m < RM; m++) {
            FragA<true> fa;
            fa.set(0, hv[0][2 * m]);
            fa.set(1, hv[0][2 * m + 1]);
            fa.set(2, hv[1][2 * m]);
            fa.set(3, hv[1][2 * m + 1]);
#pragma unroll
            for (int b = 0; b < 4; b++) mma_split<true, SP>(acc[m][b], fa, fb[b]);
        }
    }
    float* mine = red + warp * RP * 32;
#pragma unroll
    for (int m = 0; m < RM; m++)
#pragma unroll
        for (int b = 0; b < 4; b++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                mine[(2 * RM * g + 2 * m + (i >> 1)) * 32 + 4 * (2 * q + (i & 1)) + b] = acc[m][b][i];
    __syncthreads();
    T* dst = out + (int64_t)a * rank * F;
    for (int e = threadIdx.x; e < 32 * rank; e += kWarps * 32) {
        const int r = TRANS ? e % rank : e / 32, c = TRANS ? e / rank : e % 32;
        if (f0 + c >= F) continue;
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < kWarps; k++) v += red[(k * RP + r) * 32 + c];
        dst[TRANS ? (f0 + c) * rank + r : (int64_t)r * F + f0 + c] = Io<T>::narrow(v);
    }
}

// ---- host ------------------------------------------------------------------------

struct Shape {
    int64_t T, K, N;
    int n, rank, rb, mt;
    int64_t tiles_max;
    int splits_k, splits_n;  // blocks per tile that share the sum over K, over N
};

int64_t align256(int64_t b) { return (b + 255) & ~int64_t(255); }

// Places of the workspace; bytes = its size.
struct Layout {
    int64_t off, perm, tiles, tile, h, dh, bytes;
};

int rank_blocks(int rank) { return rank <= 16 ? 2 : rank <= 32 ? 4 : rank <= 64 ? 8 : 16; }

int check_shape(int64_t T, int32_t n, int32_t rank, int64_t K, int64_t N) {
    if (T < 0 || n < 0 || rank < 1 || K < 1 || N < 1) return ENGRAM_ERR_ARG;
    if (rank > kMaxRank || n > kMaxAdapters || T > (1 << 30) || K > (1 << 30) || N > (1 << 30)) return ENGRAM_ERR_RANGE;
    return ENGRAM_OK;
}

Shape shape_of(int64_t T, int n, int rank, int64_t K, int64_t N) {
    Shape s;
    s.T = T, s.K = K, s.N = N, s.n = n, s.rank = rank;
    s.rb = rank_blocks(rank);
    const int64_t groups = T < (int64_t)n + 1 ? T : (int64_t)n + 1;
    s.mt = (s.rb < 16 && groups > 0 && T / groups >= 64) ? 2 : 1;
    const int bm = 16 * s.mt;
    s.tiles_max = (T + (bm - 1) * groups) / bm;
    const auto splits = [&](int64_t width) {
        const int64_t want = s.tiles_max > 0 ? (2 * 148) / s.tiles_max : 1, most = (width + 255) / 256;
        const int64_t k = want < most ? want : most;
        return (int)(k < 1 ? 1 : k > 16 ? 16 : k);
    };
    s.splits_k = splits(K);
    s.splits_n = splits(N);
    return s;
}

Layout layout_of(const Shape& s, bool backward) {
    Layout l;
    int64_t at = 0;
    const auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += align256(bytes);
        return here;
    };
    l.off = take((int64_t)(s.n + 2) * 4);
    l.perm = take(s.T * 4);
    l.tiles = take(4);
    l.tile = take(s.tiles_max * (int64_t)sizeof(Tile));
    l.h = take((int64_t)s.splits_k * s.T * 8 * s.rb * 4);
    l.dh = backward ? take((int64_t)s.splits_n * s.T * 8 * s.rb * 4) : 0;
    l.bytes = at;
    return l;
}

Plan plan_at(uint8_t* ws, const Layout& l) {
    return Plan{reinterpret_cast<int32_t*>(ws + l.off), reinterpret_cast<int32_t*>(ws + l.perm),
                reinterpret_cast<int32_t*>(ws + l.tiles), reinterpret_cast<Tile*>(ws + l.tile)};
}

// Raises the kernel's limit of dynamic shared memory where the launch needs it.
bool allow_smem(const void* kernel, int bytes) {
    return bytes <= 48 * 1024 ||
           cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess;
}

int launched() {
    count_launches(1);
    return cudaGetLastError() == cudaSuccess ? ENGRAM_OK : ENGRAM_ERR_CUDA;
}

int run_plan(const Shape& s, const int32_t* index, const Plan& plan, cudaStream_t st) {
    const int64_t per = (s.T + 127) / 128;
    const int chunk = (int)((per + kPlanThreads - 1) / kPlanThreads) * kPlanThreads;
    const int smem = (3 * s.n + 4) * 4;
    if (!allow_smem((const void*)k_plan, smem)) return ENGRAM_ERR_CUDA;
    k_plan<<<(unsigned)((s.T + chunk - 1) / chunk), kPlanThreads, smem, st>>>(index, (int)s.T, s.n, chunk, 16 * s.mt,
                                                                              plan);
    return launched();
}

template <typename T, int RB, int MT, bool TRANS>
int run_shrink(const Shape& s, const Plan& plan, const T* x, int64_t ldx, const T* w, const float* scale, int64_t K,
               int splits, float* h, cudaStream_t st) {
    constexpr int E = 16 / sizeof(T), CH = 4 * E;
    const int64_t step = kWarps * CH, k_split = ((K + splits - 1) / splits + step - 1) / step * step;
    const bool vec = aligned16(x) && ldx % E == 0 && K % E == 0 && (TRANS || aligned16(w));
    const bool rvec = TRANS && aligned16(w) && s.rank % RB == 0;
    const int smem = kWarps * 16 * MT * 8 * RB * 4;
    if (!allow_smem((const void*)k_shrink<T, RB, MT, TRANS>, smem)) return ENGRAM_ERR_CUDA;
    k_shrink<T, RB, MT, TRANS><<<dim3((unsigned)s.tiles_max, splits), kWarps * 32, smem, st>>>(
        plan, x, ldx, w, scale, s.n, s.rank, K, k_split, s.T, vec, rvec, h);
    return launched();
}

template <typename T, int RB, int MT, bool TRANS>
int run_expand(const Shape& s, const Plan& plan, const float* h, int splits, const T* w, int64_t F, const T* base,
               int64_t ldb, T* out, int64_t ldo, cudaStream_t st) {
    constexpr int E = 16 / sizeof(T);
    // columns of a block: whole passes of its warps, about four blocks an SM
    const int64_t step = 32 * kWarps;
    const int64_t passes = (F + step - 1) / step, want = s.tiles_max > 0 ? (4 * 148 + s.tiles_max - 1) / s.tiles_max : 1;
    const int64_t blocks = want < passes ? want : passes;
    const int64_t f_block = (passes + blocks - 1) / blocks * step;
    const bool vec = (!base || (aligned16(base) && ldb % E == 0)) && aligned16(out) && ldo % E == 0 && F % 8 == 0;
    const bool wvec = aligned16(w) && (TRANS ? F % 4 == 0 : s.rank % 4 == 0);
    k_expand<T, RB, MT, TRANS><<<dim3((unsigned)s.tiles_max, (unsigned)((F + f_block - 1) / f_block)), kWarps * 32, 0,
                                 st>>>(plan, h, splits, w, s.n, s.rank, F, f_block, s.T, base, ldb, out, ldo, vec,
                                       wvec);
    return launched();
}

template <typename T, int RB, bool TRANS>
int run_weight(const Shape& s, const Plan& plan, const T* x, int64_t ldx, const float* h, int splits, int64_t F,
               T* out, cudaStream_t st) {
    const bool vec = aligned16(x) && ldx % 4 == 0 && F % 4 == 0;
    const int smem = kWarps * 8 * RB * 32 * 4;
    if (!allow_smem((const void*)k_weight<T, RB, TRANS>, smem)) return ENGRAM_ERR_CUDA;
    k_weight<T, RB, TRANS><<<dim3((unsigned)((F + 31) / 32), s.n), kWarps * 32, smem, st>>>(
        plan, x, ldx, h, splits, s.rank, F, s.T, vec, out);
    return launched();
}

struct Args {
    const void *x, *a, *b, *base, *grad;
    int64_t ldx, ldbase, ldout, ldgrad, lddx;
    const int32_t* index;
    const float* scale;
    void *out, *dx, *da, *db;
    uint8_t* ws;
    cudaStream_t st;
};

template <typename T, int RB, int MT>
int forward(const Shape& s, const Layout& l, const Args& g) {
    const Plan plan = plan_at(g.ws, l);
    float* h = reinterpret_cast<float*>(g.ws + l.h);
    int e = run_plan(s, g.index, plan, g.st);
    if (!e)
        e = run_shrink<T, RB, MT, false>(s, plan, (const T*)g.x, g.ldx, (const T*)g.a, g.scale, s.K, s.splits_k, h,
                                         g.st);
    if (!e)
        e = run_expand<T, RB, MT, false>(s, plan, h, s.splits_k, (const T*)g.b, s.N, (const T*)g.base, g.ldbase,
                                         (T*)g.out, g.ldout, g.st);
    return e;
}

template <typename T, int RB, int MT>
int backward(const Shape& s, const Layout& l, const Args& g) {
    const Plan plan = plan_at(g.ws, l);
    float *h = reinterpret_cast<float*>(g.ws + l.h), *dh = reinterpret_cast<float*>(g.ws + l.dh);
    int e = run_plan(s, g.index, plan, g.st);
    if (!e && (g.dx || g.da))
        e = run_shrink<T, RB, MT, true>(s, plan, (const T*)g.grad, g.ldgrad, (const T*)g.b, g.scale, s.N, s.splits_n,
                                        dh, g.st);
    if (!e && g.dx)
        e = run_expand<T, RB, MT, true>(s, plan, dh, s.splits_n, (const T*)g.a, s.K, (const T*)g.base, g.ldbase,
                                        (T*)g.dx, g.lddx, g.st);
    if (!e && g.da)
        e = run_weight<T, RB, false>(s, plan, (const T*)g.x, g.ldx, dh, s.splits_n, s.K, (T*)g.da, g.st);
    if (!e && g.db)
        e = run_shrink<T, RB, MT, false>(s, plan, (const T*)g.x, g.ldx, (const T*)g.a, g.scale, s.K, s.splits_k, h,
                                         g.st);
    if (!e && g.db)
        e = run_weight<T, RB, true>(s, plan, (const T*)g.grad, g.ldgrad, h, s.splits_k, s.N, (T*)g.db, g.st);
    return e;
}

template <typename T>
int by_rank(const Shape& s, const Layout& l, const Args& g, bool back) {
#define ENGRAM_CASE(RB, MT) \
    if (s.rb == RB && s.mt == MT) return back ? backward<T, RB, MT>(s, l, g) : forward<T, RB, MT>(s, l, g);
    ENGRAM_CASE(2, 1)
    ENGRAM_CASE(2, 2)
    ENGRAM_CASE(4, 1)
    ENGRAM_CASE(4, 2)
    ENGRAM_CASE(8, 1)
    ENGRAM_CASE(8, 2)
    ENGRAM_CASE(16, 1)
#undef ENGRAM_CASE
    return ENGRAM_ERR_RANGE;
}

int by_type(int32_t dtype, const Shape& s, const Layout& l, const Args& g, bool back) {
    switch (dtype) {
        case ENGRAM_DTYPE_F32: return by_rank<float>(s, l, g, back);
        case ENGRAM_DTYPE_BF16: return by_rank<__nv_bfloat16>(s, l, g, back);
        case ENGRAM_DTYPE_F16: return by_rank<__half>(s, l, g, back);
    }
    return ENGRAM_ERR_FORMAT;
}

bool aligned_to(const void* p, int32_t dtype) {
    return ((uintptr_t)p & (dtype == ENGRAM_DTYPE_F32 ? 3u : 1u)) == 0;
}

}  // namespace

extern "C" int64_t engram_adapter_workspace_bytes(int64_t T, int32_t n_adapters, int32_t rank, int64_t K, int64_t N,
                                                  int32_t backward) {
    const int e = check_shape(T, n_adapters, rank, K, N);
    if (e) return e;
    return layout_of(shape_of(T, n_adapters, rank, K, N), backward != 0).bytes;
}

extern "C" int engram_adapter_forward(int32_t dtype, const void* x, int64_t ldx, const void* a, const void* b,
                                      const int32_t* index, const float* scale, int64_t T, int32_t n_adapters,
                                      int32_t rank, int64_t K, int64_t N, const void* base, int64_t ldbase, void* out,
                                      int64_t ldout, void* workspace, int64_t workspace_bytes, void* stream) {
    const int e = check_shape(T, n_adapters, rank, K, N);
    if (e) return e;
    if (dtype < ENGRAM_DTYPE_F32 || dtype > ENGRAM_DTYPE_F16) return ENGRAM_ERR_FORMAT;
    if (T == 0) return ENGRAM_OK;
    if (!x || !index || !out || !workspace || !aligned16(workspace)) return ENGRAM_ERR_ARG;
    if (n_adapters > 0 && (!a || !b)) return ENGRAM_ERR_ARG;
    if (ldx < K || ldout < N || (base && ldbase < N) || (base == out && ldbase != ldout)) return ENGRAM_ERR_ARG;
    for (const void* p : {x, a, b, base, (const void*)out})
        if (!aligned_to(p, dtype)) return ENGRAM_ERR_ARG;
    const Shape s = shape_of(T, n_adapters, rank, K, N);
    const Layout l = layout_of(s, false);
    if (workspace_bytes < l.bytes) return ENGRAM_ERR_WORKSPACE;
    Args g = {};
    g.x = x, g.a = a, g.b = b, g.base = base, g.ldx = ldx, g.ldbase = ldbase, g.ldout = ldout;
    g.index = index, g.scale = scale, g.out = out, g.ws = (uint8_t*)workspace, g.st = (cudaStream_t)stream;
    return by_type(dtype, s, l, g, false);
}

extern "C" int engram_adapter_backward(int32_t dtype, const void* grad, int64_t ldgrad, const void* x, int64_t ldx,
                                       const void* a, const void* b, const int32_t* index, const float* scale,
                                       int64_t T, int32_t n_adapters, int32_t rank, int64_t K, int64_t N,
                                       const void* dx_base, int64_t lddx_base, void* dx, int64_t lddx, void* da,
                                       void* db, void* workspace, int64_t workspace_bytes, void* stream) {
    const int e = check_shape(T, n_adapters, rank, K, N);
    if (e) return e;
    if (dtype < ENGRAM_DTYPE_F32 || dtype > ENGRAM_DTYPE_F16) return ENGRAM_ERR_FORMAT;
    const int64_t size = dtype == ENGRAM_DTYPE_F32 ? 4 : 2;
    cudaStream_t st = (cudaStream_t)stream;
    if (T == 0) {
        for (void* p : {da, db})
            if (p && cudaMemsetAsync(p, 0, n_adapters * (int64_t)rank * (p == da ? K : N) * size, st) != cudaSuccess)
                return ENGRAM_ERR_CUDA;
        return ENGRAM_OK;
    }
    if (!grad || !x || !index || !workspace || !aligned16(workspace)) return ENGRAM_ERR_ARG;
    if (n_adapters > 0 && (!a || !b)) return ENGRAM_ERR_ARG;
    if (ldx < K || ldgrad < N || (dx && lddx < K) || (dx_base && lddx_base < K) ||
        (dx && dx_base == dx && lddx_base != lddx))
        return ENGRAM_ERR_ARG;
    for (const void* p : {grad, x, a, b, dx_base, (const void*)dx, (const void*)da, (const void*)db})
        if (!aligned_to(p, dtype)) return ENGRAM_ERR_ARG;
    const Shape s = shape_of(T, n_adapters, rank, K, N);
    const Layout l = layout_of(s, true);
    if (workspace_bytes < l.bytes) return ENGRAM_ERR_WORKSPACE;
    Args g = {};
    g.grad = grad, g.ldgrad = ldgrad, g.x = x, g.ldx = ldx, g.a = a, g.b = b, g.index = index, g.scale = scale;
    g.base = dx_base, g.ldbase = lddx_base, g.dx = dx, g.lddx = lddx;
    g.da = n_adapters ? da : nullptr, g.db = n_adapters ? db : nullptr;
    g.ws = (uint8_t*)workspace, g.st = st;
    return by_type(dtype, s, l, g, true);
}
