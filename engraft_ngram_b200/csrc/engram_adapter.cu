// engram_adapter.cu -- low-rank adapters of many requests beside a shared
// projection: out[t] = base[t] + s_i B_i (A_i x[t]) with i = index[t], A_i
// [rank, K] and B_i [N, rank], and the gradients of x, A and B.
//
// Positions are grouped by adapter, so that each tile of 16 or 128 positions
// reads one adapter's factors.  Three products are then needed:
//   shrink  h[t, :] = s_i A_i x[t]                   (a sum over a width, rank columns out)
//   expand  out[t, :] = base[t, :] + B_i h[t, :]     (a sum over the rank)
//   weight  G_i[f, :] = sum over i's positions of x[t, f] h[t, :]
// The backward uses the same three: dh = s_i B_i^T g (shrink over N), dx = A_i^T dh
// (expand), dA from (x, dh) and dB from (g, h).
//
// What bounds them is the bytes of x, base, grad and out: 2 rank flops for each
// of their elements is below what mma.sync gives at those bytes a second.  So
// each block streams its rows through a ring of shared-memory stages filled by
// cp.async, 16 bytes a thread from addresses held in registers (bulk copies of whole
// row pieces are issued one lane at a time, and cost more instructions than that);
// rows that do not start on 16 bytes, and the last stage, take a slower loop.  The
// products are mma.sync from there.  16-bit types
// use m16n8k16 in their own type; fp32 uses m16n8k8 TF32 on split operands,
// x = hi + lo with hi rounded to the 11 significant bits of TF32: hi hi + hi lo +
// lo hi.  The dropped lo lo is 2^-22 of the product at most, and lo, of 12 bits, is
// read in 11: 2^-23 of the operand.  (k_expand_wide's factors are cut to their head
// by the tensor cores, not rounded: 2^-21 for both.)  That stands beside the rounding
// of fp32 sums: 4000 positions at rank 16 are 3.4e-7 off in the 2-norm, at rank 128
// 1.1e-6, gradients of the factors 4.4e-7, where products in plain fp32, adapter by
// adapter, are 2.2e-7, 4.9e-7 and 3.3e-7 to 7.2e-7 off.
// h and dh, sums over a whole width, are kept in fp32.  Where they are an operand
// beside a 16-bit type they are split in it, h = hi + lo (16 bits for bf16, 22 for
// fp16, there after scaling by a power of two that brings the largest below 2^15):
// 2^-17 and less of h beside the half step of the result, 2^-8 and 2^-11.
// mma.sync adds to its accumulator with truncation, so fp32 sums are taken out of
// it every stage and added in fp32 proper: 12800 terms were 3e-6 off without,
// 5e-7 with it.  16-bit sums, whose results have 2^-8 or 2^-11, are taken out after
// 2^17 columns and every 2^14 positions of long lists.
#include <type_traits>

#include <cooperative_groups.h>

#include "engram_tensor.cuh"

using namespace engram;

namespace {

constexpr int kThreads = 256, kWarps = 8;
constexpr int kPlanThreads = 1024;
// Positions and adapters up to which a block finds its tile by itself.  Against k_plan, 12800 columns of fp32 at
// rank 16: 64 positions of 16 adapters 15 and 19 us, 1024 of 16 45 and 52, 1024 of 1000 202 and 203.  The
// gradients look through the positions once more, in each block of k_weight: 77 positions of 4 adapters 26.3 and
// 26.6 us (bf16 18 and 21), but 128 of 16 57 and 47 (bf16 28 and 31), 256 of 64 188 and 134, 1024 of 16 103 and 81.
constexpr int kScanMax = 1024, kScanMaxGradients = 128, kScanAdapters = 2048;
constexpr int kMaxAdapters = 16384;  // k_plan counts them in shared memory
constexpr int kMaxRank = 128;

// ---- the plan ----------------------------------------------------------------
// int32 arrays in the workspace.  off[i] = first place of adapter i in the grouped
// order, off[n] = first place of the positions without an adapter, off[n+1] = T;
// perm[p] = position; tile k covers places [start, start + rows) of one adapter.  Without k_plan (few
// positions) there is no off and no count: tile k has its own places, from k BM on, and may be empty.
struct Tile {
    int32_t adapter, start, rows, pad;
};
struct Plan {
    int32_t* off;    // [n + 2]
    int32_t* perm;   // [T]
    int32_t* tiles;  // [2]: number of tiles, of those with an adapter (they come first); null: as many as blocks
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
    // a warp whose positions share an adapter (packed prompts) adds once, another lane by lane
    constexpr int N = 4;  // loads under way a thread
    for (int t0 = 0; t0 < T; t0 += N * kPlanThreads) {
        int a[N];
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int t = t0 + j * kPlanThreads + tid;
            a[j] = t < T ? clamp_adapter(__ldg(index + t), n) : -1;
        }
#pragma unroll
        for (int j = 0; j < N; j++) {
            const bool before = t0 + j * kPlanThreads < c0;  // chunks are whole multiples of kPlanThreads
            const bool one = __all_sync(0xffffffffu, a[j] == __shfl_sync(0xffffffffu, a[j], 0));
            if (a[j] >= 0 && (!one || lane == 0)) {
                atomicAdd(cnt + a[j], one ? 32 : 1);
                if (before) atomicAdd(pre + a[j], one ? 32 : 1);
            }
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
        if (tid == 0) plan.off[n + 1] = T, plan.tiles[0] = n_tiles, plan.tiles[1] = tile0[n];
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

// Few positions need no launch for the plan: each block of the first launch looks through all indexes
// itself, and writes its tile down for the launches after it.  List, in ascending order, of the positions
// with adapter a (n: without one); every thread of the block calls it.
struct Scan {
    int32_t list[kScanMax];
    int32_t warp_count[kWarps];
};
__device__ __forceinline__ int scan_positions(Scan& s, const int32_t* __restrict__ index, int T, int n, int a) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int total = 0;
    for (int t0 = 0; t0 < T; t0 += kThreads) {
        const int t = t0 + threadIdx.x;
        const bool mine = t < T && clamp_adapter(__ldg(index + t), n) == a;
        const uint32_t m = __ballot_sync(0xffffffffu, mine);
        if (lane == 0) s.warp_count[warp] = __popc(m);
        __syncthreads();
        int before = total;
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            if (w < warp) before += s.warp_count[w];
            total += s.warp_count[w];
        }
        if (mine) s.list[before + __popc(m & ((1u << lane) - 1))] = t;
        __syncthreads();
    }
    return total;
}

// The positions of a block's tile.
template <int BM>
struct TileRows {
    int32_t row[BM];
    int32_t adapter, first, rows;
};
struct FindTile {  // used by the first launch only, where its stages come to stand later
    Scan scan;
    int32_t tiles[kScanAdapters + 1];
    int32_t warp_sum[kWarps];
};

// Tile k in the order of the adapters, found without a plan.
template <int BM>
__device__ __forceinline__ void find_tile(FindTile& f, TileRows<BM>& r, const int32_t* __restrict__ index, int T, int n,
                                          int k) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int i = tid; i <= n; i += kThreads) f.tiles[i] = 0;
    if (tid == 0) r.adapter = -1, r.first = r.rows = 0;
    __syncthreads();
    for (int t = tid; t < T; t += kThreads) atomicAdd(f.tiles + clamp_adapter(__ldg(index + t), n), 1);
    __syncthreads();
    int before = 0;  // tiles of the adapters so far
    for (int i0 = 0; i0 <= n; i0 += kThreads) {
        const int i = i0 + tid, count = i <= n ? f.tiles[i] : 0, mine = (count + BM - 1) / BM;
        int sum = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += u;
        }
        if (lane == 31) f.warp_sum[warp] = sum;
        __syncthreads();
        int at = before + sum - mine;
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            if (w < warp) at += f.warp_sum[w];
            before += f.warp_sum[w];
        }
        if (k >= at && k < at + mine) {
            r.adapter = i;
            r.first = (k - at) * BM;
            r.rows = min(BM, count - r.first);
        }
        __syncthreads();
    }
    if (r.adapter < 0) return;
    scan_positions(f.scan, index, T, n, r.adapter);
    for (int i = tid; i < BM; i += kThreads) r.row[i] = f.scan.list[r.first + min(i, r.rows - 1)];
    __syncthreads();
}

// The block's tile, or its BM positions of one shared by PARTS blocks, from the plan; false: there are none.
template <int BM, int PARTS = 1, int ROWS>
__device__ __forceinline__ bool read_tile(TileRows<ROWS>& r, const Plan& plan) {
    const int k = blockIdx.x / PARTS, from = (int)(blockIdx.x % PARTS) * BM;
    if (plan.tiles && k >= *plan.tiles) return false;
    const Tile t = plan.tile[k];
    const int rows = min(BM, t.rows - from);
    if (rows <= 0) return false;
    for (int i = threadIdx.x; i < BM; i += kThreads) r.row[i] = plan.perm[t.start + from + min(i, rows - 1)];
    if (threadIdx.x == 0) r.adapter = t.adapter, r.rows = rows;
    __syncthreads();
    return true;
}

// ---- types, stages and fragments -------------------------------------------------

template <typename T>
constexpr int kE = 16 / (int)sizeof(T);  // elements of a 16-byte unit

__device__ __forceinline__ uint32_t bits_of(float v) { return __float_as_uint(v); }
__device__ __forceinline__ float wide(float v) { return v; }
__device__ __forceinline__ float wide(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float wide(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 narrow(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half narrow(float v) { return __float2half_rn(v); }

// Two values as one register of the 16-bit type, the first in the low half.
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t u);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t u) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
}

// One 16-byte unit of a stage from src, of which `left` elements exist (the others become zero).
// vec: src is 16-byte aligned: asynchronous; else element by element.
template <typename T>
__device__ __forceinline__ void stage_unit(uint8_t* dst, const T* src, const T* valid, int64_t left, bool vec) {
    constexpr int E = kE<T>;
    if (vec) {
        const int bytes = left >= E ? 16 : left > 0 ? (int)left * (int)sizeof(T) : 0;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)),
                     "l"(bytes ? src : valid), "r"(bytes)
                     : "memory");
    } else {
        alignas(16) T v[E];
#pragma unroll
        for (int i = 0; i < E; i++) v[i] = i < left ? src[i] : narrow<T>(0.f);
        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(v);
    }
}
__device__ __forceinline__ void stage_done() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void stage_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// The units of a stage's ROWS x U that a thread copies: a fixed column, and rows 256 / U apart.
template <typename T, int ROWS, int U>
struct Units {
    static constexpr int N = (ROWS * U + kThreads - 1) / kThreads, STEP = kThreads / U;
    static_assert(kThreads % U == 0, "a thread keeps its column");
    const T* src[N];
    uint32_t bytes[N];  // 16, or 0: the unit becomes zero
    static __device__ __forceinline__ int row(int k) { return (int)threadIdx.x / U + k * STEP; }
    static __device__ __forceinline__ int column() { return (int)threadIdx.x % U; }
    static __device__ __forceinline__ bool mine(int k) { return ROWS % STEP == 0 || row(k) < ROWS; }
    __device__ __forceinline__ void copy(int k, uint32_t dst, int64_t offset) const {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src[k] + offset), "r"(bytes[k])
                     : "memory");
    }
};

__device__ __forceinline__ uint4 lds128(const void* p) { return *reinterpret_cast<const uint4*>(p); }

__device__ __forceinline__ void ldmatrix4(uint32_t* r, const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_u32(p))
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t* r, const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_u32(p))
                 : "memory");
}

template <typename T> __device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma<float>(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma<__half>(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// x = hi + lo, hi rounded to TF32 (to nearest, ties away).
__device__ __forceinline__ void split_tf32(uint32_t x, uint32_t& hi, uint32_t& lo) {
    hi = (x + 0x1000u) & 0xffffe000u;
    lo = bits_of(__uint_as_float(x) - __uint_as_float(hi));
}
// An A fragment in the operand type with its remainder, and d += a b, the small terms first.
struct Split {
    uint32_t hi[4], lo[4];
};
__device__ __forceinline__ Split split_a(uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
    Split f;
    split_tf32(a0, f.hi[0], f.lo[0]);
    split_tf32(a1, f.hi[1], f.lo[1]);
    split_tf32(a2, f.hi[2], f.lo[2]);
    split_tf32(a3, f.hi[3], f.lo[3]);
    return f;
}
// Two blocks of columns at a time: a step on one accumulator waits for the step before it.
__device__ __forceinline__ void mma_split2(float* d, float* e, const Split& a, uint32_t b0, uint32_t b1, uint32_t c0,
                                           uint32_t c1) {
    uint32_t bh[2], bl[2], ch[2], cl[2];
    split_tf32(b0, bh[0], bl[0]);
    split_tf32(b1, bh[1], bl[1]);
    split_tf32(c0, ch[0], cl[0]);
    split_tf32(c1, ch[1], cl[1]);
    mma<float>(d, a.lo, bh[0], bh[1]);
    mma<float>(e, a.lo, ch[0], ch[1]);
    mma<float>(d, a.hi, bl[0], bl[1]);
    mma<float>(e, a.hi, cl[0], cl[1]);
    mma<float>(d, a.hi, bh[0], bh[1]);
    mma<float>(e, a.hi, ch[0], ch[1]);
}

// Stages of a ring: three where that leaves room for three blocks an SM, four or three for two.
constexpr int fit_stages(int bytes) {
    return 3 * bytes <= 74 * 1024 ? 3 : 4 * bytes <= 108 * 1024 ? 4 : 3 * bytes <= 108 * 1024 ? 3
           : 2 * bytes <= 108 * 1024 ? 2 : 3 * bytes <= 216 * 1024 ? 3 : 2;
}

// What split operands make of values that are not finite, or that round to infinity in the operand's type, is NaN
// (inf - inf), never a finite number; zeros that fill a tile do the same.  So a result that is not finite is summed
// once more, term by term in fp32 up to a NaN, which gives the infinity, the NaN or the finite value that the formula
// has.  Threads find out from the sum of their results, which costs less than a look at each.
__device__ __forceinline__ bool finite(float v) { return fabsf(v) <= 3.402823466e38f; }
__device__ __forceinline__ float finite_abs(float v) { return finite(v) ? fabsf(v) : 0.f; }
struct Total {  // of many results, two at a time
    uint64_t two = 0;
    __device__ __forceinline__ void add(float a, float b) {
        asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%1, %2};\n\tadd.rn.f32x2 %0, %0, t;\n\t}" : "+l"(two) : "f"(a), "f"(b));
    }
    __device__ __forceinline__ bool ok() const {
        return finite(__uint_as_float((uint32_t)two) + __uint_as_float((uint32_t)(two >> 32)));
    }
};

// ---- shrink --------------------------------------------------------------------
// h[split, t, :] = scale_i * sum over this split's columns k of x[t, k] W_i[:, k].
// TRANS = false: W_i = A_i [rank, K] (K consecutive); true: W_i = B_i [K, rank] (rank consecutive).
// WM = 8: 64 positions of a tile of 128 a block, four warps of 16 along them; WM = 1: 16 positions.  The other
// warps share the columns and are summed, in their order, through shared memory.  (128 positions a block
// left two stages of a ring: 30 us where this takes 22 for 2048 x 12800 in fp32.)  A chunk is 64 bytes of a
// row, two steps of the MMA.  fp32 fragments come as 16-byte reads: a lane holds columns 4 q ..
// 4 q + 3 of its row, of which step s takes 2 s and 2 s + 1 (the order inside a sum is free as long as
// both operands agree).  Rows are padded so that those reads (two rows of 64 bytes a quarter warp: 64
// bytes) and ldmatrix (eight rows of 16: 16 bytes) meet no bank twice.
template <typename T, int RB, int WM, bool TRANS>
struct ShrinkCfg {
    static constexpr int E = kE<T>, RP = 8 * RB, TILE = 16 * WM, PAD = sizeof(T) == 4 ? 64 : 16;
    static constexpr int WR = WM == 8 ? 4 : 1, BM = 16 * WR, PARTS = TILE / BM, WK = kWarps / WR;  // warps along rows, columns
    static constexpr int NCH = WM == 1 ? 8 : 4, KC = NCH * 4 * E;  // chunks and columns of a stage
    static constexpr int X_PITCH = NCH * 64 + PAD, X_BYTES = BM * X_PITCH;
    static constexpr int W_PITCH = TRANS ? RP * (int)sizeof(T) + 16 : X_PITCH;
    static constexpr int W_BYTES = (TRANS ? KC : RP) * W_PITCH;
    static constexpr int STAGE = X_BYTES + W_BYTES;
    static constexpr int NS = fit_stages(STAGE);
    static constexpr int RED = WK * BM * RP * 4;
    static constexpr int MOST = NS * STAGE > RED ? NS * STAGE : RED;
    static constexpr int SMEM = MOST > (int)sizeof(FindTile) ? MOST : (int)sizeof(FindTile);
    static_assert(SMEM <= 220 * 1024, "a block's shared memory");
};

// Where a block finds its tile: k_plan's, found here and written to `plan`, or written by a launch before.
enum Tiles { PLANNED, FIND };

// One of the two sums: its operands, width and columns of a split, and where it goes.
template <typename T>
struct Shrink {
    const T* x;
    int64_t ldx;
    const T* w;
    int64_t K, k_split;
    int splits;
    bool xvec, wvec;
    float* h;
};

// A position's sum over columns k_begin .. k_end for one rank; beyond the last there is nothing.
template <bool TRANS, typename T>
__device__ __forceinline__ float plain_shrink(const T* x, const T* w, int64_t K, int rank, int r, int64_t k_begin,
                                              int64_t k_end) {
    float v = 0.f;
    if (r < rank)
#pragma unroll 1
        for (int64_t k = k_begin; k < k_end && v == v; k++) v = fmaf(wide(x[k]), wide(TRANS ? w[k * rank + r] : w[r * K + k]), v);
    return v;
}

template <typename T, int RB, int WM, bool TRANS>
__device__ __forceinline__ void shrink_tile(uint8_t* smem, TileRows<16 * WM>& tr, const Plan& plan, int tiles,
                                            const int32_t* __restrict__ index, const Shrink<T>& side,
                                            const float* __restrict__ scale, int n, int rank, int T_rows, int split) {
    using C = ShrinkCfg<T, RB, WM, TRANS>;
    constexpr int E = C::E, RP = C::RP, BM = C::BM, WK = C::WK, NCH = C::NCH, KC = C::KC, NS = C::NS;
    constexpr bool F32 = sizeof(T) == 4;
    const T* __restrict__ x = side.x;
    const T* __restrict__ w = side.w;
    const int64_t ldx = side.ldx, K = side.K, k_split = side.k_split;
    const bool xvec = side.xvec, wvec = side.wvec;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    const int wm = warp % C::WR, wk = warp / C::WR;
    int from = 0;  // this block's first position of the tile
    if (tiles == FIND) {
        let_next_start();
        const int k = blockIdx.x / C::PARTS;
        find_tile<C::TILE>(*reinterpret_cast<FindTile*>(smem), tr, index, T_rows, n, k);
        from = (int)(blockIdx.x % C::PARTS) * BM;
        if (blockIdx.y == 0 && from == 0) {
            for (int i = threadIdx.x; i < tr.rows; i += kThreads) plan.perm[k * C::TILE + i] = tr.row[i];
            if (threadIdx.x == 0) plan.tile[k] = Tile{tr.adapter, k * C::TILE, tr.rows, 0};
        }
        if (tr.rows <= from || tr.adapter >= n) return;
        __syncthreads();  // the scan's memory becomes the stages'
    } else {
        wait_for_previous();
        let_next_start();
        if (!read_tile<BM, C::PARTS>(tr, plan) || tr.adapter >= n) return;
    }
    const int adapter = tr.adapter, rows = min(BM, tr.rows - from);
    const int32_t* row_of = tr.row + from;
    const T* wi = w + (int64_t)adapter * rank * K;
    const int64_t k_begin = split * k_split, k_end = k_begin + k_split < K ? k_begin + k_split : K;
    const int stages = k_begin < k_end ? (int)((k_end - k_begin + KC - 1) / KC) : 0;

    constexpr int XU = NCH * 4, WU = TRANS ? RP / E : NCH * 4, WR = TRANS ? KC : RP;
    Units<T, BM, XU> ux;
    Units<T, WR, WU> uw;
#pragma unroll
    for (int k = 0; k < ux.N; k++) {
        const int r = ux.row(k);
        ux.src[k] = x + (int64_t)row_of[min(r, BM - 1)] * ldx + k_begin + ux.column() * E;
        ux.bytes[k] = r < rows ? 16 : 0;
    }
#pragma unroll
    for (int k = 0; k < uw.N; k++) {
        const int r = uw.row(k), c = uw.column() * E;
        const bool real = TRANS ? c < rank : r < rank;
        uw.src[k] = !real ? w : TRANS ? wi + (k_begin + r) * rank + c : wi + (int64_t)r * K + k_begin + c;
        uw.bytes[k] = real ? 16 : 0;
    }
    const auto load = [&](int i) {
        uint8_t* xs = smem + (i % NS) * C::STAGE;
        uint8_t* ws = xs + C::X_BYTES;
        const int64_t k0 = k_begin + (int64_t)i * KC, left = k_end - k0;
        if (xvec && left >= KC) {
            const uint32_t to = smem_u32(xs) + ux.row(0) * C::X_PITCH + ux.column() * 16;
#pragma unroll
            for (int k = 0; k < ux.N; k++)
                if (ux.mine(k)) ux.copy(k, to + k * ux.STEP * C::X_PITCH, (int64_t)i * KC);
        } else {
            for (int u = threadIdx.x; u < BM * XU; u += kThreads) {
                const int r = u / XU, c = u % XU;
                stage_unit<T>(xs + r * C::X_PITCH + c * 16, x + (int64_t)row_of[r] * ldx + k0 + c * E, x,
                              r < rows ? left - c * E : 0, xvec);
            }
        }
        if (wvec && left >= KC) {
            const uint32_t to = smem_u32(ws) + uw.row(0) * C::W_PITCH + uw.column() * 16;
#pragma unroll
            for (int k = 0; k < uw.N; k++)
                if (uw.mine(k))
                    uw.copy(k, to + k * uw.STEP * C::W_PITCH, uw.bytes[k] ? (int64_t)i * KC * (TRANS ? rank : 1) : 0);
        } else {
            for (int u = threadIdx.x; u < WR * WU; u += kThreads) {
                const int r = u / WU, c = u % WU;
                if constexpr (TRANS)
                    stage_unit<T>(ws + r * C::W_PITCH + c * 16, wi + (k0 + r) * rank + c * E, w,
                                  r < left ? rank - c * E : 0, wvec);
                else
                    stage_unit<T>(ws + r * C::W_PITCH + c * 16, wi + (int64_t)r * K + k0 + c * E, w,
                                  r < rank ? left - c * E : 0, wvec);
            }
        }
        stage_done();
    };

    float acc[RB][4], sum[F32 ? RB : 1][4];
#pragma unroll
    for (int b = 0; b < RB; b++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[b][i] = 0.f;
#pragma unroll
    for (int b = 0; b < (F32 ? RB : 1); b++)
#pragma unroll
        for (int i = 0; i < 4; i++) sum[b][i] = 0.f;
#pragma unroll
    for (int i = 0; i < NS - 1; i++) {
        if (i < stages) load(i);
        else stage_done();
    }
    for (int i = 0; i < stages; i++) {
        stage_wait<NS - 2>();
        __syncthreads();
        if (i + NS - 1 < stages) load(i + NS - 1);
        else stage_done();
        const uint8_t* xs = smem + (i % NS) * C::STAGE;
        const uint8_t* ws = xs + C::X_BYTES;
#pragma unroll
        for (int cc = 0; cc < NCH / WK; cc++) {
            const int ch = wk + WK * cc;
            if constexpr (F32) {
                const uint8_t* xp = xs + (16 * wm + g) * C::X_PITCH + (4 * ch + q) * 16;
                const uint4 xa = lds128(xp), xb = lds128(xp + 8 * C::X_PITCH);
                const Split f0 = split_a(xa.x, xb.x, xa.y, xb.y), f1 = split_a(xa.z, xb.z, xa.w, xb.w);
                if constexpr (!TRANS) {
#pragma unroll
                    for (int b = 0; b < RB; b += 2) {
                        const uint4 wa = lds128(ws + (8 * b + g) * C::W_PITCH + (4 * ch + q) * 16);
                        const uint4 wb = lds128(ws + (8 * b + 8 + g) * C::W_PITCH + (4 * ch + q) * 16);
                        mma_split2(acc[b], acc[b + 1], f0, wa.x, wa.y, wb.x, wb.y);
                        mma_split2(acc[b], acc[b + 1], f1, wa.z, wa.w, wb.z, wb.w);
                    }
                } else {  // a lane's column of block b is rank RB g + b
#pragma unroll
                    for (int s = 0; s < 2; s++) {
                        const uint8_t* p = ws + (16 * ch + 4 * q + 2 * s) * C::W_PITCH + RB * g * 4;
                        uint32_t wv[2][RB];
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            if constexpr (RB == 2) {
                                const uint2 v = *reinterpret_cast<const uint2*>(p + j * C::W_PITCH);
                                wv[j][0] = v.x, wv[j][1] = v.y;
                            } else {
#pragma unroll
                                for (int b = 0; b < RB; b += 4) {
                                    const uint4 v = lds128(p + j * C::W_PITCH + 4 * b);
                                    wv[j][b] = v.x, wv[j][b + 1] = v.y, wv[j][b + 2] = v.z, wv[j][b + 3] = v.w;
                                }
                            }
                        }
#pragma unroll
                        for (int b = 0; b < RB; b += 2)
                            mma_split2(acc[b], acc[b + 1], s ? f1 : f0, wv[0][b], wv[1][b], wv[0][b + 1], wv[1][b + 1]);
                    }
                }
            } else {
                const int lr = lane & 7, lm = lane >> 3;  // ldmatrix: row and matrix of this lane's address
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    uint32_t fa[4];
                    ldmatrix4(fa, xs + (16 * wm + lr + 8 * (lm & 1)) * C::X_PITCH + (4 * ch + 2 * s + (lm >> 1)) * 16);
#pragma unroll
                    for (int b = 0; b < RB; b += 2) {
                        uint32_t fb[4];
                        if constexpr (!TRANS)
                            ldmatrix4(fb, ws + (8 * b + lr + 8 * (lm >> 1)) * C::W_PITCH +
                                              (4 * ch + 2 * s + (lm & 1)) * 16);
                        else
                            ldmatrix4_trans(fb, ws + (32 * ch + 16 * s + lr + 8 * (lm & 1)) * C::W_PITCH +
                                                    (b + (lm >> 1)) * 16);
                        mma<T>(acc[b], fa, fb[0], fb[1]);
                        mma<T>(acc[b + 1], fa, fb[2], fb[3]);
                    }
                }
            }
        }
        if constexpr (F32) {
#pragma unroll
            for (int b = 0; b < RB; b++)
#pragma unroll
                for (int k = 0; k < 4; k++) sum[b][k] += acc[b][k], acc[b][k] = 0.f;
        }
    }
    const auto result = [&](int b, int k) { return F32 ? sum[F32 ? b : 0][k] : acc[b][k]; };
    const auto column = [&](int b, int j) { return F32 && TRANS ? RB * (2 * q + j) + b : 8 * b + 2 * q + j; };
    const float s = scale ? __ldg(scale + adapter) : 1.f;
    float* dst = side.h + (int64_t)split * T_rows * RP;
    stage_wait<0>();
    __syncthreads();
    float* red = reinterpret_cast<float*>(smem);  // [WK][BM][RP]
#pragma unroll
    for (int b = 0; b < RB; b++)
#pragma unroll
        for (int k = 0; k < 4; k++) red[(wk * BM + 16 * wm + g + 8 * (k >> 1)) * RP + column(b, k & 1)] = result(b, k);
    __syncthreads();
    float all = 0.f;  // of this thread's sums: not finite where one is not
    for (int e = threadIdx.x; e < rows * RP; e += kThreads) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < WK; k++) v += red[k * BM * RP + e];
        dst[(int64_t)row_of[e / RP] * RP + e % RP] = s * v;
        all += v;
    }
    if (!finite(all)) {
#pragma unroll 1
        for (int e = threadIdx.x; e < rows * RP; e += kThreads) {
            float* h = dst + (int64_t)row_of[e / RP] * RP + e % RP;
            if (!finite(*h)) *h = s * plain_shrink<TRANS>(x + (int64_t)row_of[e / RP] * ldx, wi, K, rank, e % RP, k_begin, k_end);
        }
    }
}

template <typename T, int RB, int WM>
__global__ void __launch_bounds__(kThreads, RB <= 4 ? 3 : 1) k_shrink(Plan plan, int tiles, const int32_t* __restrict__ index,
                                                                      Shrink<T> side, const float* __restrict__ scale, int n,
                                                                      int rank, int T_rows) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ TileRows<16 * WM> tr;
    shrink_tile<T, RB, WM, false>(smem, tr, plan, tiles, index, side, scale, n, rank, T_rows, (int)blockIdx.y);
}

// Both sums of the gradients, dh over grad's columns and h over x's, either of which may have no splits: blocks of
// one fill the SMs that the other's last wave leaves (two launches: 43 us for 2048 positions of 12800 + 2560 fp32).
template <typename T, int RB, int WM>
__global__ void __launch_bounds__(kThreads, RB <= 4 ? 3 : 1)
    k_shrink_both(Plan plan, int tiles, const int32_t* __restrict__ index, Shrink<T> dh, Shrink<T> h,
                  const float* __restrict__ scale, int n, int rank, int T_rows) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ TileRows<16 * WM> tr;
    const int y = (int)blockIdx.y;
    if (y < dh.splits)
        shrink_tile<T, RB, WM, true>(smem, tr, plan, tiles, index, dh, scale, n, rank, T_rows, y);
    else
        shrink_tile<T, RB, WM, false>(smem, tr, plan, tiles, index, h, scale, n, rank, T_rows, y - dh.splits);
}

// 4 consecutive ranks of a position's h, summed over the splits.
__device__ __forceinline__ float4 load_h(const float* h, int splits, int64_t stride) {
    float4 f = *reinterpret_cast<const float4*>(h);
    for (int k = 1; k < splits; k++) {
        const float4 u = *reinterpret_cast<const float4*>(h + k * stride);
        f.x += u.x, f.y += u.y, f.z += u.z, f.w += u.w;
    }
    return f;
}

// The splits' sums into the first, of two arrays, for the launches that read them often.  Rows without an
// adapter hold nothing and are summed like the others.
__global__ void __launch_bounds__(kThreads) k_sum_splits(float4* h, int h_splits, float4* dh, int dh_splits,
                                                         int64_t count4) {
    wait_for_previous();
    let_next_start();
    const int64_t i = blockIdx.x * (int64_t)kThreads + threadIdx.x;
    float4* p = blockIdx.y ? dh : h;
    const int splits = blockIdx.y ? dh_splits : h_splits;
    if (i >= count4 || splits < 2) return;
    float4 f = p[i];
#pragma unroll 4
    for (int k = 1; k < splits; k++) {
        const float4 u = p[k * count4 + i];
        f.x += u.x, f.y += u.y, f.z += u.z, f.w += u.w;
    }
    p[i] = f;
}

// The sum over ranks of a position's h and one column of factors, `step` elements apart.
template <typename T>
__device__ __forceinline__ float plain_expand(const float* h, int splits, int64_t stride, const T* w, int64_t step, int rank) {
    float y = 0.f;
#pragma unroll 1
    for (int r = 0; r < rank && y == y; r++) {
        float v = h[r];
#pragma unroll 1
        for (int k = 1; k < splits; k++) v += h[r + k * stride];
        y = fmaf(v, wide(w[r * step]), y);
    }
    return y;
}

// 2^(14 - e) for m in [2^e, 2^(e + 1)): brings m into fp16 below 2^15; 1 for zero and for what is not finite.
__device__ __forceinline__ float half_scale(float m) {
    const int e = (int)((bits_of(m) >> 23) & 255) - 127;
    return (e < -126 || e > 127) ? 1.f : __uint_as_float((uint32_t)(min(max(14 - e, -126), 126) + 127) << 23);
}

// ---- expand --------------------------------------------------------------------
// out[t, f] = base[t, f] + sum over ranks of h[t, r] W_i[f, r]; positions without an adapter get base.
// TRANS = false: W_i = B_i [F, rank]; true: W_i = A_i [rank, F].  base null: zeros.
// BIG: 64 positions, half a tile, four warps of 16 along them and two along the columns (16 bits at ranks
// over 32: the whole tile, warps of 32, which halves the reads of the factors).  Else 16 positions and
// all warps along the columns.  A
// warp keeps its positions' h fragments in registers and takes 32 columns at a time, dealt to the MMAs
// so that a lane ends up with whole 16-byte units of its rows and four lanes with 64 consecutive bytes:
// unit 4 v + q holds, for fp32, columns 2 (b % 2) + j of blocks b = 2 v, 2 v + 1 (TRANS: columns b of MMA
// column 2 q + v), for 16 bits columns 2 b + j (TRANS: 4 j + b).
template <typename T, int RB, bool BIG, bool TRANS>
struct ExpandCfg {
    static constexpr int E = kE<T>, RP = 8 * RB, SIZE = sizeof(T);
    static constexpr int MT = BIG && SIZE == 2 && RB >= 8 ? 2 : 1, WM = BIG ? 4 : 1, WF = kWarps / WM;
    static constexpr int BM = 16 * MT * WM, PARTS = BIG ? 128 / BM : 1;  // blocks of a tile
    // columns of a stage
    static constexpr int FS = BIG ? (SIZE == 2 && RB <= 4 ? 128 : 64) : RP * SIZE == 512 ? 128 : 256;
    static constexpr int FU = FS / E;  // units of a row
    static constexpr int B_PITCH = FS * SIZE + 64, B_BYTES = BM * B_PITCH;
    // B_i rows lie in the order in which the lanes of an MMA read them (row_slot), at a pitch that puts the
    // two rows of a quarter warp's 16-byte reads 64 bytes apart (fp32), the four of a half warp's 8-byte
    // reads 32 (16 bits).  A_i rows are dense, their units swapped by row number.
    static constexpr int W_PITCH = TRANS ? FS * SIZE
                                         : SIZE == 4 ? (RP == 16 ? 64 : RP * 4 + 64) : (RP == 16 ? 32 : RP * 2 + 32);
    static constexpr int W_BYTES = (TRANS ? RP : FS) * W_PITCH;
    static constexpr int STAGE = B_BYTES + W_BYTES;
    static constexpr int NS = fit_stages(STAGE);
    static constexpr int SMEM = NS * STAGE;
    static_assert(SMEM <= 220 * 1024, "a block's shared memory");
};

// Place of feature f (of each 32) of B_i in a stage: block b's eight rows follow one another.
template <typename T>
__device__ __forceinline__ int row_slot(int f) {
    if constexpr (sizeof(T) == 4)  // f = 16 v + 4 q + 2 (b % 2) + j, b = 2 v + b % 2
        return (f & ~31) + 8 * (2 * ((f >> 4) & 1) + ((f >> 1) & 1)) + 2 * ((f >> 2) & 3) + (f & 1);
    else  // f = 8 q + 2 b + j
        return (f & ~31) + 8 * ((f >> 1) & 3) + 2 * ((f >> 3) & 3) + (f & 1);
}

// Columns [f, f_end) of the rows: out = base (null: zeros).
template <typename T>
__device__ __forceinline__ void copy_rows(const int32_t* row, int rows, const T* base, int64_t ldb, T* out, int64_t ldo,
                                          int64_t f, int64_t f_end, bool vec) {
    constexpr int E = kE<T>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int r = warp; r < rows; r += kWarps) {
        const T* src = base ? base + (int64_t)row[r] * ldb : nullptr;
        T* dst = out + (int64_t)row[r] * ldo;
        for (int64_t c = f + lane * E; c < f_end; c += 32 * E) {
            if (base && vec && c + E <= f_end) {
                *reinterpret_cast<uint4*>(dst + c) = *reinterpret_cast<const uint4*>(src + c);
            } else {
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (c + e < f_end) dst[c + e] = base ? src[c + e] : narrow<T>(0.f);
            }
        }
    }
}

// The results of a lane's rows and columns (of 32) that are not finite, once more.  bs: the rows' base, or null.
template <typename T, typename C, bool TRANS>
__device__ __noinline__ void patch_piece(const int32_t* row, int rows, int first, const uint8_t* bs, const float* h, int splits,
                                         int T_rows, const T* w, int64_t F, int rank, int left, T* out, int64_t ldo) {
    constexpr int E = C::E;
    const int q = threadIdx.x & 3;
    for (int i = 0; i < 16 * C::MT; i++) {
        const int e = i % 8, r = first + 8 * (i / 8), f = (4 * (e / E) + q) * E + e % E;
        if (r >= rows || f >= left) continue;
        const int64_t t = row[r];
        if (finite(wide(out[t * ldo + f]))) continue;
        const float y = plain_expand<T>(h + t * C::RP, splits, (int64_t)T_rows * C::RP, w + (TRANS ? f : (int64_t)f * rank),
                                        TRANS ? F : 1, rank);
        out[t * ldo + f] = narrow<T>(bs ? wide(reinterpret_cast<const T*>(bs + r * C::B_PITCH)[f]) + y : y);
    }
}

template <typename T, int RB, bool BIG, bool TRANS>
__global__ void __launch_bounds__(kThreads, RB * (int)sizeof(T) <= 8 ? 3 : RB * (int)sizeof(T) <= 16 ? 2 : 1) k_expand(Plan plan, const float* h, int splits, const T* __restrict__ w,
                                                     int n, int rank, int64_t F, int64_t f_block, int T_rows,
                                                     const T* base, int64_t ldb, T* out, int64_t ldo, bool bvec,
                                                     bool wvec, bool ovec) {
    using C = ExpandCfg<T, RB, BIG, TRANS>;
    constexpr int E = C::E, RP = C::RP, BM = C::BM, MT = C::MT, FS = C::FS, FU = C::FU, NS = C::NS;
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int KS = F32 ? RP / 8 : RP / 16;  // MMA steps of the rank
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ TileRows<BM> tr;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    const int wm = warp % C::WM, wf = warp / C::WM;
    wait_for_previous();
    let_next_start();
    if (!read_tile<BM, C::PARTS>(tr, plan)) return;
    const int adapter = tr.adapter, rows = tr.rows;
    const int64_t f_begin = blockIdx.y * f_block, f_end = f_begin + f_block < F ? f_begin + f_block : F;
    if (adapter >= n) {  // no adapter: base, or zeros
        if (base != out) copy_rows<T>(tr.row, rows, base, ldb, out, ldo, f_begin, f_end, bvec && ovec);
        return;
    }
    const T* wi = w + (int64_t)adapter * rank * F;
    const int stages = f_begin < f_end ? (int)((f_end - f_begin + FS - 1) / FS) : 0;

    constexpr int WU = TRANS ? FU : RP / E, WR = TRANS ? RP : FS;
    const auto w_place = [](int r, int c) {  // where a unit of the factors stands
        if constexpr (!TRANS) return row_slot<T>(r) * C::W_PITCH + c * 16;
        else return r * C::W_PITCH + (F32 ? c ^ ((r >> 2) & 3) : c ^ (((r >> 2) & 3) << 1)) * 16;
    };
    Units<T, BM, FU> ub;
    Units<T, WR, WU> uw;
#pragma unroll
    for (int k = 0; k < ub.N; k++) {
        const int r = ub.row(k);
        ub.src[k] = base + (int64_t)tr.row[min(r, BM - 1)] * ldb + f_begin + ub.column() * E;
        ub.bytes[k] = r < rows ? 16 : 0;
    }
#pragma unroll
    for (int k = 0; k < uw.N; k++) {
        const int r = uw.row(k), c = uw.column() * E;
        const bool real = TRANS ? r < rank : c < rank;
        uw.src[k] = !real ? w : TRANS ? wi + (int64_t)r * F + f_begin + c : wi + (f_begin + r) * rank + c;
        uw.bytes[k] = real ? 16 : 0;
    }
    const auto load = [&](int i) {
        uint8_t* bs = smem + (i % NS) * C::STAGE;
        uint8_t* ws = bs + C::B_BYTES;
        const int64_t f0 = f_begin + (int64_t)i * FS, left = f_end - f0;
        if (bvec && left >= FS) {
            const uint32_t to = smem_u32(bs) + ub.row(0) * C::B_PITCH + ub.column() * 16;
#pragma unroll
            for (int k = 0; k < ub.N; k++)
                if (ub.mine(k)) ub.copy(k, to + k * ub.STEP * C::B_PITCH, (int64_t)i * FS);
        } else if (base) {
            for (int u = threadIdx.x; u < BM * FU; u += kThreads) {
                const int r = u / FU, c = u % FU;
                if (r < rows)
                    stage_unit<T>(bs + r * C::B_PITCH + c * 16, base + (int64_t)tr.row[r] * ldb + f0 + c * E, base,
                                  left - c * E, bvec);
            }
        }
        if (wvec && left >= FS) {
#pragma unroll
            for (int k = 0; k < uw.N; k++)
                if (uw.mine(k))
                    uw.copy(k, smem_u32(ws) + w_place(uw.row(k), uw.column()),
                            uw.bytes[k] ? (int64_t)i * FS * (TRANS ? 1 : rank) : 0);
        } else {
            for (int u = threadIdx.x; u < WR * WU; u += kThreads) {
                const int r = u / WU, c = u % WU;
                if constexpr (TRANS)
                    stage_unit<T>(ws + w_place(r, c), wi + (int64_t)r * F + f0 + c * E, w, r < rank ? left - c * E : 0,
                                  wvec);
                else
                    stage_unit<T>(ws + w_place(r, c), wi + (f0 + r) * rank + c * E, w, r < left ? rank - c * E : 0,
                                  wvec);
            }
        }
        stage_done();
    };
#pragma unroll
    for (int i = 0; i < NS - 1; i++) {
        if (i < stages) load(i);
        else stage_done();
    }

    // h of the warp's rows, split, and where they go
    uint32_t hi[MT][KS][4], lo[MT][KS][4];
    T* dst[2 * MT];
    float undo[2 * MT];  // fp16: the rows' scales taken back
    bool live[2 * MT];
#pragma unroll
    for (int m = 0; m < 2 * MT; m++) {
        const int r = 16 * MT * wm + 8 * m + g, t = tr.row[min(r, rows - 1)];
        live[m] = r < rows;
        dst[m] = out + (int64_t)t * ldo;
        undo[m] = 1.f;
        float v[RP / 4];  // ranks 16 c + 4 q .. + 3
        const float* hp = h + (int64_t)t * RP + 4 * q;
#pragma unroll
        for (int c = 0; c < RP / 16; c++) {
            const float4 f = load_h(hp + 16 * c, splits, (int64_t)T_rows * RP);
            v[4 * c] = f.x, v[4 * c + 1] = f.y, v[4 * c + 2] = f.z, v[4 * c + 3] = f.w;
        }
        if constexpr (std::is_same_v<T, __half>) {
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < RP / 4; i++) most = fmaxf(most, finite_abs(v[i]));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const float s = half_scale(most);
            undo[m] = 1.f / s;
#pragma unroll
            for (int i = 0; i < RP / 4; i++) v[i] *= s;
        }
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                uint32_t &a = hi[m >> 1][s][(m & 1) + 2 * k], &b = lo[m >> 1][s][(m & 1) + 2 * k];
                if constexpr (F32) {
                    split_tf32(bits_of(v[2 * s + k]), a, b);
                } else {  // ranks 4 q + 2 k, + 1 of the step: the sum's order is the factors' below
                    const float v0 = v[4 * s + 2 * k], v1 = v[4 * s + 2 * k + 1];
                    a = pack2<T>(v0, v1);
                    const float2 back = unpack2<T>(a);
                    b = pack2<T>(v0 - back.x, v1 - back.y);
                }
            }
    }

    for (int i = 0; i < stages; i++) {
        stage_wait<NS - 2>();
        __syncthreads();
        if (i + NS - 1 < stages) load(i + NS - 1);
        else stage_done();
        const uint8_t* bs = smem + (i % NS) * C::STAGE;
        const uint8_t* ws = bs + C::B_BYTES;
        const int64_t f0 = f_begin + (int64_t)i * FS;
#pragma unroll 1
        for (int fs = 32 * wf; fs < FS; fs += 32 * C::WF) {  // 32 columns from f0 + fs
            const int left = f_end - f0 - fs < 32 ? (int)(f_end - f0 - fs) : 32;
            if (left <= 0) break;
            float acc[MT][4][4];
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int b = 0; b < 4; b++)
#pragma unroll
                    for (int k = 0; k < 4; k++) acc[m][b][k] = 0.f;
            if constexpr (F32) {
#pragma unroll
                for (int c = 0; c < RP / 16; c++) {
                    uint32_t wv[2][2][4];  // step, rank of the pair, block
                    if constexpr (!TRANS) {
#pragma unroll
                        for (int b = 0; b < 4; b++) {
                            const uint4 v = lds128(ws + (fs + 8 * b + g) * C::W_PITCH + (4 * c + q) * 16);
                            wv[0][0][b] = v.x, wv[0][1][b] = v.y, wv[1][0][b] = v.z, wv[1][1][b] = v.w;
                        }
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const int u = (fs + 16 * (g & 1)) / 4 + (g >> 1);
                            const uint4 v = lds128(ws + (16 * c + 4 * q + r) * C::W_PITCH + ((u ^ q) * 16));
                            wv[r >> 1][r & 1][0] = v.x, wv[r >> 1][r & 1][1] = v.y;
                            wv[r >> 1][r & 1][2] = v.z, wv[r >> 1][r & 1][3] = v.w;
                        }
                    }
#pragma unroll
                    for (int s = 0; s < 2; s++) {
                        uint32_t wh[2][4], wl[2][4];
#pragma unroll
                        for (int b = 0; b < 4; b++) {
                            split_tf32(wv[s][0][b], wh[0][b], wl[0][b]);
                            split_tf32(wv[s][1][b], wh[1][b], wl[1][b]);
                        }
#pragma unroll
                        for (int b = 0; b < 4; b++) mma<float>(acc[0][b], lo[0][2 * c + s], wh[0][b], wh[1][b]);
#pragma unroll
                        for (int b = 0; b < 4; b++) mma<float>(acc[0][b], hi[0][2 * c + s], wl[0][b], wl[1][b]);
#pragma unroll
                        for (int b = 0; b < 4; b++) mma<float>(acc[0][b], hi[0][2 * c + s], wh[0][b], wh[1][b]);
                    }
                }
            } else {
#pragma unroll
                for (int s = 0; s < KS; s++) {
                    uint32_t w0[4], w1[4];
                    if constexpr (!TRANS) {
                        // a lane's four ranks 4 q .. 4 q + 3 of a step are the MMA's k = 2 q, 2 q + 1, 2 q + 8, 2 q + 9
#pragma unroll
                        for (int b = 0; b < 4; b++) {
                            const uint2 v = *reinterpret_cast<const uint2*>(ws + (fs + 8 * b + g) * C::W_PITCH + 32 * s + 8 * q);
                            w0[b] = v.x, w1[b] = v.y;
                        }
                    } else {
                        uint2 v[4];  // ranks 4 q .. 4 q + 3, columns 4 g .. 4 g + 3
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            v[j] = *reinterpret_cast<const uint2*>(ws + (16 * s + 4 * q + j) * C::W_PITCH +
                                                                   (((fs / 8 + (g >> 1)) ^ (q << 1)) * 16) + (g & 1) * 8);
#pragma unroll
                        for (int b = 0; b < 4; b++) {
                            const uint32_t pick = (b & 1) ? 0x7632u : 0x5410u;
                            w0[b] = __byte_perm(b < 2 ? v[0].x : v[0].y, b < 2 ? v[1].x : v[1].y, pick);
                            w1[b] = __byte_perm(b < 2 ? v[2].x : v[2].y, b < 2 ? v[3].x : v[3].y, pick);
                        }
                    }
#pragma unroll
                    for (int b = 0; b < 4; b++)
#pragma unroll
                        for (int m = 0; m < MT; m++) mma<T>(acc[m][b], lo[m][s], w0[b], w1[b]);
#pragma unroll
                    for (int b = 0; b < 4; b++)
#pragma unroll
                        for (int m = 0; m < MT; m++) mma<T>(acc[m][b], hi[m][s], w0[b], w1[b]);
                }
            }
            float all = 0.f;  // not finite where a product is not
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int b = 0; b < 4; b++) all += (acc[m][b][0] + acc[m][b][1]) + (acc[m][b][2] + acc[m][b][3]);
#pragma unroll
            for (int m = 0; m < 2 * MT; m++) {
                if (!live[m]) continue;
                const uint8_t* bp = bs + (16 * MT * wm + 8 * m + g) * C::B_PITCH + fs * (int)sizeof(T) + 16 * q;
                T* to = dst[m] + f0 + fs;
#pragma unroll
                for (int v = 0; v < 8 / E; v++) {
                    alignas(16) T o[E], d[E];
                    if (base) *reinterpret_cast<uint4*>(d) = lds128(bp + 64 * v);
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        const int b = F32 ? (TRANS ? e : 2 * v + (e >> 1)) : TRANS ? e & 3 : e >> 1;
                        const int j = F32 ? (TRANS ? v : e & 1) : TRANS ? e >> 2 : e & 1;
                        float y = acc[m >> 1][b][2 * (m & 1) + j];
                        if constexpr (std::is_same_v<T, __half>) y *= undo[m];
                        o[e] = narrow<T>(base ? wide(d[e]) + y : y);
                    }
                    const int f = (4 * v + q) * E;
                    if (ovec && f + E <= left) {
                        *reinterpret_cast<uint4*>(to + f) = *reinterpret_cast<const uint4*>(o);
                    } else {
#pragma unroll
                        for (int e = 0; e < E; e++)
                            if (f + e < left) to[f + e] = o[e];
                    }
                }
            }
            if (!finite(all))
                patch_piece<T, C, TRANS>(tr.row, rows, 16 * MT * wm + g, base ? bs + fs * (int)sizeof(T) : nullptr, h, splits, T_rows,
                                         wi + (TRANS ? 1 : rank) * (f0 + fs), F, rank, left, out + f0 + fs, ldo);
        }
    }
}

// ---- expand on the tcgen05 tensor cores -------------------------------------------
// The same product, TRANS = false, for much work at ranks over 16 (run_expand's rule), rows of base and out that start on
// 16 bytes and whole
// groups of 32 columns (fp32: 16).  What the kernel above spends its time on is instructions, 400 to 500 a
// 32 x 32 piece; here the products and the factors' way to them cost the streaming warps nothing:
//   warps 0-15  out = base + accumulator, 16 positions x 256 bytes a warp and stage, eight warps a stage in
//               turn.  A lane fetches the units of base that it will add to by cp.async into a place of
//               its own, DEPTH of its stages ahead (64 KB in flight an SM each), so base needs no barriers;
//               with base and out on TMA and mbarriers this took 1.5 to 2 times as long;
//   warp 16     the factors' tiles by TMA, NS stages ahead;
//   warp 17     one lane issues the MMAs, D [128 positions, FS columns] = H_hi W^T + H_lo W^T (fp32: in TF32,
//               H_lo W^T + H_hi W_lo^T + H_hi W^T; the tensor cores read W as its head), into four
//               accumulators in turn;
//   warp 18     h of a new tile, split, into the A operand's layout;
//   warp 19     fp32: the factors' remainders W_lo.
// An accumulator is read in the 16x256b form: a lane gets columns 2 q, 2 q + 1 of each 8 of rows g and g + 8.
// The factors' rows are loaded in an order (a five-dimensional tensor map) that makes a lane's columns of 32
// (fp32: 16) one 16-byte unit of the row: column 8 k + 2 q + j of the product is feature 8 q + 2 k + j (fp32: 4 q
// + 2 k + j).  Blocks are persistent, one an SM, and share all (tile, stage) pairs evenly in their order.
// Every wait is bounded: one that gives up (never, in a correct run) ends its warp's loop, the waits on that warp
// give up in their turn, and the results that are then missing are written as NaN.
template <typename T, int RB>
struct WideCfg {
    static constexpr int SIZE = sizeof(T), RP = 8 * RB, BM = 128;
    static constexpr bool F32 = SIZE == 4;
    static constexpr int GROUP = F32 ? 16 : 32, FS = 4 * GROUP, BLOCKS = GROUP / 8;  // columns of a warp, of a stage
    // the rank's extent in the operands: rows of SPAN bytes (the swizzle), in blocks of all rows
    static constexpr int SPAN = RP * SIZE < 128 ? RP * SIZE : 128, KB = RP * SIZE / SPAN;
    static constexpr int H_BYTES = BM * RP * SIZE, W_BYTES = FS * RP * SIZE;
    static constexpr int STAGE = W_BYTES * (F32 ? 2 : 1), NS = RP * SIZE >= 256 ? 2 : 3;
    static constexpr int FETCH = 16 * 4096;  // a stage of all sixteen warps
    static constexpr int FIT = (220 * 1024 - 2 * H_BYTES - NS * STAGE) / FETCH, DEPTH = FIT > 2 ? 2 : FIT;
    static constexpr int SMEM = 2 * H_BYTES + NS * STAGE + DEPTH * FETCH + 1024;
    static constexpr bool OK = RB >= 4 && DEPTH >= 1;  // ranks over 16: run_expand's rule
    static constexpr uint32_t SWIZZLE = SPAN == 128 ? 2 : SPAN == 64 ? 4 : 6;
};

constexpr int kWideThreads = 640;

__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %3, %3, %4}], "
        "[%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(0), "r"(y), "r"(bar)
        : "memory");
}

// Descriptor of a tile of rows of SPAN bytes along K: 8-row groups 8 SPAN apart.
template <typename C>
__device__ __forceinline__ uint64_t wide_desc(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)(8 * C::SPAN >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)C::SWIZZLE << 61);
}

template <typename T>
__device__ __forceinline__ void wide_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, uint32_t accumulate) {
    if constexpr (sizeof(T) == 4)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::tf32 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(desc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(desc), "r"(accumulate)
            : "memory");
}

// The place in the (tile, stage) order.
struct WideStep {
    int tile, stage, per_tile;
    __device__ __forceinline__ void start(int64_t at, int per) {
        tile = (int)(at / per), stage = (int)(at % per), per_tile = per;
    }
    // k steps on; true where that is another tile.
    __device__ __forceinline__ bool move(int k) {
        stage += k;
        bool other = false;
        while (stage >= per_tile) stage -= per_tile, tile++, other = true;
        return other;
    }
    // Called at step i, one by one; true where a tile begins.
    __device__ __forceinline__ bool next(int i) { return i ? move(1) : true; }
};

template <typename T, int RB>
__global__ void __launch_bounds__(kWideThreads, 1) k_expand_wide(const __grid_constant__ CUtensorMap w_map, Plan plan,
                                                                 const float* h, int splits, const T* w_all, int rank,
                                                                 int64_t F, int T_rows, const T* base, int64_t ldb, T* out,
                                                                 int64_t ldo) {
    using C = WideCfg<T, RB>;
    constexpr int RP = C::RP, FS = C::FS, NS = C::NS, SPAN = C::SPAN, KB = C::KB, SIZE = C::SIZE, BM = C::BM;
    constexpr bool F32 = SIZE == 4;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* planes = smem + NS * C::STAGE;     // H_hi, H_lo
    uint8_t* fetched = planes + 2 * C::H_BYTES;  // base: [DEPTH][warp][8][lane] units
    __shared__ uint64_t bars[3 * NS + 10];
    __shared__ uint32_t tmem_slot;
    __shared__ float undo[6][BM];  // fp16: the rows' scales taken back, of the tiles that can be in flight
    const uint32_t full = smem_u32(bars), low = full + 8 * NS, empty = low + 8 * NS, acc_full = empty + 8 * NS;
    const uint32_t acc_empty = acc_full + 32, h_full = acc_empty + 32, h_empty = h_full + 8;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < NS; i++) {
            mbar_init(full + 8 * i, 1);
            mbar_init(low + 8 * i, 1);
            mbar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 4; i++) {
            mbar_init(acc_full + 8 * i, 1);
            mbar_init(acc_empty + 8 * i, 8);
        }
        mbar_init(h_full, 1);
        mbar_init(h_empty, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 17) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                     "r"((uint32_t)(4 * FS))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_slot;
    wait_for_previous();
    let_next_start();

    // this block's share of the (tile, stage) pairs; in place, positions without an adapter stay as they are
    const int per_tile = (int)((F + FS - 1) / FS);
    const int64_t total = (int64_t)(base == out ? plan.tiles[1] : plan.tiles[0]) * per_tile;
    const int64_t begin = total * blockIdx.x / gridDim.x, end = total * (blockIdx.x + 1) / gridDim.x;
    const int steps = (int)(end - begin);
    const int real_tiles = plan.tiles[1];  // the tiles with an adapter come first
    WideStep at;
    at.start(begin, per_tile);

    if (warp < 16) {
        // rows g and g + 8 of the warp's 16, units 4 c + q of their 256 bytes; steps first, first + 2, ..
        const int quarter = warp & 3, half = (warp >> 2) & 1, first = warp >> 3, g = lane >> 2, q = lane & 3;
        constexpr int E = 16 / SIZE;
        const uint32_t place = smem_u32(fetched) + warp * 4096 + lane * 16;
        int row[2], row_ahead[2];
        const auto read_rows = [&](int (&r)[2], int tile) {
            const Tile t = plan.tile[tile];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int p = 32 * quarter + 16 * half + 8 * k + g;
                r[k] = p < t.rows ? plan.perm[t.start + p] : -1;
            }
        };
        WideStep ahead = at;
        bool there = false;  // row_ahead is ahead.tile's
        ahead.move(first);
        const auto fetch = [&](int i, int slot) {
            if (i < steps && base) {
                if (!there) read_rows(row_ahead, ahead.tile);
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const int64_t f = (int64_t)ahead.stage * FS + c * C::GROUP + q * E;
                        if (row_ahead[k] >= 0 && f < F)
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                                             place + slot * C::FETCH + (4 * k + c) * 512),
                                         "l"(base + (int64_t)row_ahead[k] * ldb + f)
                                         : "memory");
                    }
                there = !ahead.move(2);
            }
            stage_done();
        };
#pragma unroll
        for (int d = 0; d < C::DEPTH; d++) fetch(first + 2 * d, d);
        at.move(first);
        bool ok = true, fresh = true;
        int slot = 0;
        const int tile_first = (int)(begin / per_tile);
        for (int i = first; i < steps; i += 2) {
            if (fresh) read_rows(row, at.tile);
            const bool real = at.tile < real_tiles;
            const int a = i & 3;
            if (real) {
                ok = ok && mbar_wait(acc_full + 8 * a, (uint32_t)((i >> 2) & 1), nullptr);
                ok = __all_sync(0xffffffffu, ok);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            }
            stage_wait<C::DEPTH - 1>();
            Total all;  // not finite where a product is not
            float back[2] = {1.f, 1.f};
            if constexpr (std::is_same_v<T, __half>) {
                if (real)
#pragma unroll
                    for (int k = 0; k < 2; k++)
                        back[k] = undo[(at.tile - tile_first) % 6][32 * quarter + 16 * half + 8 * k + g];
            }
#pragma unroll
            for (int c2 = 0; c2 < 4; c2 += 2) {
                uint32_t r[2][4 * C::BLOCKS];  // columns 2 b + j of unit q: r[4 b + j], rows 8 below: r[4 b + 2 + j]
                if (real) {
#pragma unroll
                    for (int m = 0; m < 2; m++) {
                        const uint32_t from = tmem + ((uint32_t)(32 * quarter + 16 * half) << 16) +
                                              (uint32_t)(a * FS + (c2 + m) * C::GROUP);
                        if constexpr (F32)
                            asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                                         : "=r"(r[m][0]), "=r"(r[m][1]), "=r"(r[m][2]), "=r"(r[m][3]), "=r"(r[m][4]),
                                           "=r"(r[m][5]), "=r"(r[m][6]), "=r"(r[m][7])
                                         : "r"(from));
                        else
                            asm volatile(
                                "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
                                "%11, %12, %13, %14, %15}, [%16];"
                                : "=r"(r[m][0]), "=r"(r[m][1]), "=r"(r[m][2]), "=r"(r[m][3]), "=r"(r[m][4]),
                                  "=r"(r[m][5]), "=r"(r[m][6]), "=r"(r[m][7]), "=r"(r[m][8]), "=r"(r[m][9]),
                                  "=r"(r[m][10]), "=r"(r[m][11]), "=r"(r[m][12]), "=r"(r[m][13]), "=r"(r[m][14]),
                                  "=r"(r[m][15])
                                : "r"(from));
                    }
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                    for (int m = 0; m < 2; m++)
#pragma unroll
                        for (int j = 0; j < 4 * C::BLOCKS; j += 2)
                            all.add(__uint_as_float(r[m][j]), __uint_as_float(r[m][j + 1]));
                    if (c2 == 2) {  // the accumulator, and the rows' scales, have been read
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive(acc_empty + 8 * a);
                    }
                }
#pragma unroll
                for (int m = 0; m < 2; m++)
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const int c = c2 + m;
                        const int64_t f = (int64_t)at.stage * FS + c * C::GROUP + q * E;
                        uint4 v = make_uint4(0, 0, 0, 0);
                        if (base) v = lds128(fetched + warp * 4096 + lane * 16 + slot * C::FETCH + (4 * k + c) * 512);
                        uint32_t* w = reinterpret_cast<uint32_t*>(&v);
                        if (real) {
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                if constexpr (F32) {
                                    w[e] = bits_of(__uint_as_float(w[e]) +
                                                   __uint_as_float(r[m][4 * (e >> 1) + 2 * k + (e & 1)]));
                                } else {
                                    const float2 b = unpack2<T>(w[e]);
                                    w[e] = pack2<T>(fmaf(back[k], __uint_as_float(r[m][4 * e + 2 * k]), b.x),
                                                    fmaf(back[k], __uint_as_float(r[m][4 * e + 2 * k + 1]), b.y));
                                }
                            }
                        }
                        if (real && !ok) v = make_uint4(~0u, ~0u, ~0u, ~0u);  // NaN in every type
                        if (row[k] >= 0 && f < F) *reinterpret_cast<uint4*>(out + (int64_t)row[k] * ldo + f) = v;
                    }
            }
            if (real && ok && !all.ok()) {
                const T* wi = w_all + (int64_t)plan.tile[at.tile].adapter * F * rank;
#pragma unroll 1
                for (int u = 0; u < 8 * E; u++) {
                    const int e = u % E, unit = u / E;  // 4 k + c
                    const int t = unit < 4 ? row[0] : row[1];
                    const int64_t f = (int64_t)at.stage * FS + (unit & 3) * C::GROUP + q * E + e;
                    if (t < 0 || f >= F || finite(wide(out[(int64_t)t * ldo + f]))) continue;
                    const float y = plain_expand<T>(h + (int64_t)t * RP, splits, (int64_t)T_rows * RP, wi + f * rank, 1, rank);
                    const T* b = reinterpret_cast<const T*>(fetched + slot * C::FETCH + warp * 4096 + lane * 16 + unit * 512) + e;
                    out[(int64_t)t * ldo + f] = narrow<T>(base ? wide(*b) + y : y);
                }
            }
            fetch(i + 2 * C::DEPTH, slot);
            slot = slot + 1 == C::DEPTH ? 0 : slot + 1;
            fresh = at.move(2);
        }
    } else if (warp == 16) {
        if (lane == 0) {
            int made = 0;
            int adapter = 0;
            for (int i = 0; i < steps; i++) {
                if (at.next(i) && at.tile < real_tiles) adapter = plan.tile[at.tile].adapter;
                if (at.tile >= real_tiles) break;
                const int s = made % NS;
                if (made >= NS && !mbar_wait(empty + 8 * s, (uint32_t)((made / NS - 1) & 1), nullptr)) break;
                const uint32_t bar = full + 8 * s, to = smem_u32(smem + s * C::STAGE);
                mbar_expect_tx(bar, C::W_BYTES);
                const int y = (int)(((int64_t)adapter * F + (int64_t)at.stage * FS) / C::GROUP);
#pragma unroll
                for (int b = 0; b < KB; b++) tma_load_5d(to + b * FS * SPAN, &w_map, b * (SPAN / SIZE), y, bar);
                made++;
            }
            for (int k = made > NS ? made - NS : 0; k < made; k++)
                mbar_wait(full + 8 * (k % NS), (uint32_t)((k / NS) & 1), nullptr);
        }
    } else if (warp == 17) {
        if (lane == 0) {
            constexpr uint32_t type = F32 ? 2u : std::is_same_v<T, __nv_bfloat16> ? 1u : 0u;
            constexpr uint32_t desc =
                (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)(FS >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
            int tiles = 0, made = 0;
            bool ok = true;
            for (int i = 0; i < steps && ok; i++) {
                const bool first = at.next(i);
                if (at.tile >= real_tiles) break;
                if (first) ok = mbar_wait(h_full, (uint32_t)(tiles++ & 1), nullptr);
                const int s = made % NS, a = made & 3;
                ok = ok && mbar_wait((F32 ? low : full) + 8 * s, (uint32_t)((made / NS) & 1), nullptr);
                if (made >= 4) ok = ok && mbar_wait(acc_empty + 8 * a, (uint32_t)((made / 4 - 1) & 1), nullptr);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t hh = smem_u32(planes), hl = hh + C::H_BYTES;
                const uint32_t w = smem_u32(smem + s * C::STAGE), wl = w + C::W_BYTES, d = tmem + a * FS;
#pragma unroll
                for (int k = 0; k < RP * SIZE / 32; k++) {  // 32 bytes of the rank a step, the small terms first
                    constexpr int PER = SPAN / 32;
                    const uint32_t ho = (k / PER) * BM * SPAN + (k % PER) * 32, wo = (k / PER) * FS * SPAN + (k % PER) * 32;
                    wide_mma<T>(d, wide_desc<C>(hl + ho), wide_desc<C>(w + wo), desc, k > 0);
                    if (F32) wide_mma<T>(d, wide_desc<C>(hh + ho), wide_desc<C>(wl + wo), desc, 1);
                    wide_mma<T>(d, wide_desc<C>(hh + ho), wide_desc<C>(w + wo), desc, 1);
                }
                umma_commit(acc_full + 8 * a);
                umma_commit(empty + 8 * s);
                if (i + 1 == steps || at.stage + 1 == per_tile) umma_commit(h_empty);  // h's planes have been read
                made++;
            }
        }
        __syncwarp();
    } else if (warp == 18) {
        int tiles = 0;
        for (int i = 0; i < steps; i++) {
            if (!at.next(i)) continue;
            if (at.tile >= real_tiles) break;
            const Tile t = plan.tile[at.tile];
            if (tiles && !mbar_wait(h_empty, (uint32_t)((tiles - 1) & 1), nullptr)) break;
#pragma unroll 1
            for (int m = 0; m < BM; m += 32) {  // a row a lane
                const int r = m + lane;
                const float* hp = h + (int64_t)plan.perm[t.start + min(r, t.rows - 1)] * RP;
                float s = 1.f;
                if constexpr (std::is_same_v<T, __half>) {
                    float most = 0.f;
                    for (int c = 0; c < RP; c += 4) {
                        const float4 f = load_h(hp + c, splits, (int64_t)T_rows * RP);
                        most = fmaxf(fmaxf(most, finite_abs(f.x)), fmaxf(fmaxf(finite_abs(f.y), finite_abs(f.z)), finite_abs(f.w)));
                    }
                    s = half_scale(most);
                    undo[tiles % 6][r] = 1.f / s;
                }
#pragma unroll 4
                for (int c = 0; c < RP; c += 16 / SIZE) {
                    uint4 hi, lo;
                    uint32_t *ph = reinterpret_cast<uint32_t*>(&hi), *pl = reinterpret_cast<uint32_t*>(&lo);
                    const float4 f = load_h(hp + c, splits, (int64_t)T_rows * RP);
                    if constexpr (F32) {
                        split_tf32(bits_of(f.x), ph[0], pl[0]);
                        split_tf32(bits_of(f.y), ph[1], pl[1]);
                        split_tf32(bits_of(f.z), ph[2], pl[2]);
                        split_tf32(bits_of(f.w), ph[3], pl[3]);
                    } else {
                        const float4 e = load_h(hp + c + 4, splits, (int64_t)T_rows * RP);
                        const float v[8] = {f.x * s, f.y * s, f.z * s, f.w * s, e.x * s, e.y * s, e.z * s, e.w * s};
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            ph[k] = pack2<T>(v[2 * k], v[2 * k + 1]);
                            const float2 b = unpack2<T>(ph[k]);
                            pl[k] = pack2<T>(v[2 * k] - b.x, v[2 * k + 1] - b.y);
                        }
                    }
                    const int byte = c * SIZE, unit = (byte % SPAN) >> 4;
                    const int turn = SPAN == 128 ? r & 7 : SPAN == 64 ? (r >> 1) & 3 : (r >> 2) & 1;
                    uint8_t* to = planes + (byte / SPAN) * BM * SPAN + r * SPAN + ((unit ^ turn) << 4);
                    *reinterpret_cast<uint4*>(to) = hi;
                    *reinterpret_cast<uint4*>(to + C::H_BYTES) = lo;
                }
            }
            fence_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(h_full);
            tiles++;
        }
    } else if (warp == 19 && F32) {
        int made = 0;
        for (int i = 0; i < steps; i++) {
            at.next(i);
            if (at.tile >= real_tiles) break;
            const int s = made % NS;
            if (!mbar_wait(full + 8 * s, (uint32_t)((made / NS) & 1), nullptr)) break;
            uint8_t* w = smem + s * C::STAGE;
#pragma unroll 4
            for (int u = lane; u < C::W_BYTES / 16; u += 32) {
                uint4 v = *reinterpret_cast<const uint4*>(w + 16 * u);
                uint32_t* p = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
                for (int k = 0; k < 4; k++) p[k] = bits_of(__uint_as_float(p[k]) - __uint_as_float(p[k] & 0xffffe000u));
                *reinterpret_cast<uint4*>(w + C::W_BYTES + 16 * u) = v;
            }
            fence_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(low + 8 * s);
            made++;
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 17) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)(4 * FS))
                     : "memory");
    }
}

// ---- weight gradients ------------------------------------------------------------
// G_i = sum over adapter i's positions of x[t, f] h[t, r].  TRANS = false: G_i stored [rank, F] (dA,
// with h = dh); true: stored [F, rank] (dB, with x = the gradient of out).  Both in one launch: blocks up
// to `first` along x take the first side.  A cluster of blocks per (FC columns, adapter) shares its
// positions, 64 a stage; four warps side by side along the columns, two along the positions.  All are
// summed, in their order, through (distributed) shared memory at the end.  An adapter without positions
// gets zeros.
template <typename T>
struct Side {
    const T* x;
    int64_t ldx;
    const float* h;
    int64_t F;
    T* out;
    bool trans, vec, ovec;  // vec: rows of x start on 16 bytes; ovec: whole 16-byte units of out
};
template <typename T, int RB>
struct WeightCfg {
    // blocks of 8 columns a warp: as many as the accumulators leave room for
    static constexpr int E = kE<T>, RP = 8 * RB, NB = RB == 16 ? 2 : 4;
    static constexpr int FC = 4 * 8 * NB, FU = FC / E, TK = 64;
    static constexpr int X_BYTES = TK * FC * (int)sizeof(T);
    // h of a stage: fp32 rows at a pitch of 8 words beyond a multiple of 16; 16 bits: planes hi and lo
    static constexpr int H_PITCH = sizeof(T) == 4 ? RP * 4 + 32 : RP * 2 + 16;
    static constexpr int H_BYTES = TK * H_PITCH * (sizeof(T) == 4 ? 1 : 2);
    static constexpr int NS = 3;
    static constexpr int RED = 2 * RP * (FC + 4) * 4;
    static constexpr int SMEM = NS * X_BYTES + 2 * H_BYTES > RED ? NS * X_BYTES + 2 * H_BYTES : RED;
    static_assert(SMEM <= 220 * 1024, "a block's shared memory");
};

// The sum over the positions listed of one column of x and one rank of h.
template <typename T>
__device__ __forceinline__ float plain_weight(const T* x, int64_t ldx, const float* h, int ldh, const int32_t* list, int count) {
    float v = 0.f;
#pragma unroll 1
    for (int p = 0; p < count && v == v; p++) v = fmaf(wide(x[list[p] * ldx]), h[(int64_t)list[p] * ldh], v);
    return v;
}

template <typename T, int RB, bool LONG>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 && RB <= 4 ? 3 : 1) k_weight(Plan plan, const int32_t* __restrict__ index, Side<T> side_a,
                                                     Side<T> side_b, int first, int n, int rank, int T_rows) {
    using C = WeightCfg<T, RB>;
    constexpr int E = C::E, RP = C::RP, NB = C::NB, FC = C::FC, FU = C::FU, TK = C::TK, NS = C::NS, RM = RB / 2;
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int HV = TK * RP / 4 / kThreads;  // float4 of h a thread stages
    extern __shared__ __align__(128) uint8_t smem[];
    Scan& scan = *reinterpret_cast<Scan*>(smem + C::SMEM);  // there without a plan only
    __shared__ int32_t ids[4][C::TK];  // positions of stages i .. i + 3, -1 past the last
    __shared__ float block_max[kWarps];
    uint8_t* hs = smem + NS * C::X_BYTES;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    const int wf = warp & 3, wt = warp >> 2;
    const int a = blockIdx.y, part = blockIdx.z, parts = gridDim.z;  // the cluster is (1, 1, parts)
    const bool second = (int)blockIdx.x >= first;
    const Side<T>& side = second ? side_b : side_a;
    const T* __restrict__ x = side.x;
    const float* h = side.h;
    const int64_t ldx = side.ldx, F = side.F, f0 = (int64_t)((int)blockIdx.x - (second ? first : 0)) * FC;
    const bool xvec = side.vec;
    wait_for_previous();
    let_next_start();
    const int32_t* list;
    int count;
    if (plan.off) {
        const int p0 = plan.off[a];
        list = plan.perm + p0;
        count = plan.off[a + 1] - p0;
    } else {
        count = scan_positions(scan, index, T_rows, n, a);
        list = scan.list;
    }
    const int all = (count + TK - 1) / TK;  // stages; this block takes part, part + parts, ..
    const int stages = part < all ? (all - part + parts - 1) / parts : 0;

    float take = 1.f;  // fp16: h's scale
    if constexpr (std::is_same_v<T, __half>) {
        float m = 0.f;
        for (int64_t e = threadIdx.x; e < (int64_t)count * (RP / 4); e += kThreads) {  // count reaches 2^30
            const float4 v = load_h(h + (int64_t)list[e / (RP / 4)] * RP + 4 * (int)(e % (RP / 4)), 1, 0);
            m = fmaxf(fmaxf(fmaxf(m, fabsf(v.x)), fmaxf(fabsf(v.y), fabsf(v.z))), fabsf(v.w));
        }
        if (!finite(m)) {
            m = 0.f;
#pragma unroll 1
            for (int64_t e = threadIdx.x; e < (int64_t)count * (RP / 4); e += kThreads) {
                const float4 v = load_h(h + (int64_t)list[e / (RP / 4)] * RP + 4 * (int)(e % (RP / 4)), 1, 0);
                m = fmaxf(fmaxf(m, finite_abs(v.x)), fmaxf(fmaxf(finite_abs(v.y), finite_abs(v.z)), finite_abs(v.w)));
            }
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        if (lane == 0) block_max[warp] = m;
        __syncthreads();
        for (int k = 0; k < kWarps; k++) m = fmaxf(m, block_max[k]);
        take = half_scale(m);
    }

    // A stage's positions are read from memory four stages ahead, so that neither its rows nor its h wait
    // for them: by the first TK threads, into a register, and into their place one stage later.
    static_assert(NS == 3, "ids holds a stage more than the ring");
    const auto id_of = [&](int i) {
        const int p = (part + i * parts) * TK + (int)threadIdx.x;
        return i < stages && p < count ? list[p] : -1;
    };
    int id_next = -1;
    if (threadIdx.x < TK) {
#pragma unroll
        for (int i = 0; i < 3; i++) ids[i][threadIdx.x] = id_of(i);
        id_next = id_of(3);
    }
    __syncthreads();
    const int64_t column = f0 + threadIdx.x % FU * E;
    const int column_bytes = column >= F ? 0 : F - column >= E ? 16 : (int)(F - column) * (int)sizeof(T);
    const T* x_column = column_bytes ? x + column : x;
    const auto load_x = [&](int i) {
        uint8_t* xs = smem + (i % NS) * C::X_BYTES;
        // a thread's column is the same in all its units: kThreads is a multiple of FU
        const int c = threadIdx.x % FU, r0 = threadIdx.x / FU;
        if (xvec) {
            const uint32_t dst = smem_u32(xs);
#pragma unroll
            for (int k = 0; k < TK * FU / kThreads; k++) {
                const int r = r0 + k * (kThreads / FU), id = ids[i & 3][r];
                const int to = F32 ? c ^ ((r & 3) << 1) : c ^ (r & 7);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + (r * FU + to) * 16),
                             "l"(x_column + (int64_t)max(id, 0) * ldx), "r"(id >= 0 ? column_bytes : 0)
                             : "memory");
            }
        } else {
#pragma unroll 1
            for (int k = 0; k < TK * FU / kThreads; k++) {
                const int r = r0 + k * (kThreads / FU), id = ids[i & 3][r];
                const int to = F32 ? c ^ ((r & 3) << 1) : c ^ (r & 7);
                stage_unit<T>(xs + (r * FU + to) * 16, x + (int64_t)max(id, 0) * ldx + f0 + c * E, x,
                              id >= 0 ? F - f0 - c * E : 0, false);
            }
        }
        stage_done();
    };
    float4 hv[HV];
    const auto load_h_regs = [&](int i) {
#pragma unroll
        for (int k = 0; k < HV; k++) {
            const int e = threadIdx.x + k * kThreads, r = e / (RP / 4), c = e % (RP / 4), id = ids[i & 3][r];
            hv[k] = id >= 0 ? load_h(h + (int64_t)id * RP + 4 * c, 1, 0) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    };
    const auto store_h = [&](int i) {
        uint8_t* d = hs + (i & 1) * C::H_BYTES;
#pragma unroll
        for (int k = 0; k < HV; k++) {
            const int e = threadIdx.x + k * kThreads, r = e / (RP / 4), c = e % (RP / 4);
            if constexpr (F32) {
                *reinterpret_cast<float4*>(d + r * C::H_PITCH + 16 * c) = hv[k];
            } else {
                const float v[4] = {hv[k].x * take, hv[k].y * take, hv[k].z * take, hv[k].w * take};
                const uint2 p = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
                const float2 b0 = unpack2<T>(p.x), b1 = unpack2<T>(p.y);
                *reinterpret_cast<uint2*>(d + r * C::H_PITCH + 8 * c) = p;
                *reinterpret_cast<uint2*>(d + (TK + r) * C::H_PITCH + 8 * c) =
                    make_uint2(pack2<T>(v[0] - b0.x, v[1] - b0.y), pack2<T>(v[2] - b1.x, v[3] - b1.y));
            }
        }
    };

    // fp32 sums are taken out of the accumulators every stage.  For 16-bit results (of 8 or 11 bits) every 16384 positions
    // do (2^20 of one sign were 4e-4 off without, 2^23 3e-3), into memory: registers are what bounds the blocks an SM.
    // LONG: there may be so many (run_weight; 200 us of gradients take 203 with the look at each stage).
    constexpr int DEEP = 256;
    volatile float deep[LONG ? RM * NB * 4 : 1];
    float acc[RM][NB][4], sum[F32 ? RM : 1][NB][4];
#pragma unroll
    for (int m = 0; m < RM; m++)
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                acc[m][b][k] = 0.f;
                if (F32 || m == 0) sum[F32 ? m : 0][b][k] = 0.f;
            }
#pragma unroll
    for (int i = 0; i < NS - 1; i++) {
        if (i < stages) load_x(i);
        else stage_done();
    }
    if (stages > 0) load_h_regs(0);
    for (int i = 0; i < stages; i++) {
        store_h(i);  // its buffer was last read two stages ago, before the barrier of the last one
        stage_wait<NS - 2>();
        __syncthreads();
        if (i + NS - 1 < stages) load_x(i + NS - 1);
        else stage_done();
        if (i + 1 < stages) load_h_regs(i + 1);
        if (threadIdx.x < TK) {  // the place of stage i - 1
            ids[(i + 3) & 3][threadIdx.x] = id_next;
            id_next = id_of(i + 4);
        }
        const uint8_t* xs = smem + (i % NS) * C::X_BYTES;
        const uint8_t* hb = hs + (i & 1) * C::H_BYTES;
        if constexpr (F32) {  // lane rows g, g + 8 of block m: ranks 2 RM g + 2 m, + 1; column 8 .. of the warp: NB g + b
#pragma unroll
            for (int s = 0; s < TK / 16; s++) {
                const int t0 = 32 * wt + 8 * s + q;
                uint32_t xv[2][NB], hr[2][2 * RM];
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const int t = t0 + 4 * j;
                    if constexpr (NB == 4) {
                        const int c = 8 * wf + g;
                        const uint4 v = lds128(xs + t * (FU * 16) + ((c ^ ((t & 3) << 1)) * 16));
                        xv[j][0] = v.x, xv[j][1] = v.y, xv[j][2] = v.z, xv[j][3] = v.w;
                    } else {
                        const int c = 4 * wf + (g >> 1);
                        const uint2 v = *reinterpret_cast<const uint2*>(
                            xs + t * (FU * 16) + ((c ^ ((t & 3) << 1)) * 16) + (g & 1) * 8);
                        xv[j][0] = v.x, xv[j][1] = v.y;
                    }
                    const uint8_t* hp = hb + t * C::H_PITCH + 8 * RM * g;
                    if constexpr (RM == 1) {
                        const uint2 v = *reinterpret_cast<const uint2*>(hp);
                        hr[j][0] = v.x, hr[j][1] = v.y;
                    } else {
#pragma unroll
                        for (int r = 0; r < 2 * RM; r += 4) {
                            const uint4 v = lds128(hp + 4 * r);
                            hr[j][r] = v.x, hr[j][r + 1] = v.y, hr[j][r + 2] = v.z, hr[j][r + 3] = v.w;
                        }
                    }
                }
#pragma unroll
                for (int m = 0; m < RM; m++) {
                    const Split fa = split_a(hr[0][2 * m], hr[0][2 * m + 1], hr[1][2 * m], hr[1][2 * m + 1]);
#pragma unroll
                    for (int b = 0; b < NB; b += 2)
                        mma_split2(acc[m][b], acc[m][b + 1], fa, xv[0][b], xv[1][b], xv[0][b + 1], xv[1][b + 1]);
                }
            }
#pragma unroll
            for (int m = 0; m < RM; m++)
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int k = 0; k < 4; k++) sum[m][b][k] += acc[m][b][k], acc[m][b][k] = 0.f;
        } else {
            const int lr = lane & 7, lm = lane >> 3;
#pragma unroll
            for (int s = 0; s < TK / 32; s++) {
                const int t0 = 32 * wt + 16 * s;
                uint32_t fb[NB][2];
#pragma unroll
                for (int b = 0; b < NB; b += 2) {
                    uint32_t v[4];
                    const int t = t0 + lr + 8 * (lm & 1), c = NB * wf + b + (lm >> 1);
                    ldmatrix4_trans(v, xs + t * (FU * 16) + ((c ^ (t & 7)) * 16));
                    fb[b][0] = v[0], fb[b][1] = v[1], fb[b + 1][0] = v[2], fb[b + 1][1] = v[3];
                }
#pragma unroll
                for (int m = 0; m < RM; m++) {
                    uint32_t fh[4], fl[4];
                    const uint8_t* p = hb + (t0 + lr + 8 * (lm >> 1)) * C::H_PITCH + (2 * m + (lm & 1)) * 16;
                    ldmatrix4_trans(fh, p);
                    ldmatrix4_trans(fl, p + TK * C::H_PITCH);
#pragma unroll
                    for (int b = 0; b < NB; b++) mma<T>(acc[m][b], fl, fb[b][0], fb[b][1]);
#pragma unroll
                    for (int b = 0; b < NB; b++) mma<T>(acc[m][b], fh, fb[b][0], fb[b][1]);
                }
            }
            if (LONG && (i + 1) % DEEP == 0) {
#pragma unroll
                for (int m = 0; m < RM; m++)
#pragma unroll
                    for (int b = 0; b < NB; b++)
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            volatile float& d = deep[(m * NB + b) * 4 + k];
                            d = i < DEEP ? acc[m][b][k] : d + acc[m][b][k];
                            acc[m][b][k] = 0.f;
                        }
            }
        }
    }
    if (LONG && stages >= DEEP) {
#pragma unroll
        for (int m = 0; m < RM; m++)
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int k = 0; k < 4; k++) acc[m][b][k] += deep[(m * NB + b) * 4 + k];
    }
    stage_wait<0>();
    __syncthreads();
    constexpr int RS = FC + 4;
    float* red = reinterpret_cast<float*>(smem);  // [2][RP][RS]
    const float undo = 1.f / take;
#pragma unroll
    for (int m = 0; m < RM; m++)
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int c = 2 * q + (k & 1);
                const int r = F32 ? 2 * RM * g + 2 * m + (k >> 1) : 16 * m + g + 8 * (k >> 1);
                const int f = 8 * NB * wf + (F32 ? NB * c + b : 8 * b + c);
                if constexpr (F32) red[(wt * RP + r) * RS + f] = sum[m][b][k];
                else red[(wt * RP + r) * RS + f] = acc[m][b][k] * undo;
            }
    // each block of the cluster finishes its share of the elements, from all blocks' sums
    const cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    if (parts > 1) cluster.sync();
    else __syncthreads();
    T* dst = side.out + (int64_t)a * rank * F;
    float total = 0.f;  // of this thread's sums: not finite where one is not
    if (side.ovec) {  // 16 bytes a thread: along the columns, or along the ranks of a column
        for (int u = threadIdx.x + part * kThreads; u < FC * RP / E; u += parts * kThreads) {
            const int c = side.trans ? u % FC : u % (FC / E) * E, r = side.trans ? u / FC * E : u / (FC / E);
            if (r >= rank || f0 + c >= F) continue;
            float v[E];
#pragma unroll
            for (int j = 0; j < E; j++) v[j] = 0.f;
            for (int k = 0; k < parts; k++) {
                const float* from = (parts > 1 ? cluster.map_shared_rank(red, k) : red) + r * RS + c;
                if (side.trans) {
#pragma unroll
                    for (int j = 0; j < E; j++) v[j] += from[j * RS] + from[(RP + j) * RS];
                } else {
#pragma unroll
                    for (int j = 0; j < E; j += 4) {
                        const float4 p = *reinterpret_cast<const float4*>(from + j);
                        const float4 q4 = *reinterpret_cast<const float4*>(from + RP * RS + j);
                        v[j] += p.x + q4.x, v[j + 1] += p.y + q4.y, v[j + 2] += p.z + q4.z, v[j + 3] += p.w + q4.w;
                    }
                }
            }
            alignas(16) T o[E];
#pragma unroll
            for (int j = 0; j < E; j++) {
                total += v[j];
                o[j] = narrow<T>(v[j]);
            }
            T* to = dst + (side.trans ? (f0 + c) * rank + r : (int64_t)r * F + f0 + c);
            *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(o);
        }
        if (!finite(total)) {
#pragma unroll 1
            for (int u = threadIdx.x + part * kThreads; u < FC * RP / E; u += parts * kThreads) {
                const int c = side.trans ? u % FC : u % (FC / E) * E, r = side.trans ? u / FC * E : u / (FC / E);
                if (r >= rank || f0 + c >= F) continue;
                T* to = dst + (side.trans ? (f0 + c) * rank + r : (int64_t)r * F + f0 + c);
#pragma unroll 1
                for (int j = 0; j < E; j++)
                    if (!finite(wide(to[j])))
                        to[j] = narrow<T>(plain_weight<T>(x + f0 + c + (side.trans ? 0 : j), ldx,
                                                          h + r + (side.trans ? j : 0), RP, list, count));
            }
        }
        if (parts > 1) cluster.sync();  // its shared memory is read until here
        return;
    }
    for (int e = threadIdx.x + part * kThreads; e < FC * RP; e += parts * kThreads) {
        const int r = side.trans ? e % RP : e / FC, c = side.trans ? e / RP : e % FC;
        if (r >= rank || f0 + c >= F) continue;
        float v = 0.f;
        for (int k = 0; k < parts; k++) {
            const float* from = parts > 1 ? cluster.map_shared_rank(red, k) : red;
            v += from[r * RS + c] + from[(RP + r) * RS + c];
        }
        total += v;
        dst[side.trans ? (f0 + c) * rank + r : (int64_t)r * F + f0 + c] = narrow<T>(v);
    }
    if (!finite(total)) {
#pragma unroll 1
        for (int e = threadIdx.x + part * kThreads; e < FC * RP; e += parts * kThreads) {
            const int r = side.trans ? e % RP : e / FC, c = side.trans ? e / RP : e % FC;
            if (r >= rank || f0 + c >= F) continue;
            T* to = dst + (side.trans ? (f0 + c) * rank + r : (int64_t)r * F + f0 + c);
            if (!finite(wide(*to))) *to = narrow<T>(plain_weight<T>(x + f0 + c, ldx, h + r, RP, list, count));
        }
    }
    if (parts > 1) cluster.sync();  // its shared memory is read until here
}

// ---- host ------------------------------------------------------------------------

struct Shape {
    int64_t T, K, N;
    int n, rank, rb, wm;
    bool planned;            // by k_plan; else the first launch's blocks find their tiles
    int64_t tiles;           // blocks along x: at least the tiles there are
    int splits_k, splits_n;  // blocks per tile that share the sum over K, over N
};


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

constexpr int kSms = 148;

Shape shape_of(int64_t T, int n, int rank, int64_t K, int64_t N, bool backward) {
    Shape s;
    s.T = T, s.K = K, s.N = N, s.n = n, s.rank = rank;
    s.rb = rank_blocks(rank);
    const int64_t groups = T < (int64_t)n + 1 ? T : (int64_t)n + 1;
    // Tiles of 128 positions from 96 an adapter on, else of 16.  16 against 128, 12800 columns at rank 16: 64 an adapter
    // 68 and 76 us (2048 positions, fp32; their gradients 132 and 136), 64 and 75 (4096, bf16); 122 an adapter 44.5
    // and 45.0; 128 an adapter 117 and 108 (4096, fp32), 65 and 61 (bf16); 256 an adapter 112 and 100, 62 and 60.
    s.wm = groups > 0 && T / groups >= 96 ? 8 : 1;
    const int bm = 16 * s.wm;
    s.planned = T > (backward ? kScanMaxGradients : kScanMax) || n > kScanAdapters;
    s.tiles = (T + (bm - 1) * groups) / bm;  // as many as there can be
    // Blocks that share a sum: about two an SM.  For 2, 3, 4 and 6 an SM: gradients of 8192 positions (rank 32, bf16)
    // 193, 197, 197 and 198 us, of 2048 (rank 16, fp32) 86, 88, 87 and 92, 16384 positions (rank 64, bf16) 237, 237,
    // 246 and 280.
    const auto splits = [&](int64_t width) {
        const int64_t blocks = s.tiles * (s.wm == 8 ? 2 : 1), want = blocks > 0 ? ceil_div(2 * kSms, blocks) : 1;
        const int64_t can = ceil_div(width, 512);
        const int64_t k = want < can ? want : can;
        // and no more than 2^17 columns a split: the accumulators' sums round toward zero, 7e-5 of 2^17 / 16 of one sign
        const int64_t fewest = ceil_div(width, 1 << 17), some = k < 1 ? 1 : k > 16 ? 16 : k;
        return (int)(some < fewest ? fewest : some);
    };
    s.splits_k = splits(K);
    s.splits_n = splits(N);
    return s;
}

Layout layout_of(const Shape& s, bool backward) {
    Layout l = {};
    int64_t at = 0;
    const auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += align256(bytes);
        return here;
    };
    l.off = take((int64_t)(s.n + 2) * 4);
    l.perm = take(s.planned ? s.T * 4 : s.tiles * 16 * s.wm * 4);
    l.tiles = take(8);
    l.tile = take(s.tiles * (int64_t)sizeof(Tile));
    l.h = take((int64_t)s.splits_k * s.T * 8 * s.rb * 4);
    if (backward) l.dh = take((int64_t)s.splits_n * s.T * 8 * s.rb * 4);
    l.bytes = at;
    return l;
}

Plan plan_at(uint8_t* ws, const Shape& s, const Layout& l) {
    return Plan{s.planned ? reinterpret_cast<int32_t*>(ws + l.off) : nullptr,
                reinterpret_cast<int32_t*>(ws + l.perm),
                s.planned ? reinterpret_cast<int32_t*>(ws + l.tiles) : nullptr, reinterpret_cast<Tile*>(ws + l.tile)};
}

int run_plan(const Shape& s, const int32_t* index, const Plan& plan, cudaStream_t st) {
    if (!s.planned) return ENGRAM_OK;
    const int chunk = (int)ceil_div(ceil_div(s.T, 128), kPlanThreads) * kPlanThreads;
    return start<k_plan, (3 * kMaxAdapters + 4) * 4>(dim3((unsigned)ceil_div(s.T, chunk)), kPlanThreads, (3 * s.n + 4) * 4, false, st, index,
                 (int)s.T, s.n, chunk, 16 * s.wm, plan);
}

template <typename T>
bool row_units(const T* p, int64_t ld) {  // every row starts on 16 bytes
    return aligned16(p) && ld % kE<T> == 0;
}

template <typename T, int RB, int WM, bool TRANS>
Shrink<T> shrink_of(const Shape& s, const T* x, int64_t ldx, const T* w, int64_t K, int splits, float* h) {
    constexpr int KC = ShrinkCfg<T, RB, WM, TRANS>::KC;
    return Shrink<T>{x, ldx, w, K, splits ? ceil_div(ceil_div(K, splits), KC) * KC : 0, splits, row_units(x, ldx),
                     row_units(w, TRANS ? s.rank : K), h};
}

// The first launch after the plan; without one its blocks find their tiles, and it waits for no launch before it.
template <typename T, int RB, int WM>
int run_shrink(const Shape& s, const Plan& plan, const int32_t* index, const Shrink<T>& h, const float* scale,
               cudaStream_t st) {
    using C = ShrinkCfg<T, RB, WM, false>;
    return start<k_shrink<T, RB, WM>>(dim3((unsigned)(s.tiles * C::PARTS), (unsigned)h.splits), kThreads, C::SMEM,
                                      s.planned, st, plan, (int)(s.planned ? PLANNED : FIND), index, h, scale, s.n, s.rank,
                                      (int)s.T);
}
template <typename T, int RB, int WM>
int run_shrink_both(const Shape& s, const Plan& plan, const int32_t* index, const Shrink<T>& dh, const Shrink<T>& h,
                    const float* scale, cudaStream_t st) {
    using C = ShrinkCfg<T, RB, WM, false>;
    using B = ShrinkCfg<T, RB, WM, true>;
    constexpr int smem = C::SMEM > B::SMEM ? C::SMEM : B::SMEM;
    return start<k_shrink_both<T, RB, WM>>(dim3((unsigned)(s.tiles * C::PARTS), (unsigned)(dh.splits + h.splits)), kThreads,
                                           smem, s.planned, st, plan, (int)(s.planned ? PLANNED : FIND), index, dh, h,
                                           scale, s.n, s.rank, (int)s.T);
}

int run_sum(const Shape& s, float* h, int h_splits, float* dh, int dh_splits, cudaStream_t st) {
    if (h_splits == 1 && dh_splits == 1) return ENGRAM_OK;
    const int64_t count4 = s.T * 2 * s.rb;
    return start<k_sum_splits>(dim3((unsigned)ceil_div(count4, kThreads), 2), kThreads, 0, true, st,
                 reinterpret_cast<float4*>(h), h_splits, reinterpret_cast<float4*>(dh), dh_splits, count4);
}

template <typename T, int RB>
int run_expand_wide(const Shape& s, const Plan& plan, const float* h, int splits, const T* w, int64_t F, const T* base,
                    int64_t ldb, T* out, int64_t ldo, cudaStream_t st) {
    using C = WideCfg<T, RB>;
    constexpr CUtensorMapSwizzle span = C::SPAN == 128 ? CU_TENSOR_MAP_SWIZZLE_128B
                                        : C::SPAN == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B;
    const auto fn = encode_fn();
    if (!fn) return ENGRAM_ERR_CUDA;
    constexpr CUtensorMapDataType type = C::F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                         : std::is_same_v<T, __half> ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                     : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    // feature of a group = BLOCKS 2 q + 2 k + j, in the order (j, q, k)
    const cuuint64_t row = (cuuint64_t)s.rank * sizeof(T);
    const cuuint64_t dims[5] = {(cuuint64_t)s.rank, 2, 4, C::BLOCKS, (cuuint64_t)(s.n * F / C::GROUP)};
    const cuuint64_t strides[4] = {row, 2 * C::BLOCKS * row, 2 * row, C::GROUP * row};
    const cuuint32_t box[5] = {C::SPAN / C::SIZE, 2, 4, C::BLOCKS, 4}, step[5] = {1, 1, 1, 1, 1};
    CUtensorMap map;
    if (fn(&map, type, 5, const_cast<T*>(w), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, span,
           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return ENGRAM_ERR_CUDA;
    return start<k_expand_wide<T, RB>>(dim3((unsigned)sm_count()), kWideThreads, C::SMEM, true, st, map, plan, h,
                 splits, w, s.rank, F, (int)s.T, base, ldb, out, ldo);
}

template <typename T, int RB, int WM, bool TRANS>
int run_expand(const Shape& s, const Plan& plan, const float* h, int splits, const T* w, int64_t F, const T* base,
               int64_t ldb, T* out, int64_t ldo, cudaStream_t st) {
    using C = ExpandCfg<T, RB, WM == 8, TRANS>;
    // The tcgen05 kernel, where ranks over 16 and enough work pay for its start.  k_expand against it, the whole call
    // at 12800 columns: rank 16 never (16384 positions 187 and 198 us in bf16, 352 and 371 in fp32); rank 32 in bf16
    // 88 and 88 at 4096 positions, 154 and 125 at 8192, in fp32 211 and 220 at 8192, 407 and 384 at 16384; rank 64 in
    // bf16 87 and 94 at 2048, 136 and 126 at 4096, 380 and 238 at 16384, in fp32 148 and 154, 250 and 219, 784 and
    // 624; rank 128 in bf16 186 and 147 at 2048, 383 and 215 at 8192.
    if constexpr (WM == 8 && !TRANS && WideCfg<T, RB>::OK) {
        // More than 16 splits only widths over 2^21 have: adding them up once more for results that are not finite would
        // take milliseconds a stage, which the waits' limit leaves no room for.
        if (s.T * F >= (3ll << 30) / (8 * RB) && splits <= 16 && s.planned && s.n > 0 && F % WideCfg<T, RB>::GROUP == 0 && s.n * F / WideCfg<T, RB>::GROUP < (1ll << 31) &&
            (!base || row_units(base, ldb)) && row_units((const T*)out, ldo) && row_units(w, s.rank))
            return run_expand_wide<T, RB>(s, plan, h, splits, w, F, base, ldb, out, ldo, st);
    }
    // columns of a block: whole stages, for about eight blocks an SM
    const int64_t passes = ceil_div(F, C::FS), want = ceil_div(8 * kSms, s.tiles * C::PARTS);
    const int64_t f_block = ceil_div(passes, want < passes ? want : passes) * C::FS;
    return start<k_expand<T, RB, WM == 8, TRANS>>(dim3((unsigned)(s.tiles * C::PARTS), (unsigned)ceil_div(F, f_block)), kThreads,
                 C::SMEM, true, st, plan, h, splits, w, s.n, s.rank, F, f_block, (int)s.T, base, ldb, out, ldo,
                 base && row_units(base, ldb), row_units(w, TRANS ? F : s.rank), row_units((const T*)out, ldo));
}

constexpr int64_t kManyPositions = 1 << 17;  // 16-bit sums over as many, all of one adapter, are 7e-5 off

// Either side may be missing (out null).
template <typename T, int RB>
int run_weight(const Shape& s, const Plan& plan, const int32_t* index, const Side<T>& a, const Side<T>& b,
               cudaStream_t st) {
    using C = WeightCfg<T, RB>;
    const int64_t blocks_a = a.out ? ceil_div(a.F, C::FC) : 0, blocks_b = b.out ? ceil_div(b.F, C::FC) : 0;
    // blocks of a cluster: about two blocks an SM, while an adapter's usual share of positions has stages for them
    const int64_t want = ceil_div(2 * kSms, (blocks_a + blocks_b) * s.n), can = ceil_div(s.T, (int64_t)s.n * C::TK);
    const int64_t most = want < can ? want : can;
    const unsigned parts = most >= 8 ? 8 : most >= 4 ? 4 : most >= 2 ? 2 : 1;
    constexpr int most_smem = C::SMEM + (int)sizeof(Scan);
    const dim3 grid((unsigned)(blocks_a + blocks_b), (unsigned)s.n, parts);
    if (sizeof(T) == 2 && s.T > kManyPositions)  // planned
        return start<k_weight<T, RB, sizeof(T) == 2>, most_smem>(grid, kThreads, C::SMEM, true, st, plan, index, a, b,
                                                                 (int)blocks_a, s.n, s.rank, (int)s.T);
    return start<k_weight<T, RB, false>, most_smem>(grid, kThreads, s.planned ? C::SMEM : most_smem, true, st, plan, index, a,
                                                    b, (int)blocks_a, s.n, s.rank, (int)s.T);
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

template <typename T, int RB, int WM>
int forward(const Shape& s, const Layout& l, const Args& g) {
    const Plan plan = plan_at(g.ws, s, l);
    float* h = reinterpret_cast<float*>(g.ws + l.h);
    int e = run_plan(s, g.index, plan, g.st);
    if (!e)
        e = run_shrink<T, RB, WM>(
            s, plan, g.index, shrink_of<T, RB, WM, false>(s, (const T*)g.x, g.ldx, (const T*)g.a, s.K, s.splits_k, h),
            g.scale, g.st);
    if (!e)
        e = run_expand<T, RB, WM, false>(s, plan, h, s.splits_k, (const T*)g.b, s.N, (const T*)g.base, g.ldbase,
                                         (T*)g.out, g.ldout, g.st);
    return e;
}

template <typename T, int RB, int WM>
int backward(const Shape& s, const Layout& l, const Args& g) {
    const Plan plan = plan_at(g.ws, s, l);
    float *h = reinterpret_cast<float*>(g.ws + l.h), *dh = reinterpret_cast<float*>(g.ws + l.dh);
    const bool inner = g.dx || g.da;
    if (!inner && !g.db) return ENGRAM_OK;
    int e = run_plan(s, g.index, plan, g.st);
    if (!e)
        e = run_shrink_both<T, RB, WM>(
            s, plan, g.index,
            shrink_of<T, RB, WM, true>(s, (const T*)g.grad, g.ldgrad, (const T*)g.b, s.N, inner ? s.splits_n : 0, dh),
            shrink_of<T, RB, WM, false>(s, (const T*)g.x, g.ldx, (const T*)g.a, s.K, g.db ? s.splits_k : 0, h), g.scale,
            g.st);
    if (!e) e = run_sum(s, h, g.db ? s.splits_k : 1, dh, inner ? s.splits_n : 1, g.st);
    if (!e && g.dx)
        e = run_expand<T, RB, WM, true>(s, plan, dh, 1, (const T*)g.a, s.K, (const T*)g.base, g.ldbase, (T*)g.dx,
                                        g.lddx, g.st);
    if (!e && (g.da || g.db)) {
        const Side<T> da = {(const T*)g.x, g.ldx, dh, s.K, (T*)g.da, false, row_units((const T*)g.x, g.ldx),
                            row_units((const T*)g.da, s.K)};
        const Side<T> db = {(const T*)g.grad, g.ldgrad, h, s.N, (T*)g.db, true, row_units((const T*)g.grad, g.ldgrad),
                            row_units((const T*)g.db, s.rank)};
        e = run_weight<T, RB>(s, plan, g.index, da, db, g.st);
    }
    return e;
}

template <typename T>
int by_rank(const Shape& s, const Layout& l, const Args& g, bool back) {
#define ENGRAM_CASE(RB, WM) \
    if (s.rb == RB && s.wm == WM) return back ? backward<T, RB, WM>(s, l, g) : forward<T, RB, WM>(s, l, g);
    ENGRAM_CASE(2, 1)
    ENGRAM_CASE(2, 8)
    ENGRAM_CASE(4, 1)
    ENGRAM_CASE(4, 8)
    ENGRAM_CASE(8, 1)
    ENGRAM_CASE(8, 8)
    ENGRAM_CASE(16, 1)
    ENGRAM_CASE(16, 8)
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


}  // namespace

int64_t engram::adapter_waits_given_up() { return read_given_up(g_waits_given_up); }

extern "C" int64_t engram_adapter_workspace_bytes(int64_t T, int32_t n_adapters, int32_t rank, int64_t K, int64_t N,
                                                  int32_t backward) {
    const int e = check_shape(T, n_adapters, rank, K, N);
    if (e) return e;
    return layout_of(shape_of(T, n_adapters, rank, K, N, backward != 0), backward != 0).bytes;
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
    const Shape s = shape_of(T, n_adapters, rank, K, N, false);
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
    // dx is written before da's sum reads x and db's reads grad, and those are written while other blocks read
    if (n_adapters > 0) {
        if (dx && ((da && dx == x) || (db && dx == grad) || dx == da || dx == db)) return ENGRAM_ERR_ARG;
        for (const void* p : {(const void*)da, (const void*)db})
            if (p && (p == x || p == grad)) return ENGRAM_ERR_ARG;
        if (da && da == db) return ENGRAM_ERR_ARG;
    }
    const Shape s = shape_of(T, n_adapters, rank, K, N, true);
    const Layout l = layout_of(s, true);
    if (workspace_bytes < l.bytes) return ENGRAM_ERR_WORKSPACE;
    Args g = {};
    g.grad = grad, g.ldgrad = ldgrad, g.x = x, g.ldx = ldx, g.a = a, g.b = b, g.index = index, g.scale = scale;
    g.base = dx_base, g.ldbase = lddx_base, g.dx = dx, g.lddx = lddx;
    g.da = n_adapters ? da : nullptr, g.db = n_adapters ? db : nullptr;
    g.ws = (uint8_t*)workspace, g.st = st;
    return by_type(dtype, s, l, g, true);
}
