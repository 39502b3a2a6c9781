// Low-rank adapters of many requests beside a projection that all of them share:
//   out[t] = y[t] + scale_a * (x[t] A_a^T) B_a^T,   a = index[t]   (rows without an adapter: out[t] = y[t])
// x [T, K], y and out [T, N], A [adapters, R, K], B [adapters, N, R], an adapter's rank up to R.
//
// bfloat16: adapters_rows.cuh (decoding rows, any order of adapters) and adapters_tiles.cuh (prompts).  This file: the float32
// form (and that of ranks over 256), and the choice between them.  Tiles of 32 rows, products in float32 registers; where many rows may
// name several adapters they are put in order first (adapters_order.cuh), else the adapters that a tile's rows name are shared out to
// some CTAs ("slots"), each of which makes a pass for each of its own.  In `shrink` the
// CTAs of a cluster have a part of K each and add their sums up in their order; `expand` multiplies by the scale and adds to y: one
// rounding, of the output.
#include <algorithm>
#include "lb200/common.cuh"
#include "lb200/adapters.cuh"
#include "lb200/adapters_order.cuh"
#include "lb200/adapters_rows.cuh"
#include "lb200/adapters_tiles.cuh"
using namespace lb200;

namespace {
constexpr int kRows = 32, kCols = 64, kChunk = 32;      // rows, ranks or features of a tile; values of K or R at a time
constexpr int kThreads = 128;                           // 8 groups of 4 rows x 16 groups of 4 columns

constexpr int kMostParts = 8;
__device__ __forceinline__ void cluster_meet() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float remote(uint32_t at, uint32_t rank) {
    float v;
    asm volatile("{\n\t.reg .b32 p;\n\tmapa.shared::cluster.u32 p, %1, %2;\n\tld.shared::cluster.f32 %0, [p];\n\t}" : "=f"(v) : "r"(at), "r"(rank) : "memory");
    return v;
}
// Chunks of 32 values of both operands, row by row (rows 36 numbers apart: eight rows' pieces of 16 bytes are in different banks),
// three of them in turn: two on their way by asynchronous copies while one is multiplied.  At the end a CTA's sums.
constexpr int kStages = 3, kLd = kChunk + 4;
union Work {
    struct { float p[kRows][kLd], q[kCols][kLd]; } stage[kStages];
    float sums[kRows][kCols];
};
template <typename T> struct Operand {
    const T* at; long ld;                                 // row r at `at + r * ld`
    const int* rows;                                      // ... or at `at + rows[r] * ld` (shared memory; null: as they come)
    bool wide;                                            // 16 bytes at a time: rows lie so, and the depth is a multiple of 4
};
__device__ __forceinline__ void put(float* to, const float* from, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void put4(float* to, const float* from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void put(float* to, const __nv_bfloat16* from, bool there) { *to = there ? __bfloat162float(*from) : 0.f; }
__device__ __forceinline__ void put4(float* to, const __nv_bfloat16* from, bool there) {
#pragma unroll
    for (int i = 0; i < 4; ++i) put(to + i, from + i, there);
}
template <typename T, int ROWS, typename F>
__device__ __forceinline__ void fill(float (&to)[ROWS][kLd], const Operand<T>& o, int k0, int depth, F there) {
    if (o.wide) {
#pragma unroll
        for (int n = 0; n < ROWS * kChunk / 4 / kThreads; ++n) {
            const int i = threadIdx.x + n * kThreads, r = i / (kChunk / 4), k = i % (kChunk / 4) * 4;
            const bool ok = there(r) && k0 + k < depth;
            put4(&to[r][k], o.at + (ok ? (long)(o.rows != nullptr ? o.rows[r] : r) * o.ld + k0 + k : 0), ok);
        }
    } else {
#pragma unroll 8
        for (int n = 0; n < ROWS * kChunk / kThreads; ++n) {
            const int i = threadIdx.x + n * kThreads, r = i / kChunk, k = i % kChunk;
            const bool ok = there(r) && k0 + k < depth;
            put(&to[r][k], o.at + (ok ? (long)(o.rows != nullptr ? o.rows[r] : r) * o.ld + k0 + k : 0), ok);
        }
    }
}
// acc[i][j] += row r4 + i of P times row c + 16 j of Q, over `depth` values; rows that are not there are zeros.  `p_ready` comes
// before P is read, and behind what is asked for of Q at once.
template <typename TP, typename TQ, typename FP, typename FQ, typename Ready>
__device__ __forceinline__ void multiply(Work& w, float (&acc)[4][4], int depth, const Operand<TP>& p, FP p_there, const Operand<TQ>& q, FQ q_there, Ready p_ready) {
    const int r4 = (threadIdx.x >> 4) * 4, c = threadIdx.x & 15, chunks = (depth + kChunk - 1) / kChunk;
    auto fetch_q = [&](int n) { if (n < chunks) fill(w.stage[n % kStages].q, q, n * kChunk, depth, q_there); };
    auto fetch_p = [&](int n) {
        if (n < chunks) fill(w.stage[n % kStages].p, p, n * kChunk, depth, p_there);
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    __syncthreads();                                       // (what was there has been read)
    for (int n = 0; n < kStages - 1; ++n) fetch_q(n);
    p_ready();
    for (int n = 0; n < kStages - 1; ++n) fetch_p(n);
    for (int n = 0; n < chunks; ++n) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        __syncthreads();
        fetch_q(n + kStages - 1);
        fetch_p(n + kStages - 1);
        const auto& s = w.stage[n % kStages];
#pragma unroll
        for (int k = 0; k < kChunk; k += 4) {
            float4 u[4], v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = *reinterpret_cast<const float4*>(&s.p[r4 + i][k]);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const float4*>(&s.q[c + 16 * j][k]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[i][j] = fmaf(u[i].x, v[j].x, fmaf(u[i].y, v[j].y, fmaf(u[i].z, v[j].z, fmaf(u[i].w, v[j].w, acc[i][j]))));
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
}
template <typename T> __device__ __forceinline__ bool lies_wide(const T* p, long ld, int depth) {
    return sizeof(T) == 4 && ((uintptr_t)p & 15) == 0 && ld % 4 == 0 && depth % 4 == 0;
}

// The CTA's rows: places first .. first + rows - 1 (none: 0 rows).
struct TileOfRows {
    long first;
    int rows;
    __device__ explicit TileOfRows(const AdapterArgs& a) : first((long)blockIdx.x * kRows), rows((int)min((long)kRows, a.T - first)) {
        if (a.order == nullptr) return;
        const int4 its = (int)blockIdx.x < *a.n_tiles ? a.tiles[blockIdx.x] : make_int4(0, 0, 0, 0);
        first = its.y;
        rows = its.z;
    }
};

// grid: (row tiles, parts of K, rank tiles x slots); a cluster: the parts
template <typename T>
__global__ void __launch_bounds__(kThreads, 5) adapter_shrink_kernel(AdapterArgs a) {
    pdl_wait();
    pdl_trigger();                                         // `expand` asks for what it does not have from here
    __shared__ __align__(16) Work w;
    const TileOfRows tile(a);
    if (tile.rows <= 0) return;                            // (the whole cluster)
    const long t0 = tile.first;
    __shared__ int rows_s[kRows];                          // the tile's rows
    if (threadIdx.x < kRows) rows_s[threadIdx.x] = (int)threadIdx.x < tile.rows ? (int)row_at(a, t0 + threadIdx.x) : 0;
    const int part = blockIdx.y, j0 = (int)(blockIdx.z / a.slots) * kCols, slot = blockIdx.z % a.slots, tid = threadIdx.x;
    const int k_begin = min(part * a.part_k, a.K), depth = min(a.part_k, a.K - k_begin);
    const int mine = (tid & 31) < tile.rows ? adapter_of(a, t0 + (tid & 31)) : -1;
    const int r4 = (tid >> 4) * 4, c = tid & 15;
    Operand<T> x{(const T*)a.x + k_begin, a.ldx, rows_s, false};
    x.wide = lies_wide(x.at, a.ldx, depth);
    int turn = 0;
    for (int i = next_adapter(mine, -1); i != kNoAdapter; i = next_adapter(mine, i), ++turn) {
        if (turn % a.slots != slot) continue;
        const int rank = rank_of(a, i);
        if (j0 >= rank) continue;
        const unsigned named = __ballot_sync(0xffffffffu, mine == i);            // (bit r: row r)
        Operand<T> A{(const T*)a.A + (size_t)i * a.a_adapter + (size_t)j0 * a.a_row + k_begin, a.a_row, nullptr, false};
        A.wide = lies_wide(A.at, a.a_row, depth);
        float acc[4][4] = {};
        multiply(w, acc, depth, x, [&](int r) { return (named >> r & 1u) != 0; }, A, [&](int r) { return j0 + r < rank; }, [] {});
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) w.sums[r4 + r][c + 16 * j] = acc[r][j];
        __syncthreads();
        if (a.parts > 1) cluster_meet();
        for (int e = part * kThreads + tid; e < kRows * kCols; e += a.parts * kThreads) {
            const int r = e / kCols, j = e % kCols;
            if (!(named >> r & 1u) || j0 + j >= rank) continue;
            const uint32_t at = (uint32_t)__cvta_generic_to_shared(&w.sums[r][j]);
            float got[kMostParts], total = 0.f;
#pragma unroll
            for (int p = 0; p < kMostParts; ++p) if (p < a.parts) got[p] = a.parts > 1 ? remote(at, p) : w.sums[r][j];
#pragma unroll
            for (int p = 0; p < kMostParts; ++p) if (p < a.parts) total += got[p];
            a.h[(t0 + r) * a.R + j0 + j] = total;
        }
        if (a.parts > 1) cluster_meet();                   // (the sums have been read)
    }
}

// grid: (row tiles, feature tiles, slots)
template <typename T>
__global__ void __launch_bounds__(kThreads, 5) adapter_expand_kernel(AdapterArgs a) {
    // (what `shrink` does not make, index, y and B, is there since that kernel has begun)
    __shared__ __align__(16) Work w;
    const TileOfRows tile(a);
    if (tile.rows <= 0) {
        pdl_wait();
        return;
    }
    const long t0 = tile.first;
    const int n0 = blockIdx.y * kCols, slot = blockIdx.z, tid = threadIdx.x;
    const int mine = (tid & 31) < tile.rows ? adapter_of(a, t0 + (tid & 31)) : -1;
    const int its_row = (tid & 31) < tile.rows ? (int)row_at(a, t0 + (tid & 31)) : 0;
    long row[4];                                           // this thread's
#pragma unroll
    for (int r = 0; r < 4; ++r) row[r] = __shfl_sync(0xffffffffu, its_row, (tid >> 4) * 4 + r);
    const int r4 = (tid >> 4) * 4, c = tid & 15;
    unsigned ours = slot == 0 ? __ballot_sync(0xffffffffu, mine < 0) : 0u;       // the rows that this CTA writes
    int turn = 0;
    for (int i = next_adapter(mine, -1); i != kNoAdapter; i = next_adapter(mine, i), ++turn)
        if (turn % a.slots == slot) ours |= __ballot_sync(0xffffffffu, mine == i);
    const T* y = (const T*)a.y;
    T* out = (T*)a.out;
    float sum[4][4] = {};                                  // y first: on its way while the short sums and B come
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if ((ours >> (r4 + r) & 1u) && r4 + r < tile.rows && n0 + c + 16 * j < a.N) sum[r][j] = to_f32(y[row[r] * a.ldy + n0 + c + 16 * j]);
    turn = 0;
    for (int i = next_adapter(mine, -1); i != kNoAdapter; i = next_adapter(mine, i), ++turn) {
        if (turn % a.slots != slot) continue;
        const int rank = rank_of(a, i);
        const unsigned named = __ballot_sync(0xffffffffu, mine == i);
        const float scale = a.scales ? a.scales[i] : 1.f;
        Operand<float> h{a.h + t0 * a.R, a.R, nullptr, false};
        h.wide = lies_wide(h.at, a.R, rank);
        Operand<T> B{(const T*)a.B + (size_t)i * a.b_adapter + (size_t)n0 * a.b_row, a.b_row, nullptr, false};
        B.wide = lies_wide(B.at, a.b_row, rank);
        float acc[4][4] = {};
        multiply(w, acc, rank, h, [&](int r) { return (named >> r & 1u) != 0; }, B, [&](int r) { return n0 + r < a.N; }, [] { pdl_wait(); });
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (named >> (r4 + r) & 1u)
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[r][j] += acc[r][j] * scale;
    }
    pdl_wait();                                            // (this kernel ends behind `shrink`, with or without work)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        if (r4 + r >= tile.rows || !(ours >> (r4 + r) & 1u)) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = n0 + c + 16 * j;
            if (n < a.N) out[row[r] * a.ldo + n] = from_f32<T>(sum[r][j]);
        }
    }
}

template <typename T>
int launch_general(const AdapterArgs& a, cudaStream_t s) {
    const unsigned tiles = (unsigned)(a.order == nullptr ? (a.T + kRows - 1) / kRows : adapter_order::most_tiles(a.T, a.adapters, kRows));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(tiles, a.parts, (a.R > 0 ? (a.R + kCols - 1) / kCols : 1) * a.slots); cfg.blockDim = dim3(kThreads); cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1; attr[1].val.clusterDim.y = (unsigned)a.parts; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    int rc = launched(cudaLaunchKernelEx(&cfg, adapter_shrink_kernel<T>, a));
    if (rc == 0) rc = launch_pdl(adapter_expand_kernel<T>, dim3(tiles, (a.N + kCols - 1) / kCols, a.slots), dim3(kThreads), 0, s, a);
    return rc != 0 ? rc : launch_status();
}
}  // namespace

// How many parts K is cut into, the CTAs of a cluster: enough for the SMs, each with 64 values of K at least.
static int parts_of(long T, int K, int R) {
    const long tiles = (T + kRows - 1) / kRows * (R > 0 ? (R + kCols - 1) / kCols : 1);
    int parts = 1;
    while (parts < kMostParts && tiles * parts < 296 && K / (2 * parts) >= 64) parts *= 2;
    return parts;
}

// From so many rows on a call in bfloat16 goes to the tiles' kernel, and, where its rows may name several adapters, in their order.  Tiles
// / rows' kernel, us, 2,048 -> 4,096, rank 16: 8 adapters in random order 27 / 44 at 384 rows, 35 / 56 at 768, 37 / 84 at 1,024; 40
// adapters 51 / 45, 53 / 58, 56 / 97; portions of 8 adapters, whose order nobody knows beforehand, 29 / 12, 20 / 14, 16 / 22; 8,000 rows
// of 8 adapters in random order, 4,096 -> 12,288, rank 64, 264 / 2,892.  The form with two kernels takes rows in order from fewer on: 63 rows of 64 adapters 55 us, 84 as they come,
// 32 of 32 34 and 56; a few rows of few adapters would lose the 3 us that putting them in order takes (32 of 4: 17, 14).
constexpr long kTileRows = 384, kOrderRows = 64;
constexpr int kMostSlots = 8;
static bool two_kernels(int R, int dtype) { return dtype != kBF16 || R > adapter_rows::kMostRanks; }
static bool in_order(long T, int R, int adapters, int dtype) {
    if (adapters <= 1 || adapters > adapter_order::kMostAdapters) return false;
    return T >= (!two_kernels(R, dtype) ? kTileRows : adapters > kMostSlots ? kMostSlots + 1 : kOrderRows);
}
static long words_of_h(long T, int R, int dtype) { return two_kernels(R, dtype) ? (T * R + 3) / 4 * 4 : 0; }

static bool to_tiles(const AdapterArgs& a, int dtype) {
    return dtype == kBF16 && a.T >= kTileRows && a.adapters <= adapter_order::kMostAdapters && adapter_tiles::takes(a);
}
static long words_of_copies(const AdapterArgs& a, int dtype) { return to_tiles(a, dtype) ? adapter_tiles::words_of_copies(a, adapter_tiles::lying(a)) : 0; }

// Scratch that a call needs, in pieces of 256 bytes: copies of what does not lie on 16 bytes, the short sums [T, R] of the form with two
// kernels, the rows' order.
extern "C" int lb_adapters_scratch(const void* y, long ldy, const void* x, long ldx, const void* A, long a_adapter, long a_row, const void* B,
                                   long b_adapter, long b_row, const void* out, long ldo, long T, int K, int N, int R, int adapters, int dtype) {
    if (T <= 0 || N <= 0) return 0;
    AdapterArgs a{};
    a.y = y; a.ldy = ldy; a.out = const_cast<void*>(out); a.ldo = ldo; a.x = x; a.ldx = ldx; a.A = A; a.a_adapter = a_adapter; a.a_row = a_row; a.B = B; a.b_adapter = b_adapter; a.b_row = b_row;
    a.T = T; a.K = K; a.N = N; a.R = R; a.adapters = adapters;
    const long pieces = (words_of_copies(a, dtype) + words_of_h(T, R, dtype) + (in_order(T, R, adapters, dtype) ? adapter_order::words(T, adapters, adapter_rows::kRows) : 0) + 63) / 64;
    return (int)std::min(pieces, 0x7fffffffL);             // (so much is not to be had)
}

// Strides in elements; columns lie side by side.  out may be y.  error: the device's error word.  launches: how many kernels it were.
extern "C" int lb_add_adapters(const void* y, long ldy, const void* x, long ldx, const void* A, long a_adapter, long a_row,
                               const void* B, long b_adapter, long b_row, const int* index, const float* scales, const int* ranks,
                               void* out, long ldo, void* scratch, int* error, long T, int K, int N, int R, int adapters, int dtype,
                               int* launches, void* stream) {
    *launches = 0;
    if (T <= 0 || N <= 0) return kOk;
    if (K < 0 || R < 0 || adapters < 0) return kBadSize;
    const int parts = parts_of(T, K, R);
    if (T > 0x7fffffffL - 1024 || N > 0x3fffffff) return kTooLarge;
    if (dtype != kF32 && dtype != kBF16) return kBadDType;
    AdapterArgs a{y, ldy, x, ldx, A, a_adapter, a_row, B, b_adapter, b_row, index, scales, ranks, out, ldo, nullptr, nullptr, nullptr, nullptr, T, K, N, R, adapters,
                  parts, ((K + parts - 1) / parts + 31) / 32 * 32, std::max(1, std::min(adapters, T <= 512 ? kMostSlots : 2))};      // (tiles of more rows name one adapter or two)
    const bool ordered = in_order(T, R, adapters, dtype);
    if (ordered) a.slots = 1;                              // (one adapter in a tile)
    if ((N + kCols - 1) / kCols > 65535 || (two_kernels(R, dtype) && ((long)R + kCols - 1) / kCols * a.slots > 65535)) return kTooLarge;
    const cudaStream_t s = (cudaStream_t)stream;
    const long copies = words_of_copies(a, dtype);
    const bool tiles = to_tiles(a, dtype);
    *launches = (copies > 0) + ordered + (two_kernels(R, dtype) ? 2 : 1);
    int* words = (int*)scratch + copies;
    a.h = (float*)words;
    int* plan = ordered ? words + words_of_h(T, R, dtype) : nullptr;
    if (tiles) return adapter_tiles::launch(a, (__nv_bfloat16*)scratch, plan, error, s);
    if (plan != nullptr) {
        const int rc = adapter_order::launch(a, plan, two_kernels(R, dtype) ? kRows : adapter_rows::kRows, -1, s);
        if (rc != 0) return rc;
    }
    if (dtype == kF32) return launch_general<float>(a, s);
    return R > adapter_rows::kMostRanks ? launch_general<__nv_bfloat16>(a, s) : adapter_rows::launch(a, s);
}
