// Low-rank adapters of many requests beside a projection that all of them share:
//   out[t] = y[t] + scale_a * (x[t] A_a^T) B_a^T,   a = index[t]   (rows without an adapter: out[t] = y[t])
// x [T, K], y and out [T, N], A [adapters, R, K], B [adapters, N, R], an adapter's rank up to R.
//
// bfloat16: adapters_rows.cuh (decoding rows, any order of adapters) and adapters_tiles.cuh (prompts).  This file: the float32
// form (and that of ranks over 256), and the choice between them.  Tiles of 32 rows, one pass for each adapter that a tile's rows name, products in float32
// registers.  `shrink` leaves h = x A^T per part of K, `expand` adds the parts up in their order, multiplies by the scale and
// adds to y: one rounding, of the output.
#include "lb200/common.cuh"
#include "lb200/adapters.cuh"
#include "lb200/adapters_rows.cuh"
#include "lb200/adapters_tiles.cuh"
using namespace lb200;

namespace {
constexpr int kRows = 32, kCols = 64, kChunk = 32;      // rows, ranks or features of a tile; values of K or R at a time
constexpr int kThreads = 128;                           // 8 groups of 4 rows x 16 groups of 4 columns

// acc[4][4] += rows of `p` (kRows from its first, ld elements apart) times rows of `q` (kCols), over `depth` values
struct Tiles { float p[kChunk][kRows + 4]; float q[kChunk][kCols + 4]; };

template <typename FP, typename FQ>
__device__ __forceinline__ void multiply(Tiles& s, float (&acc)[4][4], int depth, FP p_at, FQ q_at) {
    const int tid = threadIdx.x, r4 = (tid >> 4) * 4, c4 = (tid & 15) * 4;
    for (int k0 = 0; k0 < depth; k0 += kChunk) {
        __syncthreads();
        const int k = tid & 31;
        for (int r = tid >> 5; r < kRows; r += kThreads / 32) s.p[k][r] = k0 + k < depth ? p_at(r, k0 + k) : 0.f;
        for (int c = tid >> 5; c < kCols; c += kThreads / 32) s.q[k][c] = k0 + k < depth ? q_at(c, k0 + k) : 0.f;
        __syncthreads();
#pragma unroll 8
        for (int kk = 0; kk < kChunk; ++kk) {
            const float4 u = *reinterpret_cast<const float4*>(&s.p[kk][r4]), v = *reinterpret_cast<const float4*>(&s.q[kk][c4]);
            const float pu[4] = {u.x, u.y, u.z, u.w}, pv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(pu[i], pv[j], acc[i][j]);
        }
    }
}

// grid: (row tiles, parts of K, rank tiles)
template <typename T>
__global__ void __launch_bounds__(kThreads) adapter_shrink_kernel(AdapterArgs a) {
    pdl_wait();
    __shared__ Tiles s;
    const long t0 = (long)blockIdx.x * kRows;
    const int part = blockIdx.y, j0 = blockIdx.z * kCols, tid = threadIdx.x;
    const int k_begin = part * a.part_k, k_end = min(k_begin + a.part_k, a.K);
    const int mine = adapter_of(a, t0 + (tid & 31));
    const int r4 = (tid >> 4) * 4, c4 = (tid & 15) * 4;
    const T* x = (const T*)a.x;
    for (int i = next_adapter(mine, -1); i != kNoAdapter; i = next_adapter(mine, i)) {
        const int rank = rank_of(a, i);
        if (j0 >= rank) continue;
        const T* A = (const T*)a.A + (size_t)i * a.a_adapter;
        float acc[4][4] = {};
        multiply(s, acc, k_end - k_begin,
                 [&](int r, int k) { return t0 + r < a.T ? to_f32(x[(t0 + r) * a.ldx + k_begin + k]) : 0.f; },
                 [&](int c, int k) { return j0 + c < rank ? to_f32(A[(size_t)(j0 + c) * a.a_row + k_begin + k]) : 0.f; });
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const long t = t0 + r4 + r;
            if (adapter_of(a, t) != i) continue;
            float* h = a.h + ((size_t)part * a.T + t) * a.R;
#pragma unroll
            for (int j = 0; j < 4; ++j) if (j0 + c4 + j < rank) h[j0 + c4 + j] = acc[r][j];
        }
    }
}

// grid: (row tiles, feature tiles)
template <typename T>
__global__ void __launch_bounds__(kThreads) adapter_expand_kernel(AdapterArgs a) {
    pdl_wait();
    __shared__ Tiles s;
    const long t0 = (long)blockIdx.x * kRows;
    const int n0 = blockIdx.y * kCols, tid = threadIdx.x;
    const int mine = adapter_of(a, t0 + (tid & 31));
    const int r4 = (tid >> 4) * 4, c4 = (tid & 15) * 4;
    float sum[4][4] = {};
    for (int i = next_adapter(mine, -1); i != kNoAdapter; i = next_adapter(mine, i)) {
        const int rank = rank_of(a, i);
        const T* B = (const T*)a.B + (size_t)i * a.b_adapter;
        const float scale = a.scales ? a.scales[i] : 1.f;
        float acc[4][4] = {};
        multiply(s, acc, rank,
                 [&](int r, int j) {
                     float h = 0.f;
                     if (adapter_of(a, t0 + r) == i)
                         for (int p = 0; p < a.parts; ++p) h += a.h[((size_t)p * a.T + t0 + r) * a.R + j];
                     return h * scale;
                 },
                 [&](int c, int j) { return n0 + c < a.N ? to_f32(B[(size_t)(n0 + c) * a.b_row + j]) : 0.f; });
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (adapter_of(a, t0 + r4 + r) == i)
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[r][j] = acc[r][j];
    }
    const T* y = (const T*)a.y;
    T* out = (T*)a.out;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const long t = t0 + r4 + r;
        if (t >= a.T) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = n0 + c4 + j;
            if (n < a.N) out[t * a.ldo + n] = from_f32<T>(to_f32(y[t * a.ldy + n]) + sum[r][j]);
        }
    }
}

template <typename T>
int launch_general(const AdapterArgs& a, cudaStream_t s) {
    const unsigned tiles = (unsigned)((a.T + kRows - 1) / kRows);
    int rc = launch_pdl(adapter_shrink_kernel<T>, dim3(tiles, a.parts, a.R > 0 ? (a.R + kCols - 1) / kCols : 1), dim3(kThreads), 0, s, a);
    if (rc == 0) rc = launch_pdl(adapter_expand_kernel<T>, dim3(tiles, (a.N + kCols - 1) / kCols), dim3(kThreads), 0, s, a);
    return rc != 0 ? rc : launch_status();
}
}  // namespace

// How many parts K is cut into: enough CTAs for the SMs, each with 64 values of K at least.
extern "C" int lb_adapter_parts(long T, int K, int R) {
    const long tiles = (T + kRows - 1) / kRows * (R > 0 ? (R + kCols - 1) / kCols : 1);
    const long most = K / 64 < 1 ? 1 : K / 64, want = tiles > 0 ? (296 + tiles - 1) / tiles : 1;
    return (int)(want < 1 ? 1 : want > most ? most : want > 32 ? 32 : want);
}

// From so many rows on a call goes to the tiles' kernel.
constexpr long kTileRows = 384;

// h: float32 scratch [parts, T, R].  Strides in elements; columns lie side by side.  out may be y.
// (h: float32, or ranks over 256.)  marks: int32 scratch, one per 128 rows; error: the device's error word.
extern "C" int lb_add_adapters(const void* y, long ldy, const void* x, long ldx, const void* A, long a_adapter, long a_row,
                               const void* B, long b_adapter, long b_row, const int* index, const float* scales, const int* ranks,
                               void* out, long ldo, float* h, int* marks, int* error, int parts, long T, int K, int N, int R, int adapters, int dtype,
                               void* stream) {
    if (T <= 0 || N <= 0) return kOk;
    if (K < 0 || R < 0 || adapters < 0 || parts < 1) return kBadSize;
    if (T > 0x7fffffffL - 1024 || N > 0x3fffffff) return kTooLarge;
    AdapterArgs a{y, ldy, x, ldx, A, a_adapter, a_row, B, b_adapter, b_row, index, scales, ranks, out, ldo, h, T, K, N, R, adapters,
                  parts, (K + parts - 1) / parts};
    if ((N + kCols - 1) / kCols > 65535) return kTooLarge;
    const cudaStream_t s = (cudaStream_t)stream;
    if (dtype == kF32) return launch_general<float>(a, s);
    if (dtype != kBF16) return kBadDType;
    if (R > adapter_rows::kMostRanks) return launch_general<__nv_bfloat16>(a, s);
    if (T < kTileRows || marks == nullptr || !adapter_tiles::takes(a)) return adapter_rows::launch(a, nullptr, s);
    const int rc = adapter_tiles::launch(a, marks, error, s);
    return rc != 0 ? rc : adapter_rows::launch(a, marks, s);       // what was left to it, if anything
}
