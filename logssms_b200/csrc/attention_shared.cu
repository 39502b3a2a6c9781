// Attention of a batch whose requests begin with the same tokens: the keys of the shared prefix are read once for all of them.
//
// The tokens of the batch lie in groups.  A group's queries (its tokens times the query heads of a key/value head) are the rows
// of one product with the prefix's keys, 8 to 128 rows a tile instead of the heads of one token; what is a request's own (the
// keys behind the prefix) is read token by token.  Both leave (maximum, sum, weighted values) per range of keys, in float32, and
// a third kernel puts the ranges of a row together:
//   m = max m_s,  out = sum o_s 2^(m_s - m) / sum l_s 2^(m_s - m)
//
// This file: the general form, for float32, any page size and head sizes in steps of 8 up to 256, and the merge.  Its products are
// float32 fused multiply-adds on tiles of 16 rows x 32 keys in shared memory, bound by its reads (16 bytes a lane are four of its
// cycles, also where lanes read the same): so a thread makes 4 x 4 scores of a quarter of the columns, which the four warps add up,
// and 4 rows x 4 columns of the output.  The next tile's keys and values come by asynchronous copies while one is worked on.
// 64 requests of 12 heads of 128 (2 of keys), 8,192 + 512 keys, float32: 217 us, 15 TFLOP/s; 46 tokens in 5 groups, 1,531 + 203 keys: 35.
#include <type_traits>
#include "lb200/common.cuh"
#include "lb200/attention_shared.h"
#include "lb200/attention_shared_own.cuh"
#include "lb200/attention_shared_tc.cuh"
using namespace lb200;

namespace {
constexpr int kThreads = 128, kRows = 16, kKeys = 32;

__device__ __forceinline__ float4 get4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 get4(const __nv_bfloat16* p) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
}
__device__ __forceinline__ void copy16(void* to, const void* from, bool there) {             // zeros where nothing is there
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "r"(there ? 16 : 0) : "memory");
}

// Shared memory: queries float32 [kRows][hd + 4], two stages of K and V as they are [kKeys][hd + 16 bytes], the warps' scores
// [4][kRows][kKeys + 1], the weights [kKeys][kRows + 4], the rows' factors.
template <typename T> struct Lay {
    int ld_q, ld;                                         // numbers from row to row
    size_t k, stage, s, p, all;                           // bytes: where K of stage 0 begins, a stage, the scores, the weights, the whole
    __host__ __device__ explicit Lay(int hd) {
        ld_q = hd + 4;
        ld = hd + 16 / (int)sizeof(T);
        k = (size_t)kRows * ld_q * 4;
        stage = 2 * (size_t)kKeys * ld * sizeof(T);
        s = k + 2 * stage;
        p = s + (4 * kRows * (kKeys + 1) * 4 + 15) / 16 * 16;
        all = p + (kKeys * (kRows + 4) + kRows) * 4;
    }
};

// One CTA: 16 rows (token, query head of one key/value head) x a range of keys.
//   prefix: grid (tiles of the groups' rows, kv heads, ranges); own: grid (tokens x tiles of a token's heads, kv heads, ranges)
template <typename T, bool PREFIX>
__global__ void __launch_bounds__(kThreads, 4) shared_general_kernel(SharedArgs a, int head_tiles) {
    // The own keys' launch runs beside the prefix's, of which it needs nothing; its last CTA waits for it at its end, so that the merge,
    // which waits for this launch, comes behind both.
    const bool last = !PREFIX && blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1 && blockIdx.z == gridDim.z - 1;
    if (PREFIX) { pdl_wait(); pdl_trigger(); }
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ long place[2][kKeys];                      // of a tile's keys: the row in the pool, or -1
    const int hd = a.hd, tid = threadIdx.x;
    const Lay<T> lay(hd);
    float* q_s = reinterpret_cast<float*>(smem);
    float* s_s = reinterpret_cast<float*>(smem + lay.s);
    float* p_s = reinterpret_cast<float*>(smem + lay.p);
    float* factors = p_s + kKeys * (kRows + 4);
    const int G = a.Hq / a.Hkv, kvh = blockIdx.y, split = blockIdx.z;
    int first, rows, request, begin, end;                // the rows: token first + (row0 + r) / G, head kvh * G + (row0 + r) % G
    long row0;
    if (PREFIX) {
        int n;
        if (!find_tile(a, blockIdx.x, G, kRows, &end, &row0, &first, &n)) return;
        rows = (int)min((long)kRows, (long)n * G - row0);
        request = a.token_req[first];
        begin = 0;
    } else {
        first = blockIdx.x / head_tiles;
        row0 = (long)(blockIdx.x % head_tiles) * kRows;
        rows = (int)min((long)kRows, (long)G - row0);
        int group_first;
        if (!prefix_of(a, first, &begin, &group_first)) {
            if (last) pdl_wait();
            return;
        }
        request = a.token_req[first];
        end = keys_of(a, first);
    }
    const bool known = request >= 0 && request < a.requests;
    end = known ? (int)min((long)end, (long)a.bt_cols * a.page_size) : begin;
    const int splits = PREFIX ? a.prefix_splits : a.own_splits;
    const int per = end > begin ? (((end - begin + splits - 1) / splits) + kKeys - 1) / kKeys * kKeys : 0;
    const int from = (int)min((long)begin + (long)split * per, (long)max(end, begin)), to = (int)min((long)from + per, (long)max(end, begin));
    const int* bt = a.block_table + (long)(known ? request : 0) * a.bt_stride;
    const T* kc = (const T*)a.k_cache + (size_t)kvh * hd;
    const T* vc = (const T*)a.v_cache + (size_t)kvh * hd;
    const size_t key_stride = (size_t)a.Hkv * hd;

    auto find = [&](int j0, int s) {                      // threads 0 .. 31: where the keys of the tile at j0 lie
        if (tid < kKeys) {
            long at = -1;
            if (j0 + tid < to) {
                const long page = bt[(j0 + tid) / a.page_size];
                if (page >= 0 && page < a.pages) at = page * a.page_size + (j0 + tid) % a.page_size;
            }
            place[s][tid] = at;
        }
    };
    auto fetch = [&](int s) {                             // the tile whose places are there
        T* k_s = reinterpret_cast<T*>(smem + lay.k + s * lay.stage);
        T* v_s = k_s + kKeys * lay.ld;
        constexpr int kEach = 16 / (int)sizeof(T);
        const int pieces = hd / kEach;
        for (int i = tid; i < kKeys * pieces; i += kThreads) {
            const int key = i / pieces, d = (i - key * pieces) * kEach;
            const long at = place[s][key];
            const size_t off = at >= 0 ? (size_t)at * key_stride + d : 0;
            copy16(k_s + key * lay.ld + d, kc + off, at >= 0);
            copy16(v_s + key * lay.ld + d, vc + off, at >= 0);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // the queries and positions are on their way while the places of the first keys are looked up
    constexpr int kQ = kRows * (256 / 4) / kThreads;
    const T* q = (const T*)a.q;
    T qv[kQ][4];
#pragma unroll
    for (int n = 0; n < kQ; ++n) {
        const int i = tid + n * kThreads, r = i / (hd >> 2), d = (i - r * (hd >> 2)) * 4;
        if (r < rows) {
            const int at = (int)row0 + r, token = at / G;
            const T* src = q + (first + token) * a.q_stride + (kvh * G + at - token * G) * hd + d;         // (any alignment)
#pragma unroll
            for (int e = 0; e < 4; ++e) qv[n][e] = src[e];
        }
    }
    const int r = tid >> 3, c = tid & 7;                 // this thread's row of the softmax, its keys c + 8 i
    const int warp = tid >> 5, lane = tid & 31, rg = lane >> 3, kg = lane & 7;         // of the scores: rows 4 rg + i, keys kg + 8 j
    const int o4 = (tid >> 5) * 4, col = (tid & 31) * 4; // of the output: rows o4 + i, columns col and 128 on
    const int at = (int)row0 + r;
    const int token = r < rows ? first + at / G : first;
    const int limit = r < rows ? keys_of(a, token) : 0;
    find(from, 0);
    __syncthreads();
    if (from < to) fetch(0);
    find(from + kKeys, 1);
#pragma unroll
    for (int n = 0; n < kQ; ++n) {
        const int i = tid + n * kThreads, r = i / (hd >> 2), d = (i - r * (hd >> 2)) * 4;
        if (r >= kRows) break;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < rows) v = make_float4(to_f32(qv[n][0]) * a.scale_log2, to_f32(qv[n][1]) * a.scale_log2, to_f32(qv[n][2]) * a.scale_log2, to_f32(qv[n][3]) * a.scale_log2);
        *reinterpret_cast<float4*>(q_s + r * lay.ld_q + d) = v;
    }
    float m = -INFINITY, l = 0.f;
    float4 acc[2][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i >> 2][i & 3] = make_float4(0.f, 0.f, 0.f, 0.f);
    int s_now = 0;
    for (int j0 = from; j0 < to; j0 += kKeys, s_now ^= 1) {
        const int n = min(kKeys, to - j0);
        __syncthreads();                                  // the next tile's places are there, the other stage is done with
        const bool more = j0 + kKeys < to;
        if (more) {
            fetch(s_now ^ 1);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        const bool there[4] = {place[s_now][c] >= 0, place[s_now][c + 8] >= 0, place[s_now][c + 16] >= 0, place[s_now][c + 24] >= 0};
        // the tile is there for all; and does every row see all of its keys?
        const bool clean = __syncthreads_and(r >= rows || (there[0] && there[1] && there[2] && there[3] && j0 + kKeys <= limit));
        find(j0 + 2 * kKeys, s_now);
        const T* k_s = reinterpret_cast<const T*>(smem + lay.k + s_now * lay.stage);
        const T* v_s = k_s + kKeys * lay.ld;
        {
            float part[4][4] = {};
#pragma unroll 2
            for (int d = 4 * warp; d < hd; d += 16) {
                float4 u[4], w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) u[i] = *reinterpret_cast<const float4*>(q_s + (4 * rg + i) * lay.ld_q + d);
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = get4(k_s + (kg + 8 * i) * lay.ld + d);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        part[i][j] = fmaf(u[i].x, w[j].x, fmaf(u[i].y, w[j].y, fmaf(u[i].z, w[j].z, fmaf(u[i].w, w[j].w, part[i][j]))));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) s_s[(warp * kRows + 4 * rg + i) * (kKeys + 1) + kg + 8 * j] = part[i][j];
        }
        __syncthreads();
        float s[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float* at_s = s_s + r * (kKeys + 1) + c + 8 * i;
            s[i] = (at_s[0] + at_s[kRows * (kKeys + 1)]) + (at_s[2 * kRows * (kKeys + 1)] + at_s[3 * kRows * (kKeys + 1)]);
        }
        float mx = m;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (!(there[i] && j0 + c + 8 * i < limit)) s[i] = -INFINITY;         // (no place: behind the range, or a page that is not there)
            mx = fmaxf(mx, s[i]);
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float ref = mx == -INFINITY ? 0.f : mx;    // nothing seen yet: every weight is 2^-inf = 0
        const float factor = exp2f(m - ref);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float p = exp2f(s[i] - ref);
            p_s[(c + 8 * i) * (kRows + 4) + r] = p;
            sum += p;
        }
        l = l * factor + sum;
        m = mx;
        if (c == 0) factors[r] = factor;
        __syncthreads();
        if (col < hd) {
            const float4 f = *reinterpret_cast<const float4*>(factors + o4);
            const float fs[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) { acc[h][i].x *= fs[i]; acc[h][i].y *= fs[i]; acc[h][i].z *= fs[i]; acc[h][i].w *= fs[i]; }
            auto add = [&](int key, auto guarded) {
                const float4 p4 = *reinterpret_cast<const float4*>(p_s + key * (kRows + 4) + o4);
                const float ps[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (col + 128 * h >= hd) break;
                    const float4 w = get4(v_s + key * lay.ld + col + 128 * h);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (guarded.value && ps[i] == 0.f) continue;             // (a masked key's value may be anything)
                        acc[h][i].x = fmaf(ps[i], w.x, acc[h][i].x); acc[h][i].y = fmaf(ps[i], w.y, acc[h][i].y);
                        acc[h][i].z = fmaf(ps[i], w.z, acc[h][i].z); acc[h][i].w = fmaf(ps[i], w.w, acc[h][i].w);
                    }
                }
            };
            if (clean) {
#pragma unroll 4
                for (int key = 0; key < kKeys; ++key) add(key, std::false_type());
            } else {
                for (int key = 0; key < n; ++key) add(key, std::true_type());
            }
        }
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    const int results = a.prefix_splits + a.own_splits, result = PREFIX ? split : a.prefix_splits + split;
    if (r < rows && c == 0) {
        if (l != l) m = 0.f;                             // (a NaN among the scores: the range counts, and makes the row NaN)
        const size_t slot = ((size_t)token * a.Hq + kvh * G + at % G) * results + result;
        a.part_ml[2 * slot] = m;
        a.part_ml[2 * slot + 1] = l;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (o4 + i >= rows) break;
        const int its = (int)row0 + o4 + i, of = its / G;
        const size_t slot = ((size_t)(first + of) * a.Hq + kvh * G + its - of * G) * results + result;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (col + 128 * h < hd) *reinterpret_cast<float4*>(a.part_o + slot * hd + col + 128 * h) = acc[h][i];
    }
    if (last) pdl_wait();
}

// One warp per (token, head): the ranges' weights first, a lane each, then their rows, 16 bytes a lane and several on their way.
template <typename T> __device__ __forceinline__ void store4(T* p, const float4& v);
template <> __device__ __forceinline__ void store4<float>(float* p, const float4& v) { *reinterpret_cast<float4*>(p) = v; }
template <> __device__ __forceinline__ void store4<__nv_bfloat16>(__nv_bfloat16* p, const float4& v) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// A row that stands within the prefix and has columns that are no numbers.  The tensor cores multiply the values of all of a tile's keys,
// those that the row does not see by zero, and zero times an infinity is NaN: so those columns (of `result`, the row's, where each lane
// finds what it has left there) once more, key by key, over the keys that the row sees.  A warp, four columns a lane.  It ends where every
// such column has met a NaN that the row does see, so that only values that nobody sees, and those that come late, cost a walk: 0.8 us a
// key.  It is kept as small as this for the sake of the calls that never come here: with 32 keys at a time (0.2 us a key) its registers
// and its stack cost every call 1.5 us, and 4 behind a cold cache.
template <typename T>
__device__ __noinline__ void again(const SharedArgs& a, int t, int head, int first, int keys, float4* result) {
    const int lane = threadIdx.x & 31, pieces = a.hd >> 2, request = a.token_req[first];
    const T* q = (const T*)a.q + (long)t * a.q_stride + (long)head * a.hd;
    T* out = (T*)a.out + ((size_t)t * a.Hq + head) * a.hd;
    const size_t column = (size_t)(head / (a.Hq / a.Hkv)) * a.hd;
    if (request < 0 || request >= a.requests) keys = 0;
    keys = (int)min((long)keys, (long)a.bt_cols * a.page_size);
    const float4 nothing = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int p0 = 0; p0 < pieces; p0 += 32) {              // (heads of up to 128: once)
        const bool mine = p0 + lane < pieces;
        const float4 had = mine ? result[p0 + lane] : nothing;
        float4 o = nothing;
        float m = -INFINITY, l = 0.f;
#pragma unroll 1
        for (int j = 0; j < keys; ++j) {
            auto open = [](float was, float is) { return was != was && is == is; };         // in question, and no NaN met so far
            if (!__any_sync(0xffffffffu, open(had.x, o.x) || open(had.y, o.y) || open(had.z, o.z) || open(had.w, o.w))) break;
            const long page = a.block_table[(long)request * a.bt_stride + j / a.page_size];
            if (page < 0 || page >= a.pages) continue;
            const size_t at = (size_t)(page * a.page_size + j % a.page_size) * a.Hkv * a.hd + column;
            float4 v = mine ? get4((const T*)a.v_cache + at + 4 * (p0 + lane)) : nothing;
            float score = 0.f;
#pragma unroll 1
            for (int p = lane; p < pieces; p += 32) {
                const float4 k = get4((const T*)a.k_cache + at + 4 * p);
                const T* u = q + 4 * p;                   // (any alignment)
                score = fmaf(to_f32(u[0]), k.x, fmaf(to_f32(u[1]), k.y, fmaf(to_f32(u[2]), k.z, fmaf(to_f32(u[3]), k.w, score))));
            }
            score = warp_sum(score) * a.scale_log2;
            const float top = fmaxf(m, score), ref = top == -INFINITY ? 0.f : top, before = exp2f(m - ref), w = exp2f(score - ref);
            m = top;
            l = l * before + w;
            if (w == 0.f) v = nothing;
            o.x = fmaf(o.x, before, w * v.x); o.y = fmaf(o.y, before, w * v.y);
            o.z = fmaf(o.z, before, w * v.z); o.w = fmaf(o.w, before, w * v.w);
        }
        const float inv = l != 0.f ? 1.f / l : 0.f;
        auto pick = [&](float was, float is) { return was != was ? is * inv : was; };
        // (out may be q, whose row is read for every piece: the results wait in their place until the last one)
        if (mine) result[p0 + lane] = make_float4(pick(had.x, o.x), pick(had.y, o.y), pick(had.z, o.z), pick(had.w, o.w));
    }
    for (int p = lane; p < pieces; p += 32) store4(out + 4 * p, result[p]);
}

template <typename T>
__global__ void __launch_bounds__(256, 4) shared_merge_kernel(const __grid_constant__ SharedArgs a) {
    pdl_wait();
    const long item = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (item >= (long)a.tokens * a.Hq) return;
    const int t = (int)(item / a.Hq);
    int prefix, first;
    if (!prefix_of(a, t, &prefix, &first)) return;                  // rows of no group are left as they are
    const int keys = keys_of(a, t);
    const int splits = a.prefix_splits + a.own_splits;
    const int s0 = prefix > 0 ? 0 : a.prefix_splits;     // without a prefix nobody wrote its ranges
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + (size_t)item * splits;
    const float4* po = reinterpret_cast<const float4*>(a.part_o) + (size_t)item * splits * (a.hd >> 2);
    float m = -INFINITY, l = 0.f;                        // 32 ranges at a time; what is there already is scaled to a new maximum
    float4 o[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
    const int pieces = a.hd >> 2;
    for (int base = s0; base < splits; base += 32) {
        const float2 mine = base + lane < splits ? ml[base + lane] : make_float2(-INFINITY, 0.f);
        const float top = fmaxf(m, warp_max(mine.x)), ref = top == -INFINITY ? 0.f : top;
        const float before = exp2f(m - ref), w = exp2f(mine.x - ref);
        l = l * before + warp_sum(mine.y * w);
        m = top;
#pragma unroll
        for (int h = 0; h < 2; ++h) { o[h].x *= before; o[h].y *= before; o[h].z *= before; o[h].w *= before; }
        const int n = min(32, splits - base);
        for (int s = 0; s < n; s += 4) {
            float4 v[4][2];
            float f[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                f[u] = s + u < n ? __shfl_sync(0xffffffffu, w, (s + u) & 31) : 0.f;
#pragma unroll
                for (int h = 0; h < 2; ++h)              // (a range without keys left nothing to read)
                    v[u][h] = f[u] != 0.f && lane + 32 * h < pieces ? po[(size_t)(base + s + u) * pieces + lane + 32 * h] : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    o[h].x = fmaf(v[u][h].x, f[u], o[h].x); o[h].y = fmaf(v[u][h].y, f[u], o[h].y);
                    o[h].z = fmaf(v[u][h].z, f[u], o[h].z); o[h].w = fmaf(v[u][h].w, f[u], o[h].w);
                }
        }
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;          // a row that saw no key: zeros
    if (keys < prefix && l == l) {                       // (an infinity is one that the row sees, and so is what made its sum NaN)
        const float all = (fabsf(o[0].x) + fabsf(o[0].y)) + (fabsf(o[0].z) + fabsf(o[0].w)) + ((fabsf(o[1].x) + fabsf(o[1].y)) + (fabsf(o[1].z) + fabsf(o[1].w)));
        if (__any_sync(0xffffffffu, all != all)) {
            float4* result = reinterpret_cast<float4*>(a.part_o) + (size_t)item * splits * pieces;       // (what lay there is in it)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (lane + 32 * h < pieces) result[lane + 32 * h] = make_float4(o[h].x * inv, o[h].y * inv, o[h].z * inv, o[h].w * inv);
            return again<T>(a, t, (int)(item % a.Hq), first, keys, result);
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
        if (lane + 32 * h < pieces)
            store4((T*)a.out + (size_t)item * a.hd + 4 * (lane + 32 * h), make_float4(o[h].x * inv, o[h].y * inv, o[h].z * inv, o[h].w * inv));
}

// Do the tensor-core forms take the call?  (Else: the general form; TMA has no map of a pool without pages.)
bool tc_ok(const SharedArgs& a, int dtype) {
    return dtype == kBF16 && a.pages > 0 && (a.hd == 64 || a.hd == 96 || a.hd == 128) && a.page_size % 16 == 0 && (a.pages + 1) * a.page_size < 0x7fffffffL && a.q_stride % 8 == 0 &&
           (((uintptr_t)a.q | (uintptr_t)a.k_cache | (uintptr_t)a.v_cache) & 15) == 0;
}
// How the prefix's work is laid out on the tensor cores: rows of a tile, CTAs of a cluster, clusters for a tile's keys.
struct Layout { bool two; int ranks, clusters; double us; };
Layout best_layout(long tokens, int G, int Hkv, int hd, int groups, long max_prefix, long most_ctas) {
    // us: a tile of 64 keys takes 1.1 with 256 rows and 0.6 where the groups share the tiles out (a quarter more changes no call's time
    // by more than the clock's noise); a CTA's beginning and end 8; a row of partial results is written and read at 4 TB/s.  As many CTAs at once as the GPU holds in clusters of that size.
    const long kt = max_prefix > 0 ? (max_prefix + 63) / 64 : 1;
    Layout best{false, 1, 1, 1e30};
    for (int two = 0; two < 2; ++two) {
        const long rows = two ? 256 : 128, tiles = ((tokens * G + rows - 1) / rows + (groups - 1) / 2) * Hkv;
        for (int k = 0; k < 3; ++k) {
            const int ranks = 1 << k;
            const long held = k == 2 ? 132 : 148, room = held < most_ctas ? held : most_ctas;
            long clusters = room / (tiles * ranks);
            if (clusters > (kt + ranks - 1) / ranks) clusters = (kt + ranks - 1) / ranks;
            if (clusters < 1) clusters = 1;
            if (clusters > 64) clusters = 64;
            const long per = (kt + clusters * ranks - 1) / (clusters * ranks), waves = (tiles * ranks * clusters + room - 1) / room;
            const double us = waves * (8.0 + per * (two ? 1.1 : 0.6)) + clusters * tokens * G * Hkv * hd * 8e-6 / 4.0 + 0.3 * k;
            if (us < best.us) best = {two != 0, ranks, (int)clusters, us};
        }
    }
    return best;
}
// The own keys' kernel runs beside this one, on what it leaves: it gets SMs of its own, half as many as its share of the work says
// (it is bound by memory).  256 requests, 32,768 + 2,048 keys, from a graph: 144 CTAs of the prefix's take 121 us in all, 108 115, 96 109, 84 120.
Layout layout_for(long tokens, int G, int Hkv, int hd, int groups, long max_prefix, long max_own) {
    const Layout all = best_layout(tokens, G, Hkv, hd, groups, max_prefix, 148);
    const double own = 4.0 + tokens * Hkv * hd * 4e-6 * (max_own > 0 ? max_own : 0) / 2 / 4.7;
    const long room = (long)(148 * all.us / (all.us + 0.5 * own));
    return best_layout(tokens, G, Hkv, hd, groups, max_prefix, room < 74 ? 74 : room);
}

int launch_tc(const SharedArgs& a, const Layout& y, cudaStream_t stream) {
    auto both = [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        const int rc = y.two ? shared_tc::launch_prefix<HD, true>(a, y.ranks, stream) : shared_tc::launch_prefix<HD, false>(a, y.ranks, stream);
        return rc != 0 ? rc : shared_own::launch_own<HD>(a, stream);
    };
    return a.hd == 64 ? both(std::integral_constant<int, 64>()) : a.hd == 96 ? both(std::integral_constant<int, 96>()) : both(std::integral_constant<int, 128>());
}

template <typename T>
int launch_general(const SharedArgs& a, long prefix_tiles, cudaStream_t stream) {
    static SharedLimits limits[2];
    const int G = a.Hq / a.Hkv, head_tiles = (G + kRows - 1) / kRows;
    const size_t smem = Lay<T>(a.hd).all;
    int rc = ensure_dynamic_smem(shared_general_kernel<T, true>, smem, limits[0]);
    if (rc == 0) rc = ensure_dynamic_smem(shared_general_kernel<T, false>, smem, limits[1]);
    if (rc == 0 && prefix_tiles > 0)
        rc = launch_pdl(shared_general_kernel<T, true>, dim3((unsigned)prefix_tiles, a.Hkv, a.prefix_splits), dim3(kThreads), smem, stream, a, head_tiles);
    if (rc == 0)
        rc = launch_pdl(shared_general_kernel<T, false>, dim3((unsigned)a.tokens * head_tiles, a.Hkv, a.own_splits), dim3(kThreads), smem, stream, a, head_tiles);
    return rc;
}
}  // namespace

// How many partial results a row has: (of the prefix) << 16 | (of its own keys); so many that the grids fill the SMs, each with some
// keys left.
extern "C" int lb_attention_shared_splits(const void* q, long q_stride, const void* k_cache, const void* v_cache, long pages, int tokens,
                                          int Hq, int Hkv, int hd, int page_size, int groups, long max_prefix, long max_own, int dtype) {
    if (tokens <= 0 || groups <= 0 || Hkv <= 0 || Hq < Hkv) return 1 << 16 | 1;
    SharedArgs a{};
    a.q = q; a.q_stride = q_stride; a.k_cache = k_cache; a.v_cache = v_cache; a.pages = pages; a.hd = hd; a.page_size = page_size;
    const int G = Hq / Hkv;
    const bool tc = tc_ok(a, dtype);
    const long tiles = (((long)tokens * G + kRows - 1) / kRows + (groups - 1) / 2) * Hkv, items = (long)tokens * ((G + 15) / 16) * Hkv;
    auto cut = [](long ctas, long n, long keys, long least) {
        const long most = keys / least < 1 ? 1 : keys / least, want = (ctas + n - 1) / n;
        return (int)(want > most ? (most > 64 ? 64 : most) : want > 64 ? 64 : want);
    };
    // The general form's prefix: no more CTAs than are at work at once, two an SM (float32, 64 requests of 12 heads of 128, 8,192 keys: 6
    // ranges 217 us, 7 of which some wait for a place 303, 13 255).  The own keys' are shorter and take what is left.
    auto whole_wave = [&] {
        const size_t smem = dtype == kBF16 ? Lay<__nv_bfloat16>(hd).all : Lay<float>(hd).all;
        const long n = 148 * (smem <= 113 * 1024 ? 2 : 1) / tiles, most = max_prefix / 64;
        return (int)(n > 64 && most > 64 ? 64 : n < most ? (n < 1 ? 1 : n) : most < 1 ? 1 : most);
    };
    const int prefix = tc ? layout_for(tokens, G, Hkv, hd, groups, max_prefix, max_own).clusters : whole_wave();
    return prefix << 16 | cut(tc ? 2368 : 592, items, max_own, tc ? 256 : 64);
}

// q: [tokens, Hq, hd], rows q_stride elements apart; caches [pages, page_size, Hkv, hd]; block_table [requests, bt_cols].
// part_o: float32 [tokens * Hq * (prefix_splits + own_splits) * hd], part_ml [.. * 2].  Key j of a token: page block_table[its
// request][j / page_size]; keys below its group's prefix_len through the table of the group's first token.
extern "C" int lb_attention_shared(const void* q, long q_stride, const void* k_cache, const void* v_cache, void* out,
                                   const int* block_table, long bt_stride, int bt_cols, int requests, const int* token_req,
                                   const int* positions, const int* group_start, const int* prefix_lens, int groups, float* part_o,
                                   float* part_ml, long pages, int tokens, int Hq, int Hkv, int hd, int page_size, int prefix_splits,
                                   int own_splits, long max_prefix, long max_own, float scale, int* error, int dtype,
                                   void* stream) {
    if (tokens <= 0 || groups <= 0) return kOk;
    if (Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || hd <= 0 || hd % 8 != 0 || hd > 256 || page_size <= 0 || prefix_splits < 1 || own_splits < 1) return kBadSize;
    if (Hkv > 65535 || prefix_splits > 65535 || own_splits > 65535) return kTooLarge;
    SharedArgs a{q, q_stride, k_cache, v_cache, out, block_table, bt_stride, bt_cols, requests, token_req, positions, group_start,
                 prefix_lens, groups, part_o, part_ml, pages, tokens, Hq, Hkv, hd, page_size, prefix_splits, own_splits,
                 scale * 1.4426950408889634f, error};
    const int G = Hq / Hkv;
    const long tiles = most_tiles((long)tokens * G, groups < tokens ? groups : tokens, kRows);
    if ((long)tokens * ((G + kRows - 1) / kRows) > 0x7fffffffL || tiles > 0x7fffffffL) return kTooLarge;
    const cudaStream_t s = (cudaStream_t)stream;
    int rc = kBadDType;
    const Layout y = layout_for(tokens, G, Hkv, hd, groups, max_prefix, max_own);
    LB_DISPATCH_DTYPE(dtype, rc = tc_ok(a, dtype) ? launch_tc(a, y, s) : launch_general<T>(a, tiles, s);
                      if (rc == 0) rc = launch_pdl(shared_merge_kernel<T>, dim3((unsigned)(((long)tokens * Hq + 7) / 8)), dim3(256), 0, s, a));
    return rc != 0 ? rc : launch_status();
}
