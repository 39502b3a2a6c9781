// Each request's own rules on its logits, in one pass over them:
//   l = logits[row][token], seen tokens:  l > 0 ? l / repetition : l * repetition
//   l -= frequency * count + presence * [count > 0]        (count: how often the request has answered with the token)
//   l += the row's biases of the token, in the order of its list
//   l = -inf where the row's mask does not allow the token
// All of it in 32 bits.  "Seen": in the row's history, its prompt included; "answered": in the history behind the prompt.
//
// What bounds it: reading and writing the logits (8 bytes a token), where there is a batch; for few rows the chain of dependent
// steps.  Counts are not kept as a dense state of 4 bytes a token and request (which would be read with every step and half the
// traffic again): a history of some thousand ids is counted anew every step, in shared memory.  A CTA owns a slice of the
// vocabulary, so that its counters fit; it reads the whole history (from L2) and counts what falls into its slice.  16-bit
// counters where the history's capacity allows, which makes slices twice as long and the history be read half as often.
// 256 rows of 130,048 with 16,384 ids each 62 us, 4.4 TB/s (42 us at the copy rate), 44 without a history; 64 rows with 4,096
// ids, 300 biases and masks 20 (10).  A history shared by a cluster's CTAs, with remote atomics, took 109 us where this form took 80.
#include "lb200/common.cuh"
using namespace lb200;

namespace {
constexpr int kThreads = 256;
constexpr int kUnroll = 8;                              // 16-byte pieces of the row in flight per thread

struct RuleArgs {
    const float* logits; long ld_in;
    float* out; long ld_out;
    const int* history; long ld_history; int capacity;   // null: nobody has seen anything
    const int* slots;                                   // the history's row of a row of logits (null: the same); others: none
    int n_slots;
    const int* lengths; const int* prompt_lengths;      // (null: no prompt, all of it is answer)
    const float* repetition; const float* frequency; const float* presence;     // null: 1, 0, 0
    const int* bias_start; const int* bias_ids; const float* bias_values; int n_biases;
    const unsigned* allowed; long ld_allowed; int n_masks; const int* allowed_row;      // (allowed_row null: the same)
    int rows, V, slice, slices;
};

// Counters of a slice.  The highest bit says "seen", the others count answers.  The prompt's ids come first and are plain stores (all
// of the same value); only answers need atomic additions.
struct Half {
    typedef unsigned short Raw;
    static constexpr unsigned kSeen = 0x8000u;
    static __device__ __forceinline__ void seen(unsigned* c, int i) { reinterpret_cast<Raw*>(c)[i] = (Raw)kSeen; }
    static __device__ __forceinline__ void answered(unsigned* c, int i) { atomicAdd(c + (i >> 1), 1u << ((i & 1) * 16)); }
    static __device__ __forceinline__ unsigned get(const unsigned* c, int i) { return reinterpret_cast<const Raw*>(c)[i]; }
    static __device__ __forceinline__ uint4 get4(const unsigned* c, int i) {
        const uint2 v = *reinterpret_cast<const uint2*>(c + (i >> 1));
        return make_uint4(v.x & 0xffffu, v.x >> 16, v.y & 0xffffu, v.y >> 16);
    }
    static __device__ __forceinline__ float as_float(unsigned n) { return __uint_as_float(0x4b000000u | n) - 8388608.f; }      // (below 2^23)
};
struct Whole {
    typedef unsigned Raw;
    static constexpr unsigned kSeen = 0x80000000u;
    static __device__ __forceinline__ void seen(unsigned* c, int i) { c[i] = kSeen; }
    static __device__ __forceinline__ void answered(unsigned* c, int i) { atomicAdd(c + i, 1u); }
    static __device__ __forceinline__ unsigned get(const unsigned* c, int i) { return c[i]; }
    static __device__ __forceinline__ uint4 get4(const unsigned* c, int i) { return *reinterpret_cast<const uint4*>(c + i); }
    static __device__ __forceinline__ float as_float(unsigned n) { return (float)n; }
};

// A row's penalties; `inverse`: 1 / repetition.
struct Penalties { float repetition, inverse, frequency, presence; };

// Without branches or a division: where a warp meets a token that was seen, all its tokens go through this.  The quotient is the
// product with the inverse, corrected by its remainder (where there is one: not for infinities).
template <typename C>
__device__ __forceinline__ float penalised(float l, unsigned c, const Penalties& p) {
    const float q = l * p.inverse, rest = fmaf(-q, p.repetition, l);
    const float quotient = fabsf(rest) < INFINITY ? fmaf(rest, p.inverse, q) : q;
    const unsigned n = c & (C::kSeen - 1u);
    const float less = n != 0 ? fmaf(p.frequency, C::as_float(n), p.presence) : 0.f;
    return c != 0 ? (l > 0.f ? quotient : l * p.repetition) - less : l;
}

// VEC: the row's logits and outputs lie alike within 16 bytes, and are read and written in pieces of 16.
template <typename C, bool VEC>
__global__ void __launch_bounds__(kThreads, 4) logit_rules_kernel(RuleArgs a) {
    pdl_wait();
    extern __shared__ unsigned smem[];
    __shared__ int twice;                               // a token has several biases
    unsigned* counts = smem;                            // of up to 3 tokens in front (places 0 .. 3), then the slice's, from place 4 on
    const int words = a.slice / (4 / (int)sizeof(typename C::Raw));
    unsigned* biased = smem + words + 4;                // a bit per place
    const int row = blockIdx.x / a.slices, part = blockIdx.x % a.slices, tid = threadIdx.x;
    const float* in = a.logits + (size_t)row * a.ld_in;
    float* out = a.out + (size_t)row * a.ld_out;
    // the first `skew` tokens lie in front of a 16-byte boundary; slice 0 has them as well
    const int skew = VEC ? min((int)((16 - ((uintptr_t)in & 15)) & 15) >> 2, a.V) : 0;
    const int first = skew + part * a.slice;            // the token at place 4
    const int last = min(first + a.slice, a.V);
    const int n = last - first;                         // (0 or less: only a front)
    const int lowest = part == 0 ? 0 : first;           // this CTA's tokens: lowest .. last - 1, or the front alone
    const unsigned span = (unsigned)max(max(last, part == 0 ? skew : 0) - lowest, 0);

    // the first pieces are on their way while the history is counted
    const int pieces = VEC && n > 0 ? n >> 2 : 0;
    const float4* iv = reinterpret_cast<const float4*>(in + first);
    float4 l[kUnroll];
    unsigned words_of[kUnroll];                         // the mask's word of a piece's first token
    const unsigned* mask = nullptr;
    if (a.allowed != nullptr) {
        const int m = a.allowed_row ? a.allowed_row[row] : row;
        if (m >= 0 && m < a.n_masks) mask = a.allowed + (size_t)m * a.ld_allowed;
    }
    auto fetch = [&](int p0) {                          // (nothing here uses what is loaded: a warp would wait for it)
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) if (p0 + u * kThreads < pieces) l[u] = iv[p0 + u * kThreads];
        if (mask != nullptr) {
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) if (p0 + u * kThreads < pieces) words_of[u] = mask[(first + 4 * (p0 + u * kThreads)) >> 5];
        }
    };
    if (VEC) fetch(tid);

    const float rep = a.repetition ? a.repetition[row] : 1.f;
    const float freq = a.frequency ? a.frequency[row] : 0.f, pres = a.presence ? a.presence[row] : 0.f;
    const Penalties pen{rep, 1.f / rep, freq, pres};
    const int slot = a.slots ? a.slots[row] : row;
    const bool counted = a.history != nullptr && slot >= 0 && slot < a.n_slots && !(rep == 1.f && freq == 0.f && pres == 0.f);
    const int length = counted ? min(max(a.lengths[row], 0), a.capacity) : 0;
    int b0 = 0, b1 = 0;
    if (a.bias_start != nullptr) {
        b0 = min(max(a.bias_start[row], 0), a.n_biases);
        b1 = min(max(a.bias_start[row + 1], b0), a.n_biases);
    }

    // ------------------------------------------------------------ what the row has seen, within the slice
    if (length > 0) {
        for (int i = tid; i < (words + 4) / 4; i += kThreads) reinterpret_cast<uint4*>(counts)[i] = make_uint4(0u, 0u, 0u, 0u);
        __syncthreads();
        const int prompt = a.prompt_lengths ? min(max(a.prompt_lengths[row], 0), length) : 0;
        const int* h = a.history + (size_t)slot * a.ld_history;
        auto each = [&](int from, int to, auto add) {       // of the ids from .. to - 1 those that are this CTA's, four pieces of 16 bytes on their way
            const int lead = min((int)((16 - ((uintptr_t)(h + from) & 15)) & 15) >> 2, to - from), quads = (to - from - lead) >> 2;
            auto one = [&](int id) { if ((unsigned)(id - lowest) < span) add(id - first + 4); };
            const int4* hv = reinterpret_cast<const int4*>(h + from + lead);
            for (int i0 = tid; i0 < quads; i0 += 4 * kThreads) {
                int4 v[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) v[u] = i0 + u * kThreads < quads ? hv[i0 + u * kThreads] : make_int4(-1, -1, -1, -1);
#pragma unroll
                for (int u = 0; u < 4; ++u) { one(v[u].x); one(v[u].y); one(v[u].z); one(v[u].w); }
            }
            if (tid < lead) one(h[from + tid]);
            const int rest = from + lead + 4 * quads + tid;
            if (rest < to) one(h[rest]);
        };
        if (prompt > 0) {
            each(0, prompt, [&](int i) { C::seen(counts, i); });
            __syncthreads();
        }
        if (length > prompt) each(prompt, length, [&](int i) { C::answered(counts, i); });
        __syncthreads();
    }

    // ------------------------------------------------------------ the slice
    auto allowed = [&](int token) { return mask == nullptr || ((mask[token >> 5] >> (token & 31)) & 1u) != 0; };
    auto edited = [&](float l, int token, int i) {
        if (length > 0) l = penalised<C>(l, C::get(counts, i), pen);
        return allowed(token) ? l : -INFINITY;
    };
    if (part == 0 && tid < skew) out[tid] = edited(in[tid], tid, tid - skew + 4);
    int done = 0;
    if (VEC) {
        float4* ov = reinterpret_cast<float4*>(out + first);
        for (int p0 = tid; p0 < pieces; p0 += kThreads * kUnroll) {
            if (p0 != tid) fetch(p0);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const int p = p0 + u * kThreads;
                if (p >= pieces) break;
                const int i = 4 * p;
                if (length > 0) {
                    const uint4 c = C::get4(counts, i + 4);
                    if ((c.x | c.y | c.z | c.w) != 0) {
                        l[u].x = penalised<C>(l[u].x, c.x, pen);
                        l[u].y = penalised<C>(l[u].y, c.y, pen);
                        l[u].z = penalised<C>(l[u].z, c.z, pen);
                        l[u].w = penalised<C>(l[u].w, c.w, pen);
                    }
                }
                if (mask != nullptr) {
                    const int token = first + i, bit = token & 31;
                    unsigned bits = words_of[u] >> bit;
                    if (skew != 0 && bit > 28) bits |= mask[(token >> 5) + 1] << (32 - bit);        // (a word more: its last token is below V)
                    if (!(bits & 1u)) l[u].x = -INFINITY;
                    if (!(bits & 2u)) l[u].y = -INFINITY;
                    if (!(bits & 4u)) l[u].z = -INFINITY;
                    if (!(bits & 8u)) l[u].w = -INFINITY;
                }
                ov[p] = l[u];
            }
        }
        done = pieces * 4;
    }
    for (int i0 = done + tid; i0 < n; i0 += kThreads * kUnroll) {
        float one[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) if (i0 + u * kThreads < n) one[u] = in[first + i0 + u * kThreads];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int i = i0 + u * kThreads;
            if (i < n) out[first + i] = edited(one[u], first + i, i + 4);
        }
    }
    if (b1 <= b0) return;

    // ------------------------------------------------------------ biases: added to what has been written
    // Tokens that have one bias are done by any thread; where one has several (a bit is found set), one warp goes through
    // the list in its order, so that the sum is the same every time.
    for (int i = tid; i < a.slice / 32 + 1; i += kThreads) biased[i] = 0u;
    if (tid == 0) twice = 0;
    __syncthreads();                                    // (also: the slice's outputs are there for all threads)
    auto place = [&](int id) { return (unsigned)(id - lowest) < span ? id - first + 4 : -1; };      // of a token of this CTA
    for (int j = b0 + tid; j < b1; j += kThreads) {
        const int i = place(a.bias_ids[j]);
        if (i >= 0 && (atomicOr(biased + (i >> 5), 1u << (i & 31)) >> (i & 31) & 1u)) twice = 1;
    }
    __syncthreads();
    if (!twice) {
        for (int j = b0 + tid; j < b1; j += kThreads) {
            const int id = a.bias_ids[j];
            if (place(id) >= 0 && allowed(id)) out[id] += a.bias_values[j];
        }
    } else if (tid < 32) {
        for (int j0 = b0; j0 < b1; j0 += 32) {
            const int j = j0 + tid;
            const int id = j < b1 ? a.bias_ids[j] : -1;
            const bool mine = j < b1 && place(id) >= 0 && allowed(id);
            const float v = mine ? a.bias_values[j] : 0.f;
            const unsigned same = __match_any_sync(0xffffffffu, mine ? id : -1 - tid);
            const bool leads = mine && (__ffs(same) - 1) == tid;
            float sum = leads ? out[id] : 0.f;
#pragma unroll
            for (int k = 0; k < 32; ++k) {
                const float w = __shfl_sync(0xffffffffu, v, k);
                if (leads && (same >> k & 1u)) sum += w;
            }
            if (leads) out[id] = sum;
            __syncwarp();
        }
    }
}

template <typename C, bool VEC>
int launch(const RuleArgs& a, cudaStream_t stream) {
    static SharedLimits limits;
    const size_t smem = (size_t)a.slice * sizeof(typename C::Raw) + 16 + (size_t)a.slice / 8 + 16;
    int rc = ensure_dynamic_smem(logit_rules_kernel<C, VEC>, smem, limits);
    if (rc == 0) rc = launch_pdl(logit_rules_kernel<C, VEC>, dim3((unsigned)(a.rows * a.slices)), dim3(kThreads), smem, stream, a);
    return rc != 0 ? rc : launch_status();
}
}  // namespace

// logits, out: float32 [rows, V] with row strides (out may be logits).  history: int32 [n_slots, capacity], ids outside of the
// vocabulary count nowhere.  bias_start: int32 [rows + 1] into bias_ids / bias_values.  allowed: a bit per token, row m at
// allowed + m * ld_allowed words; a row whose allowed_row is outside of [0, n_masks) has no mask.
extern "C" int lb_logit_rules(const float* logits, long ld_in, float* out, long ld_out, int rows, int V, const int* history,
                              long ld_history, int capacity, int n_slots, const int* slots, const int* lengths,
                              const int* prompt_lengths, const float* repetition, const float* frequency, const float* presence,
                              const int* bias_start, const int* bias_ids, const float* bias_values, int n_biases,
                              const int* allowed, long ld_allowed, int n_masks, const int* allowed_row, void* stream) {
    if (rows <= 0 || V <= 0) return kOk;
    if (V > (1 << 30)) return kTooLarge;
    RuleArgs a{logits, ld_in, out, ld_out, history, ld_history, capacity, slots, n_slots, lengths, prompt_lengths, repetition,
               frequency, presence, bias_start, bias_ids, bias_values, n_biases, (const unsigned*)allowed, ld_allowed, n_masks,
               allowed_row, rows, V, 0, 0};
    const bool half = capacity <= 0x7fff;               // the count of a 16-bit counter ends there
    // slices as long as the counters may be, shorter where rows are few, so that the GPU is full
    int slice = half ? 16384 : 8192;
    while (slice > 2048 && (long)rows * ((V + slice - 1) / slice) < 296) slice >>= 1;
    a.slice = slice;
    a.slices = (V + slice - 1) / slice;
    if ((long)rows * a.slices > 0x7fffffffL) return kTooLarge;
    const bool vec = (((uintptr_t)logits ^ (uintptr_t)out) & 15) == 0 && (ld_in - ld_out) % 4 == 0;
    const cudaStream_t s = (cudaStream_t)stream;
    if (half) return vec ? launch<Half, true>(a, s) : launch<Half, false>(a, s);
    return vec ? launch<Whole, true>(a, s) : launch<Whole, false>(a, s);
}
