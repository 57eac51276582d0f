// Log probability of one given token per row of logits, the row's entropy, and its k most probable tokens.
//
//   logprob = x_t - m - ln Z,  H = ln Z - (sum e_i (x_i - m)) / Z,  e_i = exp(x_i - m),  Z = sum e_i,  m = max x_i
//
// One read of the logits.  A work group takes a segment of a row (2048 pieces of 16 bytes, eight per thread, all requested before
// the first is used, and kept in registers) and leaves (m, Z, sum e (x - m)) and the segment's k best (value, index) pairs in the
// workspace; a second kernel folds a row's segments.
//
// Order of the alternatives: by value, ties to the lower index, NaN above everything (as msgl_argmax).  Value and index are one
// 64-bit key: the float's bits mapped to an unsigned number that rises with the value, then the index's complement.
#include "msgl_common.h"

namespace msgl {

constexpr int kLpThreads = 256;
constexpr int kLpLoads = 8;                        // 16-byte pieces per thread
constexpr int kLpPieces = kLpThreads * kLpLoads;   // pieces per segment
constexpr float kLog2e = 1.44269504088896340736f;

struct SegmentStats {
    double ref;  // natural units: e = exp(x - ref)
    float z;     // sum e
    float t;     // sum e (x - ref)
};

struct LogprobParams {
    const char* logits;
    int64_t row_bytes;
    const int32_t* tokens;
    float* logprobs;
    float* entropy;
    int32_t* top_ids;
    float* top_logprobs;
    SegmentStats* stats;  // [rows][segments]
    uint64_t* keys;       // [rows][segments][top]
    int vocab, top, segments;
};

constexpr uint32_t kNanKey = 0xfffffffeu;  // above +inf's 0xff800000; with index 0 still below the ~0 that stands for "nothing taken yet"
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) return kNanKey;
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);  // -0 -> +0: equal values, equal keys
    return b ^ ((int32_t)b < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
    if (k == kNanKey) return __builtin_nanf("");
    return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ uint64_t pair_key(float x, int idx) { return (uint64_t)order_key(x) << 32 | (uint32_t)~idx; }

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) x = fmaxf(x, __shfl_xor(x, d));
    return x;
}
__device__ __forceinline__ uint64_t wave_max_key(uint64_t x) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = __shfl_xor(x, d);
        x = o > x ? o : x;
    }
    return x;
}
__device__ __forceinline__ uint64_t block_max_key(uint64_t x, uint64_t* lds) {
    x = wave_max_key(x);
    __syncthreads();  // lds may still be read from the previous call
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    x = lds[0];
#pragma unroll
    for (int w = 1; w < kLpThreads / 64; ++w) x = lds[w] > x ? lds[w] : x;
    return x;
}

// element e of a 16-byte piece
template <int BYTES>
__device__ __forceinline__ float piece_value(const uint4& v, int e) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    if (BYTES == 4) return __builtin_bit_cast(float, w[e]);
    return e & 1 ? bf16_hi(w[e >> 1]) : bf16_lo(w[e >> 1]);
}

template <int BYTES>
__global__ __launch_bounds__(kLpThreads) void logprob_segment_kernel(LogprobParams p) {
    constexpr int E = 16 / BYTES;  // elements per piece
    __shared__ float lds_f[kLpThreads / 64][2];
    __shared__ uint64_t lds_k[kLpThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x / (unsigned)p.segments;
    const int seg = blockIdx.x - (unsigned)row * (unsigned)p.segments;
    // rows may start anywhere: whole aligned pieces are read (a piece with one of the row's elements in it is the row's own memory or
    // its allocation's), and what lies outside the row is left out
    const char* first = p.logits + row * p.row_bytes;
    const int lead = (int)((uintptr_t)first & 15) / BYTES;
    const char* base = first - lead * BYTES;
    const int pieces = (int)(((int64_t)lead + p.vocab + E - 1) / E);
    uint4 v[kLpLoads];
#pragma unroll
    for (int j = 0; j < kLpLoads; ++j) {
        const int g = seg * kLpPieces + j * kLpThreads + tid;
        constexpr uint32_t none = BYTES == 4 ? 0xff800000u : 0xff80ff80u;  // -inf
        v[j] = make_uint4(none, none, none, none);
        if (g < pieces) v[j] = *reinterpret_cast<const uint4*>(base + (int64_t)g * 16);
    }
    auto index = [&](int j, int e) { return (seg * kLpPieces + j * kLpThreads + tid) * E + e - lead; };
    auto inside = [&](int j, int e) { return (unsigned)index(j, e) < (unsigned)p.vocab; };
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < kLpLoads; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (inside(j, e)) m = fmaxf(m, piece_value<BYTES>(v[j], e));
    m = wave_max(m);
    if (lane == 0) lds_f[wave][0] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kLpThreads / 64; ++w) m = fmaxf(m, lds_f[w][0]);
    const float ref = m == -INFINITY ? 0.f : m;  // nothing but -inf here: every e is 0 (or NaN)
    float z = 0.f, t = 0.f;
#pragma unroll
    for (int j = 0; j < kLpLoads; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (inside(j, e)) {
                const float d = piece_value<BYTES>(v[j], e) - ref;
                const float x = fast_exp2(d * kLog2e);
                z += x;
                t += x * fmaxf(d, -200.f);  // e^-200 is 0 in 32 bits: -inf and the like add 0, not 0 * inf
            }
    z = wave_sum(z), t = wave_sum(t);
    __syncthreads();
    if (lane == 0) lds_f[wave][0] = z, lds_f[wave][1] = t;
    __syncthreads();
    if (tid == 0) {
        z = t = 0.f;
#pragma unroll
        for (int w = 0; w < kLpThreads / 64; ++w) z += lds_f[w][0], t += lds_f[w][1];
        p.stats[row * p.segments + seg] = SegmentStats{(double)ref, z, t};
    }
    // the k best: every thread offers the best of its elements that are below the last winner
    uint64_t last = ~0ull, mine = 0;
    bool stale = true;
    for (int k = 0; k < p.top; ++k) {
        if (stale) {
            mine = 0;
#pragma unroll
            for (int j = 0; j < kLpLoads; ++j)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const uint64_t key = pair_key(piece_value<BYTES>(v[j], e), index(j, e));
                    if (inside(j, e) && key < last && key > mine) mine = key;
                }
        }
        last = block_max_key(mine, lds_k);
        stale = mine == last;
        if (tid == 0) p.keys[(row * p.segments + seg) * p.top + k] = last;  // 0: the segment has fewer elements
    }
}

__global__ __launch_bounds__(kLpThreads) void logprob_row_kernel(LogprobParams p, int bytes) {
    __shared__ uint64_t lds_k[kLpThreads / 64];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x;
    const SegmentStats* st = p.stats + row * p.segments;
    double ref = -INFINITY;
    for (int s = 0; s < p.segments; ++s) ref = st[s].z > 0.f && st[s].ref > ref ? st[s].ref : ref;
    float z = 0.f, t = 0.f;
    for (int s = 0; s < p.segments; ++s) {
        if (st[s].z == 0.f) continue;
        const float d = (float)(st[s].ref - ref);
        const float f = fast_exp2(d * kLog2e);
        z += f * st[s].z;
        t += f * (st[s].t + fmaxf(d, -200.f) * st[s].z);
    }
    if (z == 0.f) z = __builtin_nanf("");  // no element above -inf
    const double lnz = (double)logf(z);
    if (tid == 0) {
        const int token = p.tokens[row];
        float x = __builtin_nanf("");
        if ((unsigned)token < (unsigned)p.vocab) {
            const char* at = p.logits + row * p.row_bytes + (int64_t)token * bytes;
            x = bytes == 4 ? *reinterpret_cast<const float*>(at) : bf16_lo(*reinterpret_cast<const uint16_t*>(at));
        }
        p.logprobs[row] = (float)(((double)x - ref) - lnz);
        p.entropy[row] = logf(z) - t / z;
    }
    const uint64_t* keys = p.keys + row * p.segments * p.top;
    uint64_t last = ~0ull;
    for (int k = 0; k < p.top; ++k) {
        uint64_t mine = 0;
        for (int i = tid; i < p.segments * p.top; i += kLpThreads) {
            const uint64_t key = keys[i];
            if (key < last && key > mine) mine = key;
        }
        last = block_max_key(mine, lds_k);
        if (tid == 0) {
            p.top_ids[row * p.top + k] = (int32_t)~(uint32_t)last;
            p.top_logprobs[row * p.top + k] = (float)(((double)key_value((uint32_t)(last >> 32)) - ref) - lnz);
        }
    }
}

static int logprob_segments(int vocab, int bytes) {
    const int64_t per = (int64_t)kLpPieces * (16 / bytes);
    return (int)(((int64_t)vocab + 16 / bytes - 1 + per - 1) / per);  // (a row's first piece may begin up to E - 1 elements early)
}

}  // namespace msgl

using namespace msgl;

extern "C" size_t msgl_token_logprobs_workspace_bytes(int rows, int vocab, int elem_bytes, int top) {
    if (rows <= 0 || vocab <= 0 || (elem_bytes != 2 && elem_bytes != 4) || top < 0) return 0;
    return (size_t)rows * logprob_segments(vocab, elem_bytes) * (sizeof(SegmentStats) + (size_t)top * sizeof(uint64_t));
}

extern "C" int msgl_token_logprobs(const void* logits, int64_t row_stride, int elem_bytes, const int32_t* token_ids, float* logprobs,
                                   float* entropy, int32_t* top_ids, float* top_logprobs, int rows, int vocab, int top, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    MSGL_REQUIRE(rows >= 0 && vocab > 0 && vocab <= (1 << 30) && (elem_bytes == 2 || elem_bytes == 4),
                 "msgl_token_logprobs: rows=%d vocab=%d elem_bytes=%d", rows, vocab, elem_bytes);
    MSGL_REQUIRE(top >= 0 && top <= MSGL_LOGPROBS_MAX_TOP && top <= vocab, "msgl_token_logprobs: top=%d outside 0..min(vocab, %d)", top,
                 MSGL_LOGPROBS_MAX_TOP);
    if (rows == 0) return MSGL_OK;
    MSGL_REQUIRE(logits && token_ids && logprobs && entropy && (top == 0 || (top_ids && top_logprobs)), "msgl_token_logprobs: null pointer argument");
    MSGL_REQUIRE(((uintptr_t)logits & (elem_bytes - 1)) == 0 && row_stride >= 0, "msgl_token_logprobs: misaligned logits or row_stride %lld",
                 (long long)row_stride);
    LogprobParams p;
    p.segments = logprob_segments(vocab, elem_bytes);
    MSGL_REQUIRE((int64_t)rows * p.segments <= 0x7fffffff, "msgl_token_logprobs: %d rows x %d segments", rows, p.segments);
    const size_t need = msgl_token_logprobs_workspace_bytes(rows, vocab, elem_bytes, top);
    if (workspace == nullptr || workspace_bytes < need) {
        set_error("msgl_token_logprobs: workspace %zu < %zu bytes", workspace_bytes, need);
        return MSGL_E_WORKSPACE;
    }
    MSGL_REQUIRE(aligned16(workspace), "msgl_token_logprobs: workspace must be 16-byte aligned");
    p.logits = static_cast<const char*>(logits), p.row_bytes = row_stride * elem_bytes, p.tokens = token_ids;
    p.logprobs = logprobs, p.entropy = entropy, p.top_ids = top_ids, p.top_logprobs = top_logprobs;
    p.stats = static_cast<SegmentStats*>(workspace);
    p.keys = reinterpret_cast<uint64_t*>(p.stats + (size_t)rows * p.segments);
    p.vocab = vocab, p.top = top;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)(rows * p.segments));
    if (elem_bytes == 2) hipLaunchKernelGGL(logprob_segment_kernel<2>, grid, dim3(kLpThreads), 0, st, p);
    else hipLaunchKernelGGL(logprob_segment_kernel<4>, grid, dim3(kLpThreads), 0, st, p);
    hipLaunchKernelGGL(logprob_row_kernel, dim3((unsigned)rows), dim3(kLpThreads), 0, st, p, elem_bytes);
    return check_launch("token_logprobs kernels");
}
