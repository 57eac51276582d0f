// Log probability of one given token per row of logits, the row's entropy, and its k most probable tokens.
//
//   logprob = x_t - m - ln Z,  H = ln Z - (sum e_i (x_i - m)) / Z,  e_i = exp(x_i - m),  Z = sum e_i,  m = max x_i
//
// One read of the logits.  A work group takes a segment of a row (LOADS pieces of 16 bytes per thread, all requested before the first is used,
// and kept in registers) and leaves (reference, Z, sum e (x - reference)) and the segment's k best (value, index) pairs in the workspace; a second
// kernel folds a row's segments.
//
// Order of the alternatives: by value, ties to the lower index, NaN above everything (as msgl_argmax).  Value and index are one
// 64-bit key: the float's bits mapped to an unsigned number that rises with the value, then the index's complement.
// The k best of a segment: the k-th largest of a wave's 64 lane maxima is no larger than the segment's k-th largest value, so the few values
// that reach it (in every wave's view: the largest of the four) are all that has to be ranked; so are those that reach the least of the waves'
// k/4-th largest, and whichever bar is higher counts (the second from kTwoBars alternatives on).  A wave's k-th largest lane maximum comes from
// bisecting its bits with ballots.  Segments where that leaves too many (long ties that are not a fill from the segment's start on, NaN, infinities)
// are taken apart winner by winner instead.
#include <type_traits>

#include "extend_common.h"
#include "msgl_common.h"

namespace msgl {

constexpr int kLpThreads = 256;
constexpr int kLpWaves = kLpThreads / 64;
constexpr int kLpCandidates = 256;  // per wave
// alternatives from which on the second bar pays for its ballots: 1000 bf16 rows of 151936 with 5, 8, 12, 20, 32 alternatives take
// 85, 88, 93, 113, 166 us with one and 88, 89, 91, 95, 103 with both
constexpr int kTwoBars = 12;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;
constexpr double kPerLog2 = 1.0 / (double)kLog2e;  // not ln 2: undoes exactly what the multiplication by the rounded kLog2e does to the reference

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
constexpr uint32_t kLowestKey = 0x007fffffu;  // of -inf
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
    for (int w = 1; w < kLpWaves; ++w) x = lds[w] > x ? lds[w] : x;
    return x;
}

// The k-th largest of the wave's 64 keys, as far as its upper `bits` bits go (the others 0); 0 if k > 64.
__device__ __forceinline__ uint32_t wave_kth(uint32_t key, int k, int bits) {
    uint32_t t = 0;
    for (int b = 31; b > 31 - bits; --b) {
        const uint32_t with = t | 1u << b;
        if (__popcll(__ballot(key >= with)) >= k) t = with;
    }
    return t;
}

// The same for two ranks at a time.
__device__ __forceinline__ uint2 wave_kth2(uint32_t key, int k0, int k1, int bits) {
    uint2 t = make_uint2(0, 0);
    for (int b = 31; b > 31 - bits; --b) {
        const uint2 with = make_uint2(t.x | 1u << b, t.y | 1u << b);
        const uint64_t at0 = __ballot(key >= with.x), at1 = __ballot(key >= with.y);
        if (__popcll(at0) >= k0) t.x = with.x;
        if (__popcll(at1) >= k1) t.y = with.y;
    }
    return t;
}

// Candidates: a list per wave, zeros behind its end up to the next eight.
struct Candidates {
    uint64_t key[kLpWaves][kLpCandidates + 8];
    int count[kLpWaves];
    // Appends the lanes' keys where `take`, in lane order; n: the wave's count so far.  What does not fit is counted only.
    __device__ __forceinline__ void append(int& n, bool take, uint64_t k) {
        const uint64_t who = __ballot(take);
        const int place = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
        if (take && place < kLpCandidates) key[threadIdx.x >> 6][place] = k;
        n += __popcll(who);
    }
    // Ends the wave's list; true if every wave's list fits.
    __device__ __forceinline__ bool close(int n) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        if (lane < 8 && n <= kLpCandidates) key[wave][n + lane] = 0;
        if (lane == 0) count[wave] = n;
        __syncthreads();
        int most = 0;
#pragma unroll
        for (int w = 0; w < kLpWaves; ++w) most = max(most, count[w]);
        return most <= kLpCandidates;
    }
    // Hands the `top` largest (all distinct) to put(rank, key); the places behind the last one get 0.  Four lanes count for a key, a list each.
    template <typename Put>
    __device__ __forceinline__ void rank(int top, Put put) {
        static_assert(kLpWaves == 4, "a lane of four per list");
        int n[kLpWaves], total = 0;
#pragma unroll
        for (int w = 0; w < kLpWaves; ++w) n[w] = count[w], total += n[w];
        const int list = threadIdx.x & 3;
        const uint64_t* mine = key[list];
        const int length = n[list];
        for (int i = threadIdx.x >> 2; i < total; i += kLpThreads / 4) {
            int at = i, w = 0;
#pragma unroll
            for (int k = 0; k < kLpWaves - 1; ++k)
                if (w == k && at >= n[k]) at -= n[k], w = k + 1;
            const uint64_t x = key[w][at];
            int above = 0;
            for (int j = 0; j < length; j += 8)
#pragma unroll
                for (int k = 0; k < 8; ++k) above += mine[j + k] > x;
            above += __shfl_xor(above, 1);
            above += __shfl_xor(above, 2);
            if (list == 0 && above < top) put(above, x);
        }
        for (int i = total + threadIdx.x; i < top; i += kLpThreads) put(i, 0);
    }
};

// element e of a 16-byte piece
template <int BYTES>
__device__ __forceinline__ float piece_value(const uint4& v, int e) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    if (BYTES == 4) return __builtin_bit_cast(float, w[e]);
    return e & 1 ? bf16_hi(w[e >> 1]) : bf16_lo(w[e >> 1]);
}

// A row's results from its sums against `ref`.
struct RowResult {
    double ref, lnz;
    __device__ __forceinline__ RowResult(const LogprobParams& p, int64_t row, int bytes, double ref_, float z, float t) : ref(ref_) {
        if (z == 0.f) z = __builtin_nanf("");  // no element above -inf
        lnz = (double)logf(z);
        if (threadIdx.x != 0) return;
        const int token = p.tokens[row];
        float x = __builtin_nanf("");
        if ((unsigned)token < (unsigned)p.vocab) {
            const char* at = p.logits + row * p.row_bytes + (int64_t)token * bytes;
            x = bytes == 4 ? *reinterpret_cast<const float*>(at) : bf16_lo(*reinterpret_cast<const uint16_t*>(at));
        }
        p.logprobs[row] = (float)(((double)x - ref) - lnz);
        p.entropy[row] = logf(z) - t / z;
    }
    __device__ __forceinline__ void put(const LogprobParams& p, int64_t row, int rank, uint64_t key) const {
        p.top_ids[row * p.top + rank] = (int32_t)~(uint32_t)key;
        p.top_logprobs[row * p.top + rank] = (float)(((double)key_value((uint32_t)(key >> 32)) - ref) - lnz);
    }
};

// WHOLE: the segment is the whole row, and its results are final.
template <int BYTES, int LOADS, bool WHOLE>
__global__ __launch_bounds__(kLpThreads) void logprob_segment_kernel(LogprobParams p) {
    constexpr int E = 16 / BYTES;                     // elements per piece
    constexpr int kPieces = kLpThreads * LOADS;       // pieces per segment
    __shared__ float lds_f[kLpWaves][2];
    __shared__ uint32_t lds_t[kLpWaves], lds_s[kLpWaves];
    __shared__ Candidates found;
    __shared__ int lds_ties[kLpWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x / (unsigned)p.segments;
    const int seg = blockIdx.x - (unsigned)row * (unsigned)p.segments;
    // rows may start anywhere: whole aligned pieces are read (a piece with one of the row's elements in it is the row's own memory or
    // its allocation's), and what lies outside the row counts as -inf
    const char* first = p.logits + row * p.row_bytes;
    const int lead = (int)((uintptr_t)first & 15) / BYTES;
    const char* base = first - lead * BYTES;
    const int pieces = (int)(((int64_t)lead + p.vocab + E - 1) / E);
    auto index = [&](int j, int e) { return (seg * kPieces + j * kLpThreads + tid) * E + e - lead; };
    auto inside = [&](int j, int e) { return (unsigned)index(j, e) < (unsigned)p.vocab; };
    uint4 v[LOADS];
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        const int g = seg * kPieces + j * kLpThreads + tid;
        constexpr uint32_t none = BYTES == 4 ? 0xff800000u : 0xff80ff80u;  // -inf
        v[j] = make_uint4(none, none, none, none);
        if (g < pieces) v[j] = *reinterpret_cast<const uint4*>(base + (int64_t)g * 16);
    }
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {  // the row's first and last piece
        if (inside(j, 0) && inside(j, E - 1)) continue;
        uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (!inside(j, e)) {
                if (BYTES == 4) w[e & 3] = 0xff800000u;
                else w[e >> 1 & 3] = e & 1 ? (w[e >> 1 & 3] & 0xffffu) | 0xff800000u : (w[e >> 1 & 3] & 0xffff0000u) | 0xff80u;
            }
        v[j] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    float best[LOADS], mine = -INFINITY;
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        best[j] = piece_value<BYTES>(v[j], 0);
#pragma unroll
        for (int e = 2; e < E; e += 2) best[j] = max3_raw(best[j], piece_value<BYTES>(v[j], e - 1), piece_value<BYTES>(v[j], e));
        best[j] = fmaxf(best[j], piece_value<BYTES>(v[j], E - 1));
        mine = fmaxf(mine, best[j]);
    }
    const float top_wave = wave_max(mine);
    // 16 bits of the thresholds are enough to leave few candidates
    uint2 bar_wave = make_uint2(0, 0);
    if (p.top >= kTwoBars) bar_wave = wave_kth2(order_key(mine), p.top, (p.top + kLpWaves - 1) / kLpWaves, 16);
    else if (p.top) bar_wave.x = wave_kth(order_key(mine), p.top, 16);
    if (lane == 0) lds_f[wave][0] = top_wave, lds_t[wave] = bar_wave.x, lds_s[wave] = bar_wave.y;
    __syncthreads();
    float m = lds_f[0][0];
    uint32_t bar = max(lds_t[0], kLowestKey), least = lds_s[0];
#pragma unroll
    for (int w = 1; w < kLpWaves; ++w) m = fmaxf(m, lds_f[w][0]), bar = max(bar, lds_t[w]), least = min(least, lds_s[w]);
    bar = max(bar, least);
    const float ref = m == -INFINITY ? 0.f : m;  // nothing but -inf here: every e is 0 (or NaN)
    float z = 0.f, t = 0.f;
    auto add = [&](auto log2_of) {
#pragma unroll
        for (int j = 0; j < LOADS; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float d = log2_of(piece_value<BYTES>(v[j], e));
                const float x = fast_exp2(d);
                z += x;
                t += x * fmaxf(d, -200.f);  // 2^-200 is 0 in 32 bits: -inf and the like add 0, not 0 * inf
            }
    };
    // (x - ref) log2 e as one multiply-add against a whole number near ref log2 e, itself the reference then (as kPerLog2 gives it: the constant's
    // rounding is then one of x - ref, not of x); huge values (a mask's lowest value
    // in every place) do not survive the multiplication and are subtracted first
    const bool tame = fabsf(ref) < 1e5f;
    const float ref2 = rintf(ref * kLog2e);
    if (tame) add([&](float x) { return __builtin_fmaf(x, kLog2e, -ref2); });
    else add([&](float x) { return (x - ref) * kLog2e; });
    z = wave_sum(z), t = wave_sum(t);
    __syncthreads();
    if (lane == 0) lds_f[wave][0] = z, lds_f[wave][1] = t;
    __syncthreads();
    z = t = 0.f;
#pragma unroll
    for (int w = 0; w < kLpWaves; ++w) z += lds_f[w][0], t += lds_f[w][1];
    const double reference = tame ? (double)ref2 * kPerLog2 : (double)ref;
    std::conditional_t<WHOLE, RowResult, SegmentStats> result = [&] {
        if constexpr (WHOLE) return RowResult(p, row, BYTES, reference, z, t * kLn2);
        else return SegmentStats{reference, z, t * kLn2};
    }();
    if constexpr (!WHOLE) {
        if (tid == 0) p.stats[row * p.segments + seg] = result;
    }
    if (p.top == 0) return;

    auto put = [&](int rank, uint64_t key) {
        if constexpr (WHOLE) result.put(p, row, rank, key);
        else p.keys[(row * p.segments + seg) * p.top + rank] = key;
    };
    bool few = z == z;  // (NaN or infinities in the segment: no sum, and no plain order)
    if (few) {
        // candidates: values at or above the bar; with `ties` only values above it, and of those at it the ones within the first pieces
        auto gather = [&](float at, auto ties) {
            int n = 0, tied = 0;  // of this wave
            // bit j E + e: this lane's element e of piece j is one; taken lane by lane, a bit per turn, so that the key's arithmetic is paid for as
            // often as the lane with the most has some, and not for every place in the pieces
            uint32_t hits = 0;
#pragma unroll
            for (int j = LOADS - 1; j >= 0; --j)
#pragma unroll
                for (int e = E - 1; e >= 0; --e) hits = hits << 1 | (piece_value<BYTES>(v[j], e) >= at ? 1u : 0u);
            while (__any(hits != 0)) {
                const int at_bit = hits ? __ffs(hits) - 1 : 0;
                const bool one = hits != 0;
                hits &= hits - 1;
                const int j = at_bit / E, e = at_bit % E;
                uint32_t w[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    w[c] = 0;
#pragma unroll
                    for (int k = 0; k < LOADS; ++k) w[c] = j == k ? (c == 0 ? v[k].x : c == 1 ? v[k].y : c == 2 ? v[k].z : v[k].w) : w[c];
                }
                const int c = BYTES == 4 ? e : e >> 1;
                const uint32_t word = c == 0 ? w[0] : c == 1 ? w[1] : c == 2 ? w[2] : w[3];
                const float x = BYTES == 4 ? __builtin_bit_cast(float, word) : e & 1 ? bf16_hi(word) : bf16_lo(word);
                const int idx = (seg * kPieces + j * kLpThreads + tid) * E + e - lead;
                bool take = one && (unsigned)idx < (unsigned)p.vocab;
                if (ties) {
                    const bool tie = x == at;
                    take = take && (!tie || (j == 0 && tid <= p.top));
                    tied += __popcll(__ballot(take && tie));
                }
                found.append(n, take, pair_key(x, idx));
            }
            if (lane == 0) lds_ties[wave] = tied;
            return found.close(n);
        };
        few = gather(key_value(bar), std::false_type{});
        if (!few) {  // the whole threshold, and ties at it by their place: a masked or constant segment
            const uint32_t full = wave_kth(order_key(mine), p.top, 32);
            __syncthreads();
            if (lane == 0) lds_t[wave] = full;
            __syncthreads();
            bar = max(lds_t[0], kLowestKey);
#pragma unroll
            for (int w = 1; w < kLpWaves; ++w) bar = max(bar, lds_t[w]);
            few = gather(key_value(bar), std::true_type{});
            int tied = 0;
#pragma unroll
            for (int w = 0; w < kLpWaves; ++w) tied += lds_ties[w];
            few = few && tied >= p.top;
        }
        if (few) found.rank(p.top, put);
    }
    if (few) return;
    // winner by winner: every thread offers the best of its elements that are below the last winner
    uint64_t last = ~0ull, offer = 0;
    bool stale = true;
    __syncthreads();
    for (int k = 0; k < p.top; ++k) {
        if (stale) {
            offer = 0;
#pragma unroll
            for (int j = 0; j < LOADS; ++j)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const uint64_t key = pair_key(piece_value<BYTES>(v[j], e), index(j, e));
                    if (inside(j, e) && key < last && key > offer) offer = key;
                }
        }
        last = block_max_key(offer, found.key[0]);
        stale = offer == last;
        if (tid == 0) put(k, last);  // 0: the segment has fewer elements
    }
}

__global__ __launch_bounds__(kLpThreads) void logprob_row_kernel(LogprobParams p, int bytes) {
    __shared__ Candidates found;
    __shared__ uint32_t lds_t;
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63;
    const SegmentStats* st = p.stats + row * p.segments;
    // every wave folds the sums for itself, a segment per lane
    double ref = -INFINITY;
    for (int s = lane; s < p.segments; s += 64) ref = st[s].z > 0.f && st[s].ref > ref ? st[s].ref : ref;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) ref = fmax(ref, __shfl_xor(ref, d));
    float z = 0.f, t = 0.f;
    for (int s = lane; s < p.segments; s += 64) {
        const SegmentStats e = st[s];
        if (e.z == 0.f) continue;
        const float d = (float)(e.ref - ref);
        const float f = fast_exp2(d * kLog2e);
        z += f * e.z;
        t += f * (e.t + fmaxf(d, -200.f) * e.z);
    }
    z = wave_sum(z), t = wave_sum(t);
    const RowResult result(p, row, bytes, ref, z, t);
    if (p.top == 0) return;
    const uint64_t* keys = p.keys + row * p.segments * p.top;
    auto put = [&](int rank, uint64_t key) { result.put(p, row, rank, key); };
    // the k-th largest of some k or more of the keys bounds the k-th largest of all from below: of the segments' best ones, as many per
    // segment as it takes
    if (tid < 64) {
        const int per = (p.top + p.segments - 1) / p.segments;
        uint32_t best = 0;
        for (int i = lane; i < p.segments * per; i += 64) best = max(best, (uint32_t)(keys[(int64_t)(i / per) * p.top + i % per] >> 32));
        const uint32_t bar = wave_kth(best, p.top, 32);
        if (lane == 0) lds_t = bar;
    }
    __syncthreads();
    const uint32_t bar = lds_t;
    int n = 0;
    for (int i0 = 0; i0 < p.segments * p.top; i0 += kLpThreads) {
        const int i = i0 + tid;
        const uint64_t key = i < p.segments * p.top ? keys[i] : 0;
        found.append(n, key != 0 && (uint32_t)(key >> 32) >= bar, key);
    }
    if (found.close(n)) {
        found.rank(p.top, put);
        return;
    }
    __syncthreads();
    uint64_t last = ~0ull;  // very long rows of ties: winner by winner
    for (int k = 0; k < p.top; ++k) {
        uint64_t offer = 0;
        for (int i = tid; i < p.segments * p.top; i += kLpThreads) {
            const uint64_t key = keys[i];
            if (key < last && key > offer) offer = key;
        }
        last = block_max_key(offer, found.key[0]);
        if (tid == 0) put(k, last);
    }
}

// Elements per thread: as many as it takes for the whole row if 32 will do (one launch instead of two: a bf16 row of 8000 tokens with five alternatives
// 7.8 -> 4.3 us, and 4.5 us of host time less), else 32, or 16 where that would be fewer than four groups per compute unit.  Measured on a vocabulary
// of 151936 with five alternatives, us with 16 / 32 / 64 elements per thread: one bf16 row 8.3 / 9.4 / 10.1, 32 rows 10.6 / 11.2 / 12.2, 64 rows 14.2 /
// 13.5 / 15.1, 1000 rows 94 / 87 / 91; fp32 with 8 / 16 / 32: one row 8.8 / 8.7 / 8.9, 32 rows 13.9 / 11.8 / 12.1, 64 rows 18.3 / 16.1 / 15.6, 1000
// rows 153 / 114 / 105.
static bool logprob_fits(int vocab, int bytes, int elements) { return (int64_t)vocab + 16 / bytes - 1 <= elements * kLpThreads; }
static int logprob_elements(int rows, int vocab, int bytes) {
    if (logprob_fits(vocab, bytes, 32)) return logprob_fits(vocab, bytes, 16) ? 16 : 32;
    const int64_t segments = ((int64_t)vocab + 32 * kLpThreads - 1) / (32 * kLpThreads);
    return rows * segments < 4 * (int64_t)device_cus() ? 16 : 32;
}
static int logprob_segments(int rows, int vocab, int bytes) {
    const int64_t per = (int64_t)kLpThreads * logprob_elements(rows, vocab, bytes);
    return (int)(((int64_t)vocab + 16 / bytes - 1 + per - 1) / per);  // (a row's first piece may begin up to 16 / bytes - 1 elements early)
}

}  // namespace msgl

using namespace msgl;

extern "C" size_t msgl_token_logprobs_workspace_bytes(int rows, int vocab, int elem_bytes, int top) {
    if (rows <= 0 || vocab <= 0 || (elem_bytes != 2 && elem_bytes != 4) || top < 0) return 0;
    const int segments = logprob_segments(rows, vocab, elem_bytes);
    return segments == 1 ? 0 : (size_t)rows * segments * (sizeof(SegmentStats) + (size_t)top * sizeof(uint64_t));
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
    p.segments = logprob_segments(rows, vocab, elem_bytes);
    MSGL_REQUIRE((int64_t)rows * p.segments <= 0xffffffffll / kLpThreads, "msgl_token_logprobs: %d rows x %d segments", rows, p.segments);
    const size_t need = msgl_token_logprobs_workspace_bytes(rows, vocab, elem_bytes, top);
    if (need && (workspace == nullptr || workspace_bytes < need)) {
        set_error("msgl_token_logprobs: workspace %zu < %zu bytes", workspace_bytes, need);
        return MSGL_E_WORKSPACE;
    }
    MSGL_REQUIRE(aligned16(workspace), "msgl_token_logprobs: workspace must be 16-byte aligned");
    const uint64_t per_row = 4 * (uint64_t)rows, per_top = per_row * (uint64_t)top;  // work groups read while others write
    const Span inputs[] = {{logits, (uint64_t)vocab * elem_bytes, (uint64_t)rows, (uint64_t)row_stride * elem_bytes}, {token_ids, per_row}};
    const Span results[] = {{logprobs, per_row}, {entropy, per_row}, {top_ids, per_top}, {top_logprobs, per_top}, {workspace, need}};
    for (const Span& result : results) {
        for (const Span& in : inputs) MSGL_REQUIRE(!spans_meet(in, result), "msgl_token_logprobs: an output or the workspace overwrites an input");
        for (const Span* other = results; other != &result; ++other) MSGL_REQUIRE(!spans_meet(*other, result), "msgl_token_logprobs: an output overwrites another");
    }
    p.logits = static_cast<const char*>(logits), p.row_bytes = row_stride * elem_bytes, p.tokens = token_ids;
    p.logprobs = logprobs, p.entropy = entropy, p.top_ids = top_ids, p.top_logprobs = top_logprobs;
    p.stats = static_cast<SegmentStats*>(workspace);
    p.keys = reinterpret_cast<uint64_t*>(p.stats + (size_t)rows * p.segments);
    p.vocab = vocab, p.top = top;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)(rows * p.segments));
    const bool most = logprob_elements(rows, vocab, elem_bytes) == 32, whole = p.segments == 1;
    auto launch = [&](auto bytes, auto loads) {
        constexpr int B = decltype(bytes)::value, L = decltype(loads)::value;
        if (whole) hipLaunchKernelGGL((logprob_segment_kernel<B, L, true>), grid, dim3(kLpThreads), 0, st, p);
        else hipLaunchKernelGGL((logprob_segment_kernel<B, L, false>), grid, dim3(kLpThreads), 0, st, p);
    };
    constexpr std::integral_constant<int, 2> two{};
    constexpr std::integral_constant<int, 4> four{};
    constexpr std::integral_constant<int, 8> eight{};
    if (elem_bytes == 2 && most) launch(two, four);
    else if (elem_bytes == 2) launch(two, two);
    else if (most) launch(four, eight);
    else launch(four, four);
    if (whole) return check_launch("logprob_segment_kernel");
    hipLaunchKernelGGL(logprob_row_kernel, dim3((unsigned)rows), dim3(kLpThreads), 0, st, p, elem_bytes);
    return check_launch("token_logprobs kernels");
}
