// The two ends of a speculative step, on the device.
//
// msgl_prepare_extend: from the cached lengths and the number of new tokens of every request to their positions, pool slots and
// page-table entries, and (for drafted trees) the mask of ancestors of every node.  What BatchInfo.prepare_for_extend does on the
// host (mini_sglang/managers/batch_info.py:135-245) with the page allocator's take-from-the-front order
// (mini_sglang/mem_cache/token2kv.py:186-196), for requests whose length is anything, page aligned or not, and whose table row may
// already be backed further than the length (slots left over from rejected drafts).
//
// msgl_accept_tree: the walk from a tree's root along the nodes the model confirms, and the move of those nodes' cache rows to
// consecutive positions in every layer.
#include "msgl_common.h"

namespace msgl {

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

struct ExtendPrepParams {
    const int32_t* req_idx;
    const int32_t* prefix;    // [bs] cached tokens
    const int32_t* new_lens;  // [bs] tokens this step adds
    const int32_t* alloc;     // [bs] positions that have a table entry
    const int32_t* free_pages;
    int32_t free_capacity;
    const int32_t* free_range;
    int32_t* r2t;
    int64_t r2t_stride;
    int32_t* r2p;
    int64_t r2p_stride;
    int32_t table_rows, max_ctx;
    const int32_t* parents;  // optional [capacity]: tree of every request, indices inside the request
    int32_t* positions;      // [capacity]
    int32_t* out_loc;        // [capacity]
    int32_t* cu;             // [bs + 1]
    int32_t* seq_lens;       // [bs]
    uint64_t* mask;          // [capacity, words]
    int32_t* alloc_out;
    int32_t* free_range_out;
    int32_t* status;
    int4* scratch;  // [bs]: prefix, alloc, page of the first page boundary at or behind alloc minus that boundary's page index, row
    int32_t capacity, words;
    int bs, ps;
};

constexpr int kScanThreads = 1024;

// Exclusive prefix sums of two counts over the work group, and their totals.  Every thread calls it.
__device__ __forceinline__ void block_scan2(int64_t a, int64_t b, int64_t (*lds)[2], int64_t& a_before, int64_t& b_before, int64_t& a_total, int64_t& b_total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t x = a, y = b;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t u = __shfl_up(x, d), v = __shfl_up(y, d);
        if (lane >= d) x += u, y += v;
    }
    __syncthreads();  // lds may still be read from the previous call
    if (lane == 63) lds[wave][0] = x, lds[wave][1] = y;
    __syncthreads();
    int64_t xb = 0, yb = 0, xt = 0, yt = 0;
#pragma unroll
    for (int w = 0; w < kScanThreads / 64; ++w) {
        const int64_t u = lds[w][0], v = lds[w][1];
        if (w < wave) xb += u, yb += v;
        xt += u, yt += v;
    }
    a_before = xb + x - a, b_before = yb + y - b, a_total = xt, b_total = yt;
}

// Positions and page-table entry of one new token: its slot.
__device__ __forceinline__ int32_t place_token(const ExtendPrepParams& p, const int4 rq, int pos) {
    const int alloc = rq.y, ps = p.ps;
    int32_t* row = p.r2t + (int64_t)rq.w * p.r2t_stride;
    if (pos < alloc) return row[pos];
    int32_t slot;
    if (pos < (alloc + ps - 1) / ps * ps) {
        slot = row[alloc - 1] + (pos - alloc + 1);  // the rest of a page that is partly backed
    } else {
        slot = p.free_pages[rq.z + pos / ps] * ps + pos % ps;
        if (p.r2p && ps > 1 && pos % ps == 0) p.r2p[(int64_t)rq.w * p.r2p_stride + pos / ps] = slot / ps;
    }
    row[pos] = slot;
    return slot;
}

// Phase 1, one work group: totals, refusal, prefix sums, the state's update.
__global__ __launch_bounds__(kScanThreads) void extend_prepare_scan_kernel(ExtendPrepParams p) {
    __shared__ int64_t lds[kScanThreads / 64][2];
    const int tid = threadIdx.x;
    const int head = p.free_range[0];
    const int end = min(p.free_range[1], p.free_capacity);
    const int earlier = *p.status;
    int64_t tokens = 0, pages = 0;
    bool too_long = false, bad = false, too_wide = false;
    for (int c0 = 0; c0 < p.bs; c0 += kScanThreads) {
        const int i = c0 + tid;
        int L = 0, n = 0, A = 0, row = 0;
        if (i < p.bs) L = p.prefix[i], n = p.new_lens[i], A = p.alloc[i], row = p.req_idx[i];
        const bool wrong = L < 0 || n < 0 || A < L || A > p.max_ctx || row < 0 || row >= p.table_rows;
        const bool longer = !wrong && (int64_t)L + n > p.max_ctx;
        bad |= wrong, too_long |= longer, too_wide |= p.words && n > p.words * 64;
        if (wrong || longer) n = 0, L = 0, A = 0, row = 0;
        const int have = (A + p.ps - 1) / p.ps;
        const int need = max(0, (L + n + p.ps - 1) / p.ps - have);
        int64_t t0, g0, tt, gt;
        block_scan2(n, need, lds, t0, g0, tt, gt);
        if (i < p.bs) {
            p.cu[i] = (int32_t)(tokens + t0);
            p.seq_lens[i] = L + n;
            p.scratch[i] = make_int4(L, A, (int32_t)(head + pages + g0 - have), row);
        }
        tokens += tt, pages += gt;
    }
    const bool any_bad = __syncthreads_or(bad), any_long = __syncthreads_or(too_long), any_wide = __syncthreads_or(too_wide);
    int refuse = earlier;
    if (!refuse) refuse = any_bad ? 3 : any_long ? 2 : (any_wide || tokens > p.capacity) ? 4 : (head < 0 || pages > (int64_t)end - head) ? 1 : 0;
    if (refuse) {  // no token at all: every cu entry 0, lengths, table and free list as they were
        for (int i = tid; i < p.bs; i += kScanThreads) {
            p.cu[i] = 0;
            p.seq_lens[i] = p.prefix[i];
            if (p.alloc_out != p.alloc) p.alloc_out[i] = p.alloc[i];
        }
        __syncthreads();  // every thread has read the status word and the free range
        if (tid == 0) {
            p.cu[p.bs] = 0;
            *p.status = refuse;
            if (p.free_range_out != p.free_range) p.free_range_out[0] = head, p.free_range_out[1] = p.free_range[1];
        }
        return;
    }
    for (int i = tid; i < p.bs; i += kScanThreads) p.alloc_out[i] = max(p.alloc[i], p.prefix[i] + p.new_lens[i]);
    const int32_t valid_end = p.free_range[1];
    __syncthreads();
    if (tid == 0) {
        p.cu[p.bs] = (int32_t)tokens;
        p.free_range_out[0] = head + (int32_t)pages;
        p.free_range_out[1] = valid_end;
    }
}

// Phase 2, plain runs of tokens: one thread per entry of the output arrays.
__global__ __launch_bounds__(256) void extend_prepare_fill_kernel(ExtendPrepParams p) {
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t >= p.capacity) return;
    if (t >= p.cu[p.bs]) {  // behind the last request: the dummy slot
        p.positions[t] = 0;
        p.out_loc[t] = 0;
        return;
    }
    int lo = 0, hi = p.bs - 1;  // last request that starts at or before t and is not empty
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.cu[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
    const int4 rq = p.scratch[lo];
    const int pos = rq.x + t - p.cu[lo];
    p.positions[t] = pos;
    p.out_loc[t] = place_token(p, rq, pos);
}

// One request's tree, by one wave: nodes in chunks of 64, a node per lane.  Inside a chunk the ancestors are collected by pointer
// doubling (a lane's pointer jumps to its pointer's pointer, collecting the nodes jumped over), so a chunk costs log2(depth) steps;
// what lies in earlier chunks is the finished mask row of the first ancestor there.
__device__ __forceinline__ void place_tree(const ExtendPrepParams& p, const int4 rq, int base, int n) {
    const int lane = threadIdx.x & 63;
    for (int c = 0; c * 64 < n; ++c) {
        const int node = c * 64 + lane;
        const bool live = node < n;
        int par = live ? p.parents[base + node] : 0;
        const int32_t slot = live ? place_token(p, rq, rq.x + node) : 0;
        if (par < 0 || par >= node) par = 0;  // anything but an earlier node hangs off the root
        const bool local = live && node > 0 && par >= c * 64;
        int ptr = local ? par - c * 64 : lane;
        const int outer = (live && node > 0 && !local) ? par : -1;
        uint64_t m = local ? 1ull << lane : 0;
        while (true) {
            const int next = __shfl(ptr, ptr);
            if (!__any(next != ptr)) break;
            m |= __shfl(m, ptr);
            ptr = next;
        }
        m |= (1ull << ptr) | (1ull << lane);
        const int up = __shfl(outer, ptr);
        int depth = __popcll(m) - 1;
        if (live) {
            uint64_t* row = p.mask + (int64_t)(base + node) * p.words;
            for (int w = 0; w < p.words; ++w) {
                uint64_t v = w == c ? m : 0;
                if (w < c && up >= 0) v = p.mask[(int64_t)(base + up) * p.words + w], depth += __popcll(v);
                row[w] = v;
            }
            p.positions[base + node] = rq.x + depth;
            p.out_loc[base + node] = slot;
        }
        if (n > 64) __threadfence_block();  // the next chunk reads these mask rows from other lanes of this wave
        __builtin_amdgcn_wave_barrier();
    }
}

// Entries behind the last request: position 0, the dummy slot, an empty mask.
__device__ __forceinline__ void clear_behind(const ExtendPrepParams& p, int total, int first, int step) {
    for (int t = total + first; t < p.capacity; t += step) {
        p.positions[t] = 0;
        p.out_loc[t] = 0;
        for (int w = 0; w < p.words; ++w) p.mask[(int64_t)t * p.words + w] = 0;
    }
}

// Phase 2, trees: a wave per request.
__global__ __launch_bounds__(256) void extend_prepare_tree_kernel(ExtendPrepParams p) {
    const int b = blockIdx.x * 4 + (threadIdx.x >> 6);
    clear_behind(p, p.cu[p.bs], blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
    if (b >= p.bs) return;
    const int base = p.cu[b];
    place_tree(p, p.scratch[b], base, min(p.cu[b + 1] - base, p.words * 64));
}

// Both phases in one launch: what bounds a step is latency, and one launch with one barrier has the least of it (4 requests of 8 nodes 4.9 + 2.4 ->
// 4.1 us, 200 prompts of 450 to 900 tokens 5.1 + 4 -> 6.2 us).  Every work group counts all requests and places its share of the tokens; the first
// writes the lengths.  In place, where a work group's inputs are the first's outputs, there is only the first, and only for steps of a few thousand
// tokens.  Counts fit 32 bits (one_launch).
constexpr int kSmallRequests = 1024, kSmallTokens = 4096, kMostSmall = 1 << 20;
static bool one_launch(int bs, int32_t capacity, int32_t max_ctx, bool in_place) {
    return bs <= kSmallRequests && capacity <= (in_place ? kSmallTokens : kMostSmall) && max_ctx <= kMostSmall;
}
__global__ __launch_bounds__(kScanThreads) void extend_prepare_small_kernel(ExtendPrepParams p) {
    __shared__ int4 req[kSmallRequests];           // prefix, alloc, page offset inside the wave's requests, table row
    __shared__ int start[kSmallRequests];          // first token inside the wave's requests
    __shared__ int sums[kScanThreads / 64][3];     // tokens, pages, refusals seen
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int head = p.free_range[0], valid_end = p.free_range[1], earlier = *p.status;
    int L = 0, n = 0, A = 0, row = 0;
    if (tid < p.bs) L = p.prefix[tid], n = p.new_lens[tid], A = p.alloc[tid], row = p.req_idx[tid];
    const bool wrong = L < 0 || n < 0 || A < L || A > p.max_ctx || row < 0 || row >= p.table_rows;
    const bool longer = !wrong && (int64_t)L + n > p.max_ctx;
    const bool wide = !wrong && ((p.words && n > p.words * 64) || n > p.capacity);
    const int counted = wrong || longer || wide ? 0 : n;
    const int have = (A + p.ps - 1) / p.ps;
    const int need = counted ? max(0, (L + counted + p.ps - 1) / p.ps - have) : 0;
    int tokens = counted, pages = need;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int u = __shfl_up(tokens, d), v = __shfl_up(pages, d);
        if (lane >= d) tokens += u, pages += v;
    }
    const int seen = (__any(wrong) ? 4 : 0) | (__any(longer) ? 2 : 0) | (__any(wide) ? 1 : 0);
    if (lane == 63) sums[wave][0] = tokens, sums[wave][1] = pages, sums[wave][2] = seen;
    if (tid < p.bs) {
        req[tid] = make_int4(L, A, pages - need - have, row);
        start[tid] = tokens - counted;
    }
    __syncthreads();
    // every wave has read the state now; the waves' totals and, for a wave's requests, what lies before them
    int total = 0, taken = 0, any = 0;
    auto before = [&](int w, int what) {
        int r = 0;
#pragma unroll
        for (int k = 0; k < kScanThreads / 64; ++k) r += k < w ? sums[k][what] : 0;
        return r;
    };
#pragma unroll
    for (int k = 0; k < kScanThreads / 64; ++k) total += sums[k][0], taken += sums[k][1], any |= sums[k][2];
    int refuse = earlier;
    if (!refuse)
        refuse = any & 4 ? 3 : any & 2 ? 2 : ((any & 1) || total > p.capacity) ? 4 : (head < 0 || taken > (int64_t)min(valid_end, p.free_capacity) - head) ? 1 : 0;
    const bool writer = blockIdx.x == 0;
    if (writer && tid < p.bs) {
        p.cu[tid] = refuse ? 0 : tokens - counted + before(wave, 0);
        p.seq_lens[tid] = refuse ? L : L + n;
        if (!refuse || p.alloc_out != p.alloc) p.alloc_out[tid] = refuse ? A : max(A, L + n);
    }
    if (writer && tid == 0) {
        p.cu[p.bs] = refuse ? 0 : total;
        if (refuse) *p.status = refuse;
        if (!refuse || p.free_range_out != p.free_range) p.free_range_out[0] = refuse ? head : head + taken, p.free_range_out[1] = valid_end;
    }
    clear_behind(p, refuse ? 0 : total, blockIdx.x * kScanThreads + tid, gridDim.x * kScanThreads);
    if (refuse) return;
    if (p.parents) {
        for (int b = blockIdx.x * (kScanThreads / 64) + wave; b < p.bs; b += gridDim.x * (kScanThreads / 64)) {
            const int4 rq = req[b];
            const int w = b >> 6, base = start[b] + before(w, 0);
            const int end = b + 1 < p.bs ? start[b + 1] + before((b + 1) >> 6, 0) : total;
            place_tree(p, make_int4(rq.x, rq.y, rq.z + head + before(w, 1), rq.w), base, end - base);
        }
    } else {
        for (int t = blockIdx.x * kScanThreads + tid; t < total; t += gridDim.x * kScanThreads) {
            int w = 0, base = 0;  // the last wave whose requests start at or before t, then the last request among them
#pragma unroll
            for (int k = 0, at = 0; k < kScanThreads / 64 - 1; ++k) {
                at += sums[k][0];
                if (at <= t && (k + 1) * 64 < p.bs) w = k + 1, base = at;
            }
            int lo = w * 64, hi = min(p.bs, lo + 64) - 1;
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (base + start[mid] <= t) lo = mid;
                else hi = mid - 1;
            }
            const int4 rq = req[lo];
            const int pos = rq.x + t - (base + start[lo]);
            p.positions[t] = pos;
            p.out_loc[t] = place_token(p, make_int4(rq.x, rq.y, rq.z + head + before(w, 1), rq.w), pos);
        }
    }
}

// ------------------------------------------------------------------------------------------------------------ acceptance
struct AcceptParams {
    const int32_t* draft;
    const int32_t* target;
    const int32_t* parents;
    const int32_t* cu;
    const int32_t* prefix;
    const int32_t* loc;
    const uint64_t* layers;  // [layers][2]: addresses of the K and the V cache
    int64_t slot_bytes;
    int32_t row_chunks;  // 16-byte chunks of one layer's K (or V) row
    int32_t* lens;
    int32_t* rows;
    int32_t* tokens;
    int32_t* next;
    int32_t* seq_lens;
    int bs, num_layers, most, layers_per_group;
};

constexpr int kMoveBatch = 8;
constexpr int kMostAccepted = 64 * MSGL_TREE_MAX_WORDS;

// Work group = one request and a run of layers.  Its first wave walks the tree: a node's child is the first later node that hangs off it and
// drafted the token the model put after it; the first 64 nodes are in registers, a node per lane, so a step is a ballot.  Then all threads move
// rows, each the same 16 bytes of every row.  Path indices rise, and row i of the path goes to node i's slot with i <= path[i]: the source of a
// later row is never an earlier row's destination, so a thread may load a batch of rows before it stores them.  What bounds this is latency
// (lengths -> tree -> rows); every group repeats the walk rather than wait for a launch of its own.
__global__ __launch_bounds__(256) void accept_tree_kernel(AcceptParams p) {
    __shared__ int2 moves[kMostAccepted];  // slots: from, to
    __shared__ int moved;
    const int lane = threadIdx.x & 63;
    const int b = blockIdx.x;
    if (threadIdx.x < 64) {
        const bool writer = blockIdx.y == 0;
        const int base = p.cu[b];
        const int n = p.cu[b + 1] - base;
        int len = 0, count = 0;
        if (n > 0) {
            int par0 = -1, tok0 = 0, tgt0 = 0, loc0 = 0;
            if (lane < n) par0 = p.parents[base + lane], tok0 = p.draft[base + lane], tgt0 = p.target[base + lane], loc0 = p.loc[base + lane];
            if (lane < n && (par0 < 0 || par0 >= lane)) par0 = 0;
            int cur = 0, want = 0;
            while (true) {
                want = cur < 64 ? __shfl(tgt0, cur) : p.target[base + cur];
                if (cur != len) {
                    const int from = cur < 64 ? __shfl(loc0, cur) : p.loc[base + cur], to = len < 64 ? __shfl(loc0, len) : p.loc[base + len];
                    if (lane == 0) moves[count] = make_int2(from, to);
                    ++count;
                }
                if (writer && lane == 0) p.rows[(int64_t)b * p.most + len] = base + cur, p.tokens[(int64_t)b * p.most + len] = want;
                if (++len == p.most) break;
                int child = -1;
                if (cur < 63) {
                    const uint64_t hit = __ballot(lane < n && lane > cur && par0 == cur && tok0 == want);
                    if (hit) child = __ffsll((unsigned long long)hit) - 1;
                }
                for (int c = max(64, (cur + 1) & ~63); child < 0 && c < n; c += 64) {
                    const int node = c + lane;
                    bool is = false;
                    if (node < n && node > cur) {
                        int par = p.parents[base + node];
                        if (par < 0 || par >= node) par = 0;
                        is = par == cur && p.draft[base + node] == want;
                    }
                    const uint64_t hit = __ballot(is);
                    if (hit) child = c + __ffsll((unsigned long long)hit) - 1;
                }
                if (child < 0) break;
                cur = child;
            }
            if (writer && lane == 0) p.next[b] = want;
        }
        if (writer) {
            for (int i = len + lane; i < p.most; i += 64) p.rows[(int64_t)b * p.most + i] = -1, p.tokens[(int64_t)b * p.most + i] = -1;
            if (lane == 0) {
                p.lens[b] = len;
                p.seq_lens[b] = p.prefix[b] + len;
            }
        }
        if (lane == 0) moved = count;
    }
    __syncthreads();
    const int count = moved;
    const int l0 = blockIdx.y * p.layers_per_group, layers = min(p.num_layers - l0, p.layers_per_group);
    for (int e = threadIdx.x; e < layers * 2 * p.row_chunks; e += 256) {  // K chunks, then V chunks, layer after layer
        const int half = e / p.row_chunks;
        char* cache = reinterpret_cast<char*>(p.layers[2 * l0 + half]) + (int64_t)(e - half * p.row_chunks) * 16;
        for (int i0 = 0; i0 < count; i0 += kMoveBatch) {
            u32x4 v[kMoveBatch];
#pragma unroll
            for (int j = 0; j < kMoveBatch; ++j) {
                v[j] = u32x4{0, 0, 0, 0};
                if (i0 + j < count) v[j] = *reinterpret_cast<const u32x4*>(cache + moves[i0 + j].x * p.slot_bytes);
            }
#pragma unroll
            for (int j = 0; j < kMoveBatch; ++j)
                if (i0 + j < count) *reinterpret_cast<u32x4*>(cache + moves[i0 + j].y * p.slot_bytes) = v[j];
        }
    }
}

}  // namespace msgl

using namespace msgl;

// (the largest sums of the one-group kernel: 1024 requests of at most `capacity` tokens and max_ctx pages)
extern "C" size_t msgl_prepare_extend_workspace_bytes(int bs, int32_t capacity, int32_t max_ctx, int in_place) {
    if (bs <= 0 || one_launch(bs, capacity, max_ctx, in_place != 0)) return 0;
    return (size_t)bs * sizeof(int4);
}

extern "C" int msgl_prepare_extend(const int32_t* req_pool_indices, const int32_t* prefix_lens, const int32_t* new_lens, const int32_t* alloc_lens,
                                   const int32_t* free_pages, int32_t free_capacity, const int32_t* free_range, int32_t* req_to_token,
                                   int64_t r2t_stride, int32_t table_rows, int32_t max_ctx, int32_t* req_to_page, int64_t r2p_stride,
                                   const int32_t* parents, uint64_t* tree_mask, int mask_words, int32_t* positions, int32_t* out_cache_loc,
                                   int32_t capacity, int32_t* cu_seqlens_q, int32_t* seq_lens, int32_t* alloc_out, int32_t* free_range_out,
                                   int32_t* status, int bs, int page_size, void* workspace, size_t workspace_bytes, void* stream) {
    MSGL_REQUIRE(bs >= 0 && page_size > 0 && free_capacity >= 0 && max_ctx > 0 && table_rows > 0 && capacity >= 0,
                 "msgl_prepare_extend: bs=%d page_size=%d free_capacity=%d max_ctx=%d table_rows=%d capacity=%d", bs, page_size, free_capacity, max_ctx,
                 table_rows, capacity);
    if (bs == 0) return MSGL_OK;
    MSGL_REQUIRE(max_ctx <= 0x7fffffff - page_size && capacity <= 1 << 30, "msgl_prepare_extend: max_ctx %d + page_size %d or capacity %d leaves 32 bits",
                 max_ctx, page_size, capacity);
    MSGL_REQUIRE(req_pool_indices && prefix_lens && new_lens && alloc_lens && (free_pages || free_capacity == 0) && free_range && req_to_token && cu_seqlens_q && seq_lens &&
                     alloc_out && free_range_out && status && (capacity == 0 || (positions && out_cache_loc)),
                 "msgl_prepare_extend: null pointer argument");
    MSGL_REQUIRE((parents == nullptr) == (tree_mask == nullptr), "msgl_prepare_extend: parents and tree_mask go together");
    MSGL_REQUIRE(parents == nullptr || (mask_words >= 1 && mask_words <= MSGL_TREE_MAX_WORDS), "msgl_prepare_extend: mask_words %d outside 1..%d",
                 mask_words, MSGL_TREE_MAX_WORDS);
    MSGL_REQUIRE(r2t_stride >= max_ctx, "msgl_prepare_extend: r2t_stride %lld < max_ctx %d", (long long)r2t_stride, max_ctx);
    MSGL_REQUIRE(req_to_page == nullptr || r2p_stride >= (max_ctx + page_size - 1) / page_size, "msgl_prepare_extend: r2p_stride %lld < pages of a row",
                 (long long)r2p_stride);
    const bool in_place = alloc_out == alloc_lens || free_range_out == free_range;
    const size_t need = msgl_prepare_extend_workspace_bytes(bs, capacity, max_ctx, in_place);
    if (need && (workspace_bytes < need || workspace == nullptr)) {
        set_error("msgl_prepare_extend: workspace %zu < %zu bytes", workspace ? workspace_bytes : (size_t)0, need);
        return MSGL_E_WORKSPACE;
    }
    MSGL_REQUIRE(aligned16(workspace), "msgl_prepare_extend: workspace must be 16-byte aligned");
    // work groups read while others write
    const uint64_t per_req = 4 * (uint64_t)bs, per_token = 4 * (uint64_t)capacity;
    const Span inputs[] = {{alloc_lens, per_req}, {free_range, 8}, {req_pool_indices, per_req}, {prefix_lens, per_req}, {new_lens, per_req},
                           {free_pages, 4 * (uint64_t)free_capacity}, {parents, per_token}};
    const Span results[] = {{alloc_out, per_req}, {free_range_out, 8}, {positions, per_token}, {out_cache_loc, per_token}, {cu_seqlens_q, per_req + 4},
                            {seq_lens, per_req}, {status, 4}, {tree_mask, 2 * per_token * (uint64_t)(parents ? mask_words : 0)},
                            {req_to_token, 4 * (uint64_t)max_ctx, (uint64_t)table_rows, 4 * (uint64_t)r2t_stride},
                            {page_size > 1 ? req_to_page : nullptr, 4 * (((uint64_t)max_ctx + page_size - 1) / page_size), (uint64_t)table_rows, 4 * (uint64_t)r2p_stride},
                            {workspace, need}};
    constexpr int kInputs = sizeof(inputs) / sizeof(Span), kResults = sizeof(results) / sizeof(Span);
    for (int j = 0; j < kResults; ++j) {
        for (int i = 0; i < kInputs; ++i)
            MSGL_REQUIRE((i == j && i < 2 && inputs[i].at == results[j].at) || !spans_meet(inputs[i], results[j]),
                         "msgl_prepare_extend: an output overwrites an input (only alloc_out may be alloc_lens, free_range_out free_range)");
        for (int i = 0; i < j; ++i) MSGL_REQUIRE(!spans_meet(results[i], results[j]), "msgl_prepare_extend: an output overwrites another");
    }
    ExtendPrepParams p;
    p.req_idx = req_pool_indices, p.prefix = prefix_lens, p.new_lens = new_lens, p.alloc = alloc_lens;
    p.free_pages = free_pages, p.free_capacity = free_capacity, p.free_range = free_range;
    p.r2t = req_to_token, p.r2t_stride = r2t_stride, p.r2p = req_to_page, p.r2p_stride = r2p_stride;
    p.table_rows = table_rows, p.max_ctx = max_ctx;
    p.parents = parents, p.positions = positions, p.out_loc = out_cache_loc, p.cu = cu_seqlens_q, p.seq_lens = seq_lens;
    p.mask = tree_mask, p.alloc_out = alloc_out, p.free_range_out = free_range_out, p.status = status;
    p.scratch = static_cast<int4*>(workspace);
    p.capacity = capacity, p.words = parents ? mask_words : 0, p.bs = bs, p.ps = page_size;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (need == 0) {
        const int share = parents ? (bs + kScanThreads / 64 - 1) / (kScanThreads / 64) : (capacity + kScanThreads - 1) / kScanThreads;
        const unsigned groups = in_place || share < 1 ? 1u : (unsigned)share;
        hipLaunchKernelGGL(extend_prepare_small_kernel, dim3(groups), dim3(kScanThreads), 0, st, p);
        return check_launch("extend_prepare_small_kernel");
    }
    hipLaunchKernelGGL(extend_prepare_scan_kernel, dim3(1), dim3(kScanThreads), 0, st, p);
    if (parents) hipLaunchKernelGGL(extend_prepare_tree_kernel, dim3((unsigned)((bs + 3) / 4)), dim3(256), 0, st, p);
    else if (capacity) hipLaunchKernelGGL(extend_prepare_fill_kernel, dim3((unsigned)((capacity + 255) / 256)), dim3(256), 0, st, p);
    return check_launch("extend_prepare kernels");
}

extern "C" int msgl_accept_tree(const int32_t* draft_tokens, const int32_t* target_tokens, const int32_t* parents, const int32_t* cu_seqlens_q,
                                const int32_t* prefix_lens, const int32_t* out_cache_loc, const uint64_t* kv_layers, int num_layers,
                                int64_t cache_stride, int Hkv, int D, int32_t* accept_lens, int32_t* accept_rows, int32_t* accept_tokens,
                                int32_t* next_tokens, int32_t* seq_lens, int bs, int max_accept, void* stream) {
    MSGL_REQUIRE(bs >= 0 && bs <= 65535 * 16 && num_layers >= 0 && num_layers <= 4096 && max_accept >= 1 && max_accept <= kMostAccepted,
                 "msgl_accept_tree: bs=%d num_layers=%d max_accept=%d", bs, num_layers, max_accept);
    if (bs == 0) return MSGL_OK;
    MSGL_REQUIRE(draft_tokens && target_tokens && parents && cu_seqlens_q && prefix_lens && out_cache_loc && accept_lens && accept_rows && accept_tokens &&
                     next_tokens && seq_lens && (num_layers == 0 || kv_layers),
                 "msgl_accept_tree: null pointer argument");
    // a request may be read by several work groups while one writes its results: no result may lie on an input (how long the nodes' arrays are is
    // known on the device only: of these the beginnings are looked at here)
    const uint64_t per_req = 4 * (uint64_t)bs;
    const Span inputs[] = {{prefix_lens, per_req}, {cu_seqlens_q, per_req + 4}, {draft_tokens, 4}, {target_tokens, 4}, {parents, 4}, {out_cache_loc, 4},
                           {kv_layers, 16 * (uint64_t)num_layers}};
    const Span results[] = {{seq_lens, per_req}, {accept_lens, per_req}, {accept_rows, per_req * (uint64_t)max_accept}, {accept_tokens, per_req * (uint64_t)max_accept},
                            {next_tokens, per_req}};
    for (const Span& result : results) {
        for (const Span& in : inputs)
            MSGL_REQUIRE((result.at == seq_lens && in.at == prefix_lens && seq_lens == prefix_lens) || !spans_meet(in, result),
                         "msgl_accept_tree: an output overwrites an input (only seq_lens may be prefix_lens)");
        for (const Span* other = results; other != &result; ++other) MSGL_REQUIRE(!spans_meet(*other, result), "msgl_accept_tree: an output overwrites another");
    }
    MSGL_REQUIRE(num_layers == 0 || (Hkv > 0 && D > 0 && (int64_t)Hkv * D % 8 == 0 && cache_stride >= (int64_t)Hkv * D && cache_stride % 8 == 0),
                 "msgl_accept_tree: Hkv=%d D=%d cache_stride=%lld (rows must be whole 16-byte pieces)", Hkv, D, (long long)cache_stride);
    AcceptParams p;
    p.draft = draft_tokens, p.target = target_tokens, p.parents = parents, p.cu = cu_seqlens_q, p.prefix = prefix_lens, p.loc = out_cache_loc;
    p.layers = kv_layers, p.slot_bytes = cache_stride * 2, p.row_chunks = num_layers ? (int32_t)((int64_t)Hkv * D / 8) : 0;
    p.lens = accept_lens, p.rows = accept_rows, p.tokens = accept_tokens, p.next = next_tokens, p.seq_lens = seq_lens;
    p.bs = bs, p.num_layers = num_layers, p.most = max_accept;
    // up to sixteen groups per compute unit, each repeating the walk (128 requests x 36 layers: 32, 22, 19, 17, 14, 13 us at 1, 2, 4, 8, 16, 32 groups
    // per unit; with one kv head, where a group moves little, 11, 9, 8, 8, 8, 11)
    const int64_t want = 16 * (int64_t)device_cus();
    const int groups = (int)((want + bs - 1) / bs);
    p.layers_per_group = (num_layers + groups - 1) / groups;
    const unsigned gy = num_layers ? (unsigned)((num_layers + p.layers_per_group - 1) / p.layers_per_group) : 1u;
    hipLaunchKernelGGL(accept_tree_kernel, dim3((unsigned)bs, gy), dim3(256), 0, static_cast<hipStream_t>(stream), p);
    return check_launch("accept_tree_kernel");
}
