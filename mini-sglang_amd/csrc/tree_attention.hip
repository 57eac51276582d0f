// Attention of drafted token trees over the paged cache (verification of a speculative step).
//
//   out[i, h] = softmax_j(scale q_ih . k_j) v_j   over the cached prefix and those nodes of the request's own tree that node i's
//   mask names; a row that sees nothing gives zeros.
//
// All nodes of a request read the same keys, so they are rows of one matrix product: the (node, head of the GQA group) pairs of a kv
// head, packed node after node, 32 to a block.  S^T = K.Q^T and O^T += V^T.P^T on v_mfma_f32_32x32x16_bf16: the row sits on the lane in
// both products (lane & 31), so maximum, sum and rescaling are in-lane plus one swap of lane halves, and the exponentiated scores,
// packed to bf16, are the second product's operand as they stand.  (That product's operand type rounds P: half a step, 2^-8 relative at most, per
// probability, unbiased, where one part holds it, 2^-16 where two do, see probability_parts; the sum is taken of the unrounded ones.)
//
// The narrow kernel, for up to 64 rows per kv head and for tiles of 32 rows of small launches: the pass over K and V bounds it (a 32-key tile
// costs a wave 512 matrix cycles per 32 rows, 768 with probabilities in two parts, where HBM takes 1250 cycles of the compute unit).  The work
// group's four waves take every fourth 32-key tile each, with RB blocks of 32 rows: tiles are private to a wave, so the loop has no barrier.
//   * K and V rows go from HBM to LDS without passing registers, 16 bytes a lane, four rows of 256 bytes an instruction; the XOR swizzles that
//     spread the fragment reads over the banks are applied to the source address.  With one block of rows a wave has room for one tile, and
//     a second work group fits on the compute unit: its loop runs beside the other's start and end (200 requests of 500 to 1000 tokens
//     x 4 to 8 nodes 130 -> 116 us; long runs the same).  With two blocks, one work group fits, and a wave has room for two tiles.
//   * The page table is read per token, also by LDS-DMA, three or four tiles ahead: any page size, no scalar path, nothing the compiler counts.
//   * All these loads are inline asm and waited for by count; their order is K0 V0 | t3 K1 V1 | t4 K2 V2 ..., two slots K0 V0 t3 K1 V1 | t4 K2 V2 ...
//     (t = table entries).
// Where requests are few or unequal, their tiles are dealt in equal shares (TreeWalk, tree_plan); runs of a request leave (O, max, sum) in the
// workspace and a second kernel joins them.
#include <cmath>
#include <type_traits>
#include <utility>

#include "msgl_common.h"
#include "extend_common.h"

namespace msgl {

constexpr int kTreeWaves = 4;
constexpr int kTreeKeys = 32;                       // keys per tile
constexpr int kTreeHalf = kTreeKeys * kHD * 2;      // bytes of a K or V tile
constexpr int tile_slots(int rb) { return rb == 1 ? 1 : 2; }                 // narrow kernel: tiles of K, and of V, a wave has room for
constexpr int tree_ring(int rb) { return 2 * tile_slots(rb) * kTreeHalf; }  // and their bytes
// bf16 parts that a probability is held in (tile_probabilities): two where up to 32 rows per kv head wait for memory anyway (64 requests of 4096 to 8192
// tokens x 4 to 8 nodes 274 us either way), as the decode kernel that such a step stands in for holds them in 32 bits; one, as in extend, where the second
// costs time: two blocks of rows (16 of 2000 to 4000 x 8 to 16 nodes, 47.2 us, would take 51.1), row tiles (1 of 1000 x 60, 14.6, would take 15.6) and
// the wide kernel, which is bound by such products.
constexpr int probability_parts(int rb, bool only_row_tile) { return rb == 1 && only_row_tile ? 2 : 1; }
constexpr int kTreeSlotRing = 4 * 256;              // per wave: table entries of four tiles (64 words each)
constexpr int kTreeMergeRow = kHD + 4;              // floats per row of the exchange at the end (spread over the banks)
constexpr int merge_bytes(int waves, int rb) { return waves * 32 * rb * (kTreeMergeRow + 2) * 4; }
constexpr int kTreeBegin = 16;                      // tiles that the start of a run is worth (TreeWalk)
constexpr int kLeastTiles = 4;                      // least tiles of a share: one per wave of the narrow kernel
constexpr float kLowestScore = -3.40282347e38f;     // reference maximum before the first score: nothing that 32 bits hold is below it
constexpr float kTameScore = 4096.f;                // log2 units up to which half a step of a reference (2^-13) is nothing beside a bf16 probability's
constexpr float kRescaleAt = 8.f;                   // log2 units a row's maximum may outgrow its reference before O is rescaled

struct TreeParams {
    const uint16_t* q;
    int64_t q_stride;
    const uint16_t* kc;
    const uint16_t* vc;
    uint32_t slot_bytes;
    const int32_t* r2t;
    int64_t r2t_stride;
    const int32_t* req_idx;
    const int32_t* cu;
    const int32_t* prefix;
    const uint64_t* mask;
    int words;
    uint16_t* out;
    int64_t out_stride;
    float* ws_o;   // [token][head][split][128]
    float* ws_ml;  // [token][head][split][2]
    int32_t* ws_n; // [token][head]: runs
    int bs, Hq, Hkv, group;
    int hq_shift, hkv_shift, group_shift;  // (all powers of two)
    int items, row_tiles, splits, shares;
    int max_q;
    float scale_log2e;
};

// Eight LDS-DMA loads of 4 rows x 256 bytes to 8 KiB at LDS byte address dst.  First waits for the wave's LDS reads: the fragments of the
// tile that these bytes held are in registers then.
template <bool NT>
__device__ __forceinline__ void dma_tile(const uint64_t (&a)[8], uint32_t dst) {
    unsigned keep;
#define MSGL_TREE_DMA(n, flag) "global_load_lds_dwordx4 %" #n ", off" flag "\n\ts_add_u32 m0, m0, 0x400\n\ts_nop 0\n\t"
    if (NT)
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\t" MSGL_TREE_DMA(2, " nt") MSGL_TREE_DMA(3, " nt")
                         MSGL_TREE_DMA(4, " nt") MSGL_TREE_DMA(5, " nt") MSGL_TREE_DMA(6, " nt") MSGL_TREE_DMA(7, " nt") MSGL_TREE_DMA(8, " nt")
                             MSGL_TREE_DMA(9, " nt") "s_mov_b32 m0, %0"
                     : "=&s"(keep)
                     : "s"(dst), "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(a[4]), "v"(a[5]), "v"(a[6]), "v"(a[7])
                     : "memory", "scc");
    else
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\t" MSGL_TREE_DMA(2, "") MSGL_TREE_DMA(3, "")
                         MSGL_TREE_DMA(4, "") MSGL_TREE_DMA(5, "") MSGL_TREE_DMA(6, "") MSGL_TREE_DMA(7, "") MSGL_TREE_DMA(8, "") MSGL_TREE_DMA(9, "")
                             "s_mov_b32 m0, %0"
                     : "=&s"(keep)
                     : "s"(dst), "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(a[4]), "v"(a[5]), "v"(a[6]), "v"(a[7])
                     : "memory", "scc");
#undef MSGL_TREE_DMA
}

// One word per lane to 256 bytes at LDS byte address dst.
__device__ __forceinline__ void dma_words(uint64_t a, uint32_t dst) {
    unsigned keep;
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %2, off\n\ts_nop 0\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "s"(dst), "v"(a)
                 : "memory");
}

template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// 32 bits of a node's mask row, from bit `off` on
__device__ __forceinline__ uint32_t mask_bits(const uint64_t* row, int words, int off) {
    const int w = off >> 6, s = off & 63;
    uint64_t v = w < words ? row[w] >> s : 0;
    if (s > 32 && w + 1 < words) v |= row[w + 1] << (64 - s);
    return (uint32_t)v;
}

// What a work group does at a time: one request's run of keys [t0, t1) against rows r0 .. of a kv head, as (node, head) pairs.
struct TreeItem {
    int b, base, n, rows, r0, prefix, t0, t1, split, nsplit;
    const int32_t* table;
};

// A request's lengths, and its tiles as far as it has rows from r0 on.
struct TreeRequest {
    int base, n, prefix, row, tiles;
    __device__ __forceinline__ TreeRequest(const TreeParams& p, int b, int r0) {
        base = p.cu[b], n = min(p.cu[b + 1] - base, p.max_q), prefix = max(p.prefix[b], 0), row = p.req_idx[b];
        tiles = n * p.group > r0 ? (prefix + n + kTreeKeys - 1) / kTreeKeys : 0;
    }
};

// Sum (maximum) of the lanes up to and including each, of values that are not negative.
template <bool MAX>
__device__ __forceinline__ int lanes_up_to(int x) {
#define MSGL_TREE_SCAN(ctrl, rows)                                               \
    {                                                                            \
        const int y = __builtin_amdgcn_update_dpp(0, x, ctrl, rows, 0xf, false); \
        x = MAX ? max(x, y) : x + y;                                             \
    }
    MSGL_TREE_SCAN(0x111, 0xf)  // within rows of 16 lanes: 1, 2, 4, 8 down
    MSGL_TREE_SCAN(0x112, 0xf)
    MSGL_TREE_SCAN(0x114, 0xf)
    MSGL_TREE_SCAN(0x118, 0xf)
    MSGL_TREE_SCAN(0x142, 0xa)  // the last lane of rows 0 and 2 into rows 1 and 3
    MSGL_TREE_SCAN(0x143, 0xc)  // the last lane of row 1 into rows 2 and 3
#undef MSGL_TREE_SCAN
    return x;
}

// The way of a work group through the batch.  splits == 1: it has request `share` to itself.  Otherwise the requests' tiles lie end to end and
// share k of them is [k len, (k + 1) len): every work group has the same number of tiles, whatever the requests' lengths are, a share holds the
// end of one request, whole ones and the beginning of another, and a request is in at most `splits` shares.  To begin with a request costs about
// as much as kTreeBegin tiles, and as many are counted in front of it; where shares of that length suffice with every request beginning a share of
// its own, it does (its last share is then the shorter).  Every wave finds all this out by itself.
struct TreeWalk {
    int share, len, begin, b, base, tiles, at, end;  // base, tiles: first tile of request b in that order, and how many; at, end: of the share's tiles left
    bool any;                                        // `it` holds a run
    __device__ __forceinline__ int span(int real) const { return real == 0 ? 0 : begin ? real + begin : (int)((unsigned)(real + len - 1) / (unsigned)len) * len; }
    __device__ __forceinline__ TreeWalk(const TreeParams& p, int k, int r0, int lane, TreeItem& it) {
        share = 0, len = 1, begin = 0, b = k, base = 0, at = 0, end = 0, any = false;
        if (p.splits == 1) {
            const TreeRequest rq(p, k, r0);
            len = max(rq.tiles, 1), end = rq.tiles;
            take(p, rq, r0, it);
            return;
        }
        begin = kTreeBegin;
        const TreeRequest mine(p, min(lane, p.bs - 1), r0);
        const int real = lane < p.bs ? mine.tiles : 0;
        int first = span(real), upto = lanes_up_to<false>(first);
        int total = __builtin_amdgcn_readlane(upto, 63), longest = first;
        for (int b0 = 64; b0 < p.bs; b0 += 64) {
            const int t = b0 + lane < p.bs ? span(TreeRequest(p, b0 + lane, r0).tiles) : 0;
            total += __builtin_amdgcn_readlane(lanes_up_to<false>(t), 63), longest = max(longest, t);
        }
        share = k;
        len = max((int)((unsigned)(total + p.shares - 1) / (unsigned)p.shares), kLeastTiles);
        if (__any(longest > (int64_t)(p.splits - 1) * len))  // (the batch is longer than the bounds said)
            len = (__builtin_amdgcn_readlane(lanes_up_to<true>(longest), 63) + p.splits - 2) / (p.splits - 1);
        if (p.bs <= 64) {
            const int own = (int)((unsigned)(real + len - 1) / (unsigned)len), own_upto = lanes_up_to<false>(own);
            const int shares = __builtin_amdgcn_readlane(own_upto, 63);
            if (shares <= p.shares) begin = 0, first = own * len, upto = own_upto * len, total = shares * len;
        }
        if ((int64_t)k * len >= total) return;
        at = k * len, end = min(total - at, len) + at;
        const uint64_t behind = __ballot(upto > at);  // the request that tile `at` belongs to
        if (behind) {
            b = __ffsll((unsigned long long)behind) - 1, base = __builtin_amdgcn_readlane(upto - first, b);
            TreeRequest rq = mine;  // (the loads above brought it already)
            rq.base = __builtin_amdgcn_readlane(mine.base, b), rq.n = __builtin_amdgcn_readlane(mine.n, b), rq.row = __builtin_amdgcn_readlane(mine.row, b);
            rq.prefix = __builtin_amdgcn_readlane(mine.prefix, b), rq.tiles = __builtin_amdgcn_readlane(mine.tiles, b);
            take(p, rq, r0, it);
            return;
        }
        base = __builtin_amdgcn_readlane(upto, 63);
        for (int b0 = 64; b0 < p.bs; b0 += 64) {
            const int own = b0 + lane < p.bs ? span(TreeRequest(p, b0 + lane, r0).tiles) : 0;
            const int sum = lanes_up_to<false>(own);
            const uint64_t there = __ballot(base + sum > at);
            if (there) {
                const int l = __ffsll((unsigned long long)there) - 1;
                b = b0 + l, base += __builtin_amdgcn_readlane(sum - own, l);
                break;
            }
            base += __builtin_amdgcn_readlane(sum, 63);
        }
        take(p, TreeRequest(p, b, r0), r0, it);
    }
    // The run of request b (rq) that begins at tile `at`.
    __device__ __forceinline__ void take(const TreeParams& p, const TreeRequest& rq, int r0, TreeItem& it) {
        const int first = base + begin;
        tiles = span(rq.tiles);
        it.t0 = max(at - first, 0) * kTreeKeys;
        const int from = (int)((unsigned)first / (unsigned)len);
        it.split = share - from, it.nsplit = (int)((unsigned)(first + rq.tiles - 1) / (unsigned)len) - from + 1;
        at = min(end, base + tiles);
        it.t1 = min(rq.prefix + rq.n, (at - first) * kTreeKeys);
        it.b = b, it.r0 = r0, it.base = rq.base, it.n = rq.n, it.rows = rq.n * p.group, it.prefix = rq.prefix;
        it.table = p.r2t + (int64_t)rq.row * p.r2t_stride;
        any = it.t0 < it.t1;
    }
    __device__ __forceinline__ void next(const TreeParams& p, int r0, TreeItem& it) {
        any = false;
        while (!any && at < end) {  // (a request without tiles is passed over)
            base += tiles, ++b;
            take(p, TreeRequest(p, b, r0), r0, it);
        }
    }
};

// block -> (item, row tile), item = (share, kv head): heads fastest, so that a token row's pieces are read at about the same time, and the row tiles
// of an item on the same XCD (block ids modulo 8), whose L2 then holds the keys for all of them.
struct TreeBlock {
    int item, row_tile;
    __device__ __forceinline__ explicit TreeBlock(const TreeParams& p) {
        const int y = blockIdx.x >> 3;
        row_tile = y % p.row_tiles;
        item = (y / p.row_tiles) * 8 + (blockIdx.x & 7);
    }
};

// The lane number, of which the compiler does not know that it is the same every time: what is derived from it is made anew for every request of a
// share, instead of occupying (and spilling) registers all along.
__device__ __forceinline__ int fresh_lane() {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    return lane;
}

// A wave's running state for RB blocks of 32 rows: O^T (dims 32 mb + 8 (i >> 2) + 4 half + (i & 3) in register i of block mb, row lane & 31),
// reference maximum in log2 units, this lane half's share of the sum.
template <int RB>
struct TreeState {
    f32x16_t o[RB][4];
    float m[RB], l[RB];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
            for (int mb = 0; mb < 4; ++mb)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[rb][mb][i] = 0.f;
            m[rb] = kLowestScore, l[rb] = 0.f;
        }
    }
};

// f(integral_constant<int, 0>) ... f(integral_constant<int, N - 1>): register arrays indexed by constants before any optimisation runs
template <int... I, typename F>
__device__ __forceinline__ void each_of(F&& f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void each(F&& f) {
    each_of(f, std::make_integer_sequence<int, N>{});
}

// Q^T fragments: lane (row lane & 31, half) holds dims 16 ks + 8 half .. + 8.  Rows behind the last one repeat it; they are never stored.
template <int RB>
__device__ __forceinline__ void load_queries(const TreeParams& p, const TreeItem& it, int row0, int h, int lane, bf16x8_t (&qf)[RB][8]) {
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const int r = min(row0 + rb * 32 + (lane & 31), it.rows - 1);
        const int node = r >> p.group_shift;
        const uint16_t* qp = p.q + (int64_t)(it.base + node) * p.q_stride + (h * p.group + (r & (p.group - 1))) * kHD + (lane >> 5) * 8;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) qf[rb][ks] = as_bf16x8(*reinterpret_cast<const uint4*>(qp + ks * 16));
    }
    // in registers before any load that the compiler does not count is under way
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) asm volatile("" : "+v"(qf[rb][ks]));
}

// K fragments of a 32-key tile: row lane & 31, piece 2 ks + half (at that piece ^ (row & 15)).
__device__ __forceinline__ void read_keys(const char* kt, int lane, bf16x8_t (&kf)[8]) {
    const int col = lane & 31, half = lane >> 5;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) kf[ks] = as_bf16x8(*reinterpret_cast<const uint4*>(kt + col * 256 + (((2 * ks + half) ^ (col & 15)) << 4)));
}

// V^T fragments: the 16 lanes of a group name 4 rows x 32 bytes and receive one dim each of those 4 rows: rows 16 ks + 8 pair + 4 half +
// (lane & 15 >> 2), dims 32 mb + 16 (lane >> 4 & 1) + (lane & 15); 16-byte piece c of row r lies at c ^ 4 (r & 3).
__device__ __forceinline__ bf16x8_t read_values(const char* vt, int lane, int mb, int ks) {
    const int q16 = lane & 15, row = 4 * (lane >> 5) + (q16 >> 2);
    const int piece = (4 * mb + 2 * (lane >> 4 & 1) + ((q16 >> 1) & 1)) ^ (4 * (row & 3));
    const char* at = vt + row * 256 + (piece << 4) + (q16 & 1) * 8;
    short4_t x[2];
#pragma unroll
    for (int pair = 0; pair < 2; ++pair)
        x[pair] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(at + (16 * ks + 8 * pair) * 256));
    return __builtin_bit_cast(bf16x8_t, (short8_t){x[0][0], x[0][1], x[0][2], x[0][3], x[1][0], x[1][1], x[1][2], x[1][3]});
}

template <int RB>
__device__ __forceinline__ void tile_scores(const bf16x8_t (&kf)[8], const bf16x8_t (&qf)[RB][8], f32x16_t (&s)[RB]) {
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[rb][i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) s[rb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[ks], qf[rb][ks], s[rb], 0, 0, 0);
    }
}

__device__ __forceinline__ const uint64_t* row_mask(const TreeParams& p, const TreeItem& it, int row) {
    return p.mask + (int64_t)(it.base + (min(row, it.rows - 1) >> p.group_shift)) * p.words;
}
// What a row sees of the tile that begins at key0: bit k for key k.  word: its mask, if that is one word.
__device__ __forceinline__ uint32_t row_sees(const TreeParams& p, const TreeItem& it, int row, uint64_t word, int key0) {
    const int rel = key0 - it.prefix;
    uint32_t see = ~0u;
    if (rel > -32) {
        const int off = max(rel, 0);
        const uint32_t bits = p.words == 1 ? (off < 64 ? (uint32_t)(word >> off) : 0) : mask_bits(row_mask(p, it, row), p.words, off);
        see = rel >= 0 ? bits : (bits << -rel) | ((1u << -rel) - 1);
    }
    if (key0 + kTreeKeys > it.t1) see &= (1u << (it.t1 - key0)) - 1;
    return see;
}

// The lanes' rows' masks where they are one word each, in registers after this.  The wide kernel reads them at the start: in its loop they would be
// waited for together with all the loads that the compiler does not count, for up to three tiles.
template <int RB>
__device__ __forceinline__ void load_masks(const TreeParams& p, const TreeItem& it, int row0, int lane, uint64_t (&word)[RB]) {
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        word[rb] = 0;
        if (p.words == 1) word[rb] = *row_mask(p, it, row0 + rb * 32 + (lane & 31));
    }
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) asm volatile("" : "+v"(word[rb]));
}

// Scales the scores of the tile that begins at key0 (log2 units from here on) and hides what the rows do not see: in this order, so that what is
// hidden is -inf for a scale of 0 too.
// s[rb][i]: key 8 (i >> 2) + 4 half + (i & 3) of the tile, row lane & 31 of the block.
template <int RB>
__device__ __forceinline__ void tile_mask(const TreeParams& p, const TreeItem& it, int row0, const uint64_t (&word)[RB], int key0, int lane, f32x16_t (&s)[RB]) {
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const uint32_t bits = row_sees(p, it, row0 + rb * 32 + (lane & 31), word[rb], key0) >> (4 * (lane >> 5));
#pragma unroll
        for (int i = 0; i < 16; ++i)
            s[rb][i] = bits >> (8 * (i >> 2) + (i & 3)) & 1 ? s[rb][i] * p.scale_log2e : -INFINITY;
    }
}

// The row's reference maximum follows the maximum of its scores (top, over this lane's keys) when that has outgrown it by 2^8 (or is the first):
// probabilities up to 2^8 are as exact in bf16 and as harmless in the sums, and O is rescaled in the first tiles only.
template <int RB>
__device__ __forceinline__ void follow_maximum(float scale_log2e, float (&top)[RB], TreeState<RB>& st) {
    bool grown = false;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        top[rb] = max_with_lane_xor32(top[rb]) * scale_log2e;
        grown |= top[rb] > st.m[rb] + kRescaleAt;
    }
    if (__any(grown)) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const float mn = fmaxf(st.m[rb], top[rb]);
            const float f = fast_exp2(st.m[rb] - mn);
            st.m[rb] = mn;
            st.l[rb] *= f;
#pragma unroll
            for (int mb = 0; mb < 4; ++mb)
#pragma unroll
                for (int i = 0; i < 16; ++i) st.o[rb][mb][i] *= f;
        }
    }
}
template <int RB>
__device__ __forceinline__ void tile_reference(float scale_log2e, const f32x16_t (&s)[RB], TreeState<RB>& st) {
    float top[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        top[rb] = s[rb][0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top[rb] = fmaxf(top[rb], s[rb][i]);
    }
    follow_maximum<RB>(scale_log2e, top, st);
}

// Scores to probabilities relative to the reference, their sum, and the second product's operand.  The scaled score is rounded before the reference is
// subtracted, as the reference was: the row's largest score then gives a power of two of a whole difference of 32-bit numbers, whatever its size (one
// multiply-add, with the product not rounded, is off by half a step of the reference: 0.5 at 2^24, beyond all numbers at 2^32).
// PARTS: the operand is bf16, so a probability is held in one part (2^-8 off at most) or in two, the second what the first left out (2^-16).
template <int PARTS, int RB>
__device__ __forceinline__ void tile_probabilities(float scale_log2e, f32x16_t (&s)[RB], TreeState<RB>& st, bf16x8_t (&pf)[PARTS][RB][2]) {
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[rb][i] = fast_exp2(s[rb][i] * scale_log2e - st.m[rb]);
            sum += s[rb][i];
        }
        st.l[rb] += sum;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = pack_bf16(s[rb][8 * ks + 2 * i], s[rb][8 * ks + 2 * i + 1]);
            pf[0][rb][ks] = as_bf16x8(make_uint4(w[0], w[1], w[2], w[3]));
            if constexpr (PARTS == 2) {
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = pack_bf16(s[rb][8 * ks + 2 * i] - bf16_lo(w[i]), s[rb][8 * ks + 2 * i + 1] - bf16_hi(w[i]));
                pf[1][rb][ks] = as_bf16x8(make_uint4(w[0], w[1], w[2], w[3]));
            }
        }
    }
}

template <int PARTS, int RB>
__device__ __forceinline__ void tile_values(const char* vt, int lane, const bf16x8_t (&pf)[PARTS][RB][2], TreeState<RB>& st) {
#pragma unroll
    for (int mb = 0; mb < 4; ++mb)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            const bf16x8_t vf = read_values(vt, lane, mb, ks);
#pragma unroll
            for (int part = 0; part < PARTS; ++part)
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) st.o[rb][mb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf[part][rb][ks], st.o[rb][mb], 0, 0, 0);
        }
}

// In a tile with hidden keys a row must not touch what it does not see: 0 * NaN and 0 * inf are NaN.  There the product is taken of the finite
// values; whether there were others (a branch of the tree that went wrong) is returned, and add_odd_values deals with them at the end.
template <int PARTS, int RB>
__device__ __forceinline__ bool tile_values_masked(const char* vt, int lane, const bf16x8_t (&pf)[PARTS][RB][2], TreeState<RB>& st) {
    bool odd = false;
#pragma unroll
    for (int mb = 0; mb < 4; ++mb)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            const uint4 x = __builtin_bit_cast(uint4, read_values(vt, lane, mb, ks));
            uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool lo = (w[i] & 0x7f80u) == 0x7f80u, hi = (w[i] & 0x7f800000u) == 0x7f800000u;
                odd |= lo || hi;
                w[i] &= (lo ? 0xffff0000u : ~0u) & (hi ? 0xffffu : ~0u);
            }
            const bf16x8_t vf = as_bf16x8(make_uint4(w[0], w[1], w[2], w[3]));
#pragma unroll
            for (int part = 0; part < PARTS; ++part)
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) st.o[rb][mb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf[part][rb][ks], st.o[rb][mb], 0, 0, 0);
        }
    return __any(odd);
}

// The values that are not finite, added to the rows that see them (a softmax weight is never 0, whatever 32 bits make of it).  o: this wave's rows in
// LDS.  Runs only where a tile had such a value.
__device__ __forceinline__ void add_odd_values(const TreeParams& p, const TreeItem& it, int row0, int rows, int h, int key0, int lane, float* o) {
    for (int r = lane; r < rows; r += 64) {
        const uint32_t see = row_sees(p, it, row0 + r, p.words == 1 ? *row_mask(p, it, row0 + r) : 0, key0);
        for (int k = 0; k < kTreeKeys && key0 + k < it.t1; ++k) {
            const uint16_t* v = reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(p.vc) + (uint64_t)(uint32_t)it.table[key0 + k] * p.slot_bytes) + h * kHD;
            for (int d = 0; d < kHD; ++d)
                if ((v[d] & 0x7f80u) == 0x7f80u && (see >> k & 1)) o[r * kTreeMergeRow + d] += bf16_lo(v[d]);
        }
    }
}

// End of a work group: groups of WPH waves hold the same rows (different keys); their states are joined through LDS and written, as the final
// rows if the request has this one run, else as the run's partial.  row0(g) / head(g): first row and kv head of wave group g; bit t of odd: this
// wave's tile at odd_key0 + t * odd_step held values that are not finite.
template <int RB, int WPH, int NW, typename Row0, typename Head>
__device__ __forceinline__ void join_and_store(const TreeParams& p, const TreeItem& it, TreeState<RB>& st, char* smem, int wave, int lane, uint64_t odd, int odd_key0,
                                               int odd_step, Row0 row0, Head head) {
    constexpr int R = 32 * RB;
    const int half = lane >> 5, col = lane & 31;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) st.l[rb] += __shfl_xor(st.l[rb], 32);
    __syncthreads();  // every wave is done with the tiles
    float* lds_o = reinterpret_cast<float*>(smem);               // [wave][row][kTreeMergeRow]
    float* lds_ml = lds_o + NW * R * kTreeMergeRow;      // [wave][row][2]
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        float* dst = lds_o + (wave * R + rb * 32 + col) * kTreeMergeRow + 4 * half;
#pragma unroll
        for (int mb = 0; mb < 4; ++mb)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float4*>(dst + 32 * mb + 8 * i) =
                    make_float4(st.o[rb][mb][4 * i], st.o[rb][mb][4 * i + 1], st.o[rb][mb][4 * i + 2], st.o[rb][mb][4 * i + 3]);
        if (half == 0) *reinterpret_cast<float2*>(lds_ml + (wave * R + rb * 32 + col) * 2) = make_float2(st.m[rb], st.l[rb]);
    }
    if (__syncthreads_or(odd != 0)) {
        for (int t = 0; odd >> t; ++t)
            if (odd >> t & 1)
                add_odd_values(p, it, row0(wave / WPH), R, head(wave / WPH), odd_key0 + t * odd_step, lane, lds_o + wave * R * kTreeMergeRow);
        __syncthreads();
    }
    for (int idx = threadIdx.x; idx < (NW / WPH) * R * 32; idx += NW * 64) {
        const int g = idx / (R * 32), r = (idx >> 5) % R, d = (idx & 31) * 4;
        const int row = row0(g) + r;
        if (row >= it.rows) continue;
        float M = kLowestScore;
#pragma unroll
        for (int w = 0; w < WPH; ++w) M = fmaxf(M, lds_ml[((g * WPH + w) * R + r) * 2]);
        float L = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WPH; ++w) {
            const float2 ml = *reinterpret_cast<const float2*>(lds_ml + ((g * WPH + w) * R + r) * 2);
            const float f = fast_exp2(ml.x - M);
            L += f * ml.y;
            const float4 x = *reinterpret_cast<const float4*>(lds_o + ((g * WPH + w) * R + r) * kTreeMergeRow + d);
            acc.x += f * x.x, acc.y += f * x.y, acc.z += f * x.z, acc.w += f * x.w;
        }
        const int node = row >> p.group_shift;
        const int hq = head(g) * p.group + (row & (p.group - 1));
        const int64_t tok = it.base + node;
        if (p.splits > 1 && it.split == 0 && d == 0) p.ws_n[tok * p.Hq + hq] = it.nsplit;
        if (it.nsplit == 1) {
            const float inv = L == 0.f ? 0.f : 1.0f / L;  // L == 0: the row sees nothing
            *reinterpret_cast<uint2*>(p.out + tok * p.out_stride + hq * kHD + d) = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
        } else {
            const int64_t at = (tok * p.Hq + hq) * p.splits + it.split;
            *reinterpret_cast<float4*>(p.ws_o + at * kHD + d) = acc;
            if (d == 0) *reinterpret_cast<float2*>(p.ws_ml + at * 2) = make_float2(M, L);
        }
    }
}

// The same where no state has to be joined and no value was odd: from the registers, eight or sixteen bytes a lane and instruction, four dims each.
// (Over LDS in whole rows this was 16 times around a loop of 60 instructions.  With the masks at hand: 1 request of 500 tokens x 60 nodes, 32 / 8 heads,
// 25.5 -> 23 us, 8 of 3000 x 90, 64 / 8 heads, 88 -> 82.5 us.)
__device__ __forceinline__ void store_rows(const TreeParams& p, const TreeItem& it, const TreeState<1>& st, int row0, int h, int lane) {
    const float l = st.l[0] + __shfl_xor(st.l[0], 32);
    const int row = row0 + (lane & 31), half = lane >> 5;
    if (row >= it.rows) return;
    const int node = row >> p.group_shift;
    const int hq = h * p.group + (row & (p.group - 1));
    const int64_t tok = it.base + node, pair = tok * p.Hq + hq;
    if (p.splits > 1 && it.split == 0 && half == 0) p.ws_n[pair] = it.nsplit;
    if (it.nsplit == 1) {
        const float inv = l == 0.f ? 0.f : 1.0f / l;  // l == 0: the row sees nothing
        uint16_t* out = p.out + tok * p.out_stride + hq * kHD + 4 * half;
#pragma unroll
        for (int mb = 0; mb < 4; ++mb)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<uint2*>(out + 32 * mb + 8 * i) = make_uint2(pack_bf16(st.o[0][mb][4 * i] * inv, st.o[0][mb][4 * i + 1] * inv),
                                                                              pack_bf16(st.o[0][mb][4 * i + 2] * inv, st.o[0][mb][4 * i + 3] * inv));
    } else {
        const int64_t at = pair * p.splits + it.split;
        float* out = p.ws_o + at * kHD + 4 * half;
#pragma unroll
        for (int mb = 0; mb < 4; ++mb)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float4*>(out + 32 * mb + 8 * i) =
                    make_float4(st.o[0][mb][4 * i], st.o[0][mb][4 * i + 1], st.o[0][mb][4 * i + 2], st.o[0][mb][4 * i + 3]);
        if (half == 0) *reinterpret_cast<float2*>(p.ws_ml + at * 2) = make_float2(st.m[0], l);
    }
}

// One run, up to 64 rows: tiles are private to a wave.  Measured: 64 requests of 8192 tokens x 8 nodes, 32 / 8 heads, 341 us = 6.3 TB/s, 0.89 of what a
// read-only stream reaches on this chip; with 16 nodes (two blocks of rows) 358 us.
template <int RB, bool NT>
__device__ __forceinline__ void narrow_run(const TreeParams& p, const TreeItem& it, int h, int wave, char* smem) {
    const int lane = fresh_lane();
    const int g4 = lane >> 4, q16 = lane & 15;
    const int all_tiles = (it.t1 - it.t0 + kTreeKeys - 1) / kTreeKeys;
    const int T = all_tiles > wave ? (all_tiles - wave + kTreeWaves - 1) / kTreeWaves : 0;  // own tiles: wave, wave + kTreeWaves, ...

    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
    constexpr int SL = tile_slots(RB), kRing = tree_ring(RB);
    constexpr int kParts = probability_parts(RB, NT);
    char* ring = smem + wave * kRing;
    char* words = smem + kTreeWaves * kRing + wave * kTreeSlotRing;
    const uint32_t ring_at = lds0 + wave * kRing;
    const uint32_t words_at = lds0 + kTreeWaves * kRing + wave * kTreeSlotRing;

    TreeState<RB> st;
    st.clear();
    uint64_t odd = 0;  // tiles behind the plain ones that held a value that is not finite
    const int plain = (max(0, (min(it.prefix, it.t1) - it.t0) / kTreeKeys - wave) + kTreeWaves - 1) / kTreeWaves;  // own tiles that every row sees whole
    if (T > 0) {
        const int32_t* table = it.table;
        // table entries of own tile j, lane (g4', i) <- key 4 i + g4' of the tile, so that a lane of the K/V loads finds its eight rows'
        // entries in 32 consecutive bytes.  Positions behind the run's last key repeat that key.
        const int word_key = 4 * (lane & 7) + ((lane >> 3) & 3);
        auto issue_words = [&](int j) {
            const int pos = min(it.t0 + (wave + j * kTreeWaves) * kTreeKeys + word_key, it.t1 - 1);
            dma_words((uint64_t)(table + pos), words_at + (j & 3) * 256);
        };
        issue_words(0);
        issue_words(1);
        issue_words(2);
        bf16x8_t qf[RB][8];
        load_queries<RB>(p, it, it.r0, h, lane, qf);
        wait_loads<0>();  // from here on the loads in flight are this kernel's to count

        // a lane loads piece q16 of rows 4 i + g4, so it fetches the piece that belongs there (read_keys, read_values)
        uint64_t kfrom[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) kfrom[i] = (uint64_t)(p.kc + h * kHD) + ((q16 ^ (4 * i + g4)) << 4);
        const uint64_t vfrom = (uint64_t)(p.vc + h * kHD) + ((q16 ^ (4 * g4)) << 4);
        auto issue_rows = [&](int j, bool values) {
            const int4 s0 = *reinterpret_cast<const int4*>(words + (j & 3) * 256 + g4 * 32), s1 = *reinterpret_cast<const int4*>(words + (j & 3) * 256 + g4 * 32 + 16);
            const uint32_t s[8] = {(uint32_t)s0.x, (uint32_t)s0.y, (uint32_t)s0.z, (uint32_t)s0.w, (uint32_t)s1.x, (uint32_t)s1.y, (uint32_t)s1.z, (uint32_t)s1.w};
            uint64_t a[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) a[i] = (uint64_t)s[i] * p.slot_bytes + (values ? vfrom : kfrom[i & 3]);
            dma_tile<NT>(a, ring_at + ((values ? SL : 0) + j % SL) * kTreeHalf);
        };
        issue_rows(0, false);
        issue_rows(0, true);
        if (SL == 2 && T > 1) {
            issue_words(3);
            issue_rows(1, false);
            issue_rows(1, true);
        }
        // two slots: outstanding behind K(j) are V(j), and if there is a next tile t(j+3), K(j+1), V(j+1); one slot: V(j)
        auto keys_of = [&](int j, f32x16_t (&s)[RB]) __attribute__((always_inline)) {
            if (SL == 2 && j + 1 < T) wait_loads<25>();
            else wait_loads<8>();
            bf16x8_t kf[8];
            read_keys(ring + j % SL * kTreeHalf, lane, kf);
            if (j + SL < T) {
                issue_words(j + SL + 2);
                issue_rows(j + SL, false);
            }
            tile_scores<RB>(kf, qf, s);
        };
        // two slots: outstanding behind V(j) are t(j+3), K(j+1), V(j+1), t(j+4), K(j+2); one slot: t(j+3), K(j+1)
        auto wait_values = [&](int j) __attribute__((always_inline)) {
            if (SL == 2 && j + 2 < T) wait_loads<26>();
            else if (j + 1 < T) wait_loads<SL == 2 ? 17 : 9>();
            else wait_loads<0>();
            return ring + (SL + j % SL) * kTreeHalf;
        };
        int j = 0;
        for (; j < plain; ++j) {
            f32x16_t s[RB];
            bf16x8_t pf[kParts][RB][2];
            keys_of(j, s);
            tile_reference<RB>(p.scale_log2e, s, st);
            tile_probabilities(p.scale_log2e, s, st, pf);
            tile_values(wait_values(j), lane, pf, st);
            if (j + SL < T) issue_rows(j + SL, true);
        }
        for (; j < T; ++j) {
            f32x16_t s[RB];
            bf16x8_t pf[kParts][RB][2];
            keys_of(j, s);
            uint64_t word[RB];  // (a wave has one such tile as a rule: asked for at the start, its mask would only make that longer)
            load_masks<RB>(p, it, it.r0, lane, word);
            tile_mask<RB>(p, it, it.r0, word, it.t0 + (wave + j * kTreeWaves) * kTreeKeys, lane, s);
            tile_reference<RB>(1.f, s, st);
            tile_probabilities(1.f, s, st, pf);
            if (tile_values_masked(wait_values(j), lane, pf, st)) odd |= 1ull << (j - plain);
            if (j + SL < T) issue_rows(j + SL, true);
        }
    }
    wait_loads<0>();
    join_and_store<RB, kTreeWaves, kTreeWaves>(p, it, st, smem, wave, lane, odd, it.t0 + (wave + plain * kTreeWaves) * kTreeKeys, kTreeWaves * kTreeKeys, [&](int) { return it.r0; },
                            [&](int) { return h; });
}
template <int RB, bool NT>
__global__ __launch_bounds__(kTreeWaves * 64, tile_slots(RB) == 1 ? 2 : 1) void tree_attention_kernel(TreeParams p) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const TreeBlock at(p);
    if (at.item >= p.items) return;
    const int r0 = at.row_tile * 32 * RB, h = at.item & (p.Hkv - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    TreeItem it;
    for (TreeWalk walk(p, at.item >> p.hkv_shift, r0, threadIdx.x & 63, it); walk.any; __syncthreads(), walk.next(p, r0, it))
        narrow_run<RB, NT>(p, it, h, wave, smem);
}

// The wide kernel, for more than 64 rows per kv head in large launches: the NW waves hold 32 rows each and share the tiles, so that K and V are read
// once per 32 NW rows.  A tile is loaded by all waves, 32 / NW keys each, SLOTS - 2 tiles ahead into a ring; a wave waits for its own loads of tile j,
// then the barrier says that everybody's have landed and that everybody is done with tile j - 2, whose slot is filled anew.  Two waves per SIMD either
// way (NW = 8 and one work group per compute unit, or NW = 4 and two): a wave issues an instruction about every eighth cycle, whatever it is, so one
// wave cannot keep softmax and matrix products side by side.  Measured: 32 requests of 16000 tokens x 64 nodes, 32 / 8 heads, 550 to 607 us = 980 to
// 890 TFLOP/s, K and V at 3.8 to 3.5 TB/s beside it (a dense product of 8192^3 reaches 1228 on this chip, whose clock gives way under such load);
// 40 requests of 4000 to 8000 x 15 to 30 nodes (four waves) 205 us = 4.8 TB/s, bound by the issue of its one wave per SIMD.
template <int NW>
struct TreeWide {
    static constexpr int kSlots = NW == 8 ? 8 : 4;
    static constexpr int kAhead = kSlots - 2;
    static constexpr int kKeys = kTreeKeys / NW;              // a wave's keys of a tile
    static constexpr int kLoads = kKeys / 4;                  // LDS-DMA loads of 4 rows for them, K and V each
    static constexpr int kBlock = 64 / kKeys;                 // tiles whose table entries one load brings
    static constexpr int kRing = kSlots * 2 * kTreeHalf;
    static constexpr int kTiles = kRing + NW * 2 * 256;       // two blocks of table entries per wave
    static constexpr int kLds = kTiles > merge_bytes(NW, 1) ? kTiles : merge_bytes(NW, 1);
    static_assert(kAhead <= kBlock - 1, "a block of table entries is refilled once its last tile has been requested");
};

// 4 rows x 256 bytes of K to 1 KiB at LDS byte address dst, and of V to the same place in the V half of the tile.
template <bool NT>
__device__ __forceinline__ void dma_rows4(uint64_t k, uint64_t v, uint32_t dst) {
    static_assert(kTreeHalf == 0x2000, "distance of the halves in the statement");
    unsigned keep;
    if (NT)
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off nt\n\ts_add_u32 m0, m0, 0x2000\n\ts_nop 0\n\t"
                     "global_load_lds_dwordx4 %3, off nt\n\ts_mov_b32 m0, %0"
                     : "=&s"(keep)
                     : "s"(dst), "v"(k), "v"(v)
                     : "memory", "scc");
    else
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off\n\ts_add_u32 m0, m0, 0x2000\n\ts_nop 0\n\t"
                     "global_load_lds_dwordx4 %3, off\n\ts_mov_b32 m0, %0"
                     : "=&s"(keep)
                     : "s"(dst), "v"(k), "v"(v)
                     : "memory", "scc");
}

// tame: long prefixes go through the steady state below, whose exponentials take one multiply-add each.  Where a row's reference then turns out to lie
// where tile_probabilities needs its two steps (or where a NaN says that it may have), nothing is stored, the result is false and the run is to be done
// again without.
template <int NW, bool NT>
__device__ __forceinline__ bool wide_run(const TreeParams& p, const TreeItem& it, int h, int wave, char* smem, bool tame) {
    using W = TreeWide<NW>;
    const int lane = fresh_lane();
    const int g4 = lane >> 4, q16 = lane & 15;
    const int row0 = it.r0 + wave * 32;
    const int T = (it.t1 - it.t0 + kTreeKeys - 1) / kTreeKeys;

    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
    char* words = smem + W::kRing + wave * 512;
    const uint32_t words_at = lds0 + W::kRing + wave * 512;
    const int32_t* table = it.table;
    // entry kKeys t + kLoads g4' + i of a block: key kKeys wave + 4 i + g4' of the block's tile t
    const int in_tile = lane % W::kKeys;
    const int word_key = lane / W::kKeys * kTreeKeys + W::kKeys * wave + 4 * (in_tile % W::kLoads) + in_tile / W::kLoads;
    auto issue_words = [&](int block) {
        const int pos = min(it.t0 + block * W::kBlock * kTreeKeys + word_key, it.t1 - 1);
        dma_words((uint64_t)(table + pos), words_at + (block & 1) * 256);
    };
    issue_words(0);
    issue_words(1);
    bf16x8_t qf[1][8];
    load_queries<1>(p, it, row0, h, lane, qf);
    uint64_t word[1];
    load_masks<1>(p, it, row0, lane, word);
    wait_loads<0>();
    uint64_t kfrom[W::kLoads];
#pragma unroll
    for (int i = 0; i < W::kLoads; ++i) kfrom[i] = (uint64_t)(p.kc + h * kHD) + ((q16 ^ ((W::kKeys * wave + 4 * i + g4) & 15)) << 4);
    const uint64_t vfrom = (uint64_t)(p.vc + h * kHD) + ((q16 ^ (4 * g4)) << 4);
    auto issue_tile = [&](int j) __attribute__((always_inline)) {
        const char* w = words + (j * W::kKeys * 4 & 511) + W::kLoads * g4 * 4;
        const uint32_t dst = lds0 + (j % W::kSlots) * 2 * kTreeHalf + wave * (W::kKeys * 256);
#pragma unroll
        for (int i = 0; i < W::kLoads; ++i) {
            const uint64_t o = (uint64_t)reinterpret_cast<const uint32_t*>(w)[i] * p.slot_bytes;
            dma_rows4<NT>(kfrom[i] + o, vfrom + o, dst + i * 1024);
        }
    };
    for (int j = 0; j < W::kAhead; ++j) issue_tile(j);

    TreeState<1> st;
    st.clear();
    uint64_t odd = 0;  // tiles behind the plain ones that held a value that is not finite
    // Tile j can be read after this.  Every call requests one tile more, behind the run's end the last key over and over, so that the count is
    // always the same (a table block among the loads only makes the wait stricter) and there is no branch.
    auto arrive = [&](int j) __attribute__((always_inline)) {
        wait_loads<2 * W::kLoads * (W::kAhead - 1)>();
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): what this wave has read of tile j - 2 is in registers
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");  // no read of the tile moves ahead of the barrier
        issue_tile(j + W::kAhead);
    };
    // the block of table entries whose last tile arrive(j) has requested is filled anew
    auto refill = [&](int j) __attribute__((always_inline)) {
        if ((j + W::kAhead + 1) % W::kBlock == 0) issue_words((j + W::kAhead) / W::kBlock + 2);
    };
    auto tile_at = [&](int j) { return smem + (j % W::kSlots) * 2 * kTreeHalf; };
    const int plain = max(0, min(it.prefix, it.t1) - it.t0) / kTreeKeys;  // tiles that every row sees whole
    int j = 0;
    if (row0 >= it.rows) {  // no rows for this wave: it loads and keeps the barriers
        for (; j < T; ++j) arrive(j), refill(j);
    } else if (tame && plain > 2) {
        // The steady state is one stream of 16 matrix instructions per tile, each a slice with its share of everything else:
        //   slices 0 .. 7     S^T of tile j + 1 (its K fragments are in registers); V^T fragments of tile j are read
        //   slices 8 .. 15    O^T of tile j; tile j + 2 arrives, its K fragments are read
        // and beside them the exponentials of tile j, sixteen in eleven slices, each pair packed the slice after, and over the last quarter the
        // maximum of the new scores.  A step is one basic block (a branch inside would let the compiler sink the exponentials behind it), and
        // four steps are unrolled: a tile's place in a 64 KiB half of the ring is then an immediate of the reads.
        f32x16_t sa[1], sb[1];
        bf16x8_t kf[8], vf[4][2], pf[1][1][2];
        float top[1];
        arrive(0);
        read_keys(tile_at(0), lane, kf);
        tile_scores<1>(kf, qf, sa);
        tile_reference<1>(p.scale_log2e, sa, st);
        arrive(1);
        refill(0), refill(1);
        read_keys(tile_at(1), lane, kf);
        typedef __attribute__((address_space(3))) char lds_char;
        uint32_t kat[8], vat[4];  // LDS addresses of the fragment reads in the ring's current half
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) kat[ks] = lds0 + (lane & 31) * 256 + (((2 * ks + (lane >> 5)) ^ (lane & 15)) << 4);
#pragma unroll
        for (int mb = 0; mb < 4; ++mb) {
            const int row = 4 * (lane >> 5) + (q16 >> 2);
            vat[mb] = lds0 + kTreeHalf + row * 256 + (((4 * mb + 2 * (g4 & 1) + ((q16 >> 1) & 1)) ^ (4 * (row & 3))) << 4) + (q16 & 1) * 8;
        }
        auto step = [&](int j, auto C, f32x16_t& s, f32x16_t& next) __attribute__((always_inline)) {
            constexpr uint32_t vimm = decltype(C)::value * 2 * kTreeHalf, kimm = ((decltype(C)::value + 2) & 3) * 2 * kTreeHalf;
            uint32_t pk[8];
            each<16>([&](auto K) __attribute__((always_inline)) {
                constexpr int k = K;
                if constexpr (k < 8) {
                    f32x16_t c;
                    if constexpr (k == 0) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) c[i] = 0.f;
                    } else {
                        c = next;
                    }
                    next = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[k], qf[0][k], c, 0, 0, 0);
                    short4_t x[2];
#pragma unroll
                    for (int pair = 0; pair < 2; ++pair)
                        x[pair] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) short4_t*)((lds_char*)(uintptr_t)vat[k & 3] + (vimm + (16 * (k >> 2) + 8 * pair) * 256)));
                    vf[k & 3][k >> 2] = __builtin_bit_cast(bf16x8_t, (short8_t){x[0][0], x[0][1], x[0][2], x[0][3], x[1][0], x[1][1], x[1][2], x[1][3]});
                } else {
                    constexpr int e = k - 8, ks = e / 4, mb = e % 4;
                    if constexpr (e == 0) arrive(j + 2);
                    st.o[0][mb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[mb][ks], pf[0][0][ks], st.o[0][mb], 0, 0, 0);
                    kf[e] = __builtin_bit_cast(bf16x8_t, *(const __attribute__((address_space(3))) u32x4_t*)((lds_char*)(uintptr_t)kat[e] + kimm));
                }
                // exponential i in slice 11 i / 16
                each<16>([&](auto U) __attribute__((always_inline)) {
                    constexpr int i = U;
                    if constexpr (i * 11 / 16 == k) s[i] = fast_exp2(__builtin_fmaf(s[i], p.scale_log2e, -st.m[0]));
                    if constexpr (i * 11 / 16 == k - 1) {
                        st.l[0] += s[i];
                        if constexpr (i % 2 == 1) pk[i / 2] = pack_bf16(s[i - 1], s[i]);
                        if constexpr (i == 7) pf[0][0][0] = as_bf16x8(make_uint4(pk[0], pk[1], pk[2], pk[3]));
                        if constexpr (i == 15) pf[0][0][1] = as_bf16x8(make_uint4(pk[4], pk[5], pk[6], pk[7]));
                    }
                });
                if constexpr (k >= 12) {  // (the last S^T instruction lies four matrix instructions back: its result is there)
                    constexpr int at = (k - 12) * 4;
                    top[0] = max3_raw(at == 0 ? next[0] : top[0], next[at], next[at + 1]);
                    top[0] = max3_raw(top[0], next[at + 2], next[at + 3]);
                }
                __builtin_amdgcn_sched_barrier(0);
            });
            follow_maximum<1>(p.scale_log2e, top, st);
            refill(j + 2);
            if constexpr (W::kSlots == 8 && decltype(C)::value == 1) {
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) kat[ks] ^= 8 * kTreeHalf;
            }
            if constexpr (W::kSlots == 8 && decltype(C)::value == 3) {
#pragma unroll
                for (int mb = 0; mb < 4; ++mb) vat[mb] ^= 8 * kTreeHalf;
            }
        };
        constexpr std::integral_constant<int, 0> c0{};
        constexpr std::integral_constant<int, 1> c1{};
        constexpr std::integral_constant<int, 2> c2{};
        constexpr std::integral_constant<int, 3> c3{};
        for (; j + 5 < plain; j += 4) {
            step(j, c0, sa[0], sb[0]);
            step(j + 1, c1, sb[0], sa[0]);
            step(j + 2, c2, sa[0], sb[0]);
            step(j + 3, c3, sb[0], sa[0]);
        }
        if (j + 2 < plain) {
            step(j, c0, sa[0], sb[0]);
            if (j + 3 < plain) {
                step(j + 1, c1, sb[0], sa[0]);
                if (j + 4 < plain) step(j + 2, c2, sa[0], sb[0]);
            }
        }
        if ((plain - 2 - j) & 1) sa[0] = sb[0];
        j = plain - 2;
        tile_probabilities(p.scale_log2e, sa, st, pf);
        tile_values(tile_at(j) + kTreeHalf, lane, pf, st);
        tile_scores<1>(kf, qf, sa);
        tile_reference<1>(p.scale_log2e, sa, st);
        tile_probabilities(p.scale_log2e, sa, st, pf);
        tile_values(tile_at(j + 1) + kTreeHalf, lane, pf, st);
        j = plain;
    }
    for (; j < T; ++j) {
        f32x16_t s[1];
        bf16x8_t kf[8], pf[1][1][2];
        arrive(j);
        refill(j);
        read_keys(tile_at(j), lane, kf);
        tile_scores<1>(kf, qf, s);
        float scale = p.scale_log2e;
        if (j >= plain) tile_mask<1>(p, it, row0, word, it.t0 + j * kTreeKeys, lane, s), scale = 1.f;
        tile_reference<1>(scale, s, st);
        tile_probabilities(scale, s, st, pf);
        if (j < plain) tile_values(tile_at(j) + kTreeHalf, lane, pf, st);
        else if (tile_values_masked(tile_at(j) + kTreeHalf, lane, pf, st)) odd |= 1ull << (j - plain);
    }
    wait_loads<0>();
    const bool wild = tame && plain > 2 && ((fabsf(st.m[0]) > kTameScore && st.m[0] != kLowestScore) || st.l[0] != st.l[0]);
    if (!__syncthreads_or(odd != 0 || wild)) {
        store_rows(p, it, st, row0, h, lane);
        return true;
    }
    if (__syncthreads_or(wild)) return false;
    join_and_store<1, 1, NW>(p, it, st, smem, wave, lane, odd, it.t0 + plain * kTreeKeys, kTreeKeys, [&](int g) { return it.r0 + g * 32; }, [&](int) { return h; });
    return true;
}
template <int NW, bool NT>
__global__ __launch_bounds__(NW * 64, 2) void tree_attention_wide_kernel(TreeParams p) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const TreeBlock at(p);
    if (at.item >= p.items) return;
    const int r0 = at.row_tile * 32 * NW, h = at.item & (p.Hkv - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    TreeItem it;
    bool tame = true;
    for (TreeWalk walk(p, at.item >> p.hkv_shift, r0, threadIdx.x & 63, it); walk.any; __syncthreads()) {
        tame = wide_run<NW, NT>(p, it, h, wave, smem, tame);
        if (tame) walk.next(p, r0, it);
    }
}

// Joins the runs of a (token, head): GROUPS half-waves per row take every GROUPS-th run, four dims per lane, and meet in LDS.
template <int GROUPS>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeParams p) {
    __shared__ float lds[8][kHD + 2];
    const int lane = threadIdx.x & 31, hw = threadIdx.x >> 5;
    const int g = hw % GROUPS;
    const int b = blockIdx.y;
    const int base = p.cu[b], n = min(p.cu[b + 1] - base, p.max_q);
    const int r = blockIdx.x * (8 / GROUPS) + hw / GROUPS;  // (node, head) pair of the request
    const int64_t pair = (int64_t)base * p.Hq + r;
    const int nsplit = r < n * p.Hq ? p.ws_n[pair] : 0;
    const bool live = nsplit > 1;  // (one run: written by the first kernel)
    const int64_t at = pair * p.splits;
    float M = kLowestScore, L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live) {
        for (int s0 = g; s0 < nsplit; s0 += 4 * GROUPS) {  // four runs' loads under way at a time
            float2 ml[4];
            float4 o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int s = min(s0 + k * GROUPS, nsplit - 1);
                ml[k] = *reinterpret_cast<const float2*>(p.ws_ml + (at + s) * 2);
                o[k] = *reinterpret_cast<const float4*>(p.ws_o + (at + s) * kHD + 4 * lane);
            }
            float top = M;
#pragma unroll
            for (int k = 0; k < 4; ++k) top = fmaxf(top, ml[k].x);
            const float f0 = fast_exp2(M - top);
            M = top;
            L *= f0, acc.x *= f0, acc.y *= f0, acc.z *= f0, acc.w *= f0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float f = s0 + k * GROUPS < nsplit ? fast_exp2(ml[k].x - M) : 0.f;
                L += f * ml[k].y;
                if (f != 0.f) acc.x += f * o[k].x, acc.y += f * o[k].y, acc.z += f * o[k].z, acc.w += f * o[k].w;
            }
        }
    }
    if (GROUPS > 1) {
        *reinterpret_cast<float2*>(&lds[hw][4 * lane]) = make_float2(acc.x, acc.y);
        *reinterpret_cast<float2*>(&lds[hw][4 * lane + 2]) = make_float2(acc.z, acc.w);
        if (lane == 0) lds[hw][kHD] = M, lds[hw][kHD + 1] = L;
        __syncthreads();
        if (g != 0) return;
        float top = kLowestScore;
#pragma unroll
        for (int k = 0; k < GROUPS; ++k) top = fmaxf(top, lds[hw + k][kHD]);
        L = 0.f;
        acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < GROUPS; ++k) {
            const float f = fast_exp2(lds[hw + k][kHD] - top);
            L += f * lds[hw + k][kHD + 1];
            acc.x += f * lds[hw + k][4 * lane], acc.y += f * lds[hw + k][4 * lane + 1];
            acc.z += f * lds[hw + k][4 * lane + 2], acc.w += f * lds[hw + k][4 * lane + 3];
        }
    }
    if (!live) return;
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    const int node = r >> p.hq_shift;
    *reinterpret_cast<uint2*>(p.out + (int64_t)(base + node) * p.out_stride + (r & (p.Hq - 1)) * kHD + 4 * lane) =
        make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
}

// Kernels that need more than the 64 KiB of LDS a kernel gets by default.
template <typename K>
static int launch_tree(K kernel, PerDeviceOnce& once, int lds, int waves, const TreeParams& p, int64_t blocks, hipStream_t stream) {
    if (!once.ensure([&] { return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds) == hipSuccess; })) {
        set_error("msgl_tree_attention: cannot reserve %d bytes of LDS", lds);
        return MSGL_E_LAUNCH;
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(waves * 64), lds, stream, p);
    return check_launch("tree_attention_kernel");
}
template <int RB, bool NT>
static int launch_narrow(const TreeParams& p, int64_t blocks, hipStream_t stream) {
    constexpr int kTiles = kTreeWaves * (tree_ring(RB) + kTreeSlotRing), kJoin = merge_bytes(kTreeWaves, RB);
    static PerDeviceOnce once;
    return launch_tree(&tree_attention_kernel<RB, NT>, once, kTiles > kJoin ? kTiles : kJoin, kTreeWaves, p, blocks, stream);
}
template <int NW, bool NT>
static int launch_wide(const TreeParams& p, int64_t blocks, hipStream_t stream) {
    static PerDeviceOnce once;
    return launch_tree(&tree_attention_wide_kernel<NW, NT>, once, TreeWide<NW>::kLds, NW, p, blocks, stream);
}

constexpr int kMaxTreeSplits = 256;
constexpr int kMostKeys = 1 << 30;  // keys of a request: positions plus a run stay inside 32 bits

// How a launch is laid out: the kernel (waves of the wide one, 0: the narrow one with rb blocks of 32 rows), its row tiles, work groups per
// (kv head, row tile), most runs of a request (1: a work group per request).
struct TreePlan {
    int waves, rb, row_tiles, shares, splits;
    double cost;  // ns
};
// The cost of a layout: a work group per request, or equal shares of all tiles, one per compute unit, whichever is done sooner, counted in tiles. A
// run costs its tiles and kTreeBegin for its start; a second kernel has to join shared requests, which is worth `join` tiles (4 to 8 us). Then
// the tiles' time, or the memory's (2.6 ns per tile of one kv head; narrow row tiles of an item drift apart and read most of it again).
// Measured, in us, work group per request | shares (two shares per unit where two work groups fit were slower: 12 requests of 8000 to 16000 x 30
// nodes, 32 / 8 heads, 126 instead of 112):
//   16 requests of 2000 to 4000 tokens x 16 nodes, 32 / 8 heads (128 work groups)      60 (equal runs of 1500 keys) | 47
//   12 of 8000 to 16000 x 30 (96)  138 (same) | 112      3 of 15000 to 30000 x 70, 16 / 4 heads (24)  124 (same) | 90
//   64 of 500 to 1000 x 8 (512)  44 | 55      48 of 4096 to 8192 x 8 (384)  243 | 207      32 of 250 to 500 x 60 (256)  34 | 41
//   1 of 1000 x 4, 16 / 8 heads (8)  15 | 20      1 of 2000 x 4 (8)  20 | 20      7 of 500 to 1000 x 4 (56)  17 | 19
static TreePlan tree_plan_of(int waves, int rb, int tile_ns, int64_t rows, int bs, int max_k, int64_t tiles, int Hkv) {
    const int64_t units = device_cus(), tile_rows = 32 * (waves ? waves : rb), row_tiles = (rows + tile_rows - 1) / tile_rows;
    // an XCD gets every eighth item, with all its row tiles
    const int64_t xcd_units = units >= 8 ? units / 8 : 1;
    const double load = (double)((((int64_t)bs * Hkv + 7) / 8) * row_tiles) / xcd_units;
    const int64_t most = ((int64_t)max_k + kTreeKeys - 1) / kTreeKeys, mean = (tiles + bs - 1) / bs, all = tiles + (int64_t)bs * kTreeBegin;
    const int64_t least = waves ? 6 : kLeastTiles, join = waves ? 6 : 28;
    int64_t shares = 8 * (xcd_units / row_tiles) / Hkv;
    if (shares < 1) shares = 1;
    if (shares > (all + least - 1) / least) shares = (all + least - 1) / least;
    const int64_t len = (all + shares - 1) / shares;
    const bool two_fit = waves == 4 || (waves == 0 && rb == 1);
    const double alone = load <= 1 ? kTreeBegin + most : (kTreeBegin + mean) * (two_fit ? load : ceil(load)) + most - mean;
    const double shared = (kTreeBegin + len) * (row_tiles > xcd_units ? (double)row_tiles / xcd_units : 1.0) + join;
    TreePlan t = {waves, rb, (int)row_tiles, bs, 1, alone * tile_ns};
    const int forced = variant(MSGL_VARIANT_TREE_SHARES);
    if (forced < 0 ? shared < alone : forced == 1) {
        const int64_t splits = (most + len - 1) / len + 1;
        t.shares = (int)shares, t.splits = (int)(splits < kMaxTreeSplits ? splits : kMaxTreeSplits), t.cost = shared * tile_ns;
    }
    const double memory = 2.6 * tiles * Hkv * (!waves && row_tiles > 1 ? 1.75 : 1.0) + kTreeBegin * tile_ns;
    if (t.cost < memory) t.cost = memory;
    return t;
}
// More than 32 rows per kv head: row tiles of 32 in the narrow kernel's smaller form, which starts soonest and fits twice on a compute unit, or the
// form that reads K and V once (64 rows) or once per 128 or 256 rows.  The tile times are those of the forms with enough to do. Measured with
// 32 / 8 heads, three sets of inputs in turn, us, row tiles of 32 | the other form:
//   requests x nodes    300 tokens    1000        4000        16000 (ragged: half to all of them)
//   1 x 16              13 | 15       14 | 21     18 | 21     21 | 28
//   16 x 16             13 | 16       16 | 24     59 | 48
//   1 x 60              13 | 22       15 | 25     20 | 32     43 | 43
//   4 x 60              13 | 23       16 | 30     35 | 41     130 | 68
//   16 x 60             25 | 25       37 | 41     112 | 73
//   100 x 30            73 | 42       130 | 81
static TreePlan tree_plan(int bs, int max_q, int max_k, int64_t total_kv, int Hq, int Hkv) {
    const TreePlan none = {0, 1, 1, bs, 1, 0};
    if (bs <= 0 || max_q <= 0 || max_k <= 0 || Hkv <= 0 || Hq < Hkv) return none;
    const int64_t rows = (int64_t)max_q * (Hq / Hkv);
    const int64_t tiles = total_kv > 0 && total_kv < (int64_t)bs * max_k ? total_kv / kTreeKeys + bs : bs * (((int64_t)max_k + kTreeKeys - 1) / kTreeKeys);
    auto of = [&](int waves, int rb, int tile_ns) { return tree_plan_of(waves, rb, tile_ns, rows, bs, max_k, tiles, Hkv); };
    TreePlan best = of(0, 1, 250);
    if (rows > 32) {
        const TreePlan other = rows <= 64 ? of(0, 2, 490) : rows <= 128 ? of(4, 1, 650) : of(8, 1, 1100);
        const int forced = variant(MSGL_VARIANT_TREE_FORM);
        if (forced < 0 ? other.cost <= best.cost : forced == 1) best = other;
    }
    if (bs > 65535) best.shares = bs, best.splits = 1;
    return best;
}

}  // namespace msgl

using namespace msgl;

extern "C" int msgl_tree_attention_splits(int bs, int max_seqlen_q, int max_seqlen_k, int64_t total_kv, int Hq, int Hkv) {
    return tree_plan(bs, max_seqlen_q, max_seqlen_k, total_kv, Hq, Hkv).splits;
}
extern "C" size_t msgl_tree_attention_workspace_bytes(int64_t total_tokens, int Hq, int D, int splits) {
    if (total_tokens <= 0 || Hq <= 0 || D <= 0 || splits <= 1) return 0;
    return (size_t)total_tokens * Hq * ((size_t)splits * (D + 2) + 1) * sizeof(float);
}

extern "C" int msgl_tree_attention(const void* q, int64_t q_stride, const void* k_cache, const void* v_cache, int64_t cache_stride,
                                   const int32_t* req_to_token, int64_t r2t_stride, const int32_t* req_pool_indices, const int32_t* cu_seqlens_q,
                                   const int32_t* prefix_lens, const uint64_t* tree_mask, int mask_words, void* out, int64_t out_stride,
                                   int64_t total_tokens, int bs, int max_seqlen_q, int max_seqlen_k, int64_t total_kv, int Hq, int Hkv, int D, float scale,
                                   void* workspace, size_t workspace_bytes, void* stream) {
    MSGL_REQUIRE(D == kHD, "msgl_tree_attention: head dim %d unsupported (built for %d)", D, kHD);
    MSGL_REQUIRE(Hkv >= 1 && Hkv <= 8 && (Hkv & (Hkv - 1)) == 0 && Hq % Hkv == 0 && (Hq / Hkv == 1 || Hq / Hkv == 2 || Hq / Hkv == 4 || Hq / Hkv == 8),
                 "msgl_tree_attention: %d query / %d kv heads unsupported", Hq, Hkv);
    MSGL_REQUIRE(bs >= 0 && total_tokens >= 0 && total_tokens <= 0x7fffffff && max_seqlen_q >= 0 && max_seqlen_k >= 0,
                 "msgl_tree_attention: bs=%d total_tokens=%lld max_seqlen_q=%d max_seqlen_k=%d", bs, (long long)total_tokens, max_seqlen_q, max_seqlen_k);
    if (bs == 0 || total_tokens == 0 || max_seqlen_q == 0) return MSGL_OK;
    MSGL_REQUIRE(mask_words >= 1 && mask_words <= MSGL_TREE_MAX_WORDS && max_seqlen_q <= 64 * mask_words,
                 "msgl_tree_attention: %d mask words for up to %d nodes (at most %d words)", mask_words, max_seqlen_q, MSGL_TREE_MAX_WORDS);
    MSGL_REQUIRE(max_seqlen_k >= 1 && max_seqlen_k <= kMostKeys, "msgl_tree_attention: max_seqlen_k %d outside 1..%d", max_seqlen_k, kMostKeys);
    MSGL_REQUIRE(q && k_cache && v_cache && req_to_token && req_pool_indices && cu_seqlens_q && prefix_lens && tree_mask && out,
                 "msgl_tree_attention: null pointer argument");
    MSGL_REQUIRE(scale >= 0.f && scale <= 1.0e38f, "msgl_tree_attention: scale must be in 0..1e38");
    MSGL_REQUIRE(q != out, "msgl_tree_attention: out overwrites q");
    MSGL_REQUIRE(q_stride >= 0 && out_stride >= (int64_t)Hq * D, "msgl_tree_attention: q_stride %lld, out_stride %lld (rows of %d elements)",
                 (long long)q_stride, (long long)out_stride, Hq * D);
    MSGL_REQUIRE(aligned16(q) && aligned16(k_cache) && aligned16(v_cache) && aligned16(out) && q_stride % 8 == 0 && out_stride % 8 == 0 && cache_stride % 8 == 0,
                 "msgl_tree_attention: tensors must be 16-byte aligned with strides in multiples of 8");
    MSGL_REQUIRE(cache_stride >= (int64_t)Hkv * D && cache_stride <= 0x7fffffff, "msgl_tree_attention: cache_stride %lld", (long long)cache_stride);
    TreeParams p;
    p.q = static_cast<const uint16_t*>(q), p.q_stride = q_stride;
    p.kc = static_cast<const uint16_t*>(k_cache), p.vc = static_cast<const uint16_t*>(v_cache), p.slot_bytes = (uint32_t)(cache_stride * 2);
    p.r2t = req_to_token, p.r2t_stride = r2t_stride, p.req_idx = req_pool_indices, p.cu = cu_seqlens_q, p.prefix = prefix_lens;
    p.mask = tree_mask, p.words = mask_words;
    p.out = static_cast<uint16_t*>(out), p.out_stride = out_stride;
    p.bs = bs, p.Hq = Hq, p.Hkv = Hkv, p.group = Hq / Hkv, p.max_q = max_seqlen_q;
    p.hq_shift = __builtin_ctz(Hq), p.hkv_shift = __builtin_ctz(Hkv), p.group_shift = __builtin_ctz(Hq / Hkv);
    TreePlan plan = tree_plan(bs, max_seqlen_q, max_seqlen_k, total_kv, Hq, Hkv);
    p.row_tiles = plan.row_tiles;
    p.scale_log2e = scale * 1.44269504088896340736f;
    if (plan.splits > 1) {  // as many runs as the workspace has room for
        const size_t per_row = workspace ? workspace_bytes / sizeof(float) / ((size_t)total_tokens * Hq) : 0;
        const size_t room = per_row ? (per_row - 1) / (D + 2) : 0;
        if ((size_t)plan.splits > room) plan.splits = (int)room;
        if (plan.splits < 2) plan.splits = 1, plan.shares = bs;
    }
    const int splits = plan.splits;
    p.splits = splits, p.shares = plan.shares;
    p.ws_o = static_cast<float*>(workspace);
    p.ws_ml = p.ws_o + (splits > 1 ? (size_t)total_tokens * Hq * splits * kHD : 0);
    p.ws_n = reinterpret_cast<int32_t*>(p.ws_ml + (splits > 1 ? (size_t)total_tokens * Hq * splits * 2 : 0));
    MSGL_REQUIRE(splits == 1 || aligned16(workspace), "msgl_tree_attention: workspace must be 16-byte aligned");
    const uint64_t tokens = (uint64_t)total_tokens, row = 2 * (uint64_t)Hq * D;  // work groups read while others write
    const Span inputs[] = {{q, row, tokens, 2 * (uint64_t)q_stride}, {req_pool_indices, 4 * (uint64_t)bs}, {cu_seqlens_q, 4 * (uint64_t)bs + 4},
                           {prefix_lens, 4 * (uint64_t)bs}, {tree_mask, 8 * tokens * (uint64_t)mask_words}};
    const Span result = {out, row, tokens, 2 * (uint64_t)out_stride}, runs = {workspace, splits > 1 ? msgl_tree_attention_workspace_bytes(total_tokens, Hq, D, splits) : 0};
    for (const Span& in : inputs) MSGL_REQUIRE(!spans_meet(in, result) && !spans_meet(in, runs), "msgl_tree_attention: an output or the workspace overwrites an input");
    MSGL_REQUIRE(!spans_meet(result, runs), "msgl_tree_attention: the workspace overwrites out");
    const int64_t items = (int64_t)plan.shares * Hkv;
    const int64_t blocks = (items + 7) / 8 * 8 * p.row_tiles;
    MSGL_REQUIRE(blocks <= 0x7fffff, "msgl_tree_attention: %lld work groups", (long long)blocks);
    p.items = (int)items;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const bool once = p.row_tiles == 1;  // K and V are read by one work group: past the caches
    int rc;
    if (plan.waves == 8) rc = once ? launch_wide<8, true>(p, blocks, st) : launch_wide<8, false>(p, blocks, st);
    else if (plan.waves == 4) rc = launch_wide<4, true>(p, blocks, st);
    else if (plan.rb == 2) rc = launch_narrow<2, true>(p, blocks, st);
    else rc = once ? launch_narrow<1, true>(p, blocks, st) : launch_narrow<1, false>(p, blocks, st);
    if (rc != MSGL_OK || splits == 1) return rc;
    // half-waves per row: as many as there are runs for, up to eight
    const unsigned rows = (unsigned)max_seqlen_q * Hq;
    if (splits <= 8) hipLaunchKernelGGL(tree_merge_kernel<1>, dim3((rows + 7) / 8, bs), dim3(256), 0, st, p);
    else if (splits <= 32) hipLaunchKernelGGL(tree_merge_kernel<4>, dim3((rows + 1) / 2, bs), dim3(256), 0, st, p);
    else hipLaunchKernelGGL(tree_merge_kernel<8>, dim3(rows, bs), dim3(256), 0, st, p);
    return check_launch("tree_merge_kernel");
}
