// Attention of drafted token trees over the paged cache (verification of a speculative step).
//
//   out[i, h] = softmax_j(scale q_ih . k_j) v_j   over the cached prefix and those nodes of the request's own tree that node i's
//   mask names; a row that sees nothing gives zeros.
//
// All nodes of a request read the same keys, so they are rows of one matrix product: the (node, head of the GQA group) pairs of a kv
// head, packed node after node, 32 to a block.  S^T = K.Q^T and O^T += V^T.P^T on v_mfma_f32_32x32x16_bf16: the row sits on the lane in
// both products (lane & 31), so maximum, sum and rescaling are in-lane plus one swap of lane halves, and the exponentiated scores,
// packed to bf16, are the second product's operand as they stand.  (P is rounded to bf16 as that product's operand type asks: half a
// step, 2^-9 relative, per probability, unbiased, and the sum is taken of the unrounded ones.)
//
// With up to 64 rows per kv head the pass over K and V bounds the kernel (a 32-key tile costs a wave 512 matrix cycles per 32 rows
// where HBM takes 1250 cycles of the compute unit).  The work group's four waves take every fourth 32-key tile each, with RB blocks of
// 32 rows: tiles are private to a wave, so the loop has no barrier.
//   * K and V rows go from HBM to LDS without passing registers, 16 bytes a lane, four rows of 256 bytes an instruction, into two tile
//     slots per wave; the XOR swizzles that spread the fragment reads over the banks are applied to the source address.
//   * The page table is read per token, also by LDS-DMA, four tiles ahead: any page size, no scalar path, nothing the compiler counts.
//   * All these loads are inline asm and waited for by count; their order is K0 V0 t3 K1 V1 | t4 K2 V2 | t5 K3 V3 ... (t = table entries).
// Long contexts are cut into runs of keys (one work group each) that leave (O, max, sum) in the workspace; a second kernel joins them.
#include "msgl_common.h"
#include "extend_common.h"

namespace msgl {

constexpr int kTreeWaves = 4;
constexpr int kTreeKeys = 32;                       // keys per tile
constexpr int kTreeHalf = kTreeKeys * kHD * 2;      // bytes of a K or V tile
constexpr int kTreeRing = 4 * kTreeHalf;            // per wave: two K tiles, two V tiles
constexpr int kTreeSlotRing = 4 * 256;              // per wave: table entries of four tiles (64 words each)
constexpr int kTreeLds = kTreeWaves * (kTreeRing + kTreeSlotRing);
constexpr int kTreeMergeRow = kHD + 4;              // floats per row of the exchange at the end (spread over the banks)
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
    int Hq, Hkv, group;
    int row_tiles, splits, chunk;
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

template <int RB, bool NT>
__global__ __launch_bounds__(kTreeWaves * 64, 1) void tree_attention_kernel(TreeParams p) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    // block -> (row tile, kv head, request, run of keys), row tile fastest
    int id = blockIdx.x;
    const int rt = id % p.row_tiles;
    id /= p.row_tiles;
    const int h = id % p.Hkv;
    id /= p.Hkv;
    const int split = id % p.splits;
    const int b = id / p.splits;
    const int base = p.cu[b];
    const int n = min(p.cu[b + 1] - base, p.max_q);
    const int G = p.group;
    const int rows = n * G;
    const int r0 = rt * 32 * RB;
    if (r0 >= rows) return;
    const int prefix = p.prefix[b];
    const int S = prefix + n;
    const int nsplit = min((S + p.chunk - 1) / p.chunk, p.splits);
    if (split >= nsplit) return;
    const int t0 = split * p.chunk;
    const int t1 = split == p.splits - 1 ? S : min(S, t0 + p.chunk);

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int half = lane >> 5, col = lane & 31;
    const int g4 = lane >> 4, q16 = lane & 15;
    const int all_tiles = (t1 - t0 + kTreeKeys - 1) / kTreeKeys;
    const int T = all_tiles > wave ? (all_tiles - wave + kTreeWaves - 1) / kTreeWaves : 0;  // own tiles: wave, wave + 4, ...

    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
    char* ring = smem + wave * kTreeRing;
    char* words = smem + kTreeWaves * kTreeRing + wave * kTreeSlotRing;
    const uint32_t ring_at = lds0 + wave * kTreeRing;
    const uint32_t words_at = lds0 + kTreeWaves * kTreeRing + wave * kTreeSlotRing;

    f32x16_t o[RB][4];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int mb = 0; mb < 4; ++mb)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[rb][mb][i] = 0.f;
    float m[RB], l[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) m[rb] = kNegBigE, l[rb] = 0.f;

    if (T > 0) {
        const int32_t* table = p.r2t + (int64_t)p.req_idx[b] * p.r2t_stride;
        // table entries of own tile j, lane (g4', i) <- key 4 i + g4' of the tile, so that a lane of the K/V loads finds its eight rows'
        // entries in 32 consecutive bytes.  Positions behind the run's last key repeat that key.
        const int word_key = 4 * (lane & 7) + ((lane >> 3) & 3);
        auto issue_words = [&](int j) {
            const int pos = min(t0 + (wave + j * kTreeWaves) * kTreeKeys + word_key, t1 - 1);
            dma_words((uint64_t)(table + pos), words_at + (j & 3) * 256);
        };
        issue_words(0);
        issue_words(1);
        issue_words(2);
        // Q^T fragments: lane (row col, half) holds dims 16 ks + 8 half .. + 8.  Rows behind the last one repeat it; they are not stored.
        bf16x8_t qf[RB][8];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const int r = min(r0 + rb * 32 + col, rows - 1);
            const int node = r / G;
            const uint16_t* qp = p.q + (int64_t)(base + node) * p.q_stride + (h * G + r - node * G) * kHD + half * 8;
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) qf[rb][ks] = as_bf16x8(*reinterpret_cast<const uint4*>(qp + ks * 16));
        }
        // everything so far has arrived, the query in registers: from here on the loads in flight are this kernel's to count
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) asm volatile("" : "+v"(qf[rb][ks]));
        wait_loads<0>();

        // K rows: 16-byte piece c of row r lies at piece c ^ (r & 15); V rows: at piece c ^ 4 (r & 3).  A lane loads piece q16 of rows
        // 4 i + g4, so it fetches the piece that belongs there.
        uint64_t kfrom[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) kfrom[i] = (uint64_t)(p.kc + h * kHD) + ((q16 ^ (4 * i + g4)) << 4);
        const uint64_t vfrom = (uint64_t)(p.vc + h * kHD) + ((q16 ^ (4 * g4)) << 4);
        auto issue_k = [&](int j) {
            const int4 s0 = *reinterpret_cast<const int4*>(words + (j & 3) * 256 + g4 * 32), s1 = *reinterpret_cast<const int4*>(words + (j & 3) * 256 + g4 * 32 + 16);
            const uint32_t s[8] = {(uint32_t)s0.x, (uint32_t)s0.y, (uint32_t)s0.z, (uint32_t)s0.w, (uint32_t)s1.x, (uint32_t)s1.y, (uint32_t)s1.z, (uint32_t)s1.w};
            uint64_t a[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) a[i] = (uint64_t)s[i] * p.slot_bytes + kfrom[i & 3];
            dma_tile<NT>(a, ring_at + (j & 1) * kTreeHalf);
        };
        auto issue_v = [&](int j) {
            const int4 s0 = *reinterpret_cast<const int4*>(words + (j & 3) * 256 + g4 * 32), s1 = *reinterpret_cast<const int4*>(words + (j & 3) * 256 + g4 * 32 + 16);
            const uint32_t s[8] = {(uint32_t)s0.x, (uint32_t)s0.y, (uint32_t)s0.z, (uint32_t)s0.w, (uint32_t)s1.x, (uint32_t)s1.y, (uint32_t)s1.z, (uint32_t)s1.w};
            uint64_t a[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) a[i] = (uint64_t)s[i] * p.slot_bytes + vfrom;
            dma_tile<NT>(a, ring_at + (2 + (j & 1)) * kTreeHalf);
        };
        issue_k(0);
        issue_v(0);
        if (T > 1) {
            issue_words(3);
            issue_k(1);
            issue_v(1);
        }
        // LDS offsets of the fragment reads: K row col, piece (2 ks + half) ^ (col & 15); V^T: the 16 lanes of a group name 4 rows x 32
        // bytes and receive one dim each of those 4 rows: rows 16 s + 8 pair + 4 half + (q16 >> 2), dims 32 mb + 16 (g4 & 1) + q16.
        const uint32_t kread = (uint32_t)col * 256, kswz = (uint32_t)(col & 15);
        const uint32_t vrow = 4 * half + (q16 >> 2);
        const uint32_t vread = vrow * 256 + (q16 & 1) * 8;
        const uint32_t vpiece = 2 * (g4 & 1) + ((q16 >> 1) & 1), vswz = 4 * (vrow & 3);

        for (int j = 0; j < T; ++j) {
            const bool more = j + 2 < T, next = j + 1 < T;
            // outstanding behind K(j): V(j), and if there is a next tile t(j+3), K(j+1), V(j+1)
            if (next) wait_loads<25>();
            else wait_loads<8>();
            const char* kt = ring + (j & 1) * kTreeHalf;
            bf16x8_t kf[8];
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) kf[ks] = as_bf16x8(*reinterpret_cast<const uint4*>(kt + kread + (((2 * ks + half) ^ kswz) << 4)));
            if (more) {
                issue_words(j + 4);
                issue_k(j + 2);
            }
            f32x16_t s[RB];
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
                for (int i = 0; i < 16; ++i) s[rb][i] = 0.f;
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) s[rb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[ks], qf[rb][ks], s[rb], 0, 0, 0);
            }
            // s[rb][i]: key 8 (i >> 2) + 4 half + (i & 3) of the tile, row col of the block
            const int key0 = t0 + (wave + j * kTreeWaves) * kTreeKeys;
            const bool masked = key0 + kTreeKeys > min(prefix, t1);
            uint32_t see[RB];
            if (masked) {
                const int rel = key0 - prefix;
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    const int node = min(r0 + rb * 32 + col, rows - 1) / G;
                    const uint64_t* row = p.mask + (int64_t)(base + node) * p.words;
                    uint32_t bits = rel >= 0 ? mask_bits(row, p.words, rel) : rel <= -32 ? ~0u : (mask_bits(row, p.words, 0) << -rel) | ((1u << -rel) - 1);
                    if (key0 + kTreeKeys > t1) bits &= (1u << (t1 - key0)) - 1;
                    see[rb] = bits;
                    bits >>= 4 * half;
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (!(bits >> (8 * (i >> 2) + (i & 3)) & 1)) s[rb][i] = -INFINITY;
                }
            }
            bf16x8_t pf[RB][2];
            float pr[RB][16];
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                float top = s[rb][0];
#pragma unroll
                for (int i = 1; i < 16; ++i) top = fmaxf(top, s[rb][i]);
                top = fmaxf(top, __shfl_xor(top, 32)) * p.scale_log2e;
                // the reference follows the maximum when that has outgrown it by 2^8, or is the first: probabilities up to 2^8 are as exact
                if (__any(top > m[rb] + kRescaleAt)) {
                    const float mn = fmaxf(m[rb], top);
                    const float f = fast_exp2(m[rb] - mn);
                    m[rb] = mn;
                    l[rb] *= f;
#pragma unroll
                    for (int mb = 0; mb < 4; ++mb)
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[rb][mb][i] *= f;
                }
                uint32_t w[8];
#pragma unroll
                for (int i = 0; i < 16; ++i) pr[rb][i] = fast_exp2(__builtin_fmaf(s[rb][i], p.scale_log2e, -m[rb]));
#pragma unroll
                for (int i = 0; i < 16; ++i) l[rb] += pr[rb][i];
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = pack_bf16(pr[rb][2 * i], pr[rb][2 * i + 1]);
                pf[rb][0] = as_bf16x8(make_uint4(w[0], w[1], w[2], w[3]));
                pf[rb][1] = as_bf16x8(make_uint4(w[4], w[5], w[6], w[7]));
            }
            // outstanding behind V(j): t(j+3), K(j+1), V(j+1), t(j+4), K(j+2)
            if (more) wait_loads<26>();
            else if (next) wait_loads<17>();
            else wait_loads<0>();
            const char* vt = ring + (2 + (j & 1)) * kTreeHalf;
            bf16x8_t vf[4][2];
#pragma unroll
            for (int mb = 0; mb < 4; ++mb)
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    short4_t x[2];
#pragma unroll
                    for (int pair = 0; pair < 2; ++pair)
                        x[pair] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(
                            vt + (16 * ks + 8 * pair) * 256 + vread + (((4 * mb + vpiece) ^ vswz) << 4)));
                    vf[mb][ks] = __builtin_bit_cast(bf16x8_t, (short8_t){x[0][0], x[0][1], x[0][2], x[0][3], x[1][0], x[1][1], x[1][2], x[1][3]});
                }
            // In a tile with hidden keys a row must not touch what it does not see: 0 * NaN and 0 * inf are NaN.  If such a value is in the
            // tile (a branch of the tree that went wrong), its products are taken key by key, by those rows that see the key.
            bool plain = true;
            if (masked) {
                bool odd = false;
#pragma unroll
                for (int mb = 0; mb < 4; ++mb)
#pragma unroll
                    for (int ks = 0; ks < 2; ++ks) {
                        const uint4 x = __builtin_bit_cast(uint4, vf[mb][ks]);
                        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) odd |= (w[i] & 0x7f80u) == 0x7f80u || (w[i] & 0x7f800000u) == 0x7f800000u;
                    }
                plain = !__any(odd);
            }
            if (plain) {
                if (more) issue_v(j + 2);
#pragma unroll
                for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                    for (int mb = 0; mb < 4; ++mb)
#pragma unroll
                        for (int ks = 0; ks < 2; ++ks) o[rb][mb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[mb][ks], pf[rb][ks], o[rb][mb], 0, 0, 0);
            } else {
#pragma unroll
                for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
#pragma unroll 1
                        for (int hh = 0; hh < 2; ++hh) {
                            const int key = 8 * (i >> 2) + 4 * hh + (i & 3);
                            const float pk = __shfl(pr[rb][i], col + 32 * hh);
                            if (see[rb] >> key & 1) {
                                const char* vr = vt + key * 256;
#pragma unroll
                                for (int mb = 0; mb < 4; ++mb)
#pragma unroll
                                    for (int d = 0; d < 16; ++d) {
                                        const int dim = 32 * mb + 8 * (d >> 2) + 4 * half + (d & 3);
                                        const uint16_t x = *reinterpret_cast<const uint16_t*>(vr + (((dim >> 3) ^ (4 * (key & 3))) << 4) + (dim & 7) * 2);
                                        o[rb][mb][d] += pk * bf16_lo(x);
                                    }
                            }
                        }
                if (more) issue_v(j + 2);
            }
        }
    }
    wait_loads<0>();
    // the waves' states, joined: O^T has dims 32 mb + 8 (i >> 2) + 4 half + (i & 3) in register i of block mb
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) l[rb] += __shfl_xor(l[rb], 32);
    __syncthreads();  // every wave is done with its ring
    float* lds_o = reinterpret_cast<float*>(smem);                              // [wave][row][kTreeMergeRow]
    float* lds_ml = lds_o + kTreeWaves * 32 * RB * kTreeMergeRow;               // [wave][row][2]
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        float* dst = lds_o + (wave * 32 * RB + rb * 32 + col) * kTreeMergeRow + 4 * half;
#pragma unroll
        for (int mb = 0; mb < 4; ++mb)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float4*>(dst + 32 * mb + 8 * i) = make_float4(o[rb][mb][4 * i], o[rb][mb][4 * i + 1], o[rb][mb][4 * i + 2], o[rb][mb][4 * i + 3]);
        if (half == 0) {
            lds_ml[(wave * 32 * RB + rb * 32 + col) * 2] = m[rb];
            lds_ml[(wave * 32 * RB + rb * 32 + col) * 2 + 1] = l[rb];
        }
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < 32 * RB * 32; idx += kTreeWaves * 64) {
        const int r = idx >> 5, d = (idx & 31) * 4;
        if (r0 + r >= rows) break;
        float M = kNegBigE;
#pragma unroll
        for (int w = 0; w < kTreeWaves; ++w) M = fmaxf(M, lds_ml[(w * 32 * RB + r) * 2]);
        float L = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kTreeWaves; ++w) {
            const float f = fast_exp2(lds_ml[(w * 32 * RB + r) * 2] - M);
            L += f * lds_ml[(w * 32 * RB + r) * 2 + 1];
            const float4 x = *reinterpret_cast<const float4*>(lds_o + (w * 32 * RB + r) * kTreeMergeRow + d);
            acc.x += f * x.x, acc.y += f * x.y, acc.z += f * x.z, acc.w += f * x.w;
        }
        const int node = (r0 + r) / G;
        const int hq = h * G + (r0 + r) - node * G;
        const int64_t tok = base + node;
        if (nsplit == 1) {
            const float inv = L == 0.f ? 0.f : 1.0f / L;  // L == 0: the row sees nothing
            *reinterpret_cast<uint2*>(p.out + tok * p.out_stride + hq * kHD + d) = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
        } else {
            const int64_t at = (tok * p.Hq + hq) * p.splits + split;
            *reinterpret_cast<float4*>(p.ws_o + at * kHD + d) = acc;
            if (d == 0) *reinterpret_cast<float2*>(p.ws_ml + at * 2) = make_float2(M, L);
        }
    }
}

// Joins the runs of one (token, head) per wave: two dims per lane.
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeParams p) {
    const int lane = threadIdx.x & 63;
    const int per = p.max_q * p.Hq;  // (node, head) pairs of a request
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int b = (int)(id / per);
    const int r = (int)(id - (int64_t)b * per);
    const int base = p.cu[b];
    const int n = min(p.cu[b + 1] - base, p.max_q);
    const int node = r / p.Hq, hq = r - node * p.Hq;
    if (node >= n) return;
    const int S = p.prefix[b] + n;
    const int nsplit = min((S + p.chunk - 1) / p.chunk, p.splits);
    if (nsplit <= 1) return;  // written by the first kernel
    const int64_t at = ((int64_t)(base + node) * p.Hq + hq) * p.splits;
    float M = kNegBigE;
    for (int s = lane; s < nsplit; s += 64) M = fmaxf(M, p.ws_ml[(at + s) * 2]);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) M = fmaxf(M, __shfl_xor(M, d));
    float L = 0.f, o0 = 0.f, o1 = 0.f;
    for (int s = 0; s < nsplit; ++s) {
        const float2 ml = *reinterpret_cast<const float2*>(p.ws_ml + (at + s) * 2);
        const float2 o = *reinterpret_cast<const float2*>(p.ws_o + (at + s) * kHD + 2 * lane);
        const float f = fast_exp2(ml.x - M);
        L += f * ml.y;
        o0 += f * o.x, o1 += f * o.y;
    }
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    *reinterpret_cast<uint32_t*>(p.out + (int64_t)(base + node) * p.out_stride + hq * kHD + 2 * lane) = pack_bf16(o0 * inv, o1 * inv);
}

template <int RB, bool NT>
static int launch_tree(const TreeParams& p, int64_t blocks, hipStream_t stream) {
    constexpr int kMerge = kTreeWaves * 32 * RB * (kTreeMergeRow + 2) * 4;
    constexpr int kLds = kTreeLds > kMerge ? kTreeLds : kMerge;
    static PerDeviceOnce once;  // more than the 64 KiB a kernel gets by default
    if (!once.ensure([] {
            return hipFuncSetAttribute(reinterpret_cast<const void*>(tree_attention_kernel<RB, NT>), hipFuncAttributeMaxDynamicSharedMemorySize, kLds) ==
                   hipSuccess;
        })) {
        set_error("msgl_tree_attention: cannot reserve %d bytes of LDS", kLds);
        return MSGL_E_LAUNCH;
    }
    hipLaunchKernelGGL((tree_attention_kernel<RB, NT>), dim3((unsigned)blocks), dim3(kTreeWaves * 64), kLds, stream, p);
    return check_launch("tree_attention_kernel");
}

constexpr int kMaxTreeSplits = 256;

static int tree_row_tiles(int max_q, int group) {
    const int rows = max_q * group;
    return (rows + 63) / 64;  // blocks of 32 rows, two to a work group where there are two
}

// Runs of keys per request: enough work groups for the chip, each at least four tiles (one per wave) long.
static int tree_splits(int bs, int max_q, int max_k, int64_t total_kv, int Hq, int Hkv) {
    if (bs <= 0 || max_q <= 0 || max_k <= 0 || Hkv <= 0 || Hq < Hkv) return 1;
    const int64_t keys = total_kv > 0 && total_kv < (int64_t)bs * max_k ? total_kv : (int64_t)bs * max_k;
    const int64_t per_key = (int64_t)Hkv * tree_row_tiles(max_q, Hq / Hkv);
    const int64_t want = 2 * (int64_t)device_cus();
    int64_t chunk = (keys * per_key + want - 1) / want;
    if (chunk < kTreeKeys * kTreeWaves) chunk = kTreeKeys * kTreeWaves;
    int64_t splits = (max_k + chunk - 1) / chunk;
    return (int)(splits < kMaxTreeSplits ? splits : kMaxTreeSplits);
}

}  // namespace msgl

using namespace msgl;

extern "C" int msgl_tree_attention_splits(int bs, int max_seqlen_q, int max_seqlen_k, int64_t total_kv, int Hq, int Hkv) {
    return tree_splits(bs, max_seqlen_q, max_seqlen_k, total_kv, Hq, Hkv);
}
extern "C" size_t msgl_tree_attention_workspace_bytes(int64_t total_tokens, int Hq, int D, int splits) {
    if (total_tokens <= 0 || Hq <= 0 || D <= 0 || splits <= 1) return 0;
    return (size_t)total_tokens * Hq * splits * (D + 2) * sizeof(float);
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
    MSGL_REQUIRE(max_seqlen_k >= 1, "msgl_tree_attention: max_seqlen_k %d", max_seqlen_k);
    MSGL_REQUIRE(q && k_cache && v_cache && req_to_token && req_pool_indices && cu_seqlens_q && prefix_lens && tree_mask && out,
                 "msgl_tree_attention: null pointer argument");
    MSGL_REQUIRE(scale >= 0.f && scale <= 3.0e38f, "msgl_tree_attention: scale must be finite and not negative");
    MSGL_REQUIRE(aligned16(q) && aligned16(k_cache) && aligned16(v_cache) && aligned16(out) && q_stride % 8 == 0 && out_stride % 8 == 0 && cache_stride % 8 == 0,
                 "msgl_tree_attention: tensors must be 16-byte aligned with strides in multiples of 8");
    MSGL_REQUIRE(cache_stride >= (int64_t)Hkv * D && cache_stride <= 0x7fffffff, "msgl_tree_attention: cache_stride %lld", (long long)cache_stride);
    TreeParams p;
    p.q = static_cast<const uint16_t*>(q), p.q_stride = q_stride;
    p.kc = static_cast<const uint16_t*>(k_cache), p.vc = static_cast<const uint16_t*>(v_cache), p.slot_bytes = (uint32_t)(cache_stride * 2);
    p.r2t = req_to_token, p.r2t_stride = r2t_stride, p.req_idx = req_pool_indices, p.cu = cu_seqlens_q, p.prefix = prefix_lens;
    p.mask = tree_mask, p.words = mask_words;
    p.out = static_cast<uint16_t*>(out), p.out_stride = out_stride;
    p.Hq = Hq, p.Hkv = Hkv, p.group = Hq / Hkv, p.max_q = max_seqlen_q;
    p.row_tiles = tree_row_tiles(max_seqlen_q, p.group);
    p.scale_log2e = scale * 1.44269504088896340736f;
    int splits = tree_splits(bs, max_seqlen_q, max_seqlen_k, total_kv, Hq, Hkv);
    // as many runs as the workspace has room for
    const size_t one = (size_t)total_tokens * Hq * (D + 2) * sizeof(float);
    const size_t room = workspace ? workspace_bytes / one : 0;
    if ((size_t)splits > room) splits = room > 1 ? (int)room : 1;
    p.splits = splits;
    p.chunk = (((max_seqlen_k + splits - 1) / splits) + kTreeKeys - 1) / kTreeKeys * kTreeKeys;
    p.ws_o = static_cast<float*>(workspace);
    p.ws_ml = p.ws_o + (splits > 1 ? (size_t)total_tokens * Hq * splits * kHD : 0);
    MSGL_REQUIRE(splits == 1 || aligned16(workspace), "msgl_tree_attention: workspace must be 16-byte aligned");
    const int64_t blocks = (int64_t)bs * splits * Hkv * p.row_tiles;
    MSGL_REQUIRE(blocks <= 0x7fffffff, "msgl_tree_attention: %lld work groups", (long long)blocks);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const bool once = p.row_tiles == 1;  // K and V are read by one work group: past the caches
    int rc;
    if (max_seqlen_q * p.group <= 32) rc = launch_tree<1, true>(p, blocks, st);
    else rc = once ? launch_tree<2, true>(p, blocks, st) : launch_tree<2, false>(p, blocks, st);
    if (rc != MSGL_OK || splits == 1) return rc;
    const int64_t waves = (int64_t)bs * max_seqlen_q * Hq;
    hipLaunchKernelGGL(tree_merge_kernel, dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, st, p);
    return check_launch("tree_merge_kernel");
}
