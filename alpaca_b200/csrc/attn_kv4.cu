// attn_kv4.cu — attention over the 4-bit KV cache (kv4.cuh).
//
//   split kernel   one CTA per SM. A unit is one KV head of one sequence with up to 4 NT of its query rows (a query row = one
//                  head of one token; the G heads of every token of the call share the KV head), cut into tiles of 64
//                  (head_dim 64) or 32 (head_dim 128) cache rows. The units' tiles lie in one row and are cut into equal
//                  chunks, each worked off by one warp with its own cp.async ring and its own running softmax. A unit inside
//                  one chunk is finished there; the parts of one that crosses chunks go to records.
//                  Both products run on mma.sync m16n8k16 with the cache as the 16-row operand: S^T = K Q^T (16 keys x 8
//                  columns) and O^T = V^T P^T (16 channels x 8 columns). A column pair is one query row: f16 high part and
//                  f16 remainder of q or p, so the f32 sum of the pair's two accumulators carries ~22 bits. Scores,
//                  maxima and sums of a query row then live in the same lanes as its outputs (lane % 4).
//                  K: codes enter as f16 denormals (c * 2^-24, one AND per pair; codes in bits 4-7 count 16 times, which
//                  the queries' halves undo), exact; a block's step and zero point are applied to the block's partial
//                  score in f32: s = sum_b step_b (acc_b - zero_b * qsum_b).
//                  V: ldmatrix with transposition sets two keys' codes side by side; (c - zero) * step is exact in f16 (kv4.cuh).
//                  P moves from accumulator to operand layout with movmatrix (no shared memory).
//   combine        one CTA per query row: rescales the parts' (m, l, acc) records to the common maximum and normalises.
//   general kernel fp32 SIMT, any head_dim that is a multiple of 32 up to 256: one warp per query row.
//
// What bounds it: a row of 64 channels is 72 bytes of K and V, so HBM would allow 50 cycles of an SM per 16 keys (199 issue
// slots); decoding and both products take about 150 (d = 64, one query row) to 190, and issue is active 67-69% of the time: the
// long calls are bound by the instructions they decode with at the rate that four warps a scheduler issue, not by one unit.
// Measured on one B200: 64 sequences of 1..8192 rows at 32/32 heads, d = 64, 118-139 us a call, 4.4-5.1 TB/s, 66-78% of the copy
// bandwidth (ALU 55%, shared-memory wavefronts 61%, FMA 42%, tensor 30%); 48 sequences of 1..16000 rows at 32/8 heads, d = 128,
// paged, 99-115 us, 59-68%. Short calls are latency: 64 sequences of 1..4096 rows at 9/3 heads 15 us (floor 4.4), one session of
// 517 rows 4.3.
//
// Scores are in log2 units. A row whose context is empty, or a token that sees no row, gives zeros.
#include <algorithm>
#include <climits>
#include <cmath>

#include "kv4.cuh"

namespace alpaca {
namespace {

constexpr int kStages = 2;          // tiles in a warp's ring
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kPShift = 7.f;      // p is held times 2^7: its f16 remainder then keeps small p to 2^-31 of the maximum
constexpr float kMaxSlack = 8.f;    // the reference maximum moves only when a score exceeds it by this much (log2): p <= 2^15

struct Kv4Args {
    const void* q;
    int64_t q_token_stride, q_seq_stride;
    void* out;
    int64_t out_token_stride, out_seq_stride;
    int q_f16, out_f16;
    Kv4View c;
    const int* ctx_lens;
    int uniform_len, max_len;
    int n_seqs, n_heads, n_kv_heads, tokens, group, q_rows, q_groups;  // q_rows = tokens * group per KV head
    int2* plan;      // [unit]: the first chunk that holds tiles of it, and how many do
    float* partial;  // [chunk + unit][query row of the group][d + 4]: accumulators, m (log2 units), l
    int chunks;
    float scale;
    unsigned* err;
};

// Visible rows of sequence s (its context after this call's tokens). An entry outside [0, max_len] is reported and
// clamped: grid and workspace were sized for max_len.
__device__ __forceinline__ int ctx_of(const Kv4Args& a, int s) {
    if (!a.ctx_lens) return a.uniform_len;
    const int L = a.ctx_lens[s];
    if (L < 0 || L > a.max_len) {
        atomicOr(a.err, kDevErrBadIndex);
        return L < 0 ? 0 : a.max_len;
    }
    return L;
}

__device__ __forceinline__ void store_out(const Kv4Args& a, int seq, int token, int head, int D, int col, float x) {
    const int64_t o = seq * a.out_seq_stride + token * a.out_token_stride + static_cast<int64_t>(head) * D + col;
    if (a.out_f16) static_cast<__half*>(a.out)[o] = __float2half_rn(x);
    else static_cast<float*>(a.out)[o] = x;
}

// ------------------------------------------------------------------------------------------------ split kernel

template <int D>
struct Kv4Geo {
    static constexpr int NB = D / 32;             // blocks per row
    static constexpr int TK = 4096 / D;           // rows of a tile
    static constexpr int GR = TK / 16;            // 16-row groups of a tile
    static constexpr int CROW = D / 2;            // code bytes of a row
    static constexpr int CPR = CROW / 16;         // 16-byte chunks of a row's codes
    static constexpr int HROW = D / 16;           // header bytes of a row
    static constexpr int CB = TK * CROW;          // 2048
    static constexpr int HB = TK * HROW;          // 256
    static constexpr int STAGE = 2 * (CB + HB);   // K codes, V codes, K headers, V headers
    static constexpr int REC = D + 4;             // floats of a partial record
    static constexpr int DEC = 2048;              // bytes of a warp's decoded headers: 1 KB for K, 1 KB for V
    static constexpr int WARP = kStages * STAGE + DEC;
    // Chunk of V row `row` in shared memory: eight rows' chunks of one index lie in different banks for ldmatrix.
    __device__ static constexpr int v_chunk(int row, int c) { return D == 64 ? c ^ ((row >> 2) & 1) : c ^ ((row >> 1) & 3); }
    // Block that lane group g decodes in V (of every 16-byte chunk), and the first of the four channels it holds of chunk c.
    __device__ static constexpr int v_block(int g) { return (g >> 1) & (NB - 1); }
    __device__ static constexpr int v_channel(int g, int c) {
        return D == 64 ? 32 * ((g >> 1) & 1) + 8 * (2 * c + (g >> 2)) + 4 * (g & 1) : 32 * (g >> 1) + 8 * c + 4 * (g & 1);
    }
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t src_bytes) {  // the rest reads as zero
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same with a zero accumulator.
__device__ __forceinline__ void mma16816_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
// x and y each as a high part of 11 bits (low half) and the f16 of what that leaves (high half): x in r0, y in r1.
__device__ __forceinline__ void split_f16_pair(float x, float y, uint32_t& r0, uint32_t& r1) {
    const float hx = __uint_as_float(__float_as_uint(x) & 0xFFFFE000u), hy = __uint_as_float(__float_as_uint(y) & 0xFFFFE000u);
    r0 = pack_half2(hx, x - hx);
    r1 = pack_half2(hy, y - hy);
}

// A lane's places in a head's rows: where its 16 bytes of a tile come from (row 0 of a contiguous cache) and go to.
struct TileCopy {
    const uint8_t* k;
    const uint8_t* v;
    const uint8_t* h;  // lanes 0-15 K headers, 16-31 V headers
    uint32_t k_dst, v_dst, h_dst;  // offsets in a stage
};
template <int D>
__device__ __forceinline__ TileCopy tile_copy(const Kv4Args& a, int64_t unit, int kvh, int lane) {
    using Ge = Kv4Geo<D>;
    const int64_t code = unit * a.c.code_unit_stride + kvh * a.c.code_head_stride + 16 * lane;
    const int64_t scale = unit * a.c.scale_unit_stride + kvh * a.c.scale_head_stride + 8 * (lane & 15);
    TileCopy c;
    c.k = a.c.k_codes + code;
    c.v = a.c.v_codes + code;
    c.h = reinterpret_cast<const uint8_t*>((lane < 16 ? a.c.k_scales : a.c.v_scales) + scale);
    c.k_dst = 16 * lane;
    c.v_dst = Ge::CB + (lane / Ge::CPR) * Ge::CROW + 16 * Ge::v_chunk(lane / Ge::CPR, lane % Ge::CPR);
    c.h_dst = 2 * Ge::CB + 16 * lane;
    return c;
}

// Where a warp's tiles lie in a paged cache whose blocks hold whole tiles: block `b` of the sequence, row `r` of it, and 32
// entries of its table from `base` on, one per lane.
struct Pages {
    int b, r, base, entry;
};
template <int D>
__device__ __forceinline__ Pages first_page(const Kv4Args& a, int row0) {
    Pages p;
    p.b = a.c.block_table ? row0 / a.c.rows : 0;
    p.r = row0 - p.b * a.c.rows;
    p.base = -64;
    p.entry = -1;
    return p;
}
// Block of the tile that the pages stand at, which then move on by `step` tiles; -1 (reported) when the entry is outside the
// pool.
template <int D>
__device__ __forceinline__ int next_page(const Kv4Args& a, Pages& p, int seq, int step, int lane) {
    if (p.b >= p.base + 32) {
        p.base = p.b;
        p.entry = p.b + lane < a.c.max_blocks ? a.c.block_table[static_cast<int64_t>(seq) * a.c.max_blocks + p.b + lane] : -1;
    }
    const int blk = __shfl_sync(0xffffffffu, p.entry, p.b - p.base);
    p.r += step * Kv4Geo<D>::TK;
    if (step == 1) {
        if (p.r >= a.c.rows) {
            p.r = 0;
            p.b++;
        }
    } else {
        for (; p.r >= a.c.rows; p.r -= a.c.rows) p.b++;
    }
    if (blk >= 0 && blk < a.c.pool_blocks) return blk;
    atomicOr(a.err, kDevErrBadIndex);
    return -1;
}

// Copies rows [row0, min(row0 + TK, row_end)) of one KV head into a stage. The rows past them, and rows of a table entry
// outside the pool, read as zero codes with step 0. Calls for a unit go from tile to tile, `step` at a time. The caller commits
// the group.
template <int D>
__device__ __forceinline__ void load_tile(const Kv4Args& a, const TileCopy& head, Pages& pages, int seq, int kvh, int row0, int row_end,
                                          int step, uint32_t stage, int lane) {
    using Ge = Kv4Geo<D>;
    const int n = row_end - row0;
    TileCopy c = head;
    int64_t unit = seq;
    int r = row0;
    bool whole = n >= Ge::TK;  // a full tile of one unit: one run of bytes per plane
    if (a.c.block_table) {
        whole = whole && a.c.rows % Ge::TK == 0;
        if (whole) {
            r = pages.r;
            unit = next_page<D>(a, pages, seq, step, lane);
            whole = unit >= 0;
            if (whole) c = tile_copy<D>(a, unit, kvh, lane);
        }
    }
    if (whole) {
        const uint8_t* k = c.k + static_cast<int64_t>(r) * Ge::CROW;
        const uint8_t* v = c.v + static_cast<int64_t>(r) * Ge::CROW;
#pragma unroll
        for (int i = 0; i < Ge::CB / 512; i++) cp_async16(stage + c.k_dst + 512 * i, k + 512 * i);
        cp_async16(stage + c.h_dst, c.h + static_cast<int64_t>(r) * Ge::HROW);
#pragma unroll
        for (int i = 0; i < Ge::CB / 512; i++) cp_async16(stage + c.v_dst + 512 * i, v + 512 * i);
    } else {  // by 16-row groups, which never leave their unit: lane i finds group i
        int64_t code = 0, scale = 0;
        bool ok = false;
        if (lane < Ge::GR && 16 * lane < n) {
            ok = kv4_locate(a.c, seq, row0 + 16 * lane, a.err, unit, r);
            if (ok) {
                code = unit * a.c.code_unit_stride + kvh * a.c.code_head_stride + static_cast<int64_t>(r) * Ge::CROW;
                scale = unit * a.c.scale_unit_stride + kvh * a.c.scale_head_stride + static_cast<int64_t>(r) * Ge::NB;
            }
        }
#pragma unroll
        for (int i = 0; i < Ge::CB / 512; i++) {
            const int row = lane / Ge::CPR + 32 / Ge::CPR * i, gr = 32 / Ge::CPR * i / 16;
            const int64_t base = __shfl_sync(0xffffffffu, code, gr);
            const bool in = __shfl_sync(0xffffffffu, static_cast<int>(ok), gr) && row < n;
            const int64_t off = base + (in ? (row - 16 * gr) * Ge::CROW + 16 * (lane % Ge::CPR) : 0);
            cp_async16(stage + c.k_dst + 512 * i, a.c.k_codes + off, in ? 16u : 0u);
            cp_async16(stage + c.v_dst + 512 * i, a.c.v_codes + off, in ? 16u : 0u);
        }
        constexpr int RPC = 16 / Ge::HROW;  // rows per chunk of headers
        const int row = (lane & 15) * RPC, gr = row / 16;
        const int64_t base = __shfl_sync(0xffffffffu, scale, gr);
        const bool in = __shfl_sync(0xffffffffu, static_cast<int>(ok), gr);
        const int bytes = in ? min(max((n - row) * Ge::HROW, 0), 16) : 0;
        const uint16_t* scales = lane < 16 ? a.c.k_scales : a.c.v_scales;
        cp_async16(stage + c.h_dst, scales + base + (bytes > 0 ? (row - 16 * gr) * Ge::NB : 0), static_cast<uint32_t>(bytes));
    }
}

// V headers of keys 2 pair (he) and 2 pair + 1 (ho), blocks 2 word and 2 word + 1, as Kv4Pairs.
template <int D>
__device__ __forceinline__ void decode_v_headers(uint32_t he, uint32_t ho, uint4* s_vd, int pair, int word) {
    const Kv4Pair p0 = kv4_pair(__byte_perm(he, ho, 0x5410)), p1 = kv4_pair(__byte_perm(he, ho, 0x7632));
    uint4* out = s_vd + ((pair >> 2) * Kv4Geo<D>::NB + 2 * word) * 4 + (pair & 3);  // [eight keys][block][pair of them]
    out[0] = make_uint4(as_u32(p0.d), as_u32(p0.z), as_u32(p0.d16), as_u32(p0.z16));
    out[4] = make_uint4(as_u32(p1.d), as_u32(p1.z), as_u32(p1.d16), as_u32(p1.z16));
}

// A tile's headers decoded once per warp: per key the (step, zero * 2^-24) of its K blocks in f32, and per pair of keys that
// meet in a V operand register (2t, 2t + 1 of eight) the pair's Kv4Pair for each block.
template <int D>
__device__ __forceinline__ void decode_headers(const uint8_t* stage, float4* s_kd, uint4* s_vd, int lane) {
    using Ge = Kv4Geo<D>;
    constexpr int WPK = Ge::NB / 2;  // header words per key
    const uint32_t* kh = reinterpret_cast<const uint32_t*>(stage + 2 * Ge::CB);
    const uint32_t* vh = kh + Ge::HB / 4;
#pragma unroll
    for (int k = 0; k < Ge::HB / 128; k++) {
        const uint32_t h = kh[lane + 32 * k];
        const float2 d = __half22float2(as_half2(h & 0xFFF0FFF0u)), z = __half22float2(as_half2(h & 0x000F000Fu));
        s_kd[lane + 32 * k] = make_float4(d.x, z.x, d.y, z.y);
    }
    const int pair = lane / WPK, word = lane % WPK;  // keys 2 pair, 2 pair + 1; blocks 2 word, 2 word + 1
    decode_v_headers<D>(vh[2 * pair * WPK + word], vh[(2 * pair + 1) * WPK + word], s_vd, pair, word);
}

// FO: with one or two query rows (and NT = 1) the columns that would stand empty serve other keys. Column pair c then is query
// row c % (4 / FO) over the 16-row groups gr with gr % FO == c / (4 / FO): a tile's scores, exponentials and their operand
// conversions shrink FO-fold, the MMAs stay as many (their B operands are zero in the other pairs' columns).
template <int NT, int FO>
__host__ __device__ constexpr int query_rows() {
    return 4 * NT / FO;
}

// State of the query rows a lane keeps: nt-th row = 4 nt + lane % 4 of the unit's (FO > 1: row lane % 4 % (4 / FO)).
template <int D, int NT, int FO>
struct RowState {
    uint32_t qb[FO][NT][D / 32][4];  // query operands, per fold
    float qsum[NT][D / 32];  // sum of a block's (scaled) queries
    float fs[NT];            // raw score -> log2 units
    float m[NT], thr[NT], negm[NT], l[NT];
    int lim[NT];             // visible rows
    float o[NT][D / 32][4];  // accumulators of the lane's four channels per chunk of V codes
};

// A tile with rows that only some of the unit's query rows see: p is 0 for the others, but 0 x NaN is NaN in the MMA. So value
// blocks without a finite step (those that read as NaN) at rows from min_lim on count as zeros, and NaN is added by hand to the
// channels of the query rows that do see them. Calls of one token, and tiles that every query row sees whole, never come here.
template <int D, int NT, int FO>
__device__ __forceinline__ void hide_nan_blocks(const uint8_t* st, uint4* s_vd, int row0, int min_lim, RowState<D, NT, FO>& s, int lane) {
    using Ge = Kv4Geo<D>;
    constexpr int WPK = Ge::NB / 2;
    const uint16_t* vh = reinterpret_cast<const uint16_t*>(st + 2 * Ge::CB + Ge::HB);
    const auto no_step = [](uint32_t h) { return (h & 0x7C00u) == 0x7C00u; };
    const int pair = lane / WPK, word = lane % WPK;  // the headers that this lane decodes
    uint32_t h[2];
    bool found = false;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int row = 2 * pair + k;
        h[k] = reinterpret_cast<const uint32_t*>(vh)[row * WPK + word];
        if (row0 + row < min_lim) continue;
        const uint32_t clear = (no_step(h[k]) ? 0xFFFFu : 0u) | (no_step(h[k] >> 16) ? 0xFFFF0000u : 0u);
        h[k] &= ~clear;
        found |= clear != 0;
    }
    if (!__any_sync(0xffffffffu, found)) return;
    decode_v_headers<D>(h[0], h[1], s_vd, pair, word);
    const int block = Ge::v_block(lane >> 2);
    for (int row = max(min_lim - row0, 0); row < Ge::TK; row++) {
        if (!no_step(vh[row * Ge::NB + block])) continue;
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
            if (row0 + row < s.lim[nt]) {
#pragma unroll
                for (int c = 0; c < Ge::CPR; c++)
#pragma unroll
                    for (int e = 0; e < 4; e++) s.o[nt][c][e] = __int_as_float(0x7FFFFFFF);
            }
    }
}

template <int D, int NT, int FO>
__device__ __forceinline__ void compute_tile(const uint8_t* st, const float4* s_kd, const uint4* s_vd, int row0, int min_lim,
                                             RowState<D, NT, FO>& s, int lane) {
    using Ge = Kv4Geo<D>;
    constexpr int NB = Ge::NB, GR = Ge::GR, CPR = Ge::CPR, SG = GR / FO, QP = 4 / FO;  // SG sets of FO groups
    static_assert(FO == 1 || NT == 1, "folding is for one group of query rows");
    const int g = lane >> 2, t = lane & 3;
    const int fold = t / QP, column_fold = (g >> 1) / QP;  // of this lane's scores; of its operand column

    float r[SG][2][NT];
#pragma unroll
    for (int sg = 0; sg < SG; sg++) {
        float acc[NB][NT][4];
#pragma unroll
        for (int f = 0; f < FO; f++) {
            uint32_t w[2][NB];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint8_t* p = st + (16 * (sg * FO + f) + 8 * h + g) * Ge::CROW + 4 * NB * t;
                if (D == 64) {
                    const uint2 u = *reinterpret_cast<const uint2*>(p);
                    w[h][0] = u.x;
                    w[h][1] = u.y;
                } else {
                    const uint4 u = *reinterpret_cast<const uint4*>(p);
                    w[h][0] = u.x; w[h][1] = u.y; w[h][NB - 2] = u.z; w[h][NB - 1] = u.w;
                }
            }
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const uint32_t a0[4] = {w[0][b] & 0x000F000Fu, w[1][b] & 0x000F000Fu, w[0][b] & 0x00F000F0u, w[1][b] & 0x00F000F0u};
                const uint32_t x0 = w[0][b] >> 8, x1 = w[1][b] >> 8;
                const uint32_t a1[4] = {x0 & 0x000F000Fu, x1 & 0x000F000Fu, x0 & 0x00F000F0u, x1 & 0x00F000F0u};
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    if (f == 0) mma16816_first(acc[b][nt], a0, s.qb[f][nt][b][0], s.qb[f][nt][b][1]);
                    else mma16816(acc[b][nt], a0, s.qb[f][nt][b][0], s.qb[f][nt][b][1]);
                    mma16816(acc[b][nt], a1, s.qb[f][nt][b][2], s.qb[f][nt][b][3]);
                }
            }
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const float4* kd = s_kd + (16 * (sg * FO + fold) + 8 * h + g) * (NB / 2);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) r[sg][h][nt] = 0.f;
#pragma unroll
            for (int i = 0; i < NB / 2; i++) {
                const float4 u = kd[i];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    r[sg][h][nt] = fmaf(u.x, fmaf(-u.y, s.qsum[nt][2 * i], acc[2 * i][nt][2 * h] + acc[2 * i][nt][2 * h + 1]), r[sg][h][nt]);
                    r[sg][h][nt] =
                        fmaf(u.z, fmaf(-u.w, s.qsum[nt][2 * i + 1], acc[2 * i + 1][nt][2 * h] + acc[2 * i + 1][nt][2 * h + 1]), r[sg][h][nt]);
                }
            }
        }
    }
    if (row0 + Ge::TK > min_lim) {  // some row of the tile is hidden from some query row
#pragma unroll
        for (int sg = 0; sg < SG; sg++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
                    if (row0 + 16 * (sg * FO + fold) + 8 * h + g >= s.lim[nt]) r[sg][h][nt] = -INFINITY;
    }

    uint32_t pb[SG][2][NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        float mx = r[0][0][nt];
#pragma unroll
        for (int sg = 0; sg < SG; sg++) mx = fmax3(mx, r[sg][0][nt], r[sg][1][nt]);
        if (__any_sync(0xffffffffu, mx > s.thr[nt])) {  // the reference maximum moves (rare after the first tile)
#pragma unroll
            for (int o = QP; o <= 16; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float mn = fmaxf(s.m[nt], mx);
            const float alpha = s.m[nt] == -INFINITY ? 0.f : ex2_approx(s.fs[nt] * (s.m[nt] - mn));
            s.l[nt] *= alpha;
#pragma unroll
            for (int c = 0; c < CPR; c++)
#pragma unroll
                for (int e = 0; e < 4; e++) s.o[nt][c][e] *= alpha;
            s.m[nt] = mn;
            s.thr[nt] = mn + kMaxSlack / s.fs[nt];
            s.negm[nt] = mn == -INFINITY ? kPShift : kPShift - s.fs[nt] * mn;
        }
#pragma unroll
        for (int sg = 0; sg < SG; sg++) {
            const float p0 = ex2_approx(fmaf(s.fs[nt], r[sg][0][nt], s.negm[nt]));  // hidden rows: 2^-inf = 0
            const float p1 = ex2_approx(fmaf(s.fs[nt], r[sg][1][nt], s.negm[nt]));
            s.l[nt] += p0;
            s.l[nt] += p1;
            uint32_t u0, u1;
            split_f16_pair(p0, p1, u0, u1);
            pb[sg][0][nt] = movmatrix(u0);
            pb[sg][1][nt] = movmatrix(u1);
        }
    }

    // V: ldmatrix with transposition hands lane (g, t) the four codes that chunk c of rows 2t, 2t + 1 of eight holds at g, the
    // two rows side by side: one register for four channels of two keys. Matrices: keys 0-7 and 8-15 of chunks c, c + 1.
    const int v_row = (lane & 7) + 8 * ((lane >> 3) & 1);
    const uint32_t s_v = smem_u32(st + Ge::CB) + v_row * Ge::CROW;
#pragma unroll
    for (int c = 0; c < CPR; c += 2) {
        float acc[2][2][NT][4];  // [chunk][channels 0, 1 / 2, 3 in operand rows g, g + 8]
        const uint32_t addr = s_v + 16 * Ge::v_chunk(v_row, c + (lane >> 4));
#pragma unroll
        for (int gr = 0; gr < GR; gr++) {
            uint32_t w[4], b0[NT], b1[NT];
            ldmatrix_x4_trans(addr + 16 * gr * Ge::CROW, w);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                b0[nt] = FO == 1 || column_fold == gr % FO ? pb[gr / FO][0][nt] : 0u;
                b1[nt] = FO == 1 || column_fold == gr % FO ? pb[gr / FO][1][nt] : 0u;
            }
            Kv4Pair p[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint4 u = s_vd[((2 * gr + h) * NB + Ge::v_block(g)) * 4 + t];
                p[h].d = as_half2(u.x);
                p[h].z = as_half2(u.y);
                p[h].d16 = as_half2(u.z);
                p[h].z16 = as_half2(u.w);
            }
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int m = 0; m < 2; m++) {
                    const uint32_t u0 = w[2 * k] >> (8 * m), u1 = w[2 * k + 1] >> (8 * m);
                    const uint32_t va[4] = {kv4_lo(u0, p[0]), kv4_hi(u0, p[0]), kv4_lo(u1, p[1]), kv4_hi(u1, p[1])};
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        if (gr == 0) mma16816_first(acc[k][m][nt], va, b0[nt], b1[nt]);
                        else mma16816(acc[k][m][nt], va, b0[nt], b1[nt]);
                    }
                }
        }
        // a tile's sums are added in f32 here: long chains of MMA accumulation lose low bits one way
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    s.o[nt][c + k][2 * m] += acc[k][m][nt][0] + acc[k][m][nt][1];
                    s.o[nt][c + k][2 * m + 1] += acc[k][m][nt][2] + acc[k][m][nt][3];
                }
    }
}

// Tiles of a (sequence, KV head, query group) unit: an empty context counts one, so that its zeros are written.
template <int D>
__device__ __forceinline__ int unit_tiles(int L) {
    return max(1, (L + Kv4Geo<D>::TK - 1) / Kv4Geo<D>::TK);
}
constexpr int kUnitCost = 2;  // what a unit costs besides its tiles (queries, first copies), in tiles

// a / b for a >= 0, b > 0, by 32-bit division where the operands allow it.
__device__ __forceinline__ int64_t div_pos(int64_t a, int64_t b) {
    return (a | b) >> 32 ? a / b : static_cast<int64_t>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b));
}

// The work of a call is its units in one row, sequence by sequence, each kUnitCost places and then one place per tile. The row
// is cut into equal chunks, one per warp: all warps of the one resident wave then have the same work, whatever the contexts are.
struct Chunk {
    int64_t begin, end, size;  // places; `size` of every chunk but the last
    int64_t first;             // first place of the unit that `begin` lies in
    int seq, head_group, L;    // that unit: sequence, kv_head * q_groups + query group, the sequence's context
};
template <int D>
__device__ __forceinline__ int unit_places(int L) {
    return kUnitCost + unit_tiles<D>(L);
}

template <int D>
__device__ __forceinline__ Chunk find_chunk(const Kv4Args& a, int64_t index, int lane) {
    Chunk c;
    const int64_t hg = static_cast<int64_t>(a.n_kv_heads) * a.q_groups;
    constexpr int HELD = 2;  // blocks of 32 contexts kept in registers: one round trip for the usual batches
    int held[HELD];
    int64_t total = 0;
    if (a.ctx_lens) {
#pragma unroll
        for (int i = 0; i < HELD; i++) held[i] = lane + 32 * i < a.n_seqs ? ctx_of(a, lane + 32 * i) : 0;
#pragma unroll
        for (int i = 0; i < HELD; i++) total += lane + 32 * i < a.n_seqs ? unit_places<D>(held[i]) : 0;
        for (int s = lane + 32 * HELD; s < a.n_seqs; s += 32) total += unit_places<D>(ctx_of(a, s));
        // a lane's sum is below 2^36: two 32-bit sums hold the warp's
        const unsigned lo = __reduce_add_sync(0xffffffffu, static_cast<unsigned>(total & 0xFFFFF));
        const unsigned hi = __reduce_add_sync(0xffffffffu, static_cast<unsigned>(total >> 20));
        total = (static_cast<int64_t>(hi) << 20) + lo;
    } else {
        total = static_cast<int64_t>(a.n_seqs) * unit_places<D>(a.uniform_len);
    }
    total *= hg;
    c.size = div_pos(total + a.chunks - 1, a.chunks);
    c.begin = index * c.size;
    c.end = min(c.begin + c.size, total);
    if (c.begin >= c.end) return c;
    if (!a.ctx_lens) {
        const int t = unit_places<D>(a.uniform_len);
        const int64_t unit = div_pos(c.begin, t);
        c.first = unit * t;
        c.seq = static_cast<int>(div_pos(unit, hg));
        c.head_group = static_cast<int>(unit - c.seq * hg);
        c.L = a.uniform_len;
        return c;
    }
    int64_t before = 0;  // places before the block of 32 sequences
    for (int s0 = 0;; s0 += 32) {
        const int s = s0 + lane;
        const int L = s0 == 0 ? held[0] : (s0 == 32 ? held[1] : (s < a.n_seqs ? ctx_of(a, s) : 0));
        static_assert(32 * (kUnitCost + (int64_t(1) << 30) / Kv4Geo<D>::TK) <= INT_MAX, "places of 32 sequences must fit 32 bits");
        const int mine = s < a.n_seqs ? unit_places<D>(L) : 0;  // contexts are at most 2^30 rows
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += x;
        }
        const unsigned past = __ballot_sync(0xffffffffu, before + incl * hg > c.begin);
        if (past) {  // begin < total: some sequence holds it
            const int src = __ffs(past) - 1;
            c.seq = s0 + src;
            c.L = __shfl_sync(0xffffffffu, L, src);
            const int64_t start = before + __shfl_sync(0xffffffffu, incl - mine, src) * hg;
            const int t = unit_places<D>(c.L);
            c.head_group = static_cast<int>(div_pos(c.begin - start, t));
            c.first = start + static_cast<int64_t>(c.head_group) * t;
            return c;
        }
        before += __shfl_sync(0xffffffffu, incl, 31) * hg;
    }
}

// Query operands of the group's rows r0 .. r0 + 4 NT - 1. Column 2 q + {0, 1} of an operand is query row q's (high part,
// remainder): lane group g holds row g >> 1 and part g & 1; lane t the channels 32 b + 8 t + .. of every block, in the order of
// the K codes' nibbles. Rows are scaled by a power of two to [2^10, 2^11) so that neither part leaves f16's normal range.
template <int D, int NT, int FO>
__device__ __forceinline__ void load_queries(const Kv4Args& a, int seq, int kvh, int r0, int L, RowState<D, NT, FO>& s, int g, int t) {
    constexpr int NB = D / 32, QP = 4 / FO;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int rr = r0 + 4 * nt + (g >> 1) % QP;
        float x[NB][8];
        float amax = 0.f;
        if (rr < a.q_rows) {
            const int token = rr / a.group, head = kvh * a.group + rr % a.group;
            const int64_t off = seq * a.q_seq_stride + token * a.q_token_stride + static_cast<int64_t>(head) * D + 8 * t;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                if (a.q_f16) {
                    const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const __half*>(a.q) + off + 32 * b);
                    const uint32_t v[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float2 f = __half22float2(as_half2(v[i]));
                        x[b][2 * i] = f.x;
                        x[b][2 * i + 1] = f.y;
                    }
                } else {
                    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + off + 32 * b);
                    const float4 u = p[0], v = p[1];
                    x[b][0] = u.x; x[b][1] = u.y; x[b][2] = u.z; x[b][3] = u.w;
                    x[b][4] = v.x; x[b][5] = v.y; x[b][6] = v.z; x[b][7] = v.w;
                }
#pragma unroll
                for (int e = 0; e < 8; e++) amax = fmaxf(amax, fabsf(x[b][e]));
            }
        } else {
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int e = 0; e < 8; e++) x[b][e] = 0.f;
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const uint32_t ex = min(max(__float_as_uint(amax) >> 23, 11u), 254u);
        const float up = __uint_as_float((264u - ex) << 23), down = __uint_as_float((ex - 10u) << 23);  // 2^(137 - ex), inverse
        const int src = 8 * t;  // lane (2t, 0): query row t of this nt
        s.fs[nt] = __shfl_sync(0xffffffffu, a.scale * kLog2e * 16777216.f * down, src);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                x[b][e] *= up;
                sum += x[b][e];
            }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            s.qsum[nt][b] = __shfl_sync(0xffffffffu, sum, src);
#pragma unroll
            for (int i = 0; i < 4; i++) {  // nibble pair (i, i + 4); codes of odd i count 16 times
                uint32_t u, v;
                split_f16_pair(x[b][i] * ((i & 1) ? 0.0625f : 1.f), x[b][i + 4] * ((i & 1) ? 0.0625f : 1.f), u, v);
                const uint32_t q = __byte_perm(u, v, (g & 1) ? 0x7632 : 0x5410);
#pragma unroll
                for (int f = 0; f < FO; f++) s.qb[f][nt][b][i] = FO == 1 || (g >> 1) / QP == f ? q : 0u;
            }
        }
        s.m[nt] = s.thr[nt] = -INFINITY;
        s.negm[nt] = kPShift;
        s.l[nt] = 0.f;
        s.lim[nt] = L - a.tokens + 1 + (r0 + 4 * nt + t % QP) / a.group;
#pragma unroll
        for (int c = 0; c < D / 32; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) s.o[nt][c][e] = 0.f;
    }
}

// Warps of a CTA, one CTA per SM: as many as the registers of the form allow (128, 168 and 255 a thread). The forms for d = 128
// spill 4 to 96 bytes of their units' state, those for d = 64 none to 56. It is not what costs them: the paged decode's form
// spills 64, the same with kMany 16, and that one is 2% slower.
__host__ __device__ constexpr int split_warps(int NT) { return NT == 4 ? 8 : (NT == 2 ? 12 : 16); }

// kCta: one CTA per unit; its warps share the unit's tiles and meet in shared memory (no records).
// kMany: for calls of several tokens, whose query rows see different rows of a tile. The one-token calls of up to four query
// rows have a form without that code (paged, d = 128: 106.0 us against 108.0; one session 4.30 against 4.35).
template <int D, int NT, int FO, bool kCta, bool kMany>
__global__ void __launch_bounds__(32 * split_warps(NT), 1) kv4_split_kernel(const __grid_constant__ Kv4Args a) {
    using Ge = Kv4Geo<D>;
    constexpr int QR = query_rows<NT, FO>();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    uint8_t* ring = smem + warp * Ge::WARP;
    float4* s_kd = reinterpret_cast<float4*>(ring + kStages * Ge::STAGE);
    uint4* s_vd = reinterpret_cast<uint4*>(ring + kStages * Ge::STAGE + Ge::DEC / 2);
    const uint32_t ring_u32 = smem_u32(ring);
    const int chunk = warp * gridDim.x + blockIdx.x;  // a call with few chunks spreads them over the SMs
    Chunk w;
    if constexpr (kCta) {
        const int hg = a.n_kv_heads * a.q_groups;
        w.seq = blockIdx.x / hg;
        w.head_group = blockIdx.x - w.seq * hg;
        w.L = ctx_of(a, w.seq);
        w.begin = w.end = w.size = w.first = 0;
    } else {
        w = find_chunk<D>(a, chunk, lane);
        if (w.begin >= w.end) return;
    }
    const int64_t chunk_begin = w.begin;
    const int step = kCta ? blockDim.x / 32 : 1;
    while (true) {  // the units of the chunk
        const int seq = w.seq, kvh = w.head_group / a.q_groups, qg = w.head_group - kvh * a.q_groups, L = w.L;
        const int r0 = qg * QR, r_last = min(r0 + QR, a.q_rows) - 1;
        const int64_t tile0 = w.first + kUnitCost;  // place of the unit's first tile
        const int ut = unit_tiles<D>(L);
        const int t0 = kCta ? warp : static_cast<int>(max(w.begin - tile0, static_cast<int64_t>(0)));
        const int t1 = kCta ? ut : static_cast<int>(min(static_cast<int64_t>(ut), w.end - tile0));
        if (!kCta && t1 <= t0) return;  // the chunk ends in the places before the unit's first tile
        // rows that query row q sees: L - tokens + 1 + its token; the last one's bounds the rows worth reading
        const int min_lim = L - a.tokens + 1 + r0 / a.group;
        const int row_end = min(L, L - a.tokens + 1 + r_last / a.group);
        const int visible = min(t1, row_end > 0 ? (row_end + Ge::TK - 1) / Ge::TK : 0);
        const int n = (max(visible - t0, 0) + step - 1) / step;  // tiles of this warp: t0, t0 + step, ..
        const TileCopy copy = tile_copy<D>(a, a.c.block_table ? 0 : seq, kvh, lane);
        Pages pages = first_page<D>(a, t0 * Ge::TK);
#pragma unroll
        for (int i = 0; i < kStages - 1; i++) {
            if (i < n) load_tile<D>(a, copy, pages, seq, kvh, (t0 + i * step) * Ge::TK, row_end, step, ring_u32 + i * Ge::STAGE, lane);
            cp_async_commit();
        }
        RowState<D, NT, FO> s;
        load_queries<D, NT, FO>(a, seq, kvh, r0, L, s, g, t);
        for (int it = 0, stage = 0; it < n; it++) {
            cp_async_wait<kStages - 2>();
            __syncwarp();  // the tile has landed for every lane, and every lane is done with the stage refilled below
            const int free_stage = stage == 0 ? kStages - 1 : stage - 1;
            if (it + kStages - 1 < n)
                load_tile<D>(a, copy, pages, seq, kvh, (t0 + (it + kStages - 1) * step) * Ge::TK, row_end, step,
                             ring_u32 + free_stage * Ge::STAGE, lane);
            cp_async_commit();
            const uint8_t* st = ring + stage * Ge::STAGE;
            decode_headers<D>(st, s_kd, s_vd, lane);
            if constexpr (kMany) {
                const int row0 = (t0 + it * step) * Ge::TK;
                if (a.tokens > 1 && row0 + Ge::TK > min_lim) hide_nan_blocks<D, NT, FO>(st, s_vd, row0, min_lim, s, lane);
            }
            __syncwarp();
            compute_tile<D, NT, FO>(st, s_kd, s_vd, (t0 + it * step) * Ge::TK, min_lim, s, lane);
            stage = stage + 1 == kStages ? 0 : stage + 1;
        }
        // A unit that lies wholly in this chunk is finished here, else its part goes to a record. Parts are numbered chunk +
        // unit: along the row of places every next part has a higher number, and a unit's parts follow one another. With one CTA
        // per unit the parts are its warps', in shared memory over the rings.
        const bool whole = !kCta && t1 - t0 == ut;
        const int64_t unit = static_cast<int64_t>(seq) * a.n_kv_heads * a.q_groups + w.head_group;
        if (!kCta && t0 == 0 && lane == 0 && a.plan) {
            a.plan[unit] = make_int2(chunk, static_cast<int>(div_pos(tile0 - chunk_begin + ut - 1, w.size)) + 1);
        }
        float* rec0 = kCta ? reinterpret_cast<float*>(smem) + warp * QR * Ge::REC : a.partial + (chunk + unit) * QR * Ge::REC;
        static_assert(sizeof(float) * QR * Ge::REC <= Ge::WARP, "a warp's record must fit its ring");
        if (kCta) __syncthreads();  // every warp is done with its ring
        else __syncwarp();                 // the next unit's copies go to stages that every lane has read
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float l = s.l[nt];
#pragma unroll
            for (int o = 4 / FO; o <= 16; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
            for (int o = 4 / FO; o < 4; o <<= 1)
#pragma unroll
                for (int c = 0; c < Ge::CPR; c++)
#pragma unroll
                    for (int e = 0; e < 4; e++) s.o[nt][c][e] += __shfl_xor_sync(0xffffffffu, s.o[nt][c][e], o);
            const int row = 4 * nt + t, rr = r0 + row;
            if (t >= 4 / FO || rr >= a.q_rows) continue;
            const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
            for (int c = 0; c < Ge::CPR; c++) {
                const int ch = Ge::v_channel(g, c);
                float (&o)[4] = s.o[nt][c];
                if (whole) {
                    const int64_t out = seq * a.out_seq_stride + (rr / a.group) * a.out_token_stride +
                                        static_cast<int64_t>(kvh * a.group + rr % a.group) * D + ch;
#pragma unroll
                    for (int e = 0; e < 4; e++) o[e] = l == 0.f ? 0.f : o[e] * inv;
                    if (a.out_f16) *reinterpret_cast<uint2*>(static_cast<__half*>(a.out) + out) = make_uint2(pack_half2(o[0], o[1]), pack_half2(o[2], o[3]));
                    else *reinterpret_cast<float4*>(static_cast<float*>(a.out) + out) = make_float4(o[0], o[1], o[2], o[3]);
                } else {
                    *reinterpret_cast<float4*>(rec0 + row * Ge::REC + ch) = make_float4(o[0], o[1], o[2], o[3]);
                }
            }
            if (!whole && g == 0)
                *reinterpret_cast<float2*>(rec0 + row * Ge::REC + D) = make_float2(s.m[nt] == -INFINITY ? -INFINITY : s.fs[nt] * s.m[nt], l);
        }
        if constexpr (kCta) {
            __syncthreads();
            // Join: a warp per row turns the parts' maxima and sums into factors, then every thread adds four channels.
            const int warps = min(step, max(row_end > 0 ? (row_end + Ge::TK - 1) / Ge::TK : 0, 1));  // those with tiles
            const float* rec = reinterpret_cast<const float*>(smem);
            float* s_f = reinterpret_cast<float*>(smem) + step * QR * Ge::REC;  // [row][warp], the sum in place 16
            static_assert(sizeof(float) * QR * (Ge::REC + 17) <= Ge::WARP, "a warp's record and factors must fit its ring");
            static_assert(split_warps(NT) <= 16, "a row's factors have 16 places");
            for (int row = warp; row < QR; row += step) {
                const float* p = rec + (lane < warps ? lane : 0) * QR * Ge::REC + row * Ge::REC + D;
                const float m = lane < warps ? p[0] : -INFINITY;
                float M = m;
#pragma unroll
                for (int o = 8; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
                const float f = m == -INFINITY ? 1.f : ex2_approx(m - M);  // without a maximum: zeros, or NaN
                float l = lane < warps ? p[1] * f : 0.f;
#pragma unroll
                for (int o = 8; o >= 1; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
                if (lane < 16) s_f[row * 17 + lane] = f;
                if (lane == 0) s_f[row * 17 + 16] = l;
            }
            __syncthreads();
            for (int i = threadIdx.x; i < QR * (D / 4); i += blockDim.x) {
                const int row = i / (D / 4), col = 4 * (i - row * (D / 4)), rr = r0 + row;
                if (rr >= a.q_rows) break;
                float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int k = 0; k < warps; k++) {
                    const float4 v = *reinterpret_cast<const float4*>(rec + (k * QR + row) * Ge::REC + col);
                    const float f = s_f[row * 17 + k];
                    o.x = fmaf(v.x, f, o.x);
                    o.y = fmaf(v.y, f, o.y);
                    o.z = fmaf(v.z, f, o.z);
                    o.w = fmaf(v.w, f, o.w);
                }
                const float l = s_f[row * 17 + 16], inv = l == 0.f ? 0.f : 1.f / l;
                if (l == 0.f) o = make_float4(0.f, 0.f, 0.f, 0.f);
                const int64_t out = seq * a.out_seq_stride + (rr / a.group) * a.out_token_stride +
                                    static_cast<int64_t>(kvh * a.group + rr % a.group) * D + col;
                if (a.out_f16)
                    *reinterpret_cast<uint2*>(static_cast<__half*>(a.out) + out) = make_uint2(pack_half2(o.x * inv, o.y * inv), pack_half2(o.z * inv, o.w * inv));
                else
                    *reinterpret_cast<float4*>(static_cast<float*>(a.out) + out) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
            }
            return;
        }
        w.first = w.begin = tile0 + ut;  // the next unit
        if (w.begin >= w.end) return;
        if (++w.head_group == a.n_kv_heads * a.q_groups) {
            w.head_group = 0;
            w.seq++;
            w.L = ctx_of(a, w.seq);
        }
    }
}

// ------------------------------------------------------------------------------------------------ combine

constexpr int kCombineHeld = 4;  // records a warp has in flight

// One CTA per query row: its W warps share the records of the row's unit, each with a running maximum.
template <int D, int QR, int W>
__global__ void __launch_bounds__(32 * W) kv4_combine_kernel(const __grid_constant__ Kv4Args a) {
    constexpr int EPL = D / 32, REC = Kv4Geo<D>::REC;
    __shared__ float s_acc[W][D];
    __shared__ float s_ml[W][2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rr = blockIdx.x % a.q_rows, kvh = (blockIdx.x / a.q_rows) % a.n_kv_heads, seq = blockIdx.x / (a.q_rows * a.n_kv_heads);
    const int64_t unit = (static_cast<int64_t>(seq) * a.n_kv_heads + kvh) * a.q_groups + rr / QR;
    // Every CTA waits for the split grid, so that a later launch which sees this grid complete sees the split kernel's
    // writes too.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int2 part = a.plan[unit];
    if (part.y <= 1) return;  // written by the split kernel
    if (part.x < 0 || part.y > a.chunks - part.x) {  // not this call's plan: the workspace was written to meanwhile
        atomicOr(a.err, kDevErrBadIndex);
        return;
    }
    const float* base = a.partial + ((part.x + unit) * QR + rr % QR) * REC;
    float m = -INFINITY, l = 0.f, acc[EPL];
#pragma unroll
    for (int e = 0; e < EPL; e++) acc[e] = 0.f;
    for (int i0 = warp; i0 < part.y; i0 += W * kCombineHeld) {
        float2 ml[kCombineHeld];
        float v[kCombineHeld][EPL];
#pragma unroll
        for (int k = 0; k < kCombineHeld; k++) {
            const int i = i0 + k * W;
            const float* p = base + static_cast<int64_t>(i) * QR * REC;
            ml[k] = make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int e = 0; e < EPL; e++) v[k][e] = 0.f;
            if (i < part.y) {
                ml[k] = *reinterpret_cast<const float2*>(p + D);
#pragma unroll
                for (int e = 0; e < EPL; e++) v[k][e] = p[lane + 32 * e];
            }
        }
        float top = m;
#pragma unroll
        for (int k = 0; k < kCombineHeld; k++) top = fmaxf(top, ml[k].x);
        const float ref = top == -INFINITY ? 0.f : top;
        const float alpha = ex2_approx(m - ref);
        l *= alpha;
#pragma unroll
        for (int e = 0; e < EPL; e++) acc[e] *= alpha;
#pragma unroll
        for (int k = 0; k < kCombineHeld; k++) {
            // a part whose maximum is -inf holds zeros, or NaN where its scores are NaN
            const float f = ml[k].x == -INFINITY ? 1.f : ex2_approx(ml[k].x - ref);
            l = fmaf(ml[k].y, f, l);
#pragma unroll
            for (int e = 0; e < EPL; e++) acc[e] = fmaf(v[k][e], f, acc[e]);
        }
        m = top;
    }
#pragma unroll
    for (int e = 0; e < EPL; e++) s_acc[warp][lane + 32 * e] = acc[e];
    if (lane == 0) {
        s_ml[warp][0] = m;
        s_ml[warp][1] = l;
    }
    __syncthreads();
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; w++) M = fmaxf(M, s_ml[w][0]);
    for (int col = threadIdx.x; col < D; col += 32 * W) {
        float o = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < W; w++) {
            const float f = s_ml[w][0] == -INFINITY ? 1.f : ex2_approx(s_ml[w][0] - M);
            o = fmaf(s_acc[w][col], f, o);
            sum = fmaf(s_ml[w][1], f, sum);
        }
        store_out(a, seq, rr / a.group, kvh * a.group + rr % a.group, D, col, sum == 0.f ? 0.f : o / sum);
    }
}

// ------------------------------------------------------------------------------------------------ general kernel
//
// For head dims without a form of the split kernel: f32 arithmetic, one warp per query row and no staging, so each query row
// decodes its cache rows again, a lane's K words lie d / 2 bytes from its neighbour's, and eight lanes load one V word. Bound by
// that latency chain, far from the bytes: 64 sequences of 1..4096 rows at 8/2 heads, d = 96, 1.44 ms (floor 4.4 us), d = 256
// 2.6 ms; a prompt of 1024 tokens 0.58 and 1.3 ms; at d = 64 the split kernel takes 15 us where this one takes 1.2 ms.

constexpr int kGenWarps = 4;
constexpr int kGenMaxD = 256;

__device__ __forceinline__ float header_step(uint32_t h) {
    return __half2float(__ushort_as_half(static_cast<unsigned short>(h & kKv4StepMask)));
}

__global__ void __launch_bounds__(32 * kGenWarps) kv4_general_kernel(const __grid_constant__ Kv4Args a, int D) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __shared__ float q_s[kGenWarps][kGenMaxD];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nb = D / 32;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kGenWarps + warp;
    const int64_t total = static_cast<int64_t>(a.n_seqs) * a.tokens * a.n_heads;
    if (row >= total) return;  // whole warp
    const int h = static_cast<int>(row % a.n_heads), t = static_cast<int>((row / a.n_heads) % a.tokens);
    const int seq = static_cast<int>(row / (static_cast<int64_t>(a.n_heads) * a.tokens)), kvh = h / a.group;
    const int vis = min(ctx_of(a, seq) - a.tokens + 1 + t, a.max_len);  // rows this token sees
    const int64_t qoff = seq * a.q_seq_stride + t * a.q_token_stride + static_cast<int64_t>(h) * D;
    for (int i = lane; i < D; i += 32)
        q_s[warp][i] = a.scale * kLog2e * (a.q_f16 ? __half2float(static_cast<const __half*>(a.q)[qoff + i])
                                                   : static_cast<const float*>(a.q)[qoff + i]);
    __syncwarp();
    float m = -INFINITY, l = 0.f, acc[kGenMaxD / 32];
#pragma unroll
    for (int e = 0; e < kGenMaxD / 32; e++) acc[e] = 0.f;
    for (int c0 = 0; c0 < vis; c0 += 32) {
        // lane j: row c0 + j
        int64_t unit = 0;
        int ur = 0;
        const bool in = c0 + lane < vis;
        const bool ok = in && kv4_locate(a.c, seq, c0 + lane, a.err, unit, ur);
        const int64_t co = unit * a.c.code_unit_stride + kvh * a.c.code_head_stride + static_cast<int64_t>(ur) * (D / 2);
        const int64_t so = unit * a.c.scale_unit_stride + kvh * a.c.scale_head_stride + static_cast<int64_t>(ur) * nb;
        float sc = in ? 0.f : -INFINITY;  // a row outside the pool reads as zero
        if (ok) {
            for (int b = 0; b < nb; b++) {
                const uint32_t hd = a.c.k_scales[so + b];
                const float zero = static_cast<float>(hd & 15u);
                float part = 0.f;
                for (int w = 0; w < 4; w++) {
                    const uint32_t word = *reinterpret_cast<const uint32_t*>(a.c.k_codes + co + 4 * (w * nb + b));
#pragma unroll
                    for (int n = 0; n < 8; n++)
                        part = fmaf(static_cast<float>((word >> (4 * n)) & 15u) - zero, q_s[warp][32 * b + 8 * w + n], part);
                }
                sc = fmaf(part, header_step(hd), sc);
            }
        }
        float cm = sc;
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) cm = fmaxf(cm, __shfl_xor_sync(0xffffffffu, cm, o));
        const float mn = fmaxf(m, cm);
        const float ref = mn == -INFINITY ? 0.f : mn;  // only NaN scores so far
        const float alpha = exp2f(m - ref);
        m = mn;
        const float p = in ? exp2f(sc - ref) : 0.f;
        l = l * alpha + p;
#pragma unroll
        for (int e = 0; e < kGenMaxD / 32; e++) acc[e] *= alpha;
        const int n = min(32, vis - c0);
        for (int j = 0; j < n; j++) {
            const float pj = __shfl_sync(0xffffffffu, p, j);
            const int64_t cj = __shfl_sync(0xffffffffu, co, j), sj = __shfl_sync(0xffffffffu, so, j);
            if (!__shfl_sync(0xffffffffu, static_cast<int>(ok), j)) continue;
#pragma unroll
            for (int e = 0; e < kGenMaxD / 32; e++) {  // channel lane + 32 e: nibble lane % 8 of word (lane / 8) * nb + e
                if (e >= nb) break;
                const uint32_t hd = a.c.v_scales[sj + e];
                const uint32_t word = *reinterpret_cast<const uint32_t*>(a.c.v_codes + cj + 4 * ((lane >> 3) * nb + e));
                const float v = (static_cast<float>((word >> (4 * (lane & 7))) & 15u) - static_cast<float>(hd & 15u)) * header_step(hd);
                acc[e] = fmaf(pj, v, acc[e]);
            }
        }
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
    for (int e = 0; e < kGenMaxD / 32; e++)
        if (e < nb) store_out(a, seq, t, h, D, lane + 32 * e, l == 0.f ? 0.f : acc[e] / l);
}

// ------------------------------------------------------------------------------------------------ host side

int max_context(const alpaca_kv4_attn_desc& d) { return d.ctx_lens ? d.max_ctx_len : d.start_position + d.tokens; }

// Query rows per unit and chunks. One or two query rows fold the columns (FO = 4 / 2; a tile of head_dim 128 has two 16-row
// groups, so at most 2); otherwise 4 NT rows, the fewest that hold the call's rows per KV head, up to 16. Chunks: one per warp of
// the machine, or one per place where the call has fewer (by its bound).
constexpr int kSms = 148;
struct SplitPlan {
    int nt, fo, q_rows, q_groups, ctas, warps, chunks;
    int64_t units;
    bool cta_units;  // one CTA per unit, no records
    bool combine;    // some unit may be split between chunks
    int rows_per_unit() const { return 4 * nt / fo; }
};
SplitPlan split_plan(const alpaca_kv4_attn_desc& d) {
    SplitPlan p;
    p.q_rows = d.tokens * (d.n_heads / d.n_kv_heads);
    p.nt = p.q_rows <= 4 ? 1 : (p.q_rows <= 8 ? 2 : 4);
    p.fo = p.q_rows == 1 ? (d.head_dim == 64 ? 4 : 2) : (p.q_rows == 2 ? 2 : 1);
    p.q_groups = (p.q_rows + p.rows_per_unit() - 1) / p.rows_per_unit();
    p.units = static_cast<int64_t>(d.n_seqs) * d.n_kv_heads * p.q_groups;
    const int tk = 4096 / d.head_dim, tiles = std::max(1, (max_context(d) + tk - 1) / tk);
    p.chunks = static_cast<int>(std::min<int64_t>(p.units * (kUnitCost + tiles), static_cast<int64_t>(kSms) * split_warps(p.nt)));
    // Few units of short contexts: one CTA per unit, one launch. With one tile a warp that wins always (9/3 heads, 517 rows:
    // 4.3 us against 5.6); with more, only where the units fill the machine: two from 32 units on (48 units of 2000 rows: 8.2
    // against 9.3; 12 units: 8.2 against 7.7), four from 96 on (128 units of 2000 rows at d = 128: 13.9 against 16.3; 48 units of
    // 4000 rows: 12.5 against 11.1).
    const int cta_tiles = p.units >= 96 ? 4 : (p.units >= 32 ? 2 : 1);
    p.cta_units = p.units <= kSms && tiles <= cta_tiles * split_warps(p.nt);
    // Warps without a tile still share the join's output elements: with one warp three units' contexts of 53 rows (9/3 heads,
    // d = 64) took 6.2 us, with eight 3.4; 16/2 heads 11.5 and 4.4.
    p.warps = p.cta_units ? std::min(std::max(tiles, std::min(8, 2 * p.rows_per_unit())), split_warps(p.nt)) : split_warps(p.nt);
    p.ctas = p.cta_units ? static_cast<int>(p.units) : std::min(p.chunks, kSms);
    p.combine = !p.cta_units && tiles > 1;
    return p;
}
size_t round_up(size_t n, size_t m) { return (n + m - 1) / m * m; }
size_t plan_bytes(const SplitPlan& p) { return p.combine ? round_up(sizeof(int2) * p.units, 256) : 0; }

cudaLaunchConfig_t pdl_config(dim3 grid, int threads, size_t smem, cudaStream_t s, cudaLaunchAttribute* attr) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    attr->id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr->val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 1 : 0;
    return cfg;
}

template <int D, int NT, int FO, bool kCta, bool kMany>
cudaError_t launch_split_form(const Kv4Args& a, const SplitPlan& p, cudaStream_t s) {
    constexpr size_t most = split_warps(NT) * Kv4Geo<D>::WARP;
    const auto fn = kv4_split_kernel<D, NT, FO, kCta, kMany>;
    cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(fn), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(most));
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = pdl_config(dim3(p.ctas, 1, 1), 32 * p.warps, p.warps * Kv4Geo<D>::WARP, s, &attr);
    e = cudaLaunchKernelEx(&cfg, fn, a);
    if (e != cudaSuccess || !p.combine) return e;
    const unsigned rows = static_cast<unsigned>(a.n_seqs) * a.n_kv_heads * a.q_rows;
    // few rows have many records each (up to one a chunk): more warps for them
    constexpr int QR = query_rows<NT, FO>();
    const int warps = rows <= 2 * kSms ? 16 : 4;
    const cudaLaunchConfig_t ccfg = pdl_config(dim3(rows, 1, 1), 32 * warps, 0, s, &attr);
    return warps == 16 ? cudaLaunchKernelEx(&ccfg, kv4_combine_kernel<D, QR, 16>, a) : cudaLaunchKernelEx(&ccfg, kv4_combine_kernel<D, QR, 4>, a);
}
template <int D, int NT, int FO>
cudaError_t launch_split_form(const Kv4Args& a, const SplitPlan& p, cudaStream_t s) {
    constexpr bool one = NT == 1, many = query_rows<NT, FO>() > 1;
    if constexpr (one && many)
        if (a.tokens > 1)
            return p.cta_units ? launch_split_form<D, NT, FO, true, true>(a, p, s) : launch_split_form<D, NT, FO, false, true>(a, p, s);
    return p.cta_units ? launch_split_form<D, NT, FO, true, !one>(a, p, s) : launch_split_form<D, NT, FO, false, !one>(a, p, s);
}

template <int D>
cudaError_t launch_split(const Kv4Args& a, const SplitPlan& p, cudaStream_t s) {
    if constexpr (D == 64)
        if (p.fo == 4) return launch_split_form<D, 1, 4>(a, p, s);
    return p.fo == 2    ? launch_split_form<D, 1, 2>(a, p, s)
           : p.nt == 1  ? launch_split_form<D, 1, 1>(a, p, s)
           : p.nt == 2  ? launch_split_form<D, 2, 1>(a, p, s)
                        : launch_split_form<D, 4, 1>(a, p, s);
}

// The prompt-chunk form: the visible rows as f16 in the workspace ([seq][row][kv_head][d], exact), then the tensor-core
// prefill over them. The f16 cache comes first in the workspace, the prefill's own after it.
struct ChunkPlan {
    alpaca_attn_desc attn;
    size_t cache_bytes;  // of K or V
};
ChunkPlan chunk_plan(const alpaca_kv4_attn_desc& d, void* ws) {
    ChunkPlan p;
    const bool varlen = (d.flags & ALPACA_ATTN_FLAG_VARLEN) != 0;
    const int64_t rows = varlen ? d.max_ctx_len : d.start_position + d.tokens;
    const int64_t row = static_cast<int64_t>(d.n_kv_heads) * d.head_dim;
    p.cache_bytes = round_up(sizeof(__half) * d.n_seqs * rows * row, 256);
    alpaca_attn_desc& a = p.attn;
    a = alpaca_attn_desc{};
    a.n_seqs = d.n_seqs;
    a.n_heads = d.n_heads;
    a.n_kv_heads = d.n_kv_heads;
    a.head_dim = d.head_dim;
    a.tokens = d.tokens;
    a.start_position = varlen ? 0 : d.start_position;
    a.max_ctx_len = varlen ? d.max_ctx_len : 0;
    a.q_dtype = d.q_dtype;
    a.kv_dtype = ALPACA_F16;
    a.out_dtype = d.out_dtype;
    a.q = d.q;
    a.q_token_stride = d.q_token_stride;
    a.q_seq_stride = d.q_seq_stride;
    a.k = ws;
    a.v = static_cast<uint8_t*>(ws) + p.cache_bytes;
    a.kv_row_stride = row;
    a.kv_seq_stride = rows * row;
    a.out = d.out;
    a.out_token_stride = d.out_token_stride;
    a.out_seq_stride = d.out_seq_stride;
    a.scale = d.scale;
    a.flags = d.flags;
    a.q_offsets = d.q_offsets;
    a.start_positions = d.start_positions;
    a.total_tokens = d.total_tokens;
    return p;
}

}  // namespace

// Estimated times (us) of the two forms, fitted by least squares of the relative error to 218 calls on a B200 (8..200 tokens, 1..4
// sequences, contexts up to 6200, five head counts at d = 64 and four at 128); over 208 others, timed later, the choice averages
// 1.3% above the better form, 26% at worst (both sets: profiles/kv4_choice.csv; the split estimates are 16-19% off by themselves,
// the prefill's 6-7%). The split kernel walks units x tiles with all warps, or (one CTA per unit) eight tiles at a time. The
// prefill form decodes the context (bytes of f16), walks the KV blocks of a work item's part and, where there are several
// parts, writes and merges their records.
// Measured split / prefill: 9/3 heads at d = 64, 4000 rows: 64 tokens 16.1 / 20.4, 128 tokens 20.6 / 21.4; 32/32 heads,
// 4 x 4000 rows: 16 tokens 30 / 76, 64 tokens 88 / 76; 32/8 heads at d = 128, 4 x 4000 rows: 16 tokens 50 / 81, 32 tokens
// 91 / 81. The split kernel's results have f32 accuracy besides.
bool kv4_split_faster(const alpaca_kv4_attn_desc& d) {
    const bool d64 = d.head_dim == 64;
    const SplitPlan p = split_plan(d);
    const double ctx = static_cast<double>(d.start_position) + d.tokens, tiles = std::ceil(ctx * d.head_dim / 4096.0);
    const double split = p.cta_units ? (d64 ? 4.0 : 3.7) + (d64 ? 3.2 : 3.9) * std::ceil(tiles / 8.0)
                                     : (d64 ? 9.8 : 11.1) + (d64 ? 2.9 : 3.4) * static_cast<double>(p.units) * tiles / (8.0 * kSms);
    const double blocks = std::ceil(ctx / (d64 ? 128.0 : 64.0)), items = static_cast<double>(d.n_seqs) * d.n_heads * std::ceil(d.tokens / 256.0);
    const double parts = std::max(1.0, std::min({8.0, std::floor(kSms / items), std::floor(blocks / 4.0)}));
    const double walk = std::ceil(blocks / parts) * std::ceil(items * parts / kSms);
    const double cache_mb = 4e-6 * d.n_seqs * ctx * d.n_kv_heads * d.head_dim;
    const double record_mb = 8e-6 * d.n_seqs * d.n_heads * static_cast<double>(d.tokens) * d.head_dim * parts;
    const double prefill = (d64 ? 6.2 : 6.8) + (d64 ? 1.24 : 1.0) * walk + (d64 ? 0.235 : 0.18) * cache_mb +
                           (parts > 1.0 ? (d64 ? 4.8 : 6.2) + (d64 ? 0.65 : 0.37) * record_mb : 0.0);
    return split <= prefill;
}

size_t kv4_workspace_bytes(const alpaca_kv4_attn_desc& d, alpaca_attn_kernel kind) {
    if (kind == ALPACA_ATTN_DECODE_SPLIT) {
        const SplitPlan p = split_plan(d);
        return p.combine ? plan_bytes(p) + sizeof(float) * (p.chunks + p.units) * p.rows_per_unit() * (d.head_dim + 4) : 0;
    }
    if (kind == ALPACA_ATTN_PREFILL_TC) {
        const ChunkPlan p = chunk_plan(d, nullptr);
        return 2 * p.cache_bytes + prefill_workspace_bytes(p.attn);
    }
    return 0;
}

cudaError_t launch_kv4_attention(const alpaca_kv4_attn_desc& d, alpaca_attn_kernel kind, float scale, void* ws, size_t ws_bytes,
                                 unsigned* err, int num_sms, cudaStream_t s) {
    if (kind == ALPACA_ATTN_PREFILL_TC) {
        const ChunkPlan p = chunk_plan(d, ws);
        const bool varlen = (d.flags & ALPACA_ATTN_FLAG_VARLEN) != 0;
        alpaca_kv4_read_desc r = {};
        r.n_seqs = d.n_seqs;
        r.n_kv_heads = d.n_kv_heads;
        r.head_dim = d.head_dim;
        r.n_rows = varlen ? d.max_ctx_len : d.start_position + d.tokens;
        r.out_dtype = ALPACA_F16;
        r.cache = d.cache;
        r.k_out = const_cast<void*>(p.attn.k);
        r.v_out = const_cast<void*>(p.attn.v);
        r.out_row_stride = p.attn.kv_row_stride;
        r.out_seq_stride = p.attn.kv_seq_stride;
        const cudaError_t e = launch_kv4_read(r, varlen ? d.start_positions : nullptr, varlen ? d.q_offsets : nullptr, err, s);
        if (e != cudaSuccess) return e;
        Call c{&p.attn, scale, err, static_cast<uint8_t*>(ws) + 2 * p.cache_bytes, ws_bytes - 2 * p.cache_bytes, num_sms};
        return launch_prefill(c, s);
    }
    Kv4Args a;
    a.q = d.q;
    a.q_token_stride = d.q_token_stride;
    a.q_seq_stride = d.q_seq_stride;
    a.out = d.out;
    a.out_token_stride = d.out_token_stride;
    a.out_seq_stride = d.out_seq_stride;
    a.q_f16 = d.q_dtype == ALPACA_F16;
    a.out_f16 = d.out_dtype == ALPACA_F16;
    a.c = kv4_view(d.cache);
    a.ctx_lens = d.ctx_lens;
    a.uniform_len = d.start_position + d.tokens;
    a.max_len = max_context(d);
    a.n_seqs = d.n_seqs;
    a.n_heads = d.n_heads;
    a.n_kv_heads = d.n_kv_heads;
    a.tokens = d.tokens;
    a.group = d.n_heads / d.n_kv_heads;
    a.plan = nullptr;
    a.partial = nullptr;
    a.scale = scale;
    a.err = err;
    if (kind == ALPACA_ATTN_DECODE_SPLIT) {
        const SplitPlan p = split_plan(d);
        a.q_rows = p.q_rows;
        a.q_groups = p.q_groups;
        a.chunks = p.chunks;
        if (p.combine) {
            a.plan = static_cast<int2*>(ws);
            a.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + plan_bytes(p));
        }
        return d.head_dim == 128 ? launch_split<128>(a, p, s) : launch_split<64>(a, p, s);
    }
    a.q_rows = a.q_groups = 0;
    a.chunks = 0;
    const int64_t rows = static_cast<int64_t>(d.n_seqs) * d.tokens * d.n_heads;
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg =
        pdl_config(dim3(static_cast<unsigned>((rows + kGenWarps - 1) / kGenWarps), 1, 1), 32 * kGenWarps, 0, s, &attr);
    return cudaLaunchKernelEx(&cfg, kv4_general_kernel, a, d.head_dim);
}

}  // namespace alpaca
