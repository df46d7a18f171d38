// attn_kv4.cu — attention over the 4-bit KV cache (kv4.cuh).
//
//   split kernel   one resident wave of warps ("workers"). A unit is one KV head of one sequence with up to 4 NT of its query
//                  rows (a query row = one head of one token; the G heads of every token of the call share the KV head),
//                  cut into tiles of 64 (head_dim 64) or 32 (head_dim 128) cache rows; the units' tiles lie in one row and
//                  every worker takes an equal run of them, with its own ring of bulk copies and its own running softmax.
//                  A unit inside one run is finished there; the parts of one that crosses runs go to records.
//                  Both products run on mma.sync m16n8k16 with the cache as the 16-row operand: S^T = K Q^T (16 keys x 8
//                  columns) and O^T = V^T P^T (16 channels x 8 columns). A column pair is one query row: f16 high part and
//                  f16 remainder of q or p, so the f32 sum of the pair's two accumulators carries ~22 bits. Scores,
//                  maxima and sums of a query row then live in the same lanes as its outputs (lane % 4).
//                  K: codes enter as f16 denormals (c * 2^-24, one AND per pair; codes in bits 4-7 count 16 times, which
//                  the queries' halves undo), exact; a block's step and zero point are applied to the block's partial
//                  score in f32: s = sum_b step_b (acc_b - zero_b * qsum_b).
//                  V: (c - zero) * step is exact in f16 (kv4.cuh), decoded for two keys side by side.
//                  P moves from accumulator to operand layout with movmatrix (no shared memory).
//   combine        one CTA per query row: rescales the parts' (m, l, acc) records to the common maximum and normalises.
//   general kernel fp32 SIMT, any head_dim that is a multiple of 32 up to 256: one warp per query row.
//
// Scores are in log2 units. A row whose context is empty, or a token that sees no row, gives zeros.
#include <algorithm>
#include <cmath>

#include "kv4.cuh"

namespace alpaca {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
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
    int64_t* plan;   // [0] tiles per worker, [1 + unit] first tile of the unit
    float* partial;  // [worker][2][query row of the group][d + 4]: accumulators, m (log2 units), l
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
    static constexpr int HROW = D / 16;           // header bytes of a row
    static constexpr int CB = TK * CROW;          // 2048
    static constexpr int HB = TK * HROW;          // 256
    static constexpr int STAGE = 2 * (CB + HB);   // K codes, V codes, K headers, V headers
    static constexpr int WX = D / 64;             // V words per lane and row
    static constexpr int REC = D + 4;             // floats of a partial record
    static constexpr int DEC = 2048;              // bytes of a warp's decoded headers: 1 KB for K, 1 KB for V
    static constexpr int WARP = kStages * STAGE + DEC;
    // Entry of block b of key pair t of 8-row half `half8` of a tile. The two blocks that a quarter warp reads at once (b = 0, 1
    // at head_dim 64; x and x + 2 at 128) are adjacent, so the 16-byte reads fall in different banks.
    __host__ __device__ static constexpr int vd_index(int half8, int b, int t) {
        return D == 64 ? (half8 * 2 + b) * 4 + t : ((half8 * 2 + (b & 1)) * 2 + (b >> 1)) * 4 + t;
    }
};

// Untiled bulk copy global -> shared completing `bytes` on `bar` (16-byte aligned ends and size; no multicast).
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
                 "r"(bytes), "r"(smem_u32(bar))
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
// x and y each as f16 value (low half) and the f16 of what that leaves (high half): x in r0, y in r1.
__device__ __forceinline__ void split_f16_pair(float x, float y, uint32_t& r0, uint32_t& r1) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    r0 = __byte_perm(as_u32(h), as_u32(l), 0x5410);
    r1 = __byte_perm(as_u32(h), as_u32(l), 0x7632);
}

// Starts the copies of rows [row0, min(row0 + TK, row_end)) of one KV head into a stage (one lane). A tile is one run of
// bytes per plane, or one per pool block it touches; headers are copied in multiples of 16 bytes (rows up to the next
// multiple of 4, which the cache's 16-row granularity covers) and the surplus is ignored by the reader. A table entry
// outside the pool reads as zero: its rows' headers are cleared.
template <int D>
__device__ __forceinline__ void load_tile(const Kv4Args& a, int seq, int kvh, int row0, int row_end, uint8_t* stage, uint64_t* bar) {
    using Ge = Kv4Geo<D>;
    const int n = min(Ge::TK, row_end - row0);
    const uint32_t st = smem_u32(stage);
    if (!a.c.block_table) {
        const int64_t code = seq * a.c.code_unit_stride + kvh * a.c.code_head_stride + static_cast<int64_t>(row0) * Ge::CROW;
        const int64_t scale = seq * a.c.scale_unit_stride + kvh * a.c.scale_head_stride + static_cast<int64_t>(row0) * Ge::NB;
        const uint32_t cb = n * Ge::CROW, hb = (n * Ge::HROW + 15) & ~15;
        mbar_arrive_expect_tx(bar, 2 * (cb + hb));
        bulk_load(st, a.c.k_codes + code, cb, bar);
        bulk_load(st + 2 * Ge::CB, a.c.k_scales + scale, hb, bar);
        bulk_load(st + Ge::CB, a.c.v_codes + code, cb, bar);
        bulk_load(st + 2 * Ge::CB + Ge::HB, a.c.v_scales + scale, hb, bar);
        return;
    }
    uint32_t total = 0;
    for (int r = 0; r < n;) {  // the copies may land before the barrier expects them: its count stays pending until the arrive
        const int row = row0 + r, b = row / a.c.rows, in = row - b * a.c.rows, m = min(n - r, a.c.rows - in);
        const int blk = b < a.c.max_blocks ? a.c.block_table[static_cast<int64_t>(seq) * a.c.max_blocks + b] : -1;
        const uint32_t cb = m * Ge::CROW, hb = (m * Ge::HROW + 15) & ~15;
        if (blk >= 0 && blk < a.c.pool_blocks) {
            const int64_t code = blk * a.c.code_unit_stride + kvh * a.c.code_head_stride + static_cast<int64_t>(in) * Ge::CROW;
            const int64_t scale = blk * a.c.scale_unit_stride + kvh * a.c.scale_head_stride + static_cast<int64_t>(in) * Ge::NB;
            bulk_load(st + r * Ge::CROW, a.c.k_codes + code, cb, bar);
            bulk_load(st + 2 * Ge::CB + r * Ge::HROW, a.c.k_scales + scale, hb, bar);
            bulk_load(st + Ge::CB + r * Ge::CROW, a.c.v_codes + code, cb, bar);
            bulk_load(st + 2 * Ge::CB + Ge::HB + r * Ge::HROW, a.c.v_scales + scale, hb, bar);
            total += 2 * (cb + hb);
        } else {
            atomicOr(a.err, kDevErrBadIndex);
            uint4* h = reinterpret_cast<uint4*>(stage + 2 * Ge::CB + r * Ge::HROW);
            for (uint32_t i = 0; i < hb / 16; i++) h[i] = h[i + Ge::HB / 16] = make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();  // before a later bulk copy into this stage
        }
        r += m;
    }
    mbar_arrive_expect_tx(bar, total);
}

// A tile's headers decoded once per warp: per key the (step, zero * 2^-24) of its K blocks in f32, and per pair of keys that
// meet in a V operand register the pair's Kv4Pair for each block. Rows at or past `n` get step 0.
template <int D>
__device__ __forceinline__ void decode_headers(const uint8_t* stage, float4* s_kd, uint4* s_vd, int n, int lane) {
    using Ge = Kv4Geo<D>;
    constexpr int WPK = Ge::NB / 2;  // header words per key
    const uint32_t* kh = reinterpret_cast<const uint32_t*>(stage + 2 * Ge::CB);
    const uint32_t* vh = kh + Ge::HB / 4;
#pragma unroll
    for (int k = 0; k < Ge::HB / 128; k++) {
        const int i = lane + 32 * k;
        const uint32_t h = i / WPK < n ? kh[i] : 0u;
        const float2 d = __half22float2(as_half2(h & 0xFFF0FFF0u)), z = __half22float2(as_half2(h & 0x000F000Fu));
        s_kd[i] = make_float4(d.x, z.x, d.y, z.y);
    }
    // pair i of the tile: rows 2t, 2t + 1 of half h of group gr (in operand order, see compute_tile); lane's word of it
    const int pair = lane / WPK, word = lane % WPK, t = pair & 3, base = (pair >> 2) * 8;
    const int ke = base + ((2 * t) ^ (t >> 1)), ko = base + ((2 * t + 1) ^ (t >> 1));
    const uint32_t he = ke < n ? vh[ke * WPK + word] : 0u, ho = ko < n ? vh[ko * WPK + word] : 0u;
    const Kv4Pair p0 = kv4_pair(__byte_perm(he, ho, 0x5410)), p1 = kv4_pair(__byte_perm(he, ho, 0x7632));
    s_vd[Kv4Geo<D>::vd_index(pair >> 2, 2 * word, t)] = make_uint4(as_u32(p0.d), as_u32(p0.z), as_u32(p0.d16), as_u32(p0.z16));
    s_vd[Kv4Geo<D>::vd_index(pair >> 2, 2 * word + 1, t)] = make_uint4(as_u32(p1.d), as_u32(p1.z), as_u32(p1.d16), as_u32(p1.z16));
}

// State of the query rows a lane keeps: nt-th row = 4 nt + lane % 4 of the CTA's group.
template <int D, int NT>
struct RowState {
    float qsum[NT][D / 32];  // sum of a block's (scaled) queries
    float fs[NT];            // raw score -> log2 units
    float m[NT], thr[NT], negm[NT], l[NT];
    int lim[NT];             // visible rows
    float o[NT][D / 64][8];  // accumulators of the lane's eight channels per V word
};

template <int D, int NT>
__device__ __forceinline__ void compute_tile(const uint8_t* st, const float4* s_kd, const uint4* s_vd, int row0, int min_lim,
                                             const uint32_t (&qb)[NT][D / 32][4], RowState<D, NT>& s, int g, int t) {
    using Ge = Kv4Geo<D>;
    constexpr int NB = Ge::NB, GR = Ge::GR, WX = Ge::WX;
    const uint8_t* s_kc = st;
    const uint8_t* s_vc = st + Ge::CB;
    // Rows of a 16-row group in operand order: operand row r < 8 is key r ^ (r >> 2), r >= 8 key 8 more. Any order serves
    // (keys meet only in sums); this one keeps both the K and the V reads free of bank conflicts.
    const int kg = g ^ (g >> 2), ke = (2 * t) ^ (t >> 1), ko = (2 * t + 1) ^ (t >> 1);

    float r[GR][2][NT];
#pragma unroll
    for (int gr = 0; gr < GR; gr++) {
        uint32_t w[2][NB];
        float dk[2][NB], zk[2][NB];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int key = 16 * gr + 8 * h + kg;
            const uint8_t* p = s_kc + key * Ge::CROW;
            if (D == 64) {
                const uint2 u = *reinterpret_cast<const uint2*>(p + 8 * t);
                w[h][0] = u.x;
                w[h][1] = u.y;
            } else {
                const uint4 u = *reinterpret_cast<const uint4*>(p + 16 * t);
                w[h][0] = u.x; w[h][1] = u.y; w[h][NB - 2] = u.z; w[h][NB - 1] = u.w;
            }
#pragma unroll
            for (int i = 0; i < NB / 2; i++) {
                const float4 u = s_kd[key * (NB / 2) + i];
                dk[h][2 * i] = u.x; zk[h][2 * i] = u.y; dk[h][2 * i + 1] = u.z; zk[h][2 * i + 1] = u.w;
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++) r[gr][0][nt] = r[gr][1][nt] = 0.f;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const uint32_t a0[4] = {w[0][b] & 0x000F000Fu, w[1][b] & 0x000F000Fu, w[0][b] & 0x00F000F0u, w[1][b] & 0x00F000F0u};
            const uint32_t x0 = w[0][b] >> 8, x1 = w[1][b] >> 8;
            const uint32_t a1[4] = {x0 & 0x000F000Fu, x1 & 0x000F000Fu, x0 & 0x00F000F0u, x1 & 0x00F000F0u};
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float acc[4];
                mma16816_first(acc, a0, qb[nt][b][0], qb[nt][b][1]);
                mma16816(acc, a1, qb[nt][b][2], qb[nt][b][3]);
                r[gr][0][nt] = fmaf(dk[0][b], fmaf(-zk[0][b], s.qsum[nt][b], acc[0] + acc[1]), r[gr][0][nt]);
                r[gr][1][nt] = fmaf(dk[1][b], fmaf(-zk[1][b], s.qsum[nt][b], acc[2] + acc[3]), r[gr][1][nt]);
            }
        }
    }
    if (row0 + Ge::TK > min_lim) {  // some row of the tile is hidden from some query row
#pragma unroll
        for (int gr = 0; gr < GR; gr++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
                    if (row0 + 16 * gr + 8 * h + kg >= s.lim[nt]) r[gr][h][nt] = -INFINITY;
    }

    uint32_t pb[GR][2][NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        float mx = r[0][0][nt];
#pragma unroll
        for (int gr = 0; gr < GR; gr++) mx = fmax3(mx, r[gr][0][nt], r[gr][1][nt]);
        if (__any_sync(0xffffffffu, mx > s.thr[nt])) {  // the reference maximum moves (rare after the first tile)
#pragma unroll
            for (int o = 4; o <= 16; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float mn = fmaxf(s.m[nt], mx);
            const float alpha = s.m[nt] == -INFINITY ? 0.f : ex2_approx(s.fs[nt] * (s.m[nt] - mn));
            s.l[nt] *= alpha;
#pragma unroll
            for (int x = 0; x < WX; x++)
#pragma unroll
                for (int e = 0; e < 8; e++) s.o[nt][x][e] *= alpha;
            s.m[nt] = mn;
            s.thr[nt] = mn + kMaxSlack / s.fs[nt];
            s.negm[nt] = mn == -INFINITY ? kPShift : kPShift - s.fs[nt] * mn;
        }
#pragma unroll
        for (int gr = 0; gr < GR; gr++) {
            const float p0 = ex2_approx(fmaf(s.fs[nt], r[gr][0][nt], s.negm[nt]));  // hidden rows: 2^-inf = 0
            const float p1 = ex2_approx(fmaf(s.fs[nt], r[gr][1][nt], s.negm[nt]));
            s.l[nt] += p0;
            s.l[nt] += p1;
            uint32_t u0, u1;
            split_f16_pair(p0, p1, u0, u1);
            pb[gr][0][nt] = movmatrix(u0);
            pb[gr][1][nt] = movmatrix(u1);
        }
    }

#pragma unroll
    for (int x = 0; x < WX; x++) {
        float acc[4][NT][4];
        const int blk = (WX * g + x) % NB;  // block of word WX g + x of a row
#pragma unroll
        for (int gr = 0; gr < GR; gr++) {
            uint32_t w[4];
            Kv4Pair p[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint4 u = s_vd[Ge::vd_index(2 * gr + h, blk, t)];
                p[h].d = as_half2(u.x);
                p[h].z = as_half2(u.y);
                p[h].d16 = as_half2(u.z);
                p[h].z16 = as_half2(u.w);
                const uint8_t* r0 = s_vc + (16 * gr + 8 * h + ke) * Ge::CROW + 4 * (WX * g + x);
                const uint8_t* r1 = s_vc + (16 * gr + 8 * h + ko) * Ge::CROW + 4 * (WX * g + x);
                w[2 * h] = *reinterpret_cast<const uint32_t*>(r0);
                w[2 * h + 1] = *reinterpret_cast<const uint32_t*>(r1);
            }
            const uint32_t lo0 = __byte_perm(w[0], w[1], 0x5410), hi0 = __byte_perm(w[0], w[1], 0x7632);
            const uint32_t lo1 = __byte_perm(w[2], w[3], 0x5410), hi1 = __byte_perm(w[2], w[3], 0x7632);
#pragma unroll
            for (int m = 0; m < 4; m++) {  // channels 2m and 2m + 1 of the word in operand rows g and g + 8
                const uint32_t u0 = (m < 2 ? lo0 : hi0) >> (8 * (m & 1)), u1 = (m < 2 ? lo1 : hi1) >> (8 * (m & 1));
                const uint32_t va[4] = {kv4_lo(u0, p[0]), kv4_hi(u0, p[0]), kv4_lo(u1, p[1]), kv4_hi(u1, p[1])};
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    if (gr == 0) mma16816_first(acc[m][nt], va, pb[gr][0][nt], pb[gr][1][nt]);
                    else mma16816(acc[m][nt], va, pb[gr][0][nt], pb[gr][1][nt]);
                }
            }
        }
        // a tile's sums are added in f32 here: long chains of MMA accumulation lose low bits one way
#pragma unroll
        for (int m = 0; m < 4; m++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                s.o[nt][x][2 * m] += acc[m][nt][0] + acc[m][nt][1];
                s.o[nt][x][2 * m + 1] += acc[m][nt][2] + acc[m][nt][3];
            }
    }
}

// Tiles of a (sequence, KV head, query group) unit: an empty context counts one, so that its zeros are written.
template <int D>
__device__ __forceinline__ int unit_tiles(int L) {
    return max(1, (L + Kv4Geo<D>::TK - 1) / Kv4Geo<D>::TK);
}

// The work of a call is its units' tiles in one row, sequence by sequence; worker (warp) w takes tiles [w C, (w + 1) C),
// C = ceil(tiles / workers), so that all workers of the one resident wave end together whatever the contexts are.
struct Range {
    int64_t begin, end, chunk;  // tiles
    int64_t first;              // first tile of the unit that `begin` lies in
    int seq, head_group;        // that unit: sequence, kv_head * q_groups + query group
    int L;                      // the sequence's context
};

template <int D>
__device__ __forceinline__ Range find_range(const Kv4Args& a, int64_t worker, int64_t workers, int lane) {
    Range r;
    const int64_t hg = static_cast<int64_t>(a.n_kv_heads) * a.q_groups;
    int64_t total = 0;
    if (a.ctx_lens) {
        for (int s = lane; s < a.n_seqs; s += 32) total += unit_tiles<D>(ctx_of(a, s));
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    } else {
        total = static_cast<int64_t>(a.n_seqs) * unit_tiles<D>(a.uniform_len);
    }
    total *= hg;
    r.chunk = (total + workers - 1) / workers;
    r.begin = worker * r.chunk;
    r.end = min(r.begin + r.chunk, total);
    if (r.begin >= r.end) return r;
    if (!a.ctx_lens) {
        const int t = unit_tiles<D>(a.uniform_len);
        const int64_t unit = r.begin / t;
        r.first = unit * t;
        r.seq = static_cast<int>(unit / hg);
        r.head_group = static_cast<int>(unit - r.seq * hg);
        r.L = a.uniform_len;
        return r;
    }
    int64_t before = 0;  // tiles (of all heads) before the chunk of 32 sequences
    for (int s0 = 0;; s0 += 32) {
        const int s = s0 + lane;
        const int L = s < a.n_seqs ? ctx_of(a, s) : 0;
        const int64_t mine = s < a.n_seqs ? unit_tiles<D>(L) * hg : 0;
        int64_t incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t x = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += x;
        }
        const unsigned past = __ballot_sync(0xffffffffu, before + incl > r.begin);
        if (past) {  // begin < total: some sequence holds it
            const int src = __ffs(past) - 1;
            r.seq = s0 + src;
            r.L = __shfl_sync(0xffffffffu, L, src);
            const int64_t start = before + __shfl_sync(0xffffffffu, incl - mine, src);
            const int t = unit_tiles<D>(r.L);
            r.head_group = static_cast<int>((r.begin - start) / t);
            r.first = start + static_cast<int64_t>(r.head_group) * t;
            return r;
        }
        before += __shfl_sync(0xffffffffu, incl, 31);
    }
}

// Query operands of the group's rows r0 .. r0 + 4 NT - 1. Column 2 q + {0, 1} of an operand is query row q's (high part,
// remainder): lane group g holds row g >> 1 and part g & 1; lane t the channels 32 b + 8 t + .. of every block, in the order of
// the K codes' nibbles. Rows are scaled by a power of two to [2^10, 2^11) so that neither part leaves f16's normal range.
template <int D, int NT>
__device__ __forceinline__ void load_queries(const Kv4Args& a, int seq, int kvh, int r0, int L, uint32_t (&qb)[NT][D / 32][4],
                                             RowState<D, NT>& s, int g, int t) {
    constexpr int NB = D / 32;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int rr = r0 + 4 * nt + (g >> 1);
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
                qb[nt][b][i] = __byte_perm(u, v, (g & 1) ? 0x7632 : 0x5410);
            }
        }
        s.m[nt] = s.thr[nt] = -INFINITY;
        s.negm[nt] = kPShift;
        s.l[nt] = 0.f;
        s.lim[nt] = L - a.tokens + 1 + (r0 + 4 * nt + t) / a.group;
#pragma unroll
        for (int x2 = 0; x2 < D / 64; x2++)
#pragma unroll
            for (int e = 0; e < 8; e++) s.o[nt][x2][e] = 0.f;
    }
}

// CTAs per SM that the registers and the shared memory are laid out for (one wave of workers is resident).
__host__ __device__ constexpr int ctas_per_sm(int D, int NT) { return NT == 4 ? 2 : (NT == 2 ? 3 : (D == 128 ? 4 : 5)); }

template <int D, int NT>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(D, NT)) kv4_split_kernel(const __grid_constant__ Kv4Args a) {
    using Ge = Kv4Geo<D>;
    constexpr int NB = Ge::NB, WX = Ge::WX, QR = 4 * NT;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ uint64_t s_bar[kWarps][kStages];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < kStages; i++) mbar_init(&s_bar[warp][i], 1);
        fence_barrier_init();
    }
    __syncwarp();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t worker = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
    Range r = find_range<D>(a, worker, static_cast<int64_t>(gridDim.x) * kWarps, lane);
    if (worker == 0 && lane == 0 && a.plan) a.plan[0] = r.chunk;
    uint8_t* ring = smem + warp * Ge::WARP;
    float4* s_kd = reinterpret_cast<float4*>(ring + kStages * Ge::STAGE);
    uint4* s_vd = reinterpret_cast<uint4*>(ring + kStages * Ge::STAGE + Ge::DEC / 2);
    const int64_t range_begin = r.begin;
    uint32_t count = 0;  // tiles consumed from the ring so far
    while (r.begin < r.end) {
        const int seq = r.seq, kvh = r.head_group / a.q_groups, qg = r.head_group - kvh * a.q_groups, L = r.L;
        const int r0 = qg * QR, r_last = min(r0 + QR, a.q_rows) - 1;
        const int ut = unit_tiles<D>(L), t0 = static_cast<int>(r.begin - r.first);
        const int t1 = static_cast<int>(min(static_cast<int64_t>(ut), t0 + (r.end - r.begin)));
        // rows that query row q sees: L - tokens + 1 + its token; the last one's bounds the rows worth reading
        const int min_lim = L - a.tokens + 1 + r0 / a.group;
        const int row_end = min(L, L - a.tokens + 1 + r_last / a.group);
        const int n = min(t1, row_end > 0 ? (row_end + Ge::TK - 1) / Ge::TK : 0) - t0;  // tiles with visible rows
        if (lane == 0) {
            for (int i = 0; i < min(kStages, n); i++)
                load_tile<D>(a, seq, kvh, (t0 + i) * Ge::TK, row_end, ring + ((count + i) % kStages) * Ge::STAGE,
                             &s_bar[warp][(count + i) % kStages]);
        }
        uint32_t qb[NT][NB][4];
        RowState<D, NT> s;
        load_queries<D, NT>(a, seq, kvh, r0, L, qb, s, g, t);
        for (int it = 0; it < n; it++, count++) {
            const int stage = count % kStages, row0 = (t0 + it) * Ge::TK;
            uint8_t* st = ring + stage * Ge::STAGE;
            int gone = 0;
            const AbortState ab{&gone, a.err, kWaitLimitNs};
            if (!__all_sync(0xffffffffu, mbar_wait(&s_bar[warp][stage], (count / kStages) & 1, ab))) {
                // given up (reported): none of this warp's copies may still be in flight when the CTA ends
                for (int j = 0; j < min(kStages, n - it); j++) {
                    int late = 0;
                    mbar_wait(&s_bar[warp][(count + j) % kStages], ((count + j) / kStages) & 1, AbortState{&late, a.err, kWaitLimitNs});
                }
                return;
            }
            decode_headers<D>(st, s_kd, s_vd, row_end - row0, lane);
            __syncwarp();
            compute_tile<D, NT>(st, s_kd, s_vd, row0, min_lim, qb, s, g, t);
            __syncwarp();  // every lane is done with the stage and the decoded headers
            if (lane == 0 && it + kStages < n)
                load_tile<D>(a, seq, kvh, row0 + kStages * Ge::TK, row_end, st, &s_bar[warp][stage]);
        }
        // A unit that lies wholly in this worker's range is finished here; else its part goes to a record: slot 0 for the part
        // that starts the range, slot 1 for one that starts within it.
        const bool whole = t1 - t0 == ut;
        if (t0 == 0 && lane == 0 && a.plan) a.plan[1 + (static_cast<int64_t>(seq) * a.n_kv_heads + kvh) * a.q_groups + qg] = r.first;
        float* rec0 = a.partial + (worker * 2 + (r.begin > range_begin ? 1 : 0)) * QR * Ge::REC;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float l = s.l[nt];
#pragma unroll
            for (int o = 4; o <= 16; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
            const int row = 4 * nt + t, rr = r0 + row;
            if (rr >= a.q_rows) continue;
            const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
            for (int x = 0; x < WX; x++) {
                const int ch = 32 * ((WX * g + x) % NB) + 8 * (g >> 1);
                float (&o)[8] = s.o[nt][x];
                if (whole) {
                    const int64_t at = seq * a.out_seq_stride + (rr / a.group) * a.out_token_stride +
                                       static_cast<int64_t>(kvh * a.group + rr % a.group) * D + ch;
#pragma unroll
                    for (int e = 0; e < 8; e++) o[e] = l == 0.f ? 0.f : o[e] * inv;
                    if (a.out_f16) {
                        *reinterpret_cast<uint4*>(static_cast<__half*>(a.out) + at) =
                            make_uint4(pack_half2(o[0], o[1]), pack_half2(o[2], o[3]), pack_half2(o[4], o[5]), pack_half2(o[6], o[7]));
                    } else {
                        float4* p = reinterpret_cast<float4*>(static_cast<float*>(a.out) + at);
                        p[0] = make_float4(o[0], o[1], o[2], o[3]);
                        p[1] = make_float4(o[4], o[5], o[6], o[7]);
                    }
                } else {
                    float4* p = reinterpret_cast<float4*>(rec0 + row * Ge::REC + ch);
                    p[0] = make_float4(o[0], o[1], o[2], o[3]);
                    p[1] = make_float4(o[4], o[5], o[6], o[7]);
                }
            }
            if (!whole && g == 0)
                *reinterpret_cast<float2*>(rec0 + row * Ge::REC + D) =
                    make_float2(s.m[nt] == -INFINITY ? -INFINITY : s.fs[nt] * s.m[nt], l);
        }
        r.begin += t1 - t0;
        if (r.begin >= r.end) break;
        r.first = r.begin;  // the next unit
        if (++r.head_group == a.n_kv_heads * a.q_groups) {
            r.head_group = 0;
            r.seq++;
            r.L = ctx_of(a, r.seq);
        }
    }
}

// ------------------------------------------------------------------------------------------------ combine

// One CTA per query row: its warps sum every fourth record of the row's unit, rescaled to the common maximum.
template <int D, int NT>
__global__ void __launch_bounds__(kThreads) kv4_combine_kernel(const __grid_constant__ Kv4Args a) {
    constexpr int EPL = D / 32, REC = Kv4Geo<D>::REC, QR = 4 * NT;
    __shared__ float s_acc[kWarps][D];
    __shared__ float s_ml[kWarps][2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // Every CTA waits for the split grid, so that a later launch which sees this grid complete sees the split kernel's
    // writes too.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int rr = blockIdx.x % a.q_rows, kvh = (blockIdx.x / a.q_rows) % a.n_kv_heads, seq = blockIdx.x / (a.q_rows * a.n_kv_heads);
    const int64_t chunk = a.plan[0], first = a.plan[1 + (static_cast<int64_t>(seq) * a.n_kv_heads + kvh) * a.q_groups + rr / QR];
    const int tiles = unit_tiles<D>(ctx_of(a, seq));
    const int64_t w0 = first / chunk, w1 = (first + tiles - 1) / chunk;
    if (w0 == w1) return;  // written by the split kernel
    const int n = static_cast<int>(w1 - w0) + 1;
    const auto record = [&](int i) {  // part i: in the first worker's slot 1 unless the unit starts that worker's range
        const int64_t w = w0 + i;
        return a.partial + ((w * 2 + (i == 0 && first > w0 * chunk ? 1 : 0)) * QR + rr % QR) * REC;
    };
    float m = -INFINITY;
    for (int i = warp + kWarps * lane; i < n; i += kWarps * 32) m = fmaxf(m, record(i)[D]);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float acc[EPL], l = 0.f;
#pragma unroll
    for (int e = 0; e < EPL; e++) acc[e] = 0.f;
#pragma unroll 4
    for (int i = warp; i < n; i += kWarps) {
        const float* p = record(i);
        const float2 ml = *reinterpret_cast<const float2*>(p + D);
        const float f = m == -INFINITY ? 1.f : ex2_approx(ml.x - m);
        l = fmaf(ml.y, f, l);
#pragma unroll
        for (int e = 0; e < EPL; e++) acc[e] = fmaf(p[lane + 32 * e], f, acc[e]);
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
    for (int w = 0; w < kWarps; w++) M = fmaxf(M, s_ml[w][0]);
    for (int col = threadIdx.x; col < D; col += kThreads) {
        float o = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            const float f = M == -INFINITY ? 1.f : ex2_approx(s_ml[w][0] - M);
            o = fmaf(s_acc[w][col], f, o);
            sum = fmaf(s_ml[w][1], f, sum);
        }
        store_out(a, seq, rr / a.group, kvh * a.group + rr % a.group, D, col, sum == 0.f ? 0.f : o / sum);
    }
}

// ------------------------------------------------------------------------------------------------ general kernel

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

// Query rows per worker (4 NT: the fewest that hold the call's rows per KV head, up to 16) and workers: one resident wave, or
// one per tile where the call has fewer (by its bound).
constexpr int kSms = 148;
struct SplitPlan {
    int nt, q_rows, q_groups;
    int64_t units, workers;
    bool combine;  // some unit may be split between workers
};
SplitPlan split_plan(const alpaca_kv4_attn_desc& d) {
    SplitPlan p;
    p.q_rows = d.tokens * (d.n_heads / d.n_kv_heads);
    p.nt = p.q_rows <= 4 ? 1 : (p.q_rows <= 8 ? 2 : 4);
    p.q_groups = (p.q_rows + 4 * p.nt - 1) / (4 * p.nt);
    p.units = static_cast<int64_t>(d.n_seqs) * d.n_kv_heads * p.q_groups;
    const int tk = 4096 / d.head_dim, tiles = std::max(1, (max_context(d) + tk - 1) / tk);
    p.workers = std::min<int64_t>(p.units * tiles, kSms * kWarps * ctas_per_sm(d.head_dim, p.nt));
    p.workers = (p.workers + kWarps - 1) / kWarps * kWarps;
    p.combine = tiles > 1;
    return p;
}
size_t round_up(size_t n, size_t m) { return (n + m - 1) / m * m; }
size_t plan_bytes(const SplitPlan& p) { return p.combine ? round_up(sizeof(int64_t) * (1 + p.units), 256) : 0; }

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

template <int D, int NT>
cudaError_t launch_split_nt(const Kv4Args& a, const SplitPlan& p, cudaStream_t s) {
    constexpr size_t smem = kWarps * Kv4Geo<D>::WARP;
    const auto fn = kv4_split_kernel<D, NT>;
    cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(fn), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    e = cudaFuncSetAttribute(reinterpret_cast<const void*>(fn), cudaFuncAttributePreferredSharedMemoryCarveout,
                             static_cast<int>(cudaSharedmemCarveoutMaxShared));
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg =
        pdl_config(dim3(static_cast<unsigned>(p.workers / kWarps), 1, 1), kThreads, smem, s, &attr);
    e = cudaLaunchKernelEx(&cfg, fn, a);
    if (e != cudaSuccess || !p.combine) return e;
    const unsigned rows = static_cast<unsigned>(a.n_seqs) * a.n_kv_heads * a.q_rows;
    const cudaLaunchConfig_t ccfg = pdl_config(dim3(rows, 1, 1), kThreads, 0, s, &attr);
    return cudaLaunchKernelEx(&ccfg, kv4_combine_kernel<D, NT>, a);
}

template <int D>
cudaError_t launch_split(const Kv4Args& a, const SplitPlan& p, cudaStream_t s) {
    return p.nt == 1   ? launch_split_nt<D, 1>(a, p, s)
           : p.nt == 2 ? launch_split_nt<D, 2>(a, p, s)
                       : launch_split_nt<D, 4>(a, p, s);
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

size_t kv4_workspace_bytes(const alpaca_kv4_attn_desc& d, alpaca_attn_kernel kind) {
    if (kind == ALPACA_ATTN_DECODE_SPLIT) {
        const SplitPlan p = split_plan(d);
        return p.combine ? plan_bytes(p) + sizeof(float) * p.workers * 2 * 4 * p.nt * (d.head_dim + 4) : 0;
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
        if (p.combine) {
            a.plan = static_cast<int64_t*>(ws);
            a.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + plan_bytes(p));
        }
        return d.head_dim == 128 ? launch_split<128>(a, p, s) : launch_split<64>(a, p, s);
    }
    a.q_rows = a.q_groups = 0;
    const int64_t rows = static_cast<int64_t>(d.n_seqs) * d.tokens * d.n_heads;
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg =
        pdl_config(dim3(static_cast<unsigned>((rows + kGenWarps - 1) / kGenWarps), 1, 1), 32 * kGenWarps, 0, s, &attr);
    return cudaLaunchKernelEx(&cfg, kv4_general_kernel, a, d.head_dim);
}

}  // namespace alpaca
