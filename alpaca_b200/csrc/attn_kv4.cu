// attn_kv4.cu — attention over the 4-bit KV cache (kv4.cuh).
//
//   split kernel   grid (kv_heads x query groups x splits, seqs), 4 warps. A CTA owns up to `split_rows` consecutive rows
//                  of one KV head of one sequence and serves 4 NT of its query rows (a query row = one head of one token;
//                  the G heads of every token of the call share the KV head). Each warp walks tiles of 64 (head_dim 64)
//                  or 32 (head_dim 128) rows with its own cp.async ring and its own running softmax; the warps meet once,
//                  at the end.
//                  Both products run on mma.sync m16n8k16 with the cache as the 16-row operand: S^T = K Q^T (16 keys x 8
//                  columns) and O^T = V^T P^T (16 channels x 8 columns). A column pair is one query row: f16 high part and
//                  f16 remainder of q or p, so the f32 sum of the pair's two accumulators carries ~22 bits. Scores,
//                  maxima and sums of a query row then live in the same lanes as its outputs (lane % 4).
//                  K: codes enter as f16 denormals (c * 2^-24, one AND per pair; codes in bits 4-7 count 16 times, which
//                  the queries' halves undo), exact; a block's step and zero point are applied to the block's partial
//                  score in f32: s = sum_b step_b (acc_b - zero_b * qsum_b).
//                  V: (c - zero) * step is exact in f16 (kv4.cuh), decoded for two keys side by side.
//                  P moves from accumulator to operand layout with movmatrix (no shared memory).
//   combine        one warp per query row: rescales the splits' (m, l, acc) records to the common maximum and normalises.
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
constexpr int kStages = 3;          // tiles in a warp's ring
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
    int max_splits, split_rows;
    float* partial;  // [seq][kv_head][query row][split][d + 4]: accumulators, m (log2 units), l
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
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t src_bytes) {  // the rest reads as zero
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
// x as its f16 value (low half) and the f16 of what that leaves (high half).
__device__ __forceinline__ uint32_t split_f16(float x) {
    const __half h = __float2half_rn(x);
    const __half l = __float2half_rn(x - __half2float(h));
    return static_cast<uint32_t>(__half_as_ushort(h)) | static_cast<uint32_t>(__half_as_ushort(l)) << 16;
}

// 16-byte chunk of a row's codes in shared memory: head_dim 128 rows swap chunk pairs by bit 1 of the row, so the V reads
// of a quarter warp (keys 0, 2, 5, 7 at one word) fall in different banks.
template <int D>
__device__ __forceinline__ int chunk_at(int row, int c) {
    return D == 128 ? (c ^ (((row >> 1) & 1) << 1)) : c;
}

// Where one 16-row group of a tile starts in global memory.
struct GroupBase {
    int64_t code, scale;
    bool ok;
};
template <int D>
__device__ __forceinline__ GroupBase group_base(const Kv4Args& a, int seq, int kvh, int row) {
    GroupBase b;
    int64_t unit;
    int r;
    b.ok = kv4_locate(a.c, seq, row, a.err, unit, r);  // a group never leaves its block: rows per block are a multiple of 16
    b.code = b.ok ? unit * a.c.code_unit_stride + kvh * a.c.code_head_stride + static_cast<int64_t>(r) * Kv4Geo<D>::CROW : 0;
    b.scale = b.ok ? unit * a.c.scale_unit_stride + kvh * a.c.scale_head_stride + static_cast<int64_t>(r) * Kv4Geo<D>::NB : 0;
    return b;
}

// Copies rows [row0, min(row0 + TK, row_end)) of one KV head into a stage; the rows past them read as zero (step 0).
template <int D>
__device__ __forceinline__ void load_tile(const Kv4Args& a, int seq, int kvh, int row0, int row_end, uint32_t stage, int lane) {
    using Ge = Kv4Geo<D>;
    constexpr int CPR = Ge::CROW / 16;  // chunks per row
    const int n = row_end - row0;
    GroupBase mine;
    mine.code = mine.scale = 0;
    mine.ok = false;
    if (lane < Ge::GR && 16 * lane < n) mine = group_base<D>(a, seq, kvh, row0 + 16 * lane);
#pragma unroll
    for (int k = 0; k < Ge::CB / 512; k++) {
        const int i = lane + 32 * k, row = i / CPR, c = i % CPR;
        const int gr = (32 * k / CPR) / 16;  // the group of this step's rows (the same for all lanes)
        const int64_t base = __shfl_sync(0xffffffffu, mine.code, gr);
        const bool ok = __shfl_sync(0xffffffffu, static_cast<int>(mine.ok), gr) && row < n;
        const int64_t off = base + (ok ? (row - 16 * gr) * Ge::CROW + 16 * c : 0);
        const uint32_t dst = stage + row * Ge::CROW + 16 * chunk_at<D>(row, c);
        cp_async16(dst, a.c.k_codes + off, ok ? 16u : 0u);
        cp_async16(dst + Ge::CB, a.c.v_codes + off, ok ? 16u : 0u);
    }
    {  // headers: lanes 0-15 K, 16-31 V, RPC rows each
        constexpr int RPC = 16 / Ge::HROW;
        const int c = lane & 15, row = c * RPC, gr = row / 16;
        const int64_t base = __shfl_sync(0xffffffffu, mine.scale, gr);
        const bool ok = __shfl_sync(0xffffffffu, static_cast<int>(mine.ok), gr);
        const int bytes = ok ? min(max((n - row) * Ge::HROW, 0), 16) : 0;
        const uint16_t* src = (lane < 16 ? a.c.k_scales : a.c.v_scales) + base + (bytes > 0 ? (row - 16 * gr) * Ge::NB : 0);
        cp_async16(stage + 2 * Ge::CB + (lane < 16 ? 0 : Ge::HB) + 16 * c, src, static_cast<uint32_t>(bytes));
    }
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
__device__ __forceinline__ void compute_tile(const uint8_t* st, int row0, int min_lim, const uint32_t (&qb)[NT][D / 32][4],
                                             RowState<D, NT>& s, int g, int t) {
    using Ge = Kv4Geo<D>;
    constexpr int NB = Ge::NB, GR = Ge::GR, WX = Ge::WX;
    const uint8_t* s_kc = st;
    const uint8_t* s_vc = st + Ge::CB;
    const uint8_t* s_kh = st + 2 * Ge::CB;
    const uint8_t* s_vh = s_kh + Ge::HB;
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
            uint32_t hd[NB / 2];
            if (D == 64) {
                const uint2 u = *reinterpret_cast<const uint2*>(p + 8 * t);
                w[h][0] = u.x;
                w[h][1] = u.y;
                hd[0] = *reinterpret_cast<const uint32_t*>(s_kh + key * Ge::HROW);
            } else {
                const uint4 u = *reinterpret_cast<const uint4*>(p + 16 * chunk_at<D>(key, t));
                w[h][0] = u.x; w[h][1] = u.y; w[h][NB - 2] = u.z; w[h][NB - 1] = u.w;
                const uint2 v = *reinterpret_cast<const uint2*>(s_kh + key * Ge::HROW);
                hd[0] = v.x;
                hd[NB / 2 - 1] = v.y;
            }
#pragma unroll
            for (int i = 0; i < NB / 2; i++) {
                const float2 d2 = __half22float2(as_half2(hd[i] & 0xFFF0FFF0u));
                const float2 z2 = __half22float2(as_half2(hd[i] & 0x000F000Fu));  // zero point * 2^-24
                dk[h][2 * i] = d2.x;
                dk[h][2 * i + 1] = d2.y;
                zk[h][2 * i] = z2.x;
                zk[h][2 * i + 1] = z2.y;
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
                float acc[4] = {0.f, 0.f, 0.f, 0.f};
                mma16816(acc, a0, qb[nt][b][0], qb[nt][b][1]);
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
        for (int gr = 0; gr < GR; gr++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const float p = ex2_approx(fmaf(s.fs[nt], r[gr][h][nt], s.negm[nt]));  // hidden rows: 2^-inf = 0
                s.l[nt] += p;
                pb[gr][h][nt] = movmatrix(split_f16(p));
            }
    }

#pragma unroll
    for (int x = 0; x < WX; x++) {
        float acc[4][NT][4];
#pragma unroll
        for (int m = 0; m < 4; m++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++) acc[m][nt][0] = acc[m][nt][1] = acc[m][nt][2] = acc[m][nt][3] = 0.f;
        // word WX g + x of a row: block (WX g + x) % NB; its header among the row's
        const int blk = (WX * g + x) % NB;
#pragma unroll
        for (int gr = 0; gr < GR; gr++) {
            uint32_t w[4], hd[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int key = 16 * gr + 8 * (i >> 1) + ((i & 1) ? ko : ke);
                const uint8_t* p = s_vc + key * Ge::CROW;
                w[i] = D == 64 ? *reinterpret_cast<const uint32_t*>(p + 4 * g)
                               : *reinterpret_cast<const uint32_t*>(p + 16 * chunk_at<D>(key, g >> 1) + 8 * (g & 1) + 4 * x);
                hd[i] = *reinterpret_cast<const uint16_t*>(s_vh + key * Ge::HROW + 2 * blk);
            }
            const Kv4Pair p0 = kv4_pair(hd[0] | hd[1] << 16), p1 = kv4_pair(hd[2] | hd[3] << 16);
            const uint32_t lo0 = __byte_perm(w[0], w[1], 0x5410), hi0 = __byte_perm(w[0], w[1], 0x7632);
            const uint32_t lo1 = __byte_perm(w[2], w[3], 0x5410), hi1 = __byte_perm(w[2], w[3], 0x7632);
#pragma unroll
            for (int m = 0; m < 4; m++) {  // channels 2m and 2m + 1 of the word in operand rows g and g + 8
                const uint32_t u0 = (m < 2 ? lo0 : hi0) >> (8 * (m & 1)), u1 = (m < 2 ? lo1 : hi1) >> (8 * (m & 1));
                const uint32_t va[4] = {kv4_lo(u0, p0), kv4_hi(u0, p0), kv4_lo(u1, p1), kv4_hi(u1, p1)};
#pragma unroll
                for (int nt = 0; nt < NT; nt++) mma16816(acc[m][nt], va, pb[gr][0][nt], pb[gr][1][nt]);
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

template <int D, int NT>
__global__ void __launch_bounds__(kThreads) kv4_split_kernel(const __grid_constant__ Kv4Args a) {
    using Ge = Kv4Geo<D>;
    constexpr int NB = Ge::NB, WX = Ge::WX, QR = 4 * NT;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ __align__(16) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int kvh = blockIdx.x % a.n_kv_heads, rest = blockIdx.x / a.n_kv_heads;
    const int qg = rest % a.q_groups, split = rest / a.q_groups, seq = blockIdx.y;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int L = ctx_of(a, seq);
    const int nsplits = max(1, (L + a.split_rows - 1) / a.split_rows);
    if (split >= nsplits) return;
    const int first_row = split * a.split_rows;
    const int r0 = qg * QR, r_last = min(r0 + QR, a.q_rows) - 1;
    // rows that query row r sees: L - tokens + 1 + its token
    const int min_lim = L - a.tokens + 1 + r0 / a.group;
    const int row_end = min(min(L, first_row + a.split_rows), L - a.tokens + 1 + r_last / a.group);
    const int ntiles = row_end > first_row ? (row_end - first_row + Ge::TK - 1) / Ge::TK : 0;

    uint8_t* ring = smem + warp * (kStages * Ge::STAGE);
    const uint32_t ring_u32 = smem_u32(ring);
#pragma unroll
    for (int i = 0; i < kStages - 1; i++) {
        const int tile = warp + kWarps * i;
        if (tile < ntiles)
            load_tile<D>(a, seq, kvh, first_row + tile * Ge::TK, row_end, ring_u32 + i * Ge::STAGE, lane);
        cp_async_commit();
    }

    // Query operands. Column 2 q + {0, 1} of an operand is query row q's (high part, remainder): lane group g holds row
    // g >> 1 and part g & 1; lane t the channels 32 b + 8 t + .. of every block, in the order of the K codes' nibbles.
    // Rows are scaled by a power of two to [2^10, 2^11) so that neither part leaves f16's normal range.
    uint32_t qb[NT][NB][4];
    RowState<D, NT> s;
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
                const uint32_t u = split_f16(x[b][i] * ((i & 1) ? 0.0625f : 1.f));
                const uint32_t v = split_f16(x[b][i + 4] * ((i & 1) ? 0.0625f : 1.f));
                qb[nt][b][i] = __byte_perm(u, v, (g & 1) ? 0x7632 : 0x5410);
            }
        }
        s.m[nt] = s.thr[nt] = -INFINITY;
        s.negm[nt] = kPShift;
        s.l[nt] = 0.f;
        s.lim[nt] = L - a.tokens + 1 + (r0 + 4 * nt + t) / a.group;
#pragma unroll
        for (int x2 = 0; x2 < WX; x2++)
#pragma unroll
            for (int e = 0; e < 8; e++) s.o[nt][x2][e] = 0.f;
    }

    for (int tile = warp, it = 0; tile < ntiles; tile += kWarps, it++) {
        cp_async_wait<kStages - 2>();
        __syncwarp();  // the tile has landed for every lane, and every lane is done with the stage refilled below
        const int next = tile + kWarps * (kStages - 1);
        if (next < ntiles)
            load_tile<D>(a, seq, kvh, first_row + next * Ge::TK, row_end,
                         ring_u32 + ((it + kStages - 1) % kStages) * Ge::STAGE, lane);
        cp_async_commit();
        compute_tile<D, NT>(ring + (it % kStages) * Ge::STAGE, first_row + tile * Ge::TK, min_lim, qb, s, g, t);
    }
    cp_async_wait<0>();
    __syncthreads();  // every warp is done with its ring: the records below lie over it

    // Records of the warps: [warp][query row][d] accumulators, [warp][query row] m, l.
    float* s_o = reinterpret_cast<float*>(smem);
    float* s_m = s_o + kWarps * QR * D;
    float* s_l = s_m + kWarps * QR;
    static_assert(sizeof(float) * kWarps * QR * (D + 2) <= kWarps * kStages * Ge::STAGE, "records must fit the rings");
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        float l = s.l[nt];
#pragma unroll
        for (int o = 4; o <= 16; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        const int row = warp * QR + 4 * nt + t;
        if (g == 0) {
            s_m[row] = s.m[nt] == -INFINITY ? -INFINITY : s.fs[nt] * s.m[nt];
            s_l[row] = l;
        }
#pragma unroll
        for (int x = 0; x < WX; x++) {
            const int ch = 32 * ((WX * g + x) % NB) + 8 * (g >> 1);
            float4* p = reinterpret_cast<float4*>(s_o + row * D + ch);
            p[0] = make_float4(s.o[nt][x][0], s.o[nt][x][1], s.o[nt][x][2], s.o[nt][x][3]);
            p[1] = make_float4(s.o[nt][x][4], s.o[nt][x][5], s.o[nt][x][6], s.o[nt][x][7]);
        }
    }
    __syncthreads();
    for (int i = tid; i < QR * D; i += kThreads) {
        const int row = i / D, col = i - row * D, rr = r0 + row;
        if (rr >= a.q_rows) break;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; w++) M = fmaxf(M, s_m[w * QR + row]);
        float o = 0.f, l = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            const float f = s_m[w * QR + row] == -INFINITY ? 0.f : ex2_approx(s_m[w * QR + row] - M);
            if (s_l[w * QR + row] != 0.f) {  // a warp without rows holds zeros
                o = fmaf(s_o[(w * QR + row) * D + col], M == -INFINITY ? 1.f : f, o);
                l = fmaf(s_l[w * QR + row], M == -INFINITY ? 1.f : f, l);
            }
        }
        if (nsplits == 1) {
            store_out(a, seq, rr / a.group, kvh * a.group + rr % a.group, D, col, l == 0.f ? 0.f : o / l);
        } else {
            float* rec = a.partial + (((static_cast<int64_t>(seq) * a.n_kv_heads + kvh) * a.q_rows + rr) * a.max_splits + split) * Ge::REC;
            rec[col] = o;
            if (col == 0) {
                rec[D] = M;
                rec[D + 1] = l;
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ combine

template <int D>
__global__ void __launch_bounds__(kThreads) kv4_combine_kernel(const __grid_constant__ Kv4Args a) {
    constexpr int EPL = D / 32, REC = Kv4Geo<D>::REC;
    const int lane = threadIdx.x & 31;
    const int64_t rows = static_cast<int64_t>(a.n_seqs) * a.n_kv_heads * a.q_rows;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
    // Every CTA waits for the split grid, so that a later launch which sees this grid complete sees the split kernel's
    // writes too.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (row >= rows) return;
    const int rr = static_cast<int>(row % a.q_rows);
    const int kvh = static_cast<int>((row / a.q_rows) % a.n_kv_heads);
    const int seq = static_cast<int>(row / (static_cast<int64_t>(a.q_rows) * a.n_kv_heads));
    const int L = ctx_of(a, seq);
    const int nsp = (L + a.split_rows - 1) / a.split_rows;
    if (nsp <= 1) return;  // written by the split kernel
    const float* base = a.partial + row * a.max_splits * REC;
    float M = -INFINITY;
    for (int sp = lane; sp < nsp; sp += 32) M = fmaxf(M, base[static_cast<int64_t>(sp) * REC + D]);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    float acc[EPL], l = 0.f;
#pragma unroll
    for (int e = 0; e < EPL; e++) acc[e] = 0.f;
#pragma unroll 4
    for (int sp = 0; sp < nsp; sp++) {
        const float* r = base + static_cast<int64_t>(sp) * REC;
        const float2 ml = *reinterpret_cast<const float2*>(r + D);
        const float f = M == -INFINITY ? 1.f : ex2_approx(ml.x - M);
        l = fmaf(ml.y, f, l);
#pragma unroll
        for (int e = 0; e < EPL; e++) acc[e] = fmaf(r[lane + 32 * e], f, acc[e]);
    }
#pragma unroll
    for (int e = 0; e < EPL; e++)
        store_out(a, seq, rr / a.group, kvh * a.group + rr % a.group, D, lane + 32 * e, l == 0.f ? 0.f : acc[e] / l);
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

struct SplitPlan {
    int nt, q_rows, q_groups, split_rows, max_splits;
};

int max_context(const alpaca_kv4_attn_desc& d) { return d.ctx_lens ? d.max_ctx_len : d.start_position + d.tokens; }

// Query rows per CTA and rows per split. Splits are as long as the call's CTAs allow: kTargetCtas CTAs over the bound of
// the call's rows, at least one tile per warp each.
constexpr int kTargetCtas = 148 * 8;
SplitPlan split_plan(const alpaca_kv4_attn_desc& d) {
    SplitPlan p;
    const int group = d.n_heads / d.n_kv_heads, tk = 4096 / d.head_dim, unit = kWarps * tk;
    p.q_rows = d.tokens * group;
    p.nt = p.q_rows <= 4 ? 1 : (p.q_rows <= 8 ? 2 : 4);
    p.q_groups = (p.q_rows + 4 * p.nt - 1) / (4 * p.nt);
    const int64_t L = std::max(max_context(d), 1);
    const int64_t heads = static_cast<int64_t>(d.n_seqs) * d.n_kv_heads * p.q_groups;
    const int64_t rows = (heads * L + kTargetCtas - 1) / kTargetCtas;
    const int64_t units = std::max<int64_t>(1, (rows + unit - 1) / unit);
    p.split_rows = static_cast<int>(std::min<int64_t>(units * unit, 1 << 20));
    p.max_splits = static_cast<int>((L + p.split_rows - 1) / p.split_rows);
    return p;
}

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
cudaError_t launch_split_nt(const Kv4Args& a, cudaStream_t s) {
    constexpr size_t smem = kWarps * kStages * Kv4Geo<D>::STAGE;
    const auto fn = kv4_split_kernel<D, NT>;
    cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(fn), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    e = cudaFuncSetAttribute(reinterpret_cast<const void*>(fn), cudaFuncAttributePreferredSharedMemoryCarveout,
                             static_cast<int>(cudaSharedmemCarveoutMaxShared));
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg =
        pdl_config(dim3(static_cast<unsigned>(a.n_kv_heads * a.q_groups * a.max_splits), a.n_seqs, 1), kThreads, smem, s, &attr);
    return cudaLaunchKernelEx(&cfg, fn, a);
}

template <int D>
cudaError_t launch_split(const Kv4Args& a, int nt, cudaStream_t s) {
    cudaError_t e = nt == 1   ? launch_split_nt<D, 1>(a, s)
                    : nt == 2 ? launch_split_nt<D, 2>(a, s)
                              : launch_split_nt<D, 4>(a, s);
    if (e != cudaSuccess || a.max_splits <= 1) return e;
    const int64_t rows = static_cast<int64_t>(a.n_seqs) * a.n_kv_heads * a.q_rows;
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = pdl_config(dim3(static_cast<unsigned>((rows + kWarps - 1) / kWarps), 1, 1), kThreads, 0, s, &attr);
    return cudaLaunchKernelEx(&cfg, kv4_combine_kernel<D>, a);
}

size_t round_up(size_t n, size_t m) { return (n + m - 1) / m * m; }

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
        if (p.max_splits <= 1) return 0;
        return sizeof(float) * static_cast<size_t>(d.n_seqs) * d.n_kv_heads * p.q_rows * p.max_splits * (d.head_dim + 4);
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
    a.partial = static_cast<float*>(ws);
    a.scale = scale;
    a.err = err;
    if (kind == ALPACA_ATTN_DECODE_SPLIT) {
        const SplitPlan p = split_plan(d);
        a.q_rows = p.q_rows;
        a.q_groups = p.q_groups;
        a.split_rows = p.split_rows;
        a.max_splits = p.max_splits;
        return d.head_dim == 128 ? launch_split<128>(a, p.nt, s) : launch_split<64>(a, p.nt, s);
    }
    a.q_rows = a.q_groups = a.split_rows = a.max_splits = 0;
    const int64_t rows = static_cast<int64_t>(d.n_seqs) * d.tokens * d.n_heads;
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg =
        pdl_config(dim3(static_cast<unsigned>((rows + kGenWarps - 1) / kGenWarps), 1, 1), 32 * kGenWarps, 0, s, &attr);
    return cudaLaunchKernelEx(&cfg, kv4_general_kernel, a, d.head_dim);
}

}  // namespace alpaca
