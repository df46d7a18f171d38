// kv4_cache.cu — writing new rows into a KV cache with head norms, RoPE and (4-bit caches) quantisation in one pass, and
// reading rows of a 4-bit cache back.
//
// qkv_append_kernel: one CTA per `tpc` tokens of a sequence; a row (one head of one token) is handled by LP lanes, eight or
// sixteen channels each, so norms, rotations and block extremes are register work and shuffles within LP lanes and nothing
// passes through shared memory but the (cos, sin) table and the norm weights. A warp's rows are of one kind. The first loads
// are in flight while that table is computed. Per row:
//   norm       x * (1 / sqrt(mean(x^2) + eps)) * w, f32, the sum of squares over the row's lanes
//   rotation   as in rope_kv.cu: angle, cos and sin in double, rounded once to f32; products rounded separately
//   write      f16 / f32 row, or the blocks' steps, zero points and codes (kv4.cuh)
// A row moves 4 d or 2 d bytes in and 0.56 d .. 4 d out. Prompts are bounded by instruction issue and memory waits about
// equally (8 x 2048 tokens of 32/8 heads at d = 128 with norms, f16 in, 4-bit cache: 73-78 us, 354 MB, 4.5-4.9 TB/s, 70% issue);
// 4096 tokens of 9/3 heads at d = 64, f32 in: 5.8 us, one wave's latency; 64 tokens 2.7 us.
//
// kv4_read_kernel: four lanes per head row, f16 or f32 out in the [seq][row][head][d] layout of the f16 cache. It moves
// 0.56 d + 2 d (f16) bytes per row and is bounded by its writes: 8 x 4096 rows of 5 heads at d = 64 in 11.9 us, 4.5 TB/s.
#include <cmath>

#include "kv4.cuh"

namespace alpaca {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kAppendBatch = 4;   // sets of eight channels in flight per lane
constexpr int kAppendTokens = 8;  // most tokens per CTA

struct AppendArgs {
    const void* q;
    const void* k;
    const void* v;
    void* q_out;
    int64_t q_seq_stride, kv_seq_stride, out_seq_stride;
    int q_token_stride, kv_token_stride, out_token_stride;  // at most kMaxTokenStride
    const float* q_norm;
    const float* k_norm;
    float eps, inv_d, inv_heads, inv_kv_heads;  // inv_x = 1 / x
    float one;  // 1, unknown to the compiler: by a known 1 it contracts a rounded product into the sum that follows
    int in_f16, out_f16, interleaved;
    const int* positions;
    int start, n_heads, n_kv_heads, d, tokens, tpc;
    // f16 / f32 row caches
    void* k_cache;
    void* v_cache;
    int64_t cache_row_stride, cache_seq_stride, block_stride;
    const int* block_table;
    int block_rows, max_blocks, pool_blocks, cache_rows;
    Kv4View kv4;  // 4-bit cache
    unsigned* err;
    double freq[128];  // theta^(-2i/d), host-computed in double
};

// Minimum / maximum that return NaN when either operand is one.
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Eight channels as loaded (f16: u[0] only) and as f32 pairs.
struct Raw8 {
    uint4 u[2];
};
__device__ __forceinline__ Raw8 load_raw(const void* p, int64_t off, int f16) {
    Raw8 r;
    if (f16) {
        r.u[0] = *reinterpret_cast<const uint4*>(static_cast<const __half*>(p) + off);
        r.u[1] = make_uint4(0, 0, 0, 0);
    } else {
        const uint4* q = reinterpret_cast<const uint4*>(static_cast<const float*>(p) + off);
        r.u[0] = q[0];
        r.u[1] = q[1];
    }
    return r;
}
__device__ __forceinline__ void unpack8(const Raw8& r, int f16, float2 (&x)[4]) {
    if (f16) {
        x[0] = __half22float2(as_half2(r.u[0].x));
        x[1] = __half22float2(as_half2(r.u[0].y));
        x[2] = __half22float2(as_half2(r.u[0].z));
        x[3] = __half22float2(as_half2(r.u[0].w));
    } else {
        x[0] = make_float2(__uint_as_float(r.u[0].x), __uint_as_float(r.u[0].y));
        x[1] = make_float2(__uint_as_float(r.u[0].z), __uint_as_float(r.u[0].w));
        x[2] = make_float2(__uint_as_float(r.u[1].x), __uint_as_float(r.u[1].y));
        x[3] = make_float2(__uint_as_float(r.u[1].z), __uint_as_float(r.u[1].w));
    }
}
__device__ __forceinline__ void store8(void* p, int64_t off, int f16, const float2 (&x)[4]) {
    if (f16) {
        *reinterpret_cast<uint4*>(static_cast<__half*>(p) + off) =
            make_uint4(pack_half2(x[0].x, x[0].y), pack_half2(x[1].x, x[1].y), pack_half2(x[2].x, x[2].y), pack_half2(x[3].x, x[3].y));
    } else {
        float4* f = reinterpret_cast<float4*>(static_cast<float*>(p) + off);
        f[0] = make_float4(x[0].x, x[0].y, x[1].x, x[1].y);
        f[1] = make_float4(x[2].x, x[2].y, x[3].x, x[3].y);
    }
}

// sin and cos of x (|x| < 2^50, tested to 2^33) to about 2e-16, for one rounding to f32: the nearest multiple of pi/2 taken off in two FMAs
// against a 106-bit pi/2 (Cody and Waite's reduction), then the Taylor series on [-pi/4, pi/4] (next terms below 5e-17).
// The call it replaces takes some 700 instructions, most of an append's work at few heads; this takes about 50.
__device__ __forceinline__ float2 sincos_f32(double x) {  // (cos, sin)
    const double shifted = fma(x, 0.63661977236758134308, 6755399441055744.0);  // x * 2/pi + 1.5 * 2^52: rounds to an integer
    const int quadrant = __double2loint(shifted);
    const double n = shifted - 6755399441055744.0;
    double r = fma(-n, 1.5707963267948966192, x);
    r = fma(-n, 6.1232339957367658860e-17, r);
    const double z = r * r;
    double s = -1.0 / 1307674368000.0;  // 1 / 15!
    s = fma(s, z, 1.0 / 6227020800.0);
    s = fma(s, z, -1.0 / 39916800.0);
    s = fma(s, z, 1.0 / 362880.0);
    s = fma(s, z, -1.0 / 5040.0);
    s = fma(s, z, 1.0 / 120.0);
    s = fma(s, z, -1.0 / 6.0);
    s = fma(s * z, r, r);
    double c = 1.0 / 20922789888000.0;  // 1 / 16!
    c = fma(c, z, -1.0 / 87178291200.0);
    c = fma(c, z, 1.0 / 479001600.0);
    c = fma(c, z, -1.0 / 3628800.0);
    c = fma(c, z, 1.0 / 40320.0);
    c = fma(c, z, -1.0 / 720.0);
    c = fma(c, z, 1.0 / 24.0);
    c = fma(c, z, -0.5);
    c = fma(c, z, 1.0);
    const float fs = static_cast<float>(s), fc = static_cast<float>(c);
    const float a = (quadrant & 1) ? fc : fs, b = (quadrant & 1) ? fs : fc;
    return make_float2(((quadrant + 1) & 2) ? -b : b, (quadrant & 2) ? -a : a);
}

// Form of the append kernel: head_dim (0: a.d), lanes per row, alpaca_cache_kind, and the two choices that its inner code
// depends on. At head_dim 64 and 128 lane j of a row holds two sets of eight channels, 8 j .. and d/2 + 8 j ..: both halves of
// its rotation pairs in either convention, and whole quarters of blocks. Other head dims: one set, 8 j .. .
template <int D_, int LP_, int kKind_, bool kInter_, bool kF16_>
struct Form {
    static constexpr int D = D_, LP = LP_, kKind = kKind_, SETS = D_ ? 2 : 1;
    static constexpr bool kInter = kInter_, kF16 = kF16_;
    __device__ static __forceinline__ int dim(const AppendArgs& a) { return D ? D : a.d; }
};

// Position of pair i in the (cos, sin) table. Split halves: a lane reads pairs 8 j .. 8 j + 7 as two 16-byte pieces; the
// first pieces of all lanes lie together, then the second ones, so that a row's lanes read consecutive banks.
template <bool kInter>
__device__ __forceinline__ int table_at(int i, int half) {
    return kInter ? i : ((i >> 2) & 1) * (half / 2) + (i >> 3) * 4 + (i & 3);
}

// What the row loop of a CTA needs.
struct Cta {
    int seq, pos0;
    const char* q_at;  // this lane's channels of row 0 of the CTA's first token
    const char* k_at;
    const char* v_at;
    char* out_at;
    const float* s_cos;
    const float* s_sin;
    const float* s_w;  // norm weights of the query heads, then of the key heads
};

// Writes the codes and headers of this lane's sets of a K or V row.
template <typename F, int K>
__device__ __forceinline__ void quantise_row(const AppendArgs& a, const Cta& c, int tt, int head, bool active, int j, float2 (&x)[F::SETS][4]) {
    const int d = F::dim(a), nb = d / 32, t = j & 3;
    uint32_t word[F::SETS], header[F::SETS];
#pragma unroll
    for (int s = 0; s < F::SETS; s++) {
        float lo = 0.f, hi = 0.f;  // block extremes, with 0 in the range: four lanes hold a block
#pragma unroll
        for (int e = 0; e < 4; e++) {
            lo = min_nan(min_nan(lo, x[s][e].x), x[s][e].y);
            hi = max_nan(max_nan(hi, x[s][e].x), x[s][e].y);
        }
#pragma unroll
        for (int o = 1; o <= 2; o <<= 1) {
            lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        const Kv4Block q = kv4_block(lo, hi);
        if (q.wide) {  // keep quotients in the range of the integer rounding; the codes end at 0 and 15 long before
#pragma unroll
            for (int e = 0; e < 4; e++) {
                x[s][e].x = fminf(fmaxf(x[s][e].x, -32.f * kKv4MaxStep), 32.f * kKv4MaxStep);
                x[s][e].y = fminf(fmaxf(x[s][e].y, -32.f * kKv4MaxStep), 32.f * kKv4MaxStep);
            }
        }
        word[s] = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) word[s] += kv4_code_pair(x[s][e], q) << (8 * e);
        if (q.step == 0.f) word[s] = 0;
        header[s] = q.header;
    }
    int64_t unit;
    int ur;
    if (!active || !kv4_locate(a.kv4, c.seq, c.pos0 + tt, a.err, unit, ur)) return;
    uint32_t* codes = reinterpret_cast<uint32_t*>((K == 1 ? a.kv4.k_codes : a.kv4.v_codes) + unit * a.kv4.code_unit_stride +
                                                  head * a.kv4.code_head_stride + static_cast<int64_t>(ur) * (d / 2));
    uint16_t* scales = (K == 1 ? a.kv4.k_scales : a.kv4.v_scales) + unit * a.kv4.scale_unit_stride +
                       head * a.kv4.scale_head_stride + static_cast<int64_t>(ur) * nb;
    if constexpr (F::SETS == 2 && F::D == 64) {  // blocks 0 and 1
        *reinterpret_cast<uint2*>(codes + 2 * t) = make_uint2(word[0], word[1]);
        if (t == 0) *reinterpret_cast<uint32_t*>(scales) = header[0] | header[1] << 16;
    } else {
#pragma unroll
        for (int s = 0; s < F::SETS; s++) {
            const int blk = (j >> 2) + s * nb / 2;
            codes[t * nb + blk] = word[s];
            if (t == 0) scales[blk] = static_cast<uint16_t>(header[s]);
        }
    }
}

// One head row, LP lanes: norm, rotation, write. K: 0 query, 1 key, 2 value, the same for the whole warp. Lanes without a row
// (`active` false) hold zeros, point at the row of token 0, and take part in the shuffles only.
template <typename F, int K>
__device__ __forceinline__ void finish_row(const AppendArgs& a, const Cta& c, int tt, int head, bool active, int j, float2 (&x)[F::SETS][4]) {
    constexpr int LP = F::LP, SETS = F::SETS;
    const int d = F::dim(a), half = d / 2, c0 = 8 * j;
    if (K < 2 && (K == 0 ? a.q_norm : a.k_norm) != nullptr) {
        float2 s2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int s = 0; s < SETS; s++)
#pragma unroll
            for (int e = 0; e < 4; e++) s2 = __ffma2_rn(x[s][e], x[s][e], s2);
        float ss = s2.x + s2.y;
#pragma unroll
        for (int o = LP / 2; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        // 1 / sqrt(mean + eps): the hardware's approximation and one Newton step. Where the squares' sum is past f32, inf * 0 is
        // NaN there; fmaxf drops it, and the result is 0 as 1 / sqrt(inf) is (a NaN sum stays one through y).
        const float m = fmaf(ss, a.inv_d, a.eps), y = rsqrtf(m);
        const float inv = fmaf(y * 0.5f, fmaf(-fmaxf(m * y, 0.f), y, 1.f), y);
#pragma unroll
        for (int s = 0; s < SETS; s++) {
            const float4* w = reinterpret_cast<const float4*>(c.s_w + (K == 0 ? 0 : d) + s * half + c0);
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float4 u = w[e];
                x[s][2 * e] = __fmul2_rn(__fmul2_rn(x[s][2 * e], make_float2(inv, inv)), make_float2(u.x, u.y));
                x[s][2 * e + 1] = __fmul2_rn(__fmul2_rn(x[s][2 * e + 1], make_float2(inv, inv)), make_float2(u.z, u.w));
            }
        }
    }
    if constexpr (K < 2 && F::kInter) {
#pragma unroll
        for (int s = 0; s < SETS; s++) {
            const int at = tt * half + (s * half + c0) / 2;
            const float4 cv = *reinterpret_cast<const float4*>(c.s_cos + at), sv = *reinterpret_cast<const float4*>(c.s_sin + at);
            const float cs[4] = {cv.x, cv.y, cv.z, cv.w}, sn[4] = {sv.x, sv.y, sv.z, sv.w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float x0 = x[s][e].x, x1 = x[s][e].y;
                x[s][e].x = __fsub_rn(__fmul_rn(x0, cs[e]), __fmul_rn(x1, sn[e]));
                x[s][e].y = __fadd_rn(__fmul_rn(x0, sn[e]), __fmul_rn(x1, cs[e]));
            }
        }
    }
    if constexpr (K < 2 && !F::kInter) {
        // channel i pairs with i + d/2: the lane's second set, or (one set) held by the lane d/16 further on.
        // first: x c - partner s; second: x c + partner s. The products are rounded before the sum: adding sign * product in an
        // FMA rounds as the sum does.
        const int lane = threadIdx.x & 31, hl = d / 16;
        const bool first = j < hl;
        const int other = first ? lane + hl : lane - hl;
        const float minus = SETS == 1 && !first ? a.one : -a.one;
        const float2 sign = make_float2(minus, minus), plus = make_float2(a.one, a.one);
        const int at = tt * half + 4 * (SETS == 2 || first ? j : j - hl);
        float2 p[4];
        if constexpr (SETS == 1) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                p[e].x = __shfl_sync(0xffffffffu, x[0][e].x, other);
                p[e].y = __shfl_sync(0xffffffffu, x[0][e].y, other);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) p[e] = x[SETS - 1][e];
        }
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const float4 c4 = *reinterpret_cast<const float4*>(c.s_cos + at + e * (half / 2));
            const float4 s4 = *reinterpret_cast<const float4*>(c.s_sin + at + e * (half / 2));
            const float2 cs[2] = {make_float2(c4.x, c4.y), make_float2(c4.z, c4.w)}, sn[2] = {make_float2(s4.x, s4.y), make_float2(s4.z, s4.w)};
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const float2 x0 = x[0][2 * e + k], x1 = p[2 * e + k];
                x[0][2 * e + k] = __ffma2_rn(__fmul2_rn(x1, sn[k]), sign, __fmul2_rn(x0, cs[k]));
                if constexpr (SETS == 2) x[SETS - 1][2 * e + k] = __ffma2_rn(__fmul2_rn(x0, sn[k]), plus, __fmul2_rn(x1, cs[k]));
            }
        }
    }
    if constexpr (K == 0) {
        const int64_t off = tt * a.out_token_stride + head * d;
        if (active) {
#pragma unroll
            for (int s = 0; s < SETS; s++) store8(c.out_at + (off + s * half) * (a.out_f16 ? 2 : 4), 0, a.out_f16, x[s]);
        }
    } else if constexpr (F::kKind == ALPACA_CACHE_KV4) {
        quantise_row<F, K>(a, c, tt, head, active, j, x);
    } else if (active) {
        const int pos = c.pos0 + tt;
        int64_t off;
        bool ok = true;
        if (!a.block_table) {
            ok = pos >= 0 && pos < a.cache_rows;
            off = c.seq * a.cache_seq_stride + static_cast<int64_t>(pos) * a.cache_row_stride;
        } else {
            const int n = pos >= 0 ? pos / a.block_rows : -1;
            const int blk = (n >= 0 && n < a.max_blocks) ? a.block_table[static_cast<int64_t>(c.seq) * a.max_blocks + n] : -1;
            ok = blk >= 0 && blk < a.pool_blocks;
            off = static_cast<int64_t>(blk) * a.block_stride + static_cast<int64_t>(pos - n * a.block_rows) * a.cache_row_stride;
        }
        if (ok) {
#pragma unroll
            for (int s = 0; s < SETS; s++)
                store8(K == 1 ? a.k_cache : a.v_cache, off + head * d + s * half + c0, F::kKind == ALPACA_CACHE_F16, x[s]);
        } else {
            atomicOr(a.err, kDevErrBadIndex);
        }
    }
}

template <typename F>
__global__ void __launch_bounds__(kAppendThreads, 4) qkv_append_kernel(const __grid_constant__ AppendArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ __align__(16) float s_table[];  // cos [tpc][d/2], sin [tpc][d/2], norm weights [2][d]
    constexpr int LP = F::LP, RPW = 32 / LP, kWarps = kAppendThreads / 32, kSize = F::kF16 ? 2 : 4, SETS = F::SETS;
    constexpr int B = kAppendBatch / SETS;
    const int t0 = blockIdx.x * a.tpc, seq = blockIdx.y, tid = threadIdx.x, warp = tid / 32;
    const int d = F::dim(a), ntok = min(a.tpc, a.tokens - t0), half = d / 2;
    float* s_cos = s_table;
    float* s_sin = s_table + a.tpc * half;
    float* s_w = s_sin + a.tpc * half;
    const int sub = (tid % 32) / LP, lane_j = tid % LP;
    const bool in = 8 * SETS * lane_j < d;  // lanes past the row (d not a power of two) only take part in the shuffles
    const int j = in ? lane_j : 0;
    const auto table = [&](int pos0) {
        for (int i = tid; i < ntok * half; i += kAppendThreads) {
            const int tt = i / half, at = tt * half + table_at<F::kInter>(i - tt * half, half);
            const float2 w = sincos_f32(static_cast<double>(pos0 + tt) * a.freq[i - tt * half]);
            s_cos[at] = w.x;
            s_sin[at] = w.y;
        }
    };
    // A uniform start needs no global data: its table is computed while the previous kernel drains.
    if (!a.positions) table(a.start + t0);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t kv_at = (seq * a.kv_seq_stride + static_cast<int64_t>(t0) * a.kv_token_stride + 8 * j) * kSize;
    Cta c;
    c.seq = seq;
    c.pos0 = (a.positions ? a.positions[seq] : a.start) + t0;
    c.q_at = static_cast<const char*>(a.q) + (seq * a.q_seq_stride + static_cast<int64_t>(t0) * a.q_token_stride + 8 * j) * kSize;
    c.k_at = static_cast<const char*>(a.k) + kv_at;
    c.v_at = static_cast<const char*>(a.v) + kv_at;
    c.out_at = static_cast<char*>(a.q_out) +
               (seq * a.out_seq_stride + static_cast<int64_t>(t0) * a.out_token_stride + 8 * j) * (a.out_f16 ? 2 : 4);
    c.s_cos = s_cos;
    c.s_sin = s_sin;
    c.s_w = s_w;
    for (int i = tid; i < 2 * d; i += kAppendThreads) {
        const float* w = i < d ? a.q_norm : a.k_norm;
        if (w) s_w[i] = w[i < d ? i : i - d];
    }
    // The CTA's rows in groups of RPW (a warp's), each of one kind: all query rows, then the key rows, then the value rows.
    const int nq = ntok * a.n_heads, nk = ntok * a.n_kv_heads;
    const int gq = (nq + RPW - 1) / RPW, gk = (nk + RPW - 1) / RPW, groups = gq + 2 * gk;
    bool first = true;
    for (int g0 = warp; first || g0 < groups; g0 += kWarps * B) {
        Raw8 raw[B][SETS];
        int tt[B], head[B];
        bool active[B];
#pragma unroll
        for (int b = 0; b < B; b++) {  // B groups in flight; a kind's row i is head i % heads of token i / heads
            const int g = g0 + b * kWarps;
            const bool q = g < gq, k = g < gq + gk;
            const int i = (g - (q ? 0 : (k ? gq : gq + gk))) * RPW + sub, heads = q ? a.n_heads : a.n_kv_heads;
            active[b] = in && g < groups && i < (q ? nq : nk);
            const int row = active[b] ? i : 0;
            // i < 2^19 and the quotient at most 8, so half a unit of slack covers the rounding of the reciprocal
            tt[b] = static_cast<int>((static_cast<float>(row) + 0.5f) * (q ? a.inv_heads : a.inv_kv_heads));
            head[b] = row - tt[b] * heads;
            // offsets within a CTA's tokens fit 32 bits
            const int64_t off = tt[b] * (q ? a.q_token_stride : a.kv_token_stride) + head[b] * d;
#pragma unroll
            for (int s = 0; s < SETS; s++) {
                raw[b][s].u[0] = raw[b][s].u[1] = make_uint4(0, 0, 0, 0);
                if (active[b]) raw[b][s] = load_raw((q ? c.q_at : (k ? c.k_at : c.v_at)) + (off + s * half) * kSize, 0, F::kF16);
            }
        }
        if (first) {
            if (a.positions) table(c.pos0);
            __syncthreads();  // every thread passes here once
            first = false;
        }
#pragma unroll
        for (int b = 0; b < B; b++) {
            const int g = g0 + b * kWarps;
            if (g >= groups) break;
            float2 x[SETS][4];
#pragma unroll
            for (int s = 0; s < SETS; s++) unpack8(raw[b][s], F::kF16, x[s]);
            if (g < gq) finish_row<F, 0>(a, c, tt[b], head[b], active[b], j, x);
            else if (g < gq + gk) finish_row<F, 1>(a, c, tt[b], head[b], active[b], j, x);
            else finish_row<F, 2>(a, c, tt[b], head[b], active[b], j, x);
        }
    }
}

template <int D, int LP, bool kInter, bool kF16>
cudaError_t launch_append(const AppendArgs& a, int kind, const cudaLaunchConfig_t& cfg) {
    switch (kind) {
        case ALPACA_CACHE_KV4: return cudaLaunchKernelEx(&cfg, qkv_append_kernel<Form<D, LP, ALPACA_CACHE_KV4, kInter, kF16>>, a);
        case ALPACA_CACHE_F16: return cudaLaunchKernelEx(&cfg, qkv_append_kernel<Form<D, LP, ALPACA_CACHE_F16, kInter, kF16>>, a);
        default: return cudaLaunchKernelEx(&cfg, qkv_append_kernel<Form<D, LP, ALPACA_CACHE_F32, kInter, kF16>>, a);
    }
}

template <int D, int LP>
cudaError_t launch_append(const AppendArgs& a, int kind, const cudaLaunchConfig_t& cfg) {
    if (a.interleaved) return a.in_f16 ? launch_append<D, LP, true, true>(a, kind, cfg) : launch_append<D, LP, true, false>(a, kind, cfg);
    return a.in_f16 ? launch_append<D, LP, false, true>(a, kind, cfg) : launch_append<D, LP, false, false>(a, kind, cfg);
}

// ------------------------------------------------------------------------------------------------ read back

constexpr int kReadThreads = 256;
constexpr int kReadBatch = 2;  // head rows in flight per lane group
constexpr int kReadRows = kReadThreads / 4 * kReadBatch;  // head rows per CTA

struct ReadArgs {
    Kv4View c;
    void* k_out;
    void* v_out;
    int64_t out_row_stride, out_seq_stride;
    const int* row_starts;
    // ragged prefill: the first start_positions[s] + (q_offsets[s + 1] - q_offsets[s]) rows of each sequence (null: n_rows)
    const int* start_positions;
    const int* q_offsets;
    int start, n_rows, n_kv_heads, out_f16;
    unsigned* err;
};

// NB = d / 32. Four lanes hold a head row, lane t the words t * NB .. of all blocks: channels 32 b + 8 t .. + 7.
template <int NB>
__global__ void __launch_bounds__(kReadThreads) kv4_read_kernel(const __grid_constant__ ReadArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int seq = blockIdx.y, t = threadIdx.x & 3;
    const uint8_t* codes = blockIdx.z ? a.c.v_codes : a.c.k_codes;
    const uint16_t* scales = blockIdx.z ? a.c.v_scales : a.c.k_scales;
    void* out = blockIdx.z ? a.v_out : a.k_out;
    const int start = a.row_starts ? a.row_starts[seq] : a.start;
    int rows = a.n_rows;
    if (a.q_offsets) {  // entries out of bounds are reported by the prefill's plan kernel, which skips the sequence
        const int64_t n = static_cast<int64_t>(a.q_offsets[seq + 1]) - a.q_offsets[seq];
        rows = n > 0 ? static_cast<int>(max(min(a.start_positions[seq] + n, static_cast<int64_t>(a.n_rows)), static_cast<int64_t>(0))) : 0;
    }
    uint32_t w[kReadBatch][NB], h[kReadBatch][NB];
    int64_t at[kReadBatch];
#pragma unroll
    for (int b = 0; b < kReadBatch; b++) {
        const int64_t i = static_cast<int64_t>(blockIdx.x) * kReadRows + b * (kReadThreads / 4) + threadIdx.x / 4;
        const int row = static_cast<int>(i >> 32 ? i / a.n_kv_heads : static_cast<uint32_t>(i) / static_cast<uint32_t>(a.n_kv_heads));
        const int head = static_cast<int>(i - static_cast<int64_t>(row) * a.n_kv_heads);
        at[b] = -1;
#pragma unroll
        for (int k = 0; k < NB; k++) w[b][k] = h[b][k] = 0;
        if (row >= rows) continue;
        at[b] = seq * a.out_seq_stride + row * a.out_row_stride + head * (32 * NB) + 8 * t;
        int64_t unit;
        int ur;
        if (!kv4_locate(a.c, seq, start + row, a.err, unit, ur)) continue;  // reads as zero
        const uint32_t* c = reinterpret_cast<const uint32_t*>(codes + unit * a.c.code_unit_stride + head * a.c.code_head_stride +
                                                              static_cast<int64_t>(ur) * (16 * NB)) + t * NB;
        const uint16_t* s = scales + unit * a.c.scale_unit_stride + head * a.c.scale_head_stride + static_cast<int64_t>(ur) * NB;
        if constexpr (NB % 4 == 0) {
#pragma unroll
            for (int k = 0; k < NB; k += 4) {
                const uint4 u = *reinterpret_cast<const uint4*>(c + k);
                w[b][k] = u.x; w[b][k + 1] = u.y; w[b][k + 2] = u.z; w[b][k + 3] = u.w;
                const uint2 v = *reinterpret_cast<const uint2*>(s + k);
                h[b][k] = v.x & 0xFFFFu; h[b][k + 1] = v.x >> 16; h[b][k + 2] = v.y & 0xFFFFu; h[b][k + 3] = v.y >> 16;
            }
        } else if constexpr (NB % 2 == 0) {
#pragma unroll
            for (int k = 0; k < NB; k += 2) {
                const uint2 u = *reinterpret_cast<const uint2*>(c + k);
                w[b][k] = u.x; w[b][k + 1] = u.y;
                const uint32_t v = *reinterpret_cast<const uint32_t*>(s + k);
                h[b][k] = v & 0xFFFFu; h[b][k + 1] = v >> 16;
            }
        } else {
#pragma unroll
            for (int k = 0; k < NB; k++) {
                w[b][k] = c[k];
                h[b][k] = s[k];
            }
        }
    }
#pragma unroll
    for (int b = 0; b < kReadBatch; b++) {
        if (at[b] < 0) continue;
#pragma unroll
        for (int k = 0; k < NB; k++) {
            const uint4 u = kv4_word_values(w[b][k], h[b][k]);
            if (a.out_f16) {
                *reinterpret_cast<uint4*>(static_cast<__half*>(out) + at[b] + 32 * k) = u;
            } else {
                float4* o = reinterpret_cast<float4*>(static_cast<float*>(out) + at[b] + 32 * k);
                const float2 f0 = __half22float2(as_half2(u.x)), f1 = __half22float2(as_half2(u.y));
                const float2 f2 = __half22float2(as_half2(u.z)), f3 = __half22float2(as_half2(u.w));
                o[0] = make_float4(f0.x, f0.y, f1.x, f1.y);
                o[1] = make_float4(f2.x, f2.y, f3.x, f3.y);
            }
        }
    }
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

// Lanes of a head row: 16 channels each at head_dim 64 and 128, else 8.
int append_lanes(int head_dim) {
    if (head_dim == 64 || head_dim == 128) return head_dim / 16;
    return head_dim <= 32 ? 4 : (head_dim <= 128 ? 16 : 32);
}

// Tokens per CTA: the power of two up to kAppendTokens with the least waves x time of a CTA, which is about 1.75 us (its wait,
// its angles, its loads' latency) and 0.0057 us per lane of work (fitted to the calls below; a B200 holds four CTAs an SM). It
// ranks the choices; the time of a single wave it overstates up to twice. Measured at 1 / 2 / 4 / 8 tokens, us: 64 tokens of
// 32/8 heads at d = 128 2.7 / 3.5 / 5.4 / 9.0; 1024 tokens 8.8 / 9.0 / 14.8 / 20.6; 16384 tokens 92 / 78 / 73 / 76; 4096 tokens
// of 9/3 heads at d = 64 17 / 10 / 7.1 / 5.9; 2048 tokens 9.9 / 5.5 / 4.2 / 5.4.
int append_tokens(const alpaca_qkv_desc& d, int row_lanes) {
    const double token_lanes = static_cast<double>(d.n_heads + 2 * d.n_kv_heads) * row_lanes;
    constexpr int64_t resident = 148 * 4;
    double best = 0;
    int tokens = 0;
    for (int t = 1; t <= kAppendTokens; t *= 2) {
        const int64_t ctas = (static_cast<int64_t>(d.tokens) + t - 1) / t * d.n_seqs;
        const double us = static_cast<double>((ctas + resident - 1) / resident) * (1.75 + 0.0057 * t * token_lanes);
        if (tokens == 0 || us < best) {
            best = us;
            tokens = t;
        }
        if (t >= d.tokens) break;
    }
    return tokens;
}

}  // namespace

cudaError_t launch_qkv_append(const alpaca_qkv_desc& d, unsigned* err, cudaStream_t s) {
    AppendArgs a;
    a.q = d.q;
    a.k = d.k;
    a.v = d.v;
    a.q_out = d.q_out;
    a.q_token_stride = static_cast<int>(d.q_token_stride);
    a.q_seq_stride = d.q_seq_stride;
    a.kv_token_stride = static_cast<int>(d.kv_token_stride);
    a.kv_seq_stride = d.kv_seq_stride;
    a.out_token_stride = static_cast<int>(d.q_out_token_stride);
    a.out_seq_stride = d.q_out_seq_stride;
    a.q_norm = d.q_norm;
    a.k_norm = d.k_norm;
    a.eps = d.eps;
    a.one = 1.f;
    a.inv_d = 1.f / static_cast<float>(d.head_dim);
    a.inv_heads = 1.f / static_cast<float>(d.n_heads > 0 ? d.n_heads : 1);
    a.inv_kv_heads = 1.f / static_cast<float>(d.n_kv_heads > 0 ? d.n_kv_heads : 1);
    a.in_f16 = d.in_dtype == ALPACA_F16;
    a.out_f16 = d.q_out_dtype == ALPACA_F16;
    a.interleaved = d.interleaved;
    a.positions = d.positions;
    a.start = d.start_position;
    a.n_heads = d.n_heads;
    a.n_kv_heads = d.n_kv_heads;
    a.d = d.head_dim;
    a.tokens = d.tokens;
    const int row_lanes = append_lanes(d.head_dim);
    a.tpc = append_tokens(d, row_lanes);
    a.k_cache = d.k_cache;
    a.v_cache = d.v_cache;
    a.cache_row_stride = d.cache_row_stride;
    a.cache_seq_stride = d.cache_seq_stride;
    a.block_stride = d.block_stride;
    a.block_table = d.block_table;
    a.block_rows = d.block_rows;
    a.max_blocks = d.max_blocks;
    a.pool_blocks = d.pool_blocks;
    a.cache_rows = d.cache_rows;
    a.kv4 = kv4_view(d.kv4);
    a.err = err;
    const double theta = static_cast<double>(d.theta);
    for (int i = 0; i < 128; i++)
        a.freq[i] = i < d.head_dim / 2 ? std::pow(theta, -2.0 * static_cast<double>(i) / static_cast<double>(d.head_dim)) : 0.0;
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = pdl_config(dim3((d.tokens + a.tpc - 1) / a.tpc, d.n_seqs, 1), kAppendThreads,
                                              sizeof(float) * (a.tpc + 2) * d.head_dim, s, &attr);
    return d.head_dim == 64    ? launch_append<64, 4>(a, d.cache_kind, cfg)
           : d.head_dim == 128 ? launch_append<128, 8>(a, d.cache_kind, cfg)
           : row_lanes == 4    ? launch_append<0, 4>(a, d.cache_kind, cfg)
           : row_lanes == 16   ? launch_append<0, 16>(a, d.cache_kind, cfg)
                               : launch_append<0, 32>(a, d.cache_kind, cfg);
}

cudaError_t launch_kv4_read(const alpaca_kv4_read_desc& d, const int* start_positions, const int* q_offsets, unsigned* err,
                            cudaStream_t s) {
    ReadArgs a;
    a.c = kv4_view(d.cache);
    a.k_out = d.k_out;
    a.v_out = d.v_out;
    a.out_row_stride = d.out_row_stride;
    a.out_seq_stride = d.out_seq_stride;
    a.row_starts = d.row_starts;
    a.start_positions = start_positions;
    a.q_offsets = q_offsets;
    a.start = d.start_row;
    a.n_rows = d.n_rows;
    a.n_kv_heads = d.n_kv_heads;
    a.out_f16 = d.out_dtype == ALPACA_F16;
    a.err = err;
    const int64_t rows = static_cast<int64_t>(d.n_rows) * d.n_kv_heads;
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg =
        pdl_config(dim3(static_cast<unsigned>((rows + kReadRows - 1) / kReadRows), d.n_seqs, 2), kReadThreads, 0, s, &attr);
    switch (d.head_dim / 32) {
        case 1: return cudaLaunchKernelEx(&cfg, kv4_read_kernel<1>, a);
        case 2: return cudaLaunchKernelEx(&cfg, kv4_read_kernel<2>, a);
        case 3: return cudaLaunchKernelEx(&cfg, kv4_read_kernel<3>, a);
        case 4: return cudaLaunchKernelEx(&cfg, kv4_read_kernel<4>, a);
        case 5: return cudaLaunchKernelEx(&cfg, kv4_read_kernel<5>, a);
        case 6: return cudaLaunchKernelEx(&cfg, kv4_read_kernel<6>, a);
        case 7: return cudaLaunchKernelEx(&cfg, kv4_read_kernel<7>, a);
        default: return cudaLaunchKernelEx(&cfg, kv4_read_kernel<8>, a);
    }
}

}  // namespace alpaca
