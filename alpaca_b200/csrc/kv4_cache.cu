// kv4_cache.cu — writing new rows into a KV cache with head norms, RoPE and (4-bit caches) quantisation in one pass, and
// reading rows of a 4-bit cache back.
//
// qkv_append_kernel: one CTA per `tpc` tokens of a sequence; a row (one head of one token) is handled by LP lanes, eight
// consecutive channels each (LP = d/8 rounded up to a power of two), so norms, rotations and block extremes are
// shuffles within LP lanes and nothing passes through shared memory but the (cos, sin) table. The first batch of 16-byte
// loads is in flight while that table is computed. Per row:
//   norm       x * (1 / sqrt(mean(x^2) + eps)) * w, f32, the sum of squares over the row's lanes
//   rotation   the arithmetic of rope_kv.cu: angle, cos and sin in double, rounded once to f32; products rounded
//              separately, so rows without a norm equal alpaca_rope_kv_append's bit for bit
//   write      f16 / f32 row, or the blocks' steps, zero points and codes (kv4.cuh)
// A row moves 4 d or 2 d bytes in and 0.56 d .. 4 d out: HBM for prompts, latency for one token per sequence.
//
// kv4_read_kernel: four lanes per head row, f16 or f32 out in the [seq][row][head][d] layout of the f16 cache. It moves 0.56 d + 2 d (f16) bytes per row: HBM-bound.
#include <cmath>

#include "kv4.cuh"

namespace alpaca {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kAppendBatch = 2;   // rows in flight per lane group
constexpr int kAppendTokens = 8;  // most tokens per CTA

struct AppendArgs {
    const void* q;
    const void* k;
    const void* v;
    void* q_out;
    int64_t q_token_stride, q_seq_stride, kv_token_stride, kv_seq_stride, out_token_stride, out_seq_stride;
    const float* q_norm;
    const float* k_norm;
    float eps, inv_d;  // inv_d = 1 / d
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

__device__ __forceinline__ void load8(const void* p, int64_t off, int f16, float (&x)[8]) {
    if (f16) {
        const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const __half*>(p) + off);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(as_half2(w[i]));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    } else {
        const float4* f = reinterpret_cast<const float4*>(static_cast<const float*>(p) + off);
        const float4 a = f[0], b = f[1];
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
}

__device__ __forceinline__ void store8(void* p, int64_t off, int f16, const float (&x)[8]) {
    if (f16) {
        *reinterpret_cast<uint4*>(static_cast<__half*>(p) + off) =
            make_uint4(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]), pack_half2(x[4], x[5]), pack_half2(x[6], x[7]));
    } else {
        float4* f = reinterpret_cast<float4*>(static_cast<float*>(p) + off);
        f[0] = make_float4(x[0], x[1], x[2], x[3]);
        f[1] = make_float4(x[4], x[5], x[6], x[7]);
    }
}

// Rows of a CTA's tokens in order: row `i` (query heads, key heads, value heads) of its token `tt`. Lane groups step through
// them by the CTA's rows per pass, without a division per row.
struct RowAt {
    int tt, i;
    __device__ __forceinline__ void step(int tokens, int rows, int per) {
        tt += tokens;
        i += rows;
        if (i >= per) {
            i -= per;
            tt++;
        }
    }
};

__device__ __forceinline__ void load_row(const AppendArgs& a, int seq, int t0, const RowAt& r, int c0, float (&x)[8]) {
    const int64_t t = t0 + r.tt;
    if (r.i < a.n_heads) {
        load8(a.q, seq * a.q_seq_stride + t * a.q_token_stride + r.i * a.d + c0, a.in_f16, x);
    } else {
        const int h = r.i - a.n_heads;
        const bool k = h < a.n_kv_heads;
        load8(k ? a.k : a.v, seq * a.kv_seq_stride + t * a.kv_token_stride + (k ? h : h - a.n_kv_heads) * a.d + c0, a.in_f16, x);
    }
}

// Position of pair i in the (cos, sin) table. Split halves: a lane reads pairs 8 j .. 8 j + 7 as two 16-byte pieces; the
// first pieces of all lanes lie together, then the second ones, so that a row's lanes read consecutive banks.
__device__ __forceinline__ int table_at(int i, int half, int interleaved) {
    return interleaved ? i : ((i >> 2) & 1) * (half / 2) + (i >> 3) * 4 + (i & 3);
}

// kKind: alpaca_cache_kind. LP: lanes per row. qw / kw: this lane's norm weights.
template <int LP, int kKind>
__device__ __forceinline__ void finish_row(const AppendArgs& a, int seq, int t0, int pos0, const RowAt& r, bool active, int j,
                                           const float* s_cos, const float* s_sin, const float (&qw)[8], const float (&kw)[8],
                                           float (&x)[8]) {
    const int half = a.d / 2, c0 = 8 * j;
    const bool is_q = r.i < a.n_heads, is_k = !is_q && r.i < a.n_heads + a.n_kv_heads;
    const bool norm = active && (is_q ? a.q_norm != nullptr : (is_k && a.k_norm != nullptr));
    if (__any_sync(0xffffffffu, norm)) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e++) ss = fmaf(x[e], x[e], ss);
#pragma unroll
        for (int o = LP / 2; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (norm) {
            // 1 / sqrt(mean + eps): the hardware's approximation and one Newton step
            const float m = fmaf(ss, a.inv_d, a.eps), y = rsqrtf(m);
            const float inv = fmaf(y * 0.5f, fmaf(-m * y, y, 1.f), y);
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = __fmul_rn(__fmul_rn(x[e], inv), is_q ? qw[e] : kw[e]);
        }
    }
    const bool rotate = active && (is_q || is_k);
    if (__any_sync(0xffffffffu, rotate)) {
        const float* cs = s_cos + r.tt * half;
        const float* sn = s_sin + r.tt * half;
        if (a.interleaved) {
            if (rotate) {
                const float4 c = *reinterpret_cast<const float4*>(cs + c0 / 2);
                const float4 s = *reinterpret_cast<const float4*>(sn + c0 / 2);
                const float cv[4] = {c.x, c.y, c.z, c.w}, sv[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float x0 = x[2 * e], x1 = x[2 * e + 1];
                    x[2 * e] = __fsub_rn(__fmul_rn(x0, cv[e]), __fmul_rn(x1, sv[e]));
                    x[2 * e + 1] = __fadd_rn(__fmul_rn(x0, sv[e]), __fmul_rn(x1, cv[e]));
                }
            }
        } else {
            // channel i pairs with i + d/2: the lane d/16 further on holds the partners of this lane's eight channels.
            // first: x c - partner s; second: partner s + x c. One sign covers both.
            const int lane = threadIdx.x & 31, hl = a.d / 16;
            const bool first = j < hl;
            const int other = active ? (first ? lane + hl : lane - hl) : lane;
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; e++) p[e] = __shfl_sync(0xffffffffu, x[e], other);
            if (rotate) {
                const int at = 4 * (first ? j : j - hl);
#pragma unroll
                for (int e4 = 0; e4 < 2; e4++) {
                    const float4 c = *reinterpret_cast<const float4*>(cs + at + e4 * (half / 2));
                    const float4 s = *reinterpret_cast<const float4*>(sn + at + e4 * (half / 2));
                    const float cv[4] = {c.x, c.y, c.z, c.w}, sv[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float ps = __fmul_rn(p[4 * e4 + e], sv[e]);
                        x[4 * e4 + e] = __fadd_rn(__fmul_rn(x[4 * e4 + e], cv[e]), first ? -ps : ps);
                    }
                }
            }
        }
    }
    float lo = 0.f, hi = 0.f;
    if (kKind == ALPACA_CACHE_KV4 && __any_sync(0xffffffffu, active && !is_q)) {
        // block extremes, with 0 in the range: four lanes hold a block
#pragma unroll
        for (int e = 0; e < 8; e++) {
            lo = min_nan(lo, x[e]);
            hi = max_nan(hi, x[e]);
        }
#pragma unroll
        for (int o = 1; o <= 2; o <<= 1) {
            lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
    }
    if (!active) return;
    const int64_t t = t0 + r.tt;
    if (is_q) {
        store8(a.q_out, seq * a.out_seq_stride + t * a.out_token_stride + r.i * a.d + c0, a.out_f16, x);
        return;
    }
    const int pos = pos0 + r.tt, head = r.i - a.n_heads - (is_k ? 0 : a.n_kv_heads);
    if (kKind == ALPACA_CACHE_KV4) {
        int64_t unit;
        int ur;
        if (!kv4_locate(a.kv4, seq, pos, a.err, unit, ur)) return;
        const Kv4Block q = kv4_block(lo, hi);
        if (q.wide) {  // keep quotients in the range of the integer rounding; the codes end at 0 and 15 long before
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = fminf(fmaxf(x[e], -32.f * kKv4MaxStep), 32.f * kKv4MaxStep);
        }
        uint32_t word = 0;
        if (q.step > 0.f) {
#pragma unroll
            for (int e = 0; e < 8; e++) word += kv4_code(x[e], q) << (4 * e);
        }
        const int nb = a.d / 32, b = j >> 2, tw = j & 3;
        uint8_t* codes = (is_k ? a.kv4.k_codes : a.kv4.v_codes) + unit * a.kv4.code_unit_stride +
                         head * a.kv4.code_head_stride + static_cast<int64_t>(ur) * (a.d / 2);
        *reinterpret_cast<uint32_t*>(codes + 4 * (tw * nb + b)) = word;
        if (tw == 0) {
            uint16_t* scales = (is_k ? a.kv4.k_scales : a.kv4.v_scales) + unit * a.kv4.scale_unit_stride +
                               head * a.kv4.scale_head_stride + static_cast<int64_t>(ur) * nb;
            scales[b] = static_cast<uint16_t>(q.header);
        }
    } else {
        int64_t off;
        if (!a.block_table) {
            if (pos < 0 || pos >= a.cache_rows) {
                atomicOr(a.err, kDevErrBadIndex);
                return;
            }
            off = seq * a.cache_seq_stride + static_cast<int64_t>(pos) * a.cache_row_stride;
        } else {
            const int b = pos >= 0 ? pos / a.block_rows : -1;
            const int blk = (b >= 0 && b < a.max_blocks) ? a.block_table[static_cast<int64_t>(seq) * a.max_blocks + b] : -1;
            if (blk < 0 || blk >= a.pool_blocks) {
                atomicOr(a.err, kDevErrBadIndex);
                return;
            }
            off = static_cast<int64_t>(blk) * a.block_stride + static_cast<int64_t>(pos - b * a.block_rows) * a.cache_row_stride;
        }
        store8(is_k ? a.k_cache : a.v_cache, off + static_cast<int64_t>(head) * a.d + c0, kKind == ALPACA_CACHE_F16, x);
    }
}

template <int LP, int kKind>
__global__ void __launch_bounds__(kAppendThreads, 3) qkv_append_kernel(const __grid_constant__ AppendArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ __align__(16) float s_table[];  // cos [tpc][d/2], sin [tpc][d/2]
    const int t0 = blockIdx.x * a.tpc, seq = blockIdx.y, tid = threadIdx.x;
    const int ntok = min(a.tpc, a.tokens - t0), half = a.d / 2;
    float* s_cos = s_table;
    float* s_sin = s_table + a.tpc * half;
    constexpr int RP = kAppendThreads / LP;  // rows per pass of the CTA
    const int sub = tid / LP, j = tid % LP, per = a.n_heads + 2 * a.n_kv_heads;
    const int step_tokens = RP / per, step_rows = RP - step_tokens * per;
    const bool in = 8 * j < a.d;  // lanes past the row (d not a power of two) only take part in the shuffles
    const auto table = [&](int pos0) {
        for (int i = tid; i < ntok * half; i += kAppendThreads) {
            const int tt = i / half, at = tt * half + table_at(i - tt * half, half, a.interleaved);
            double sn, cs;
            sincos(static_cast<double>(pos0 + tt) * a.freq[i - tt * half], &sn, &cs);
            s_cos[at] = static_cast<float>(cs);
            s_sin[at] = static_cast<float>(sn);
        }
    };
    // A uniform start needs no global data: its table is computed while the previous kernel drains.
    if (!a.positions) table(a.start + t0);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int pos0 = (a.positions ? a.positions[seq] : a.start) + t0;
    float qw[8], kw[8];
#pragma unroll
    for (int e = 0; e < 8; e++) qw[e] = kw[e] = 1.f;
    if (in && a.q_norm) load8(a.q_norm, 8 * j, 0, qw);
    if (in && a.k_norm) load8(a.k_norm, 8 * j, 0, kw);
    RowAt r;
    r.tt = sub / per;
    r.i = sub - r.tt * per;
    float x[kAppendBatch][8];
    const int passes = (ntok * per + RP * kAppendBatch - 1) / (RP * kAppendBatch);
    for (int p = 0; p < passes; p++) {
        RowAt at[kAppendBatch];
#pragma unroll
        for (int b = 0; b < kAppendBatch; b++) {
            at[b] = r;
            r.step(step_tokens, step_rows, per);
#pragma unroll
            for (int e = 0; e < 8; e++) x[b][e] = 0.f;
            if (in && at[b].tt < ntok) load_row(a, seq, t0, at[b], 8 * j, x[b]);
        }
        if (p == 0) {
            if (a.positions) table(pos0);
            __syncthreads();  // once, by every thread
        }
#pragma unroll
        for (int b = 0; b < kAppendBatch; b++)
            finish_row<LP, kKind>(a, seq, t0, pos0, at[b], in && at[b].tt < ntok, j, s_cos, s_sin, qw, kw, x[b]);
    }
}

template <int LP>
cudaError_t launch_append(const AppendArgs& a, int kind, const cudaLaunchConfig_t& cfg) {
    switch (kind) {
        case ALPACA_CACHE_KV4: return cudaLaunchKernelEx(&cfg, qkv_append_kernel<LP, ALPACA_CACHE_KV4>, a);
        case ALPACA_CACHE_F16: return cudaLaunchKernelEx(&cfg, qkv_append_kernel<LP, ALPACA_CACHE_F16>, a);
        default: return cudaLaunchKernelEx(&cfg, qkv_append_kernel<LP, ALPACA_CACHE_F32>, a);
    }
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
    int start, n_rows, n_kv_heads, d, out_f16;
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
        const int row = static_cast<int>(i / a.n_kv_heads), head = static_cast<int>(i - static_cast<int64_t>(row) * a.n_kv_heads);
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

}  // namespace

cudaError_t launch_qkv_append(const alpaca_qkv_desc& d, unsigned* err, cudaStream_t s) {
    AppendArgs a;
    a.q = d.q;
    a.k = d.k;
    a.v = d.v;
    a.q_out = d.q_out;
    a.q_token_stride = d.q_token_stride;
    a.q_seq_stride = d.q_seq_stride;
    a.kv_token_stride = d.kv_token_stride;
    a.kv_seq_stride = d.kv_seq_stride;
    a.out_token_stride = d.q_out_token_stride;
    a.out_seq_stride = d.q_out_seq_stride;
    a.q_norm = d.q_norm;
    a.k_norm = d.k_norm;
    a.eps = d.eps;
    a.inv_d = 1.f / static_cast<float>(d.head_dim);
    a.in_f16 = d.in_dtype == ALPACA_F16;
    a.out_f16 = d.q_out_dtype == ALPACA_F16;
    a.interleaved = d.interleaved;
    a.positions = d.positions;
    a.start = d.start_position;
    a.n_heads = d.n_heads;
    a.n_kv_heads = d.n_kv_heads;
    a.d = d.head_dim;
    a.tokens = d.tokens;
    a.tpc = d.tokens < kAppendTokens ? d.tokens : kAppendTokens;
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
                                              sizeof(float) * a.tpc * d.head_dim, s, &attr);
    const int lanes = d.head_dim / 8;
    return lanes <= 4    ? launch_append<4>(a, d.cache_kind, cfg)
           : lanes <= 8  ? launch_append<8>(a, d.cache_kind, cfg)
           : lanes <= 16 ? launch_append<16>(a, d.cache_kind, cfg)
                         : launch_append<32>(a, d.cache_kind, cfg);
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
    a.d = d.head_dim;
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
