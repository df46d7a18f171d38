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
// kv4_read_kernel: eight values of a row per thread and step, f16 or f32 out in the [seq][row][head][d] layout of the
// f16 cache. It moves 0.56 d + 2 d (f16) bytes per row: HBM-bound.
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
    float eps;
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

// Row `row` of the CTA's tokens: its token, kind and head.
struct RowAt {
    int tt, head;
    bool q, k;
};
__device__ __forceinline__ RowAt row_at(const AppendArgs& a, int row) {
    const int per = a.n_heads + 2 * a.n_kv_heads;
    RowAt r;
    r.tt = row / per;
    const int i = row - r.tt * per;
    r.q = i < a.n_heads;
    r.k = !r.q && i < a.n_heads + a.n_kv_heads;
    r.head = r.q ? i : (r.k ? i - a.n_heads : i - a.n_heads - a.n_kv_heads);
    return r;
}

__device__ __forceinline__ void load_row(const AppendArgs& a, int seq, int t0, int row, int c0, float (&x)[8]) {
    const RowAt r = row_at(a, row);
    const int64_t t = t0 + r.tt;
    if (r.q) load8(a.q, seq * a.q_seq_stride + t * a.q_token_stride + static_cast<int64_t>(r.head) * a.d + c0, a.in_f16, x);
    else load8(r.k ? a.k : a.v, seq * a.kv_seq_stride + t * a.kv_token_stride + static_cast<int64_t>(r.head) * a.d + c0, a.in_f16, x);
}

// kKind: alpaca_cache_kind. LP: lanes per row.
template <int LP, int kKind>
__device__ __forceinline__ void finish_row(const AppendArgs& a, int seq, int t0, int pos0, int row, bool active, int j,
                                           const float* s_cos, const float* s_sin, float (&x)[8]) {
    const RowAt r = row_at(a, active ? row : 0);
    const int half = a.d / 2, c0 = 8 * j;
    const float* w = r.q ? a.q_norm : (r.k ? a.k_norm : nullptr);
    if (a.q_norm || a.k_norm) {  // the same for the whole grid: every lane takes part in the shuffles
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e++) ss = fmaf(x[e], x[e], ss);
#pragma unroll
        for (int o = LP / 2; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (w && active) {
            const float inv = 1.f / sqrtf(ss / static_cast<float>(a.d) + a.eps);
            const float4 w0 = *reinterpret_cast<const float4*>(w + c0), w1 = *reinterpret_cast<const float4*>(w + c0 + 4);
            const float wv[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = __fmul_rn(__fmul_rn(x[e], inv), wv[e]);
        }
    }
    const bool rotate = active && (r.q || r.k);
    if (a.interleaved) {
        if (rotate) {
            const float4 c = *reinterpret_cast<const float4*>(s_cos + r.tt * half + c0 / 2);
            const float4 s = *reinterpret_cast<const float4*>(s_sin + r.tt * half + c0 / 2);
            const float cv[4] = {c.x, c.y, c.z, c.w}, sv[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float x0 = x[2 * e], x1 = x[2 * e + 1];
                x[2 * e] = __fsub_rn(__fmul_rn(x0, cv[e]), __fmul_rn(x1, sv[e]));
                x[2 * e + 1] = __fadd_rn(__fmul_rn(x0, sv[e]), __fmul_rn(x1, cv[e]));
            }
        }
    } else {
        // channel i pairs with i + d/2: the lane d/16 further on holds the partners of this lane's eight channels
        const int lane = threadIdx.x & 31, hl = a.d / 16;
        const bool first = j < hl;
        const int other = active ? (first ? lane + hl : lane - hl) : lane;
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; e++) p[e] = __shfl_sync(0xffffffffu, x[e], other);
        if (rotate) {
            const int i0 = r.tt * half + (first ? c0 : c0 - half);
#pragma unroll
            for (int e4 = 0; e4 < 8; e4 += 4) {
                const float4 c = *reinterpret_cast<const float4*>(s_cos + i0 + e4);
                const float4 s = *reinterpret_cast<const float4*>(s_sin + i0 + e4);
                const float cv[4] = {c.x, c.y, c.z, c.w}, sv[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float own = x[e4 + e], par = p[e4 + e];
                    x[e4 + e] = first ? __fsub_rn(__fmul_rn(own, cv[e]), __fmul_rn(par, sv[e]))
                                      : __fadd_rn(__fmul_rn(par, sv[e]), __fmul_rn(own, cv[e]));
                }
            }
        }
    }
    float lo = 0.f, hi = 0.f;
    if (kKind == ALPACA_CACHE_KV4) {  // block extremes, with 0 in the range: four lanes hold a block
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
    if (r.q) {
        store8(a.q_out, seq * a.out_seq_stride + t * a.out_token_stride + static_cast<int64_t>(r.head) * a.d + c0, a.out_f16, x);
        return;
    }
    const int pos = pos0 + r.tt;
    if (kKind == ALPACA_CACHE_KV4) {
        int64_t unit;
        int ur;
        if (!kv4_locate(a.kv4, seq, pos, a.err, unit, ur)) return;
        float step, zero;
        const uint32_t header = kv4_header(lo, hi, step, zero);
        uint32_t word = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) word |= kv4_code(x[e], step, zero) << (4 * e);
        const int nb = a.d / 32, b = j >> 2, tw = j & 3;
        uint8_t* codes = (r.k ? a.kv4.k_codes : a.kv4.v_codes) + unit * a.kv4.code_unit_stride +
                         r.head * a.kv4.code_head_stride + static_cast<int64_t>(ur) * (a.d / 2);
        *reinterpret_cast<uint32_t*>(codes + 4 * (tw * nb + b)) = word;
        if (tw == 0) {
            uint16_t* scales = (r.k ? a.kv4.k_scales : a.kv4.v_scales) + unit * a.kv4.scale_unit_stride +
                               r.head * a.kv4.scale_head_stride + static_cast<int64_t>(ur) * nb;
            scales[b] = static_cast<uint16_t>(header);
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
        store8(r.k ? a.k_cache : a.v_cache, off + static_cast<int64_t>(r.head) * a.d + c0, kKind == ALPACA_CACHE_F16, x);
    }
}

template <int LP, int kKind>
__global__ void __launch_bounds__(kAppendThreads) qkv_append_kernel(const __grid_constant__ AppendArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ __align__(16) float s_table[];  // cos [tpc][d/2], sin [tpc][d/2]
    const int t0 = blockIdx.x * a.tpc, seq = blockIdx.y, tid = threadIdx.x;
    const int ntok = min(a.tpc, a.tokens - t0), half = a.d / 2;
    const int total = ntok * (a.n_heads + 2 * a.n_kv_heads);
    float* s_cos = s_table;
    float* s_sin = s_table + a.tpc * half;
    constexpr int RP = kAppendThreads / LP;  // rows per pass of the CTA
    const int sub = tid / LP, j = tid % LP;
    const bool in = 8 * j < a.d;  // lanes past the row (d not a power of two) only take part in the shuffles
    const auto table = [&](int pos0) {
        for (int i = tid; i < ntok * half; i += kAppendThreads) {
            const int tt = i / half;
            double sn, cs;
            sincos(static_cast<double>(pos0 + tt) * a.freq[i - tt * half], &sn, &cs);
            s_cos[i] = static_cast<float>(cs);
            s_sin[i] = static_cast<float>(sn);
        }
    };
    // A uniform start needs no global data: its table is computed while the previous kernel drains.
    if (!a.positions) table(a.start + t0);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int pos0 = (a.positions ? a.positions[seq] : a.start) + t0;
    float x[kAppendBatch][8];
    for (int base = 0; base < total; base += RP * kAppendBatch) {
#pragma unroll
        for (int b = 0; b < kAppendBatch; b++) {
            const int row = base + b * RP + sub;
#pragma unroll
            for (int e = 0; e < 8; e++) x[b][e] = 0.f;
            if (in && row < total) load_row(a, seq, t0, row, 8 * j, x[b]);
        }
        if (base == 0) {
            if (a.positions) table(pos0);
            __syncthreads();  // once: `base` is the same in every thread
        }
#pragma unroll
        for (int b = 0; b < kAppendBatch; b++) {
            const int row = base + b * RP + sub;
            finish_row<LP, kKind>(a, seq, t0, pos0, row, in && row < total, j, s_cos, s_sin, x[b]);
        }
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
constexpr int kReadBatch = 4;  // words in flight per thread

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

__global__ void __launch_bounds__(kReadThreads) kv4_read_kernel(const __grid_constant__ ReadArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int seq = blockIdx.y, nb = a.d / 32, lpr = a.d / 8, per_row = a.n_kv_heads * lpr;
    const uint8_t* codes = blockIdx.z ? a.c.v_codes : a.c.k_codes;
    const uint16_t* scales = blockIdx.z ? a.c.v_scales : a.c.k_scales;
    void* out = blockIdx.z ? a.v_out : a.k_out;
    const int start = a.row_starts ? a.row_starts[seq] : a.start;
    int rows = a.n_rows;
    if (a.q_offsets) {  // entries out of bounds are reported by the prefill's plan kernel, which skips the sequence
        const int64_t n = static_cast<int64_t>(a.q_offsets[seq + 1]) - a.q_offsets[seq];
        rows = n > 0 ? static_cast<int>(max(min(a.start_positions[seq] + n, static_cast<int64_t>(a.n_rows)), static_cast<int64_t>(0))) : 0;
    }
    const int64_t total = static_cast<int64_t>(rows) * per_row;
    const int64_t i0 = static_cast<int64_t>(blockIdx.x) * (kReadThreads * kReadBatch) + threadIdx.x;
    uint32_t w[kReadBatch], h[kReadBatch];
    int64_t at[kReadBatch];
#pragma unroll
    for (int b = 0; b < kReadBatch; b++) {
        const int64_t i = i0 + b * kReadThreads;
        at[b] = -1;
        w[b] = h[b] = 0;
        if (i < total) {
            const int row = static_cast<int>(i / per_row), rem = static_cast<int>(i - static_cast<int64_t>(row) * per_row);
            const int head = rem / lpr, j = rem - head * lpr;
            at[b] = seq * a.out_seq_stride + row * a.out_row_stride + static_cast<int64_t>(head) * a.d + 8 * j;
            int64_t unit;
            int ur;
            if (kv4_locate(a.c, seq, start + row, a.err, unit, ur)) {  // else the row reads as zero
                w[b] = *reinterpret_cast<const uint32_t*>(codes + unit * a.c.code_unit_stride + head * a.c.code_head_stride +
                                                          static_cast<int64_t>(ur) * (a.d / 2) + 4 * ((j & 3) * nb + (j >> 2)));
                h[b] = scales[unit * a.c.scale_unit_stride + head * a.c.scale_head_stride + static_cast<int64_t>(ur) * nb + (j >> 2)];
            }
        }
    }
#pragma unroll
    for (int b = 0; b < kReadBatch; b++) {
        if (at[b] < 0) continue;
        const uint4 u = kv4_word_values(w[b], h[b]);
        if (a.out_f16) {
            *reinterpret_cast<uint4*>(static_cast<__half*>(out) + at[b]) = u;
        } else {
            float4* o = reinterpret_cast<float4*>(static_cast<float*>(out) + at[b]);
            const float2 f0 = __half22float2(as_half2(u.x)), f1 = __half22float2(as_half2(u.y));
            const float2 f2 = __half22float2(as_half2(u.z)), f3 = __half22float2(as_half2(u.w));
            o[0] = make_float4(f0.x, f0.y, f1.x, f1.y);
            o[1] = make_float4(f2.x, f2.y, f3.x, f3.y);
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
    const int64_t words = static_cast<int64_t>(d.n_rows) * d.n_kv_heads * (d.head_dim / 8);
    const int64_t per = kReadThreads * kReadBatch;
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg =
        pdl_config(dim3(static_cast<unsigned>((words + per - 1) / per), d.n_seqs, 2), kReadThreads, 0, s, &attr);
    return cudaLaunchKernelEx(&cfg, kv4_read_kernel, a);
}

}  // namespace alpaca
