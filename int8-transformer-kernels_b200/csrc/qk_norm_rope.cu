// Queries and keys of a grouped-head layer between the QKV projection and attention: per-head RMS norm,
// position rotation and (optionally) the per-token INT8 quantiser, in one pass over the projection.
//
//   y = x * rsqrt(mean(x^2) + eps) * w                    per (token, head) row of D channels; no norm: y = x
//   (y_a, y_b) -> (y_a c - y_b s, y_b c + y_a s)          pairs (d, d + R/2), or (2i, 2i+1) when interleaved, of the
//                                                         first R channels; c, s from the table row of the position
//   quantised: scale = max(max|y|, 1e-8) / 127, code = rne(y / scale)
//
// All in fp32 from the 16-bit input, one rounding at the end (to the input's type, or to the code).
//
// Memory moves 2 bytes in and 2 (or 1) out per channel; at that rate an SM has about 15 instruction slots of a lane
// per channel, so the arithmetic is what has to be kept short:
// * norm, weight and rotation are u = x * (w c) + z * (w' s) and y = r u, where z is the partner channel and w' its
//   weight.  The products with the weights are made once for the rows of a warp, which are heads of one kind (query,
//   key or value) of ONE token; the partner comes by one shuffle of the raw 16-bit pair (half split) or by swapping
//   the halves of a word (interleaved).  Packed fp32 pairs throughout.
// * r never touches the channels in the quantised form: it goes into the scale.
// * Rounding is the addition of 1.5 * 2^23, the code is the low byte of the sum.
// A row is held by D/8 lanes, eight channels (one 16-byte load) each; a warp has kRows rows per lane group in flight.
// Measured: 8192 bf16 tokens, 32/8 heads, D 128, quantised: 42-44 us for 156 MB, 69 % of the issue slots (84 us before the
// norm, weight and rotation were joined and the kinds of rotation split).
#include "pairs16.cuh"

namespace i8tk {
namespace {

constexpr int kRows = 4;          // rows of one token per lane group
constexpr int kThreads = 128;

struct QkArgs {
    const void* qkv;              // [tokens] rows of (heads + 2 kv_heads) * D channels, row_stride channels apart
    long long row_stride;
    const float* q_weight;        // [D] or null: no norm
    const float* k_weight;
    const int* positions;         // [tokens] or null: no rotation
    const float* rope;            // [rope_rows][R]: cosines of the R/2 frequencies, then their sines
    int rope_rows;
    int R;
    int interleaved;
    float eps;
    long long tokens;
    int heads, kv_heads;
    int q_units, k_units, units;  // warps per token: of query heads, of key heads, in all
    void* out;                    // [tokens][heads + kv_heads][D] in the input's type (float form), or
    int8_t* codes;                // [tokens][heads + 2 kv_heads][D]
    float* scales;                // [tokens][heads + 2 kv_heads]
    void* k_out;                  // [tokens][kv_heads][D] in the input's type, or null (quantised form)
};

__device__ __forceinline__ uint32_t narrow(const __half*, float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t narrow(const __nv_bfloat16*, float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// maximum that is NaN when an operand is
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// ROT: 0 no rotation, 1 half-split pairs, 2 interleaved pairs.
template <typename T, int D, bool QUANT, int ROT>
__global__ void __launch_bounds__(kThreads, 8)
qk_norm_rope_kernel(const QkArgs a) {
    constexpr int LPR = D / 8;                       // lanes per row
    constexpr int GROUPS = 32 / LPR;                 // rows a warp holds side by side
    constexpr int PER = kRows * GROUPS;              // rows of a warp
    const T* tag = nullptr;
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, sub = lane % LPR, d0 = sub * 8;
    const unsigned chunk = blockIdx.x / (unsigned)a.units;
    const int unit = (int)(blockIdx.x - chunk * (unsigned)a.units);
    const long long t = (long long)chunk * (kThreads / 32) + (threadIdx.x >> 5);
    if (t >= a.tokens) return;                       // whole warps leave
    // units of query heads first, then of key heads, then of value heads
    const int kind = unit < a.q_units ? 0 : unit < a.q_units + a.k_units ? 1 : 2;
    const int head0 = kind == 0 ? 0 : kind == 1 ? a.heads : a.heads + a.kv_heads;
    const int count = kind == 0 ? a.heads : a.kv_heads;
    const int unit0 = (unit - (kind == 0 ? 0 : kind == 1 ? a.q_units : a.q_units + a.k_units)) * PER;    // first head of the warp
    const int left = count - unit0 - lane / LPR;     // heads from this group's first one on
    const int total = a.heads + a.kv_heads * (QUANT ? 2 : 1);
    const int first = head0 + unit0 + lane / LPR;    // this group's first head of the token

    const T* row = static_cast<const T*>(a.qkv) + t * a.row_stride + (first * D + d0);
    uint4 raw[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i)
        raw[i] = i * GROUPS < left ? *reinterpret_cast<const uint4*>(row + i * GROUPS * D) : make_uint4(0u, 0u, 0u, 0u);

    const long long at = t * total + first;
    T* out = static_cast<T*>(a.out) + at * D + d0;
    int8_t* codes = a.codes + at * D + d0;
    float* scales = a.scales + at;
    const f32x2 magic = pack2(12582912.f, 12582912.f), minus = pack2(-1.f, -1.f);
    auto store_codes = [&](int i, const f32x2* q, float scale) {
        if (i * GROUPS < left) {
            const uint32_t b0 = prmt(__float_as_uint(q[0].x), __float_as_uint(q[0].y), 0x0040), b1 = prmt(__float_as_uint(q[1].x), __float_as_uint(q[1].y), 0x0040);
            const uint32_t b2 = prmt(__float_as_uint(q[2].x), __float_as_uint(q[2].y), 0x0040), b3 = prmt(__float_as_uint(q[3].x), __float_as_uint(q[3].y), 0x0040);
            *reinterpret_cast<uint2*>(codes + i * GROUPS * D) = make_uint2(prmt(b0, b1, 0x5410), prmt(b2, b3, 0x5410));
            if (sub == 0) scales[i * GROUPS] = scale;
        }
    };

    if (QUANT && (kind == 2 || (ROT == 0 && a.q_weight == nullptr))) {
        // rows that are only quantised get exactly the per-token quantiser: a quotient next to a tie is divided
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            if (unit0 + i * GROUPS >= count) break;  // the whole warp is past the last head
            const f32x2 u[4] = {widen(tag, raw[i].x), widen(tag, raw[i].y), widen(tag, raw[i].z), widen(tag, raw[i].w)};
            float mx = max3(max3(fabsf(u[0].x), fabsf(u[0].y), fabsf(u[1].x)), fabsf(u[1].y),
                            max3(fabsf(u[2].x), fabsf(u[2].y), fmaxf(fabsf(u[3].x), fabsf(u[3].y))));
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            mx = fmaxf(mx, 1e-8f);
            const float scale = mx < INFINITY ? div_by<127>(mx) : mx, inv = rcp_approx(scale);
            const f32x2 inv2 = pack2(inv, inv);
            f32x2 q[4];
            float off = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                q[k] = fma2(u[k], inv2, magic);
                const f32x2 d = fma2(u[k], inv2, fma2(q[k], minus, magic));      // the quotient less its rounding
                off = max3(off, fabsf(d.x), fabsf(d.y));
            }
            if (off > 0.4999f) {
#pragma unroll
                for (int k = 0; k < 4; ++k) q[k] = pack2(rintf(__fdiv_rn(u[k].x, scale)) + 12582912.f, rintf(__fdiv_rn(u[k].y, scale)) + 12582912.f);
            }
            store_codes(i, q, scale);
            if (kind == 1 && a.k_out != nullptr && i * GROUPS < left)
                *reinterpret_cast<uint4*>(static_cast<T*>(a.k_out) + (t * a.kv_heads + (first - head0) + i * GROUPS) * D + d0) = raw[i];
        }
        return;
    }

    // ---- what the rows share: w c and w' s of this lane's channels ----
    f32x2 wc[4], ws[4];
    const int half_r = a.R >> 1;
    const bool norm = a.q_weight != nullptr;
    const bool turn = ROT != 0 && d0 < a.R;          // R is a multiple of 16: all of a lane's channels or none
    const int partner = d0 < half_r ? sub + half_r / 8 : sub - half_r / 8;     // lane of the half-split partner
    const int from = lane - sub + (ROT == 1 && turn ? partner : sub);
    bool known = true;                               // a position without a table row shows in the result
    {
        const float* weight = kind == 0 ? a.q_weight : a.k_weight;
        float w[8], wp[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] = wp[k] = 1.0f;
        if (norm) {
            const float* own = weight + d0;
            const float* other = weight + (ROT == 1 && turn ? partner * 8 : d0);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float4 x = *reinterpret_cast<const float4*>(own + 4 * k), y = *reinterpret_cast<const float4*>(other + 4 * k);
                w[4 * k] = x.x, w[4 * k + 1] = x.y, w[4 * k + 2] = x.z, w[4 * k + 3] = x.w;
                wp[4 * k] = y.x, wp[4 * k + 1] = y.y, wp[4 * k + 2] = y.z, wp[4 * k + 3] = y.w;
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) wc[k] = pack2(w[2 * k], w[2 * k + 1]), ws[k] = pack2(0.f, 0.f);
        if constexpr (ROT != 0) {
            const int pos = a.positions[t];
            known = pos >= 0 && pos < a.rope_rows;
            const float* tab = a.rope + (long long)(known ? pos : 0) * a.R;
            if (ROT == 2 && turn) {                  // four pairs of this lane: the partner is the other half of a word
                const float4 c = *reinterpret_cast<const float4*>(tab + (d0 >> 1)), s = *reinterpret_cast<const float4*>(tab + half_r + (d0 >> 1));
                const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    wc[k] = pack2(w[2 * k] * cs[k], w[2 * k + 1] * cs[k]);
                    ws[k] = pack2(-w[2 * k + 1] * sn[k], w[2 * k] * sn[k]);
                }
            } else if (turn) {
                const float* c0 = tab + (d0 < half_r ? d0 : d0 - half_r);
                const float sign = d0 < half_r ? -1.0f : 1.0f;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float4 c = *reinterpret_cast<const float4*>(c0 + 4 * k), s = *reinterpret_cast<const float4*>(c0 + half_r + 4 * k);
                    wc[2 * k] = pack2(w[4 * k] * c.x, w[4 * k + 1] * c.y), wc[2 * k + 1] = pack2(w[4 * k + 2] * c.z, w[4 * k + 3] * c.w);
                    ws[2 * k] = pack2(wp[4 * k] * (sign * s.x), wp[4 * k + 1] * (sign * s.y));
                    ws[2 * k + 1] = pack2(wp[4 * k + 2] * (sign * s.z), wp[4 * k + 3] * (sign * s.w));
                }
            }
            if (turn && !known) {
#pragma unroll
                for (int k = 0; k < 4; ++k) wc[k] = pack2(__int_as_float(0x7fc00000), __int_as_float(0x7fc00000));
            }
        }
    }

#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        if (unit0 + i * GROUPS >= count) break;      // the whole warp is past the last head
        const uint32_t x4[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
        f32x2 u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) u[k] = widen(tag, x4[k]);
        f32x2 sq = mul2(u[0], u[0]);
#pragma unroll
        for (int k = 1; k < 4; ++k) sq = fma2(u[k], u[k], sq);
        float ss = sq.x + sq.y;
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float r = norm ? rsqrtf(ss * (1.0f / D) + a.eps) : 1.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) u[k] = mul2(u[k], wc[k]);
        if constexpr (ROT != 0) {
            uint32_t z4[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) z4[k] = ROT == 2 ? prmt(x4[k], 0u, 0x1032u) : __shfl_sync(0xffffffffu, x4[k], from);
            if (turn) {                              // (a lane outside the rotated channels must not see 0 * infinity)
#pragma unroll
                for (int k = 0; k < 4; ++k) u[k] = fma2(widen(tag, z4[k]), ws[k], u[k]);
            }
        }
        const f32x2 r2 = pack2(r, r);
        if constexpr (!QUANT) {
#pragma unroll
            for (int k = 0; k < 4; ++k) u[k] = mul2(u[k], r2);
            if (i * GROUPS < left)
                *reinterpret_cast<uint4*>(out + i * GROUPS * D) =
                    make_uint4(narrow(tag, u[0].x, u[0].y), narrow(tag, u[1].x, u[1].y), narrow(tag, u[2].x, u[2].y), narrow(tag, u[3].x, u[3].y));
        } else {
            // a NaN or an infinity anywhere in the head makes the scale NaN (the product with r = 0 of an infinity is NaN, and
            // so is div_by of one)
            float mx = max3_nan(max3_nan(fabsf(u[0].x), fabsf(u[0].y), fabsf(u[1].x)), fabsf(u[1].y),
                                max3_nan(fabsf(u[2].x), fabsf(u[2].y), max_nan(fabsf(u[3].x), fabsf(u[3].y))));
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float scale = known ? div_by<127>(max_nan(mx * r, 1e-8f)) : __int_as_float(0x7fc00000);
            const float inv = rcp_approx(scale) * r;
            const f32x2 inv2 = pack2(inv, inv);
            f32x2 q[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) q[k] = fma2(u[k], inv2, magic);
            store_codes(i, q, scale);
            if (kind == 1 && a.k_out != nullptr && i * GROUPS < left) {
#pragma unroll
                for (int k = 0; k < 4; ++k) u[k] = mul2(u[k], r2);
                *reinterpret_cast<uint4*>(static_cast<T*>(a.k_out) + (t * a.kv_heads + (first - head0) + i * GROUPS) * D + d0) =
                    make_uint4(narrow(tag, u[0].x, u[0].y), narrow(tag, u[1].x, u[1].y), narrow(tag, u[2].x, u[2].y), narrow(tag, u[3].x, u[3].y));
            }
        }
    }
}

template <typename T, int D, bool QUANT>
cudaError_t launch_rot(const QkArgs& a, dim3 grid, cudaStream_t st) {
    if (a.positions == nullptr) return launch_after(qk_norm_rope_kernel<T, D, QUANT, 0>, grid, dim3(kThreads), 0, st, a);
    if (!a.interleaved) return launch_after(qk_norm_rope_kernel<T, D, QUANT, 1>, grid, dim3(kThreads), 0, st, a);
    return launch_after(qk_norm_rope_kernel<T, D, QUANT, 2>, grid, dim3(kThreads), 0, st, a);
}

template <typename T, bool QUANT>
int launch_qk(QkArgs a, int D, cudaStream_t st) {
    const int per_warp = kRows * (256 / D);          // rows of one token a warp takes
    a.q_units = (a.heads + per_warp - 1) / per_warp;
    a.k_units = (a.kv_heads + per_warp - 1) / per_warp;
    a.units = a.q_units + a.k_units * (QUANT ? 2 : 1);
    const long long blocks = (a.tokens + kThreads / 32 - 1) / (kThreads / 32) * a.units;
    I8TK_REQUIRE(blocks < (1ll << 31), I8TK_ERR_UNSUPPORTED, "too many tokens");
    const dim3 grid((unsigned)blocks);
    I8TK_CUDA((D == 64 ? launch_rot<T, 64, QUANT>(a, grid, st) : D == 128 ? launch_rot<T, 128, QUANT>(a, grid, st) : launch_rot<T, 256, QUANT>(a, grid, st)));
    return I8TK_OK;
}

int check_qk(const QkArgs& a, int dtype, int D) {
    I8TK_REQUIRE(a.qkv != nullptr, I8TK_ERR_INVALID_ARGUMENT, "null pointer argument");
    I8TK_REQUIRE(dtype == I8TK_F16 || dtype == I8TK_BF16, I8TK_ERR_INVALID_ARGUMENT, "dtype must be I8TK_F16 or I8TK_BF16");
    I8TK_REQUIRE(a.tokens > 0 && a.heads > 0 && a.kv_heads > 0, I8TK_ERR_INVALID_ARGUMENT, "sizes must be positive");
    I8TK_REQUIRE(D == 64 || D == 128 || D == 256, I8TK_ERR_UNSUPPORTED, "head_dim must be 64, 128 or 256 (got %d)", D);
    I8TK_REQUIRE((long long)a.heads + 2ll * a.kv_heads < (1 << 20), I8TK_ERR_UNSUPPORTED, "too many heads");
    I8TK_REQUIRE(a.row_stride >= ((long long)a.heads + 2ll * a.kv_heads) * D && a.row_stride % 8 == 0, I8TK_ERR_INVALID_ARGUMENT,
                 "row_stride must cover a row and be a multiple of 8");
    I8TK_REQUIRE((a.q_weight == nullptr) == (a.k_weight == nullptr), I8TK_ERR_INVALID_ARGUMENT,
                 "q_weight and k_weight are given together or not at all");
    I8TK_REQUIRE((a.positions == nullptr) == (a.rope == nullptr), I8TK_ERR_INVALID_ARGUMENT,
                 "positions and the rotation table are given together or not at all");
    I8TK_REQUIRE(a.positions == nullptr || (a.R > 0 && a.R <= D && a.R % 16 == 0 && a.rope_rows > 0), I8TK_ERR_UNSUPPORTED,
                 "rotary_dim must be a multiple of 16, at most head_dim, and the table must have rows");
    I8TK_REQUIRE(aligned_to(a.qkv, 16) && aligned_to(a.out, 16) && aligned_to(a.codes, 16) && aligned_to(a.k_out, 16) &&
                     aligned_to(a.rope, 16) && aligned_to(a.q_weight, 16) && aligned_to(a.k_weight, 16),
                 I8TK_ERR_ALIGNMENT, "qkv, the outputs, the table and the weights must be 16-byte aligned");
    return I8TK_OK;
}

}  // namespace
}  // namespace i8tk

using namespace i8tk;

extern "C" int i8tk_qk_norm_rope(const void* qkv, int dtype, int64_t row_stride, const float* q_weight, const float* k_weight,
                                 const int32_t* positions, const float* rope_table, int rope_rows, int rotary_dim,
                                 int interleaved, float eps, void* out, int64_t tokens, int heads, int kv_heads,
                                 int head_dim, i8tk_stream_t stream) {
    QkArgs a{qkv, row_stride, q_weight, k_weight, positions, rope_table, rope_rows, rotary_dim, interleaved, eps, tokens,
             heads, kv_heads, 0, 0, 0, out, nullptr, nullptr, nullptr};
    const int rc = check_qk(a, dtype, head_dim);
    if (rc != I8TK_OK) return rc;
    I8TK_REQUIRE(out != nullptr, I8TK_ERR_INVALID_ARGUMENT, "null pointer argument");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == I8TK_F16 ? launch_qk<__half, false>(a, head_dim, st) : launch_qk<__nv_bfloat16, false>(a, head_dim, st);
}

extern "C" int i8tk_qk_norm_rope_quantize(const void* qkv, int dtype, int64_t row_stride, const float* q_weight,
                                          const float* k_weight, const int32_t* positions, const float* rope_table,
                                          int rope_rows, int rotary_dim, int interleaved, float eps, int8_t* codes,
                                          float* scales, void* k_out, int64_t tokens, int heads, int kv_heads,
                                          int head_dim, i8tk_stream_t stream) {
    QkArgs a{qkv, row_stride, q_weight, k_weight, positions, rope_table, rope_rows, rotary_dim, interleaved, eps, tokens,
             heads, kv_heads, 0, 0, 0, nullptr, codes, scales, k_out};
    const int rc = check_qk(a, dtype, head_dim);
    if (rc != I8TK_OK) return rc;
    I8TK_REQUIRE(codes && scales, I8TK_ERR_INVALID_ARGUMENT, "null pointer argument");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == I8TK_F16 ? launch_qk<__half, true>(a, head_dim, st) : launch_qk<__nv_bfloat16, true>(a, head_dim, st);
}
