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
// Bound by memory: 2 bytes read and 2 (or 1) written per channel.  A row is held by D/8 lanes, eight channels
// (one 16-byte load) each, so the norm and the row maximum are shuffles and the partner of a half-split rotation is
// one shuffle away.  A warp works on kRows rows per lane group of ONE token: their loads are in flight together, and
// the eight cosines and sines a lane needs (64 bytes, four times the data of a row) are read once for all of them.
#include "common.cuh"

#include <cuda_bf16.h>

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
    int units;                    // warps per token
    void* out;                    // [tokens][heads + kv_heads][D] in the input's type (float form), or
    int8_t* codes;                // [tokens][heads + 2 kv_heads][D]
    float* scales;                // [tokens][heads + 2 kv_heads]
    void* k_out;                  // [tokens][kv_heads][D] in the input's type, or null (quantised form)
};

__device__ __forceinline__ float2 widen(const __half*, uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
__device__ __forceinline__ float2 widen(const __nv_bfloat16*, uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
__device__ __forceinline__ uint32_t narrow(const __half*, float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t narrow(const __nv_bfloat16*, float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// round half to even of y / s as the quantiser defines it: the product with the rounded reciprocal is within a few
// ulps of the quotient, so only quotients next to a tie need the division itself
__device__ __forceinline__ int code_of(float y, float s, float inv) {
    const float t = y * inv;
    float r = rintf(t);
    if (fabsf(t - r) > 0.4999f) r = rintf(__fdiv_rn(y, s));
    return (int)r;
}

template <typename T, int D, bool QUANT>
__global__ void __launch_bounds__(kThreads)
qk_norm_rope_kernel(const QkArgs a) {
    constexpr int LPR = D / 8;                       // lanes per row
    constexpr int GROUPS = 32 / LPR;                 // rows a warp holds side by side
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const long long unit = (long long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    const long long t = unit / a.units;
    if (t >= a.tokens) return;                       // whole warps leave
    const int first = (int)(unit - t * a.units) * (kRows * GROUPS) + lane / LPR;   // this group's first head
    const int sub = lane % LPR;
    const int d0 = sub * 8;
    const int rotated = a.heads + a.kv_heads;        // heads that are normed and rotated; the rest are values
    const int total = QUANT ? rotated + a.kv_heads : rotated;

    const T* row = static_cast<const T*>(a.qkv) + t * a.row_stride + d0;
    uint4 raw[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int h = first + i * GROUPS;
        raw[i] = h < total ? *reinterpret_cast<const uint4*>(row + (long long)h * D) : make_uint4(0u, 0u, 0u, 0u);
    }
    float c[8], s[8];
    const bool turn = a.positions != nullptr;
    const int half_r = a.R >> 1;
    const bool mine = turn && d0 < a.R;              // R is a multiple of 16: a lane's channels are all in or all out
    if (mine) {
        const int pos = a.positions[t];
        const bool known = pos >= 0 && pos < a.rope_rows;
        if (a.interleaved) {                         // four pairs of this lane
            const float* tab = a.rope + (long long)(known ? pos : 0) * a.R + (d0 >> 1);
            const float4 cc = *reinterpret_cast<const float4*>(tab), ss = *reinterpret_cast<const float4*>(tab + half_r);
            c[0] = cc.x, c[1] = cc.y, c[2] = cc.z, c[3] = cc.w;
            s[0] = ss.x, s[1] = ss.y, s[2] = ss.z, s[3] = ss.w;
        } else {
            const float* tab = a.rope + (long long)(known ? pos : 0) * a.R + (d0 < half_r ? d0 : d0 - half_r);
            const float sign = d0 < half_r ? -1.0f : 1.0f;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float4 cc = *reinterpret_cast<const float4*>(tab + 4 * k), ss = *reinterpret_cast<const float4*>(tab + half_r + 4 * k);
                c[4 * k] = cc.x, c[4 * k + 1] = cc.y, c[4 * k + 2] = cc.z, c[4 * k + 3] = cc.w;
                s[4 * k] = sign * ss.x, s[4 * k + 1] = sign * ss.y, s[4 * k + 2] = sign * ss.z, s[4 * k + 3] = sign * ss.w;
            }
        }
        if (!known) {                                // a position without a table row shows in the result
#pragma unroll
            for (int k = 0; k < 8; ++k) c[k] = s[k] = __int_as_float(0x7fc00000);
        }
    }
    // the partner lane of a half-split rotation
    const int partner = lane - sub + (d0 < half_r ? sub + half_r / 8 : sub - half_r / 8);
    const int from = mine ? partner : lane;

#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int h = first + i * GROUPS;
        const uint32_t w4[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
        float y[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 v = widen(static_cast<const T*>(nullptr), w4[k]);
            y[2 * k] = v.x, y[2 * k + 1] = v.y;
        }
        const bool is_qk = h < rotated;
        const float* weight = h < a.heads ? a.q_weight : a.k_weight;
        float ss = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) ss = fmaf(y[k], y[k], ss);
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (is_qk && weight != nullptr) {
            const float r = rsqrtf(ss * (1.0f / D) + a.eps);
            const float4 wa = *reinterpret_cast<const float4*>(weight + d0), wb = *reinterpret_cast<const float4*>(weight + d0 + 4);
            y[0] *= r * wa.x, y[1] *= r * wa.y, y[2] *= r * wa.z, y[3] *= r * wa.w;
            y[4] *= r * wb.x, y[5] *= r * wb.y, y[6] *= r * wb.z, y[7] *= r * wb.w;
        }
        if (turn) {
            if (a.interleaved) {
                if (mine && is_qk) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float u = y[2 * k], v = y[2 * k + 1];
                        y[2 * k] = u * c[k] - v * s[k];
                        y[2 * k + 1] = v * c[k] + u * s[k];
                    }
                }
            } else {
                float z[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) z[k] = __shfl_sync(0xffffffffu, y[k], from);
                if (mine && is_qk) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) y[k] = y[k] * c[k] + z[k] * s[k];
                }
            }
        }
        if constexpr (!QUANT) {
            if (h < total) {
                const T* tag = nullptr;
                *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (t * total + h) * D + d0) =
                    make_uint4(narrow(tag, y[0], y[1]), narrow(tag, y[2], y[3]), narrow(tag, y[4], y[5]), narrow(tag, y[6], y[7]));
            }
        } else {
            float mx = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) mx = fmaxf(mx, fabsf(y[k]));
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            // a row whose position has no table entry is NaN throughout its rotated part: its scale says so
            float scale = __fdiv_rn(fmaxf(mx, 1e-8f), 127.0f);
            const bool bad = mine && is_qk && c[0] != c[0];
            if (__any_sync(0xffffffffu, bad)) {
                const unsigned who = __ballot_sync(0xffffffffu, bad);
                const unsigned group = (LPR == 32 ? 0xffffffffu : ((1u << LPR) - 1u) << (lane - sub));
                if (who & group) scale = __int_as_float(0x7fc00000);
            }
            const float inv = __frcp_rn(scale);
            int q[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) q[k] = code_of(y[k], scale, inv);
            if (h < total) {
                const uint32_t lo = prmt(prmt(q[0], q[1], 0x0040), prmt(q[2], q[3], 0x0040), 0x5410);
                const uint32_t hi = prmt(prmt(q[4], q[5], 0x0040), prmt(q[6], q[7], 0x0040), 0x5410);
                *reinterpret_cast<uint2*>(a.codes + (t * total + h) * D + d0) = make_uint2(lo, hi);
                if (sub == 0) a.scales[t * total + h] = scale;
                if (a.k_out != nullptr && h >= a.heads && is_qk) {
                    const T* tag = nullptr;
                    *reinterpret_cast<uint4*>(static_cast<T*>(a.k_out) + (t * a.kv_heads + (h - a.heads)) * D + d0) =
                        make_uint4(narrow(tag, y[0], y[1]), narrow(tag, y[2], y[3]), narrow(tag, y[4], y[5]), narrow(tag, y[6], y[7]));
                }
            }
        }
    }
}

template <typename T, bool QUANT>
int launch_qk(QkArgs a, int D, cudaStream_t st) {
    const int per_warp = kRows * (256 / D);          // rows of one token a warp takes
    const int total = a.heads + a.kv_heads * (QUANT ? 2 : 1);
    a.units = (total + per_warp - 1) / per_warp;
    const long long warps = a.tokens * a.units;
    const long long blocks = (warps + kThreads / 32 - 1) / (kThreads / 32);
    I8TK_REQUIRE(blocks < (1ll << 31), I8TK_ERR_UNSUPPORTED, "too many tokens");
    const dim3 grid((unsigned)blocks), block(kThreads);
    if (D == 64) I8TK_CUDA(launch_after(qk_norm_rope_kernel<T, 64, QUANT>, grid, block, 0, st, a));
    else if (D == 128) I8TK_CUDA(launch_after(qk_norm_rope_kernel<T, 128, QUANT>, grid, block, 0, st, a));
    else I8TK_CUDA(launch_after(qk_norm_rope_kernel<T, 256, QUANT>, grid, block, 0, st, a));
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
             heads, kv_heads, 0, out, nullptr, nullptr, nullptr};
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
             heads, kv_heads, 0, nullptr, codes, scales, k_out};
    const int rc = check_qk(a, dtype, head_dim);
    if (rc != I8TK_OK) return rc;
    I8TK_REQUIRE(codes && scales, I8TK_ERR_INVALID_ARGUMENT, "null pointer argument");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == I8TK_F16 ? launch_qk<__half, true>(a, head_dim, st) : launch_qk<__nv_bfloat16, true>(a, head_dim, st);
}
