// Writing rows into the 4-bit paged cache, and reading them back (layout: kv4.cuh).
//
//   per 64 channels:  scale  = fp16((max - min) / 15)
//                     centre = fp16(min + 8 * scale)
//                     code   = clamp(rne((x - centre) / scale), -8, 7) + 8       (scale 0: code 8)
//
// Every step is one IEEE operation in fp32 on 16-bit inputs, so the result does not depend on the order of anything.
//
// Bound by memory: 2 bytes read and 9/16 written per channel (read back: the other way round).  Eight lanes hold a
// group of 64 channels, one 16-byte load each; minimum and maximum are three shuffles, a lane's eight codes are
// exactly one word of the row.  A thread takes the key row and the value row of a token together.
// Measured: 16384 tokens, 8 heads, D 128 (86 MB): append 29-30 us, read-back 16-18 us, both at 74 % of the issue slots.
#include "kv4.cuh"
#include "pairs16.cuh"

namespace i8tk {
namespace {

constexpr int kThreads = 128;

// minimum of the pairs in two words; the sign bits of a word flipped
__device__ __forceinline__ uint32_t min2(const __half*, uint32_t a, uint32_t b) {
    const __half2 m = __hmin2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ uint32_t min2(const __nv_bfloat16*, uint32_t a, uint32_t b) {
    const __nv_bfloat162 m = __hmin2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
}

// Codes and pair of the eight channels of this lane in its group of eight lanes.
template <typename T>
__device__ __forceinline__ uint32_t quantize8(uint4 raw, __half2& pair) {
    const T* tag = nullptr;
    constexpr uint32_t kSigns = 0x80008000u;
    // minimum of the values and of their negatives, both as 16-bit numbers: exact, and one word to shuffle
    const uint32_t lo2 = min2(tag, min2(tag, raw.x, raw.y), min2(tag, raw.z, raw.w));
    const uint32_t hi2 = min2(tag, min2(tag, raw.x ^ kSigns, raw.y ^ kSigns), min2(tag, raw.z ^ kSigns, raw.w ^ kSigns));
    uint32_t both = min2(tag, prmt(lo2, hi2, 0x5410u), prmt(lo2, hi2, 0x7632u));
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) both = min2(tag, both, __shfl_xor_sync(0xffffffffu, both, o));
    // the pair is fp16: a range that does not fit saturates
    const float lo = fminf(fmaxf(widen(tag, both).x, -65504.f), 65504.f), hi = fminf(fmaxf(-widen(tag, both).y, -65504.f), 65504.f);
    const __half sh = __float2half_rn(div_by<15>(__fsub_rn(hi, lo)));
    const float s = __half2float(sh);
    const __half zh = __float2half_rn(__fadd_rn(lo, 8.0f * s));
    const float z = __half2float(zh);
    pair = __halves2half2(sh, zh);
    const float inv = s > 0.f ? rcp_approx(s) : 0.f;
    const f32x2 inv2 = pack2(inv, inv), nz2 = pack2(-z, -z);
    // code + 8 in the low bits of 1.5 * 2^23 + 8 + (x - z) / s; the product with the approximate reciprocal is within
    // a few ulps of the quotient, so only next to a tie is it divided (and clamped, where the range saturated: then a
    // quotient may lie far outside)
    const f32x2 magic = pack2(12582920.f, 12582920.f), minus = pack2(-1.f, -1.f);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    f32x2 d[4], q[4];
    float off = fmaxf(fabsf(lo), fabsf(hi)) < 65504.f ? 0.f : 1.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        d[k] = add2(widen(tag, w[k]), nz2);
        const f32x2 t = mul2(d[k], inv2);
        q[k] = add2(t, magic);
        const f32x2 e = add2(t, fma2(q[k], minus, magic));           // the quotient less its rounding
        off = max3(off, fabsf(e.x), fabsf(e.y));
    }
    if (off > 0.4999f && s > 0.f) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            q[k] = pack2(fminf(fmaxf(rintf(__fdiv_rn(d[k].x, s)), -8.f), 7.f) + 12582920.f, fminf(fmaxf(rintf(__fdiv_rn(d[k].y, s)), -8.f), 7.f) + 12582920.f);
    }
    // channels e and e + 4 side by side in 16 bits each, clamped to 0..15, four nibbles apart
    uint32_t word = 0;
    const float qe[8] = {q[0].x, q[0].y, q[1].x, q[1].y, q[2].x, q[2].y, q[3].x, q[3].y};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t p = __vimin_s16x2_relu(prmt(__float_as_uint(qe[e]), __float_as_uint(qe[e + 4]), 0x5410u), 0x000f000fu);
        word += p << (4 * e);
    }
    return word;
}

// Where row (slot, head) lives: its block, and its position in the page; null when the slot is outside the pool.
__device__ __forceinline__ unsigned char* block_of(unsigned char* pool, long long slot, long long slots, int page_shift, unsigned kv_heads,
                                                   unsigned h, int block_bytes, int& at) {
    if (slot < 0 || slot >= slots) return nullptr;
    at = (int)(slot & ((1 << page_shift) - 1));
    return pool + ((slot >> page_shift) * kv_heads + h) * (long long)block_bytes;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads)
kv4_append_kernel(const T* __restrict__ k, const T* __restrict__ v, long long k_stride, long long v_stride,
                  unsigned char* __restrict__ pool, const long long* __restrict__ slots, long long num_slots, int page_shift,
                  unsigned rows, unsigned kv_heads) {
    constexpr int G = D / 64, LPR = D / 8;
    pdl_wait();
    pdl_launch_dependents();
    const int page = 1 << page_shift;
    const int block_bytes = kv4_block_bytes(page, D);
    const int sub = threadIdx.x % LPR, g = sub >> 3, u = sub & 7;
    const unsigned row = (unsigned)blockIdx.x * (kThreads / LPR) + threadIdx.x / LPR;
    const bool there = row < rows;
    const unsigned t = there ? row / kv_heads : 0u, h = there ? row - t * kv_heads : 0u;
    uint4 kr = make_uint4(0u, 0u, 0u, 0u), vr = kr;
    int at = 0;
    unsigned char* block = nullptr;
    if (there) {
        block = block_of(pool, slots[t], num_slots, page_shift, kv_heads, h, block_bytes, at);
        kr = *reinterpret_cast<const uint4*>(k + (long long)t * k_stride + h * D + sub * 8);
        vr = *reinterpret_cast<const uint4*>(v + (long long)t * v_stride + h * D + sub * 8);
    }
    __half2 kp, vp;
    const uint32_t kw = quantize8<T>(kr, kp), vw = quantize8<T>(vr, vp);
    if (block == nullptr) return;
    unsigned char* codes = block + at * kv4_row_bytes(D) + (u * G + g) * 4;
    *reinterpret_cast<uint32_t*>(codes) = kw;
    *reinterpret_cast<uint32_t*>(codes + page * kv4_row_bytes(D)) = vw;
    if (u == 0) {
        __half2* pairs = reinterpret_cast<__half2*>(block + page * D) + at * G + g;
        pairs[0] = kp;
        pairs[page * G] = vp;
    }
}

// Two rows per thread, a block apart: the slot and the codes of both are on their way together.
template <int D>
__global__ void __launch_bounds__(kThreads)
kv4_dequantize_kernel(const unsigned char* __restrict__ pool, const long long* __restrict__ slots, long long num_slots,
                      int page_shift, __half* __restrict__ k, __half* __restrict__ v, unsigned rows, unsigned kv_heads) {
    constexpr int G = D / 64, LPR = D / 8, PER = kThreads / LPR;
    pdl_wait();
    pdl_launch_dependents();
    const int page = 1 << page_shift;
    const int sub = threadIdx.x % LPR, g = sub >> 3, u = sub & 7;
    const unsigned row0 = (unsigned)blockIdx.x * (2 * PER) + threadIdx.x / LPR;
    long long slot[2];
    unsigned h[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const unsigned row = row0 + i * PER, t = row / kv_heads;
        h[i] = row - t * kv_heads;
        slot[i] = row < rows ? slots[t] : -1;
    }
    uint32_t w[2][2];
    __half2 pair[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        int at = 0;
        const unsigned char* block = block_of(const_cast<unsigned char*>(pool), slot[i], num_slots, page_shift, kv_heads, h[i], kv4_block_bytes(page, D), at);
        w[i][0] = w[i][1] = 0u;
        pair[i][0] = pair[i][1] = __floats2half2_rn(0.f, 0.f);
        if (block != nullptr) {
            const unsigned char* codes = block + at * kv4_row_bytes(D) + (u * G + g) * 4;
            const __half2* pairs = reinterpret_cast<const __half2*>(block + page * D) + at * G + g;
            w[i][0] = *reinterpret_cast<const uint32_t*>(codes);
            w[i][1] = *reinterpret_cast<const uint32_t*>(codes + page * kv4_row_bytes(D));
            pair[i][0] = pairs[0];
            pair[i][1] = pairs[page * G];
        }
    }
    const __half2 bias = __floats2half2_rn(1032.f, 1032.f), top = __floats2half2_rn(65504.f, 65504.f), bottom = __floats2half2_rn(-65504.f, -65504.f);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const unsigned row = row0 + i * PER;
        if (row >= rows) return;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const __half2 s = __low2half2(pair[i][m]), z = __high2half2(pair[i][m]);
            uint32_t v4[4];                          // channels e and e + 4
#pragma unroll
            for (int e = 0; e < 4; ++e) {            // 1024 + code as a half, less 1032: exact
                const uint32_t c = ((w[i][m] >> (4 * e)) & 0x000f000fu) | 0x64006400u;
                // one rounding, of scale * (code - 8) + centre; the top code of a group that reaches the end of the fp16
                // range may lie half a step beyond it
                __half2 x = __hfma2(__hsub2(*reinterpret_cast<const __half2*>(&c), bias), s, z);
                x = __hmax2(__hmin2(x, top), bottom);
                v4[e] = *reinterpret_cast<const uint32_t*>(&x);
            }
            *reinterpret_cast<uint4*>((m == 0 ? k : v) + (long long)row * D + sub * 8) =
                make_uint4(prmt(v4[0], v4[1], 0x5410u), prmt(v4[2], v4[3], 0x5410u), prmt(v4[0], v4[1], 0x7632u), prmt(v4[2], v4[3], 0x7632u));
        }
    }
}

int check_kv4(const void* pool, const int64_t* slots, int64_t tokens, int kv_heads, int head_dim, int page_size, int64_t num_pages) {
    I8TK_REQUIRE(pool && slots, I8TK_ERR_INVALID_ARGUMENT, "null pointer argument");
    I8TK_REQUIRE(tokens > 0 && kv_heads > 0 && num_pages > 0, I8TK_ERR_INVALID_ARGUMENT, "sizes must be positive");
    I8TK_REQUIRE(head_dim == 64 || head_dim == 128, I8TK_ERR_UNSUPPORTED, "head_dim must be 64 or 128 (got %d)", head_dim);
    I8TK_REQUIRE(kv4_page_ok(page_size), I8TK_ERR_UNSUPPORTED, "page_size must be 16, 32, 64 or 128 (got %d)", page_size);
    I8TK_REQUIRE(tokens < (1ll << 31) && num_pages < (1ll << 31) && kv_heads < (1 << 16) && tokens * kv_heads < (1ll << 31) - 1024,
                 I8TK_ERR_UNSUPPORTED, "too many rows");
    I8TK_REQUIRE(aligned_to(pool, 16), I8TK_ERR_ALIGNMENT, "the pool must be 16-byte aligned");
    return I8TK_OK;
}

int shift_of(int page) { return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7; }

template <typename T>
int launch_append(const void* k, const void* v, int64_t ks, int64_t vs, void* pool, const int64_t* slots, int64_t tokens,
                  int kv_heads, int D, int page, int64_t num_pages, cudaStream_t st) {
    const long long rows = tokens * kv_heads, blocks = (rows * (D / 8) + kThreads - 1) / kThreads;
    const dim3 grid((unsigned)blocks), block(kThreads);
    if (D == 64)
        I8TK_CUDA(launch_after(kv4_append_kernel<T, 64>, grid, block, 0, st, static_cast<const T*>(k), static_cast<const T*>(v), ks, vs,
                               static_cast<unsigned char*>(pool), reinterpret_cast<const long long*>(slots), num_pages * page,
                               shift_of(page), (unsigned)rows, (unsigned)kv_heads));
    else
        I8TK_CUDA(launch_after(kv4_append_kernel<T, 128>, grid, block, 0, st, static_cast<const T*>(k), static_cast<const T*>(v), ks, vs,
                               static_cast<unsigned char*>(pool), reinterpret_cast<const long long*>(slots), num_pages * page,
                               shift_of(page), (unsigned)rows, (unsigned)kv_heads));
    return I8TK_OK;
}

}  // namespace
}  // namespace i8tk

using namespace i8tk;

extern "C" int64_t i8tk_kv4_block_bytes(int page_size, int head_dim) {
    if (!kv4_page_ok(page_size) || (head_dim != 64 && head_dim != 128)) return 0;
    return kv4_block_bytes(page_size, head_dim);
}

extern "C" int i8tk_kv4_append(const void* k_new, const void* v_new, int dtype, int64_t k_stride, int64_t v_stride, void* pool,
                               const int64_t* slots, int64_t tokens, int kv_heads, int head_dim, int page_size,
                               int64_t num_pages, i8tk_stream_t stream) {
    const int rc = check_kv4(pool, slots, tokens, kv_heads, head_dim, page_size, num_pages);
    if (rc != I8TK_OK) return rc;
    I8TK_REQUIRE(k_new && v_new, I8TK_ERR_INVALID_ARGUMENT, "null pointer argument");
    I8TK_REQUIRE(dtype == I8TK_F16 || dtype == I8TK_BF16, I8TK_ERR_INVALID_ARGUMENT, "dtype must be I8TK_F16 or I8TK_BF16");
    I8TK_REQUIRE(k_stride >= (int64_t)kv_heads * head_dim && v_stride >= (int64_t)kv_heads * head_dim && k_stride % 8 == 0 &&
                     v_stride % 8 == 0,
                 I8TK_ERR_INVALID_ARGUMENT, "token strides must cover a token's heads and be multiples of 8");
    I8TK_REQUIRE(aligned_to(k_new, 16) && aligned_to(v_new, 16), I8TK_ERR_ALIGNMENT, "k_new and v_new must be 16-byte aligned");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == I8TK_F16)
        return launch_append<__half>(k_new, v_new, k_stride, v_stride, pool, slots, tokens, kv_heads, head_dim, page_size, num_pages, st);
    return launch_append<__nv_bfloat16>(k_new, v_new, k_stride, v_stride, pool, slots, tokens, kv_heads, head_dim, page_size, num_pages, st);
}

extern "C" int i8tk_kv4_dequantize(const void* pool, const int64_t* slots, void* k_f16, void* v_f16, int64_t tokens, int kv_heads,
                                   int head_dim, int page_size, int64_t num_pages, i8tk_stream_t stream) {
    const int rc = check_kv4(pool, slots, tokens, kv_heads, head_dim, page_size, num_pages);
    if (rc != I8TK_OK) return rc;
    I8TK_REQUIRE(k_f16 && v_f16, I8TK_ERR_INVALID_ARGUMENT, "null pointer argument");
    I8TK_REQUIRE(aligned_to(k_f16, 16) && aligned_to(v_f16, 16), I8TK_ERR_ALIGNMENT, "k and v must be 16-byte aligned");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const long long rows = tokens * kv_heads, per = 2 * kThreads / (head_dim / 8), blocks = (rows + per - 1) / per;
    const dim3 grid((unsigned)blocks), block(kThreads);
    const unsigned char* p = static_cast<const unsigned char*>(pool);
    const long long* sl = reinterpret_cast<const long long*>(slots);
    if (head_dim == 64)
        I8TK_CUDA(launch_after(kv4_dequantize_kernel<64>, grid, block, 0, st, p, sl, num_pages * page_size, shift_of(page_size),
                               static_cast<__half*>(k_f16), static_cast<__half*>(v_f16), (unsigned)rows, (unsigned)kv_heads));
    else
        I8TK_CUDA(launch_after(kv4_dequantize_kernel<128>, grid, block, 0, st, p, sl, num_pages * page_size, shift_of(page_size),
                               static_cast<__half*>(k_f16), static_cast<__half*>(v_f16), (unsigned)rows, (unsigned)kv_heads));
    return I8TK_OK;
}
