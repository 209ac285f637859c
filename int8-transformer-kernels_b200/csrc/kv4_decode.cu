// Decode attention (one query token per request) over the paged 4-bit cache of kv4.cuh, with grouped heads.
//
//   score_j = (q . k_j) * sQ / sqrt(D),   k_j = s (c - 8) + z per 64 channels,   out = softmax(score) . v
//
// q is INT8 with one scale per head, so q . c is an integer sum and
//   q . k_j = sum over the groups of  s_j ((q . c_j) - 8 Q) + z_j Q,      Q = sum of the group's query codes;
//   out     = sum over the groups of  [sum_j P_j c_j] - 8 [sum_j P_j] + sum_j p_j z_j,      P_j = fp16(p_j s_j).
// The - 8 is applied to the sums: with P rounded, sum P (c - 8) is what comes out, without the cancellation that
// unsigned codes would otherwise bring into the rounding error of P.
//
// Bound by memory: D + D/8 bytes per position and key head, read once for all the query heads that share them
// (D=128: 144 bytes; FP16 would be 512).  What has to be kept out of the way is the unpacking, 2 D codes a position:
// * Both products are tensor-core instructions (m16n8k16) in the orientation where the CACHE is the 16-row operand
//   and the query heads are the 8 columns, so a group of up to 8 heads costs one instruction per 16x16 codes.
// * A code needs no conversion to fp16: the bits of a nibble in the low bits of a half are the subnormal c * 2^-24
//   (bits 4-7: 16 c * 2^-24), which the tensor core multiplies exactly.  A key word is four ANDs and a shift for
//   eight codes, the 1/16 of the high nibbles sits in the query operand; a value word pairs two positions with a byte
//   permute first, its 1/16 is applied to the accumulators at the end.
// * The scores come out with positions as rows; the probabilities turn around for the second product with one
//   8x8 transposing move per eight positions.
//
// The tiles (128 positions) of all (request, key head) rows, in that order, are one sequence, cut into equal runs for
// the CTAs from the lengths on the device: a short request costs what it reads.  Every CTA adds the lengths up itself
// (they are a few hundred words), so nothing runs ahead of the scan.  In a CTA one warp brings pages by bulk copies,
// one copy per page and head, into a ring; four warps take 32 positions of a tile each and meet only where a row ends.
// A row that one CTA scans whole is written there; a row cut between CTAs leaves at most two partial rows per CTA,
// merged by a second kernel that is launched behind the first one's tail.
#include "kv4.cuh"

#include <cmath>

namespace i8tk {
namespace {

constexpr int kTile = 128;                  // positions
constexpr int kWarps = 4;                   // scanning warps, 32 positions each
constexpr int kScanThreads = (kWarps + 1) * 32;
constexpr float kLazy = 2.0f;               // log2 units a row's maximum may run ahead of its reference: p <= 4, and
                                            // 4 * (largest scale, 131008 / 15) is still an fp16 number

template <int D, int NT>                    // NT: blocks of 8 query heads per key head
struct Kv4Cfg {
    static constexpr int G = D / 64;
    static constexpr int TILE_BYTES = kTile * (D + D / 8);
    static constexpr int STAGES = D == 64 ? 4 : 3;
    static constexpr int CTAS = NT == 1 ? 3 : 2;                  // per SM
    static constexpr int HEADS = NT * 8;
    static constexpr int ROW = D + 4;                             // floats of a partial row: acc[D], m, l, -, -
    static constexpr int OFF_MERGE = STAGES * TILE_BYTES;         // [kWarps][HEADS][ROW]
    static constexpr int OFF_BARS = OFF_MERGE + kWarps * HEADS * ROW * 4;
    static constexpr int SMEM = OFF_BARS + STAGES * 16;
    static_assert(SMEM * CTAS <= 227 * 1024, "shared memory of an SM");
};

constexpr uint32_t kNotedBadIndex = 1u, kNotedTimeout = 2u;

struct Kv4Args {
    const int8_t* Q;                        // rows of heads * D codes, q_stride apart
    const float* sQ;                        // rows of heads scales, sq_stride apart
    long long q_stride, sq_stride;
    const unsigned char* pool;
    const int* table;                       // [B][max_pages]
    const int* lens;                        // [B]
    __half* out;                            // [B][heads][D]
    int B, kv_heads, group, max_len, page_shift, max_pages, num_pages;
    float score_scale;                      // log2(e) / sqrt(D)
    uint32_t* status;
    int* prefix;                            // [B + 1] tiles per key head of the requests before
    uint32_t* noted;                        // [CTAs] kNoted* of a CTA; the merging kernel makes the call's status word of them
    float* parts;                           // [CTAs][2][group][D + 4]
};

__device__ __forceinline__ void note(const Kv4Args& a, uint32_t what, uint32_t count) {
    atomicOr(a.noted + blockIdx.x, what);
    atomicAdd(a.status + 1, count);
}
__device__ __forceinline__ int row_len(const Kv4Args& a, int b) {
    return min(max(__ldg(a.lens + b), 0), a.max_len);
}
__device__ __forceinline__ int row_tiles(const Kv4Args& a, int b) { return (row_len(a, b) + kTile - 1) / kTile; }
// The first n CTAs have a run each, none of them empty: n is the grid or, with fewer tiles than that, their number.
// First tile of CTA c's run, and the CTA that a tile belongs to.
__device__ __forceinline__ int runs_of(long long total, int ctas) { return total < ctas ? (int)total : ctas; }
__device__ __forceinline__ long long run_start(long long total, int c, int n) { return total * c / n; }
__device__ __forceinline__ int run_owner(long long total, long long tile, int n) { return (int)(((tile + 1) * n - 1) / total); }

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <int W>
__device__ __forceinline__ void lds_words(uint32_t addr, uint32_t (&w)[W]) {
    if constexpr (W == 1) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
    if constexpr (W == 2) asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
    if constexpr (W == 4)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
}
__device__ __forceinline__ float2 pair_of(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// Position of the sequence of tiles: request, key head, tile of the row.
struct Cursor {
    int b, h, tile, tiles, len;
};
__device__ __forceinline__ void load_row(const Kv4Args& a, Cursor& c) {
    c.len = row_len(a, c.b);
    c.tiles = (c.len + kTile - 1) / kTile;
}
// to the next tile; called only while tiles remain, the bound on b is for lengths that changed under the kernel
__device__ __forceinline__ void advance(const Kv4Args& a, Cursor& c) {
    if (++c.tile < c.tiles) return;
    c.tile = 0;
    if (++c.h < a.kv_heads) return;
    c.h = 0;
    while (c.b + 1 < a.B) {
        ++c.b;
        load_row(a, c);
        if (c.tiles > 0) return;
    }
}

template <int D, int NT>
__global__ void __launch_bounds__(kScanThreads, Kv4Cfg<D, NT>::CTAS)
kv4_scan_kernel(const Kv4Args a) {
    using Cfg = Kv4Cfg<D, NT>;
    constexpr int G = Cfg::G, ROW = Cfg::ROW;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int s_warp[kWarps + 1];
    __shared__ int s_start[2];
    const uint32_t base = smem_u32(smem), bars = base + Cfg::OFF_BARS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto full = [&](int s) { return bars + 16u * s; };
    auto empty = [&](int s) { return bars + 16u * s + 8u; };
    if (threadIdx.x == 0) {
        for (int s = 0; s < Cfg::STAGES; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), kWarps);
        }
        fence_mbar_init();
        s_start[0] = 0, s_start[1] = 0;
    }
    pdl_wait();
    pdl_launch_dependents();

    // ---- tiles per key head in all, and where this CTA's run starts ----
    const int per = (a.B + kScanThreads - 1) / kScanThreads;
    const int lo = min(a.B, (int)threadIdx.x * per), hi = min(a.B, lo + per);
    int mine = 0;
    for (int b = lo; b < hi; ++b) mine += row_tiles(a, b);
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    int before = inc - mine, sum = 0;
#pragma unroll
    for (int w = 0; w <= kWarps; ++w) {
        if (w < warp) before += s_warp[w];
        sum += s_warp[w];
    }
    const long long total = (long long)sum * a.kv_heads;
    const int runs = runs_of(total, gridDim.x);
    const bool busy = (int)blockIdx.x < runs;
    const long long first = busy ? run_start(total, blockIdx.x, runs) : 0;
    const int run = busy ? (int)(run_start(total, blockIdx.x + 1, runs) - first) : 0;
    if (mine > 0 && (long long)before * a.kv_heads <= first && first < (long long)(before + mine) * a.kv_heads) {
        int at = before;
        for (int b = lo; b < hi; ++b) {
            const int n = row_tiles(a, b);
            if (first < (long long)(at + n) * a.kv_heads) {
                s_start[0] = b, s_start[1] = at;
                break;
            }
            at += n;
        }
    }
    if (blockIdx.x == 0) {                   // for the merging kernel
        int at = before;
        for (int b = lo; b < hi; ++b) {
            a.prefix[b] = at;
            at += row_tiles(a, b);
        }
        if (threadIdx.x == 0) a.prefix[a.B] = sum;
    }
    if (threadIdx.x == 0) a.noted[blockIdx.x] = 0u;
    __syncthreads();
    if (run == 0) return;
    Cursor cur;
    cur.b = s_start[0];
    load_row(a, cur);
    {
        const long long in = first - (long long)s_start[1] * a.kv_heads;
        cur.h = (int)(in / max(cur.tiles, 1));
        cur.tile = (int)(in - (long long)cur.h * cur.tiles);
    }
    const int page = 1 << a.page_shift, block_bytes = kv4_block_bytes(page, D);

    if (warp == kWarps) {
        // ================= one warp brings the pages =================
        const int per_tile = kTile >> a.page_shift;          // pages of a tile: 1 to 8, a lane each
        bool ok = true;
        int i = 0, bad = 0;
        for (; i < run && ok; ++i) {
            const int s = i % Cfg::STAGES;
            const int p = cur.tile * per_tile + lane;
            const bool use = lane < per_tile && p * page < cur.len;
            int id = 0;
            if (use) {
                id = __ldg(a.table + (long long)cur.b * a.max_pages + p);
                if ((unsigned)id >= (unsigned)a.num_pages) id = 0, ++bad;      // never followed
            }
            const int pages = __popc(__ballot_sync(0xffffffffu, use));
            const bool got = mbar_wait_bounded(empty(s), ((i / Cfg::STAGES) & 1) ^ 1);
            ok = __all_sync(0xffffffffu, got);
            if (!ok) break;
            if (lane == 0) mbar_expect_tx(full(s), pages * block_bytes);
            __syncwarp();
            if (use)
                bulk_g2s(base + s * Cfg::TILE_BYTES + lane * block_bytes, a.pool + ((long long)id * a.kv_heads + cur.h) * block_bytes,
                         block_bytes, full(s));
            if (i + 1 < run) advance(a, cur);
        }
        if (!ok) {                           // copies still in flight land before this block lets go of its memory
            if (lane == 0) note(a, kNotedTimeout, 1u);
            for (int k = max(0, i - Cfg::STAGES); k < i; ++k) mbar_wait_bounded(full(k % Cfg::STAGES), (k / Cfg::STAGES) & 1, 64u);
        }
        bad = __reduce_add_sync(0xffffffffu, bad);
        if (lane == 0 && bad > 0) note(a, kNotedBadIndex, (uint32_t)bad);
        return;
    }

    // ================= four warps scan, 32 positions of a tile each =================
    const int gid = lane >> 2, tig = lane & 3;
    const int row = gid ^ ((gid >> 1) & 1);                  // row gid of an operand holds this position of eight: the two
                                                             // lanes groups of a shared-memory phase then differ in parity
    const int vrow = (2 * tig) ^ (tig & 1);                  // the same order seen from the second product
    float* merge = reinterpret_cast<float*>(smem + Cfg::OFF_MERGE);
    const int heads = a.kv_heads * a.group;

    uint32_t q[NT][G * 2][4];                                // per word of a key row: code pairs (0,4) (1,5)/16 (2,6) (3,7)/16
    f32x2 to_log2[NT], qz[NT][G], q8[NT][G];                 // heads 2 tig, 2 tig + 1
    float acc[NT][G][4][4], ones[NT][G][4];
    f32x2 m_ref[NT], l2[NT], w2[NT][G];

    auto begin_row = [&]() {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int j = n * 8 + gid;                       // this lane's query head in the group
            const bool real = j < a.group;
            int sums[G];
#pragma unroll
            for (int g = 0; g < G; ++g) sums[g] = 0;
#pragma unroll
            for (int w = 0; w < 2 * G; ++w) {                // words in row order: unit 2 tig + w / G, group w % G
                uint2 c = make_uint2(0u, 0u);
                if (real)
                    c = __ldg(reinterpret_cast<const uint2*>(a.Q + cur.b * a.q_stride + (long long)(cur.h * a.group + j) * D +
                                                             64 * (w % G) + 8 * (2 * tig + w / G)));
                float e[8];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int x = (int)(int8_t)(c.x >> (8 * k)), y = (int)(int8_t)(c.y >> (8 * k));
                    sums[w % G] += x + y;
                    e[k] = (float)x, e[k + 4] = (float)y;
                }
                q[n][w][0] = pack_half2(e[0], e[4]);
                q[n][w][1] = pack_half2(e[1] * 0.0625f, e[5] * 0.0625f);
                q[n][w][2] = pack_half2(e[2], e[6]);
                q[n][w][3] = pack_half2(e[3] * 0.0625f, e[7] * 0.0625f);
            }
            const float sc = real ? __ldg(a.sQ + cur.b * a.sq_stride + cur.h * a.group + j) * a.score_scale : 0.f;
            const float c0 = __shfl_sync(0xffffffffu, sc, 8 * tig), c1 = __shfl_sync(0xffffffffu, sc, 8 * tig + 4);
            to_log2[n] = pack2(c0 * 16777216.0f, c1 * 16777216.0f);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                sums[g] += __shfl_xor_sync(0xffffffffu, sums[g], 1);
                sums[g] += __shfl_xor_sync(0xffffffffu, sums[g], 2);
                const float x = (float)__shfl_sync(0xffffffffu, sums[g], 8 * tig) * c0;
                const float y = (float)__shfl_sync(0xffffffffu, sums[g], 8 * tig + 4) * c1;
                qz[n][g] = pack2(x, y);
                q8[n][g] = pack2(-8.f * x, -8.f * y);
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc[n][g][t][k] = 0.f;
#pragma unroll
                for (int k = 0; k < 4; ++k) ones[n][g][k] = 0.f;
                w2[n][g] = pack2(0.f, 0.f);
            }
            m_ref[n] = pack2(-INFINITY, -INFINITY);
            l2[n] = pack2(0.f, 0.f);
        }
    };

    bool ok = true;
    int seg_first = cur.tile;                                // first tile of the row in this run
    begin_row();
    for (int i = 0; i < run; ++i) {
        const int s = i % Cfg::STAGES;
        if (ok) {
            const bool got = mbar_wait_bounded(full(s), (i / Cfg::STAGES) & 1);
            ok = __all_sync(0xffffffffu, got);
            if (!ok && lane == 0) note(a, kNotedTimeout, 1u);
        }
        const int left = cur.len - cur.tile * kTile - warp * 32;     // positions of this warp's 32 that exist
        if (ok && left > 0) {
            // ---- scores of 2 x 16 positions ----
            f32x2 sc[2][2][NT];                              // [16 positions][row gid, gid + 8][8 heads]
            uint32_t vp[2][2][G];                            // the values' pairs of the same positions
            uint32_t blk[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int p0 = warp * 32 + u * 16;
                blk[u] = base + s * Cfg::TILE_BYTES + (p0 >> a.page_shift) * block_bytes;
                const int r = (p0 & (page - 1)) + row;
                uint32_t wa[2 * G], wb[2 * G];
                lds_words(blk[u] + r * (D / 2) + tig * (D / 8), wa);
                lds_words(blk[u] + (r + 8) * (D / 2) + tig * (D / 8), wb);
                float dot[NT][G][4];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int g = 0; g < G; ++g)
#pragma unroll
                        for (int k = 0; k < 4; ++k) dot[n][g][k] = 0.f;
#pragma unroll
                for (int w = 0; w < 2 * G; ++w) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const uint32_t x = wa[w] >> (8 * half), y = wb[w] >> (8 * half);
                        const uint32_t a0 = x & 0x000f000fu, a1 = y & 0x000f000fu, a2 = x & 0x00f000f0u, a3 = y & 0x00f000f0u;
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma_16816(dot[n][w % G], a0, a1, a2, a3, q[n][w][2 * half], q[n][w][2 * half + 1]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    uint32_t kp[G];
                    const uint32_t pairs = blk[u] + page * D + (r + 8 * e) * (G * 4);
                    lds_words(pairs, kp);
                    lds_words(pairs + page * (G * 4), vp[u][e]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) sc[u][e][n] = pack2(0.f, 0.f);
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const float2 sz = pair_of(kp[g]);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const f32x2 t = fma2(pack2(dot[n][g][2 * e], dot[n][g][2 * e + 1]), to_log2[n], q8[n][g]);
                            sc[u][e][n] = fma2(pack2(sz.x, sz.x), t, sc[u][e][n]);
                            sc[u][e][n] = fma2(pack2(sz.y, sz.y), qz[n][g], sc[u][e][n]);
                        }
                    }
                    if (u * 16 + 8 * e + row >= left) {      // no such position: whatever the page holds there
#pragma unroll
                        for (int n = 0; n < NT; ++n) sc[u][e][n] = pack2(-INFINITY, -INFINITY);
#pragma unroll
                        for (int g = 0; g < G; ++g) vp[u][e][g] = 0u;
                    }
                }
            }
            // ---- reference maximum: moved only when a score runs ahead of it ----
            bool ahead = false;
            f32x2 mx[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                mx[n].x = fmaxf(fmaxf(sc[0][0][n].x, sc[0][1][n].x), fmaxf(sc[1][0][n].x, sc[1][1][n].x));
                mx[n].y = fmaxf(fmaxf(sc[0][0][n].y, sc[0][1][n].y), fmaxf(sc[1][0][n].y, sc[1][1][n].y));
                ahead |= mx[n].x > m_ref[n].x + kLazy || mx[n].y > m_ref[n].y + kLazy;
            }
            if (__any_sync(0xffffffffu, ahead)) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) {
                        mx[n].x = fmaxf(mx[n].x, __shfl_xor_sync(0xffffffffu, mx[n].x, o));
                        mx[n].y = fmaxf(mx[n].y, __shfl_xor_sync(0xffffffffu, mx[n].y, o));
                    }
                    const float nx = fmaxf(m_ref[n].x, mx[n].x), ny = fmaxf(m_ref[n].y, mx[n].y);
                    const float cx = m_ref[n].x == nx ? 1.f : ex2_approx(m_ref[n].x - nx), cy = m_ref[n].y == ny ? 1.f : ex2_approx(m_ref[n].y - ny);
                    m_ref[n] = pack2(nx, ny);
                    l2[n] = mul2(l2[n], pack2(cx, cy));
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        w2[n][g] = mul2(w2[n][g], pack2(cx, cy));
                        ones[n][g][0] *= cx, ones[n][g][1] *= cy;
#pragma unroll
                        for (int t = 0; t < 4; ++t) acc[n][g][t][0] *= cx, acc[n][g][t][1] *= cy, acc[n][g][t][2] *= cx, acc[n][g][t][3] *= cy;
                    }
                }
            }
            // ---- probabilities, and the second product ----
            f32x2 neg[NT];                                   // a row without a finite score yet: every p is 2^-inf
#pragma unroll
            for (int n = 0; n < NT; ++n)
                neg[n] = pack2(m_ref[n].x == -INFINITY ? 0.f : -m_ref[n].x, m_ref[n].y == -INFINITY ? 0.f : -m_ref[n].y);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                if (u == 1 && left <= 16) break;
                uint32_t pb[NT][G][2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    f32x2 p[NT];
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const f32x2 x = add2(sc[u][e][n], neg[n]);
                        p[n] = pack2(ex2_approx(x.x), ex2_approx(x.y));
                        l2[n] = add2(l2[n], p[n]);
                    }
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const float2 sz = pair_of(vp[u][e][g]);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            w2[n][g] = fma2(p[n], pack2(sz.y, sz.y), w2[n][g]);
                            const f32x2 ps = mul2(p[n], pack2(sz.x, sz.x));
                            pb[n][g][e] = transpose8x8(pack_half2(ps.x, ps.y));
                        }
                    }
                }
                const int r = ((warp * 32 + u * 16) & (page - 1)) + vrow;
                const uint32_t vaddr = blk[u] + page * (D / 2) + r * (D / 2) + gid * (G * 4);
                const int next = ((vrow ^ 1) - vrow) * (D / 2);      // the odd position of the pair
                uint32_t v0[G], v1[G], v2[G], v3[G];
                lds_words(vaddr, v0);
                lds_words(vaddr + next, v1);
                lds_words(vaddr + 8 * (D / 2), v2);
                lds_words(vaddr + 8 * (D / 2) + next, v3);
#pragma unroll
                for (int g = 0; g < G; ++g) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        mma_16816(ones[n][g], 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, pb[n][g][0], pb[n][g][1]);
#pragma unroll
                    for (int hw = 0; hw < 2; ++hw) {         // channels 0..3, 4..7 of the word
                        const uint32_t sel = hw ? 0x7632u : 0x5410u;
                        const uint32_t x = prmt(v0[g], v1[g], sel), y = prmt(v2[g], v3[g], sel);
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const uint32_t xs = x >> (8 * half), ys = y >> (8 * half);
#pragma unroll
                            for (int n = 0; n < NT; ++n)
                                mma_16816(acc[n][g][2 * hw + half], xs & 0x000f000fu, xs & 0x00f000f0u, ys & 0x000f000fu,
                                          ys & 0x00f000f0u, pb[n][g][0], pb[n][g][1]);
                        }
                    }
                }
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty(s));

        const bool row_ends = cur.tile + 1 == cur.tiles, seg_ends = row_ends || i + 1 == run;
        if (seg_ends) {
            // ---- the four warps' rows become one ----
            float* mine_rows = merge + warp * (Cfg::HEADS * ROW);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) {
                    l2[n].x += __shfl_xor_sync(0xffffffffu, l2[n].x, o), l2[n].y += __shfl_xor_sync(0xffffffffu, l2[n].y, o);
#pragma unroll
                    for (int g = 0; g < G; ++g)
                        w2[n][g].x += __shfl_xor_sync(0xffffffffu, w2[n][g].x, o), w2[n][g].y += __shfl_xor_sync(0xffffffffu, w2[n][g].y, o);
                }
                float* r0 = mine_rows + (n * 8 + 2 * tig) * ROW;     // heads 2 tig, 2 tig + 1
                float* r1 = r0 + ROW;
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const float k0 = fmaf(-8.f, ones[n][g][0], w2[n][g].x), k1 = fmaf(-8.f, ones[n][g][1], w2[n][g].y);
                    const int d = 64 * g + 8 * gid;
#pragma unroll
                    for (int t = 0; t < 4; ++t) {            // rows gid: an even channel; rows gid + 8: the odd one, 16 times
                        r0[d + 2 * t] = fmaf(acc[n][g][t][0], 16777216.0f, k0), r1[d + 2 * t] = fmaf(acc[n][g][t][1], 16777216.0f, k1);
                        r0[d + 2 * t + 1] = fmaf(acc[n][g][t][2], 1048576.0f, k0), r1[d + 2 * t + 1] = fmaf(acc[n][g][t][3], 1048576.0f, k1);
                    }
                }
                if (gid == 0) {
                    r0[D] = m_ref[n].x, r0[D + 1] = l2[n].x;
                    r1[D] = m_ref[n].y, r1[D + 1] = l2[n].y;
                }
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
            const bool whole = seg_first == 0 && row_ends;
            float* part = a.parts + ((long long)blockIdx.x * 2 + (seg_first == 0 ? 1 : 0)) * a.group * ROW;
            __half* out = a.out + ((long long)cur.b * heads + (long long)cur.h * a.group) * D;
            for (int e = threadIdx.x; e < a.group * (D / 4); e += kWarps * 32) {
                const int j = e / (D / 4), d = (e - j * (D / 4)) * 4;
                const float* r = merge + j * ROW;
                float m = -INFINITY;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) m = fmaxf(m, r[w * (Cfg::HEADS * ROW) + D]);
                float l = 0.f;
                float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float* rw = r + w * (Cfg::HEADS * ROW);
                    const float f = rw[D] == -INFINITY && rw[D + 1] == 0.f ? 0.f : ex2_approx(rw[D] - (m == -INFINITY ? 0.f : m));
                    // a row whose scores were all NaN has no maximum but its sum is NaN: it stays in
                    const float keep = rw[D + 1] != rw[D + 1] ? 1.f : f;
                    const float4 x = *reinterpret_cast<const float4*>(rw + d);
                    l = fmaf(keep, rw[D + 1], l);
                    o.x = fmaf(keep, x.x, o.x), o.y = fmaf(keep, x.y, o.y), o.z = fmaf(keep, x.z, o.z), o.w = fmaf(keep, x.w, o.w);
                }
                if (whole) {
                    const float inv = 1.0f / l;
                    *reinterpret_cast<uint2*>(out + (long long)j * D + d) = make_uint2(pack_half2(o.x * inv, o.y * inv), pack_half2(o.z * inv, o.w * inv));
                } else {
                    *reinterpret_cast<float4*>(part + j * ROW + d) = o;
                    if (d == 0) part[j * ROW + D] = m, part[j * ROW + D + 1] = l;
                }
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
            if (i + 1 < run) {
                advance(a, cur);
                seg_first = cur.tile;
                begin_row();
            }
        } else {
            ++cur.tile;
        }
    }
}

// One CTA per (request, key head) row and query head: adds up the partial rows the scan left for it, if it left any;
// a request without positions gets zeros.
template <int D>
__global__ void __launch_bounds__(128)
kv4_merge_kernel(const Kv4Args a, int nctas) {
    constexpr int ROW = D + 4, LPR = D / 4, PER = 128 / LPR;     // lanes of a row, rows side by side
    __shared__ float s_o[PER][D];
    __shared__ float s_l[PER], s_m[4];
    pdl_wait();
    pdl_launch_dependents();
    const int r = blockIdx.x, b = r / a.kv_heads, h = r - b * a.kv_heads, j = blockIdx.y;
    if (r == 0 && j == 0) {                  // what the scan's CTAs met, as the status word of this call
        uint32_t any = 0u;
        for (int c = threadIdx.x; c < nctas; c += 128) any |= a.noted[c];
        const int late = __syncthreads_or((int)(any & kNotedTimeout)), bad = __syncthreads_or((int)(any & kNotedBadIndex));
        if (threadIdx.x == 0) *a.status = late ? kDeviceTimeoutMagic : bad ? kDeviceBadIndexMagic : 0u;
    }
    const int p0 = a.prefix[b], tiles = a.prefix[b + 1] - p0;
    __half* out = a.out + (((long long)b * a.kv_heads + h) * a.group + j) * D;
    if (tiles == 0) {
        if (threadIdx.x < D / 8) *reinterpret_cast<uint4*>(out + threadIdx.x * 8) = make_uint4(0u, 0u, 0u, 0u);
        return;
    }
    const long long total = (long long)a.prefix[a.B] * a.kv_heads;
    const long long t0 = (long long)p0 * a.kv_heads + (long long)h * tiles;
    const int runs = runs_of(total, nctas);
    const int c0 = run_owner(total, t0, runs), c1 = run_owner(total, t0 + tiles - 1, runs);
    if (c0 == c1) return;
    const int parts = c1 - c0 + 1;
    // the first CTA left its piece in slot 1 (the row began there), the others in slot 0
    auto part_of = [&](int i) { return a.parts + ((long long)((c0 + i) * 2 + (i == 0 ? 1 : 0)) * a.group + j) * ROW; };
    float m = -INFINITY;
    for (int i = threadIdx.x; i < parts; i += 128) m = fmaxf(m, part_of(i)[D]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((threadIdx.x & 31) == 0) s_m[threadIdx.x >> 5] = m;
    __syncthreads();
    m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    const float ref = m == -INFINITY ? 0.f : m;
    const int k = threadIdx.x / LPR, d = (threadIdx.x % LPR) * 4;
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = k; i < parts; i += PER) {
        const float* p = part_of(i);
        const float4 x = *reinterpret_cast<const float4*>(p + d);
        const float2 ml = *reinterpret_cast<const float2*>(p + D);
        const float f = ml.y != ml.y ? 1.f : ex2_approx(ml.x - ref);
        l = fmaf(f, ml.y, l);
        o.x = fmaf(f, x.x, o.x), o.y = fmaf(f, x.y, o.y), o.z = fmaf(f, x.z, o.z), o.w = fmaf(f, x.w, o.w);
    }
    *reinterpret_cast<float4*>(&s_o[k][d]) = o;
    if (d == 0) s_l[k] = l;
    __syncthreads();
    if (threadIdx.x < D / 2) {
        const int e = threadIdx.x * 2;
        float x = 0.f, y = 0.f, ls = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) x += s_o[i][e], y += s_o[i][e + 1], ls += s_l[i];
        const float inv = 1.0f / ls;
        *reinterpret_cast<uint32_t*>(out + e) = pack_half2(x * inv, y * inv);
    }
}

// ---- host ----------------------------------------------------------------------------------------------
int sms() {
    static int cached[64] = {0};
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    if (cached[dev] == 0 && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess) cached[dev] = n;
    return cached[dev] > 0 ? cached[dev] : 148;
}

struct Kv4Layout {
    int ctas;
    size_t prefix_off, noted_off, parts_off, total;
};

int blocks_of_8(int group) { return group <= 8 ? 1 : 2; }

Kv4Layout kv4_layout(int B, int kv_heads, int group, int max_len, int D) {
    Kv4Layout y;
    const long long tiles = (long long)B * kv_heads * ((max_len + kTile - 1) / kTile);
    const long long resident = (long long)sms() * (blocks_of_8(group) == 1 ? Kv4Cfg<128, 1>::CTAS : Kv4Cfg<128, 2>::CTAS);
    y.ctas = (int)(tiles < resident ? tiles : resident);
    y.prefix_off = 256;
    y.noted_off = y.prefix_off + round_up((size_t)(B + 1) * 4, 256);
    y.parts_off = y.noted_off + round_up((size_t)y.ctas * 4, 256);
    y.total = y.parts_off + round_up((size_t)y.ctas * 2 * group * (D + 4) * 4, 256);
    return y;
}

bool kv4_shape_ok(int B, int heads, int kv_heads, int max_len, int D) {
    return B > 0 && kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && heads / kv_heads <= 16 && max_len > 0 && (D == 64 || D == 128) &&
           (long long)B * kv_heads * ((max_len + kTile - 1) / kTile) < (1ll << 31) && (long long)B * kv_heads < (1ll << 31);
}

template <int D, int NT>
int launch_kv4(const Kv4Args& a, int ctas, cudaStream_t st) {
    using Cfg = Kv4Cfg<D, NT>;
    static bool attr_done[64] = {false};
    int dev = 0;
    I8TK_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !attr_done[dev]) {
        I8TK_CUDA(cudaFuncSetAttribute(kv4_scan_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM));
        if (dev >= 0 && dev < 64) attr_done[dev] = true;
    }
    I8TK_CUDA(launch_after(kv4_scan_kernel<D, NT>, dim3((unsigned)ctas), dim3(kScanThreads), Cfg::SMEM, st, a));
    I8TK_CUDA(launch_after(kv4_merge_kernel<D>, dim3((unsigned)(a.B * a.kv_heads), (unsigned)a.group), dim3(128), 0, st, a, ctas));
    return I8TK_OK;
}

}  // namespace
}  // namespace i8tk

using namespace i8tk;

extern "C" size_t i8tk_decode_kv4_workspace_bytes(int batch, int heads, int kv_heads, int max_seq_len, int head_dim) {
    if (!kv4_shape_ok(batch, heads, kv_heads, max_seq_len, head_dim)) return 0;
    return kv4_layout(batch, kv_heads, heads / kv_heads, max_seq_len, head_dim).total;
}

extern "C" int i8tk_decode_attention_kv4(const int8_t* Q, int64_t q_stride, const float* sQ, int64_t sq_stride, const void* pool,
                                         const int32_t* page_table, const int32_t* seq_lens, void* out_f16, int batch, int heads,
                                         int kv_heads, int max_seq_len, int page_size, int max_pages_per_seq, int head_dim,
                                         int64_t num_pages, void* workspace, size_t workspace_bytes, i8tk_stream_t stream) {
    I8TK_REQUIRE(Q && sQ && pool && page_table && seq_lens && out_f16, I8TK_ERR_INVALID_ARGUMENT, "null pointer argument");
    I8TK_REQUIRE(batch > 0 && heads > 0 && kv_heads > 0 && max_seq_len > 0 && max_pages_per_seq > 0 && num_pages > 0,
                 I8TK_ERR_INVALID_ARGUMENT, "sizes must be positive");
    I8TK_REQUIRE(head_dim == 64 || head_dim == 128, I8TK_ERR_UNSUPPORTED, "head_dim must be 64 or 128 (got %d)", head_dim);
    I8TK_REQUIRE(kv4_page_ok(page_size), I8TK_ERR_UNSUPPORTED, "page_size must be 16, 32, 64 or 128 (got %d)", page_size);
    I8TK_REQUIRE(heads % kv_heads == 0 && heads / kv_heads <= 16, I8TK_ERR_UNSUPPORTED,
                 "heads must be a multiple of kv_heads, at most 16 times as many");
    I8TK_REQUIRE(kv4_shape_ok(batch, heads, kv_heads, max_seq_len, head_dim) && num_pages < (1ll << 31), I8TK_ERR_UNSUPPORTED, "shape too large");
    I8TK_REQUIRE((long long)max_pages_per_seq * page_size >= max_seq_len, I8TK_ERR_INVALID_ARGUMENT,
                 "max_seq_len %d does not fit %d pages of %d", max_seq_len, max_pages_per_seq, page_size);
    I8TK_REQUIRE(q_stride >= (int64_t)heads * head_dim && q_stride % 16 == 0 && sq_stride >= heads, I8TK_ERR_INVALID_ARGUMENT,
                 "q_stride must cover a request's heads and be a multiple of 16, sq_stride must cover its scales");
    I8TK_REQUIRE(aligned_to(Q, 16) && aligned_to(pool, 16) && aligned_to(out_f16, 16), I8TK_ERR_ALIGNMENT,
                 "Q, the pool and out must be 16-byte aligned");
    const int group = heads / kv_heads;
    const Kv4Layout y = kv4_layout(batch, kv_heads, group, max_seq_len, head_dim);
    I8TK_REQUIRE(workspace != nullptr && workspace_bytes >= y.total, I8TK_ERR_WORKSPACE,
                 "decode workspace too small: need %zu bytes, got %zu", y.total, workspace_bytes);
    I8TK_REQUIRE(aligned_to(workspace, 256), I8TK_ERR_ALIGNMENT, "workspace must be 256-byte aligned");
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    int shift = 4;
    while ((1 << shift) < page_size) ++shift;
    const Kv4Args a{Q, sQ, q_stride, sq_stride, static_cast<const unsigned char*>(pool), page_table, seq_lens,
                    static_cast<__half*>(out_f16), batch, kv_heads, group, max_seq_len, shift, max_pages_per_seq, (int)num_pages,
                    1.4426950408889634f / sqrtf((float)head_dim), reinterpret_cast<uint32_t*>(ws),
                    reinterpret_cast<int*>(ws + y.prefix_off), reinterpret_cast<uint32_t*>(ws + y.noted_off), reinterpret_cast<float*>(ws + y.parts_off)};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (blocks_of_8(group) == 1)
        return head_dim == 64 ? launch_kv4<64, 1>(a, y.ctas, st) : launch_kv4<128, 1>(a, y.ctas, st);
    return head_dim == 64 ? launch_kv4<64, 2>(a, y.ctas, st) : launch_kv4<128, 2>(a, y.ctas, st);
}
