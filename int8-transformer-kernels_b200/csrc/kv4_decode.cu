// Decode attention (one query token per request) over the paged 4-bit cache of kv4.cuh, with grouped heads.
//
//   score_j = (q . k_j) * sQ / sqrt(D),   k_j = s (c - 8) + z per 64 channels,   out = softmax(score) . v
//
// q is INT8 with one scale per head, so q . c is an integer sum and
//   q . k_j = sum over the groups of  s_j ((q . c_j) - 8 Q) + z_j Q,      Q = sum of the group's query codes;
//   out     = sum over the groups of  [sum_j P_j c_j] - 8 [sum_j P_j] + sum_j p_j z_j,      P_j = fp16(p_j s_j).
// The - 8 is applied to the sums: with P rounded, sum P (c - 8) is what comes out, without the cancellation that
// unsigned codes would otherwise bring into the rounding error of P.  The tensor core cuts a sum's last bits, always
// downwards; so sum P 8 is made of the code 8 in the same form as the codes and cut alike, and it leaves the sums every 256
// positions, before they are large.  (8 requests of 58915, 28/4 heads, D 64: error 3.4e-4 of the result's norm, of which
// fp16 results alone make 2.1e-4; with sums of P against the number 1, subtracted at the end, 4.3e-4.  1 % of the time.)
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
// * With 4 heads or fewer in a group, the 8 columns are W = 2 or 4 copies of the heads, and copy w takes every W-th
//   octet of positions: the products cost the same, but the work per score -- scales, exponentials, packing -- is done
//   for one octet per lane instead of for W of which only one has heads in the lane.  A copy keeps a maximum and sums of
//   its own, as a row apart, and the copies are merged with the warps' rows.
//
// The tiles (128 positions, 256 at head_dim 64) of all (request, key head) rows, in that order, are one sequence, cut into equal runs for
// the CTAs from the lengths on the device: a short request costs what it reads.  Every CTA adds the lengths up itself
// (they are a few hundred words), so nothing runs ahead of the scan.  A CTA is four warps, a quarter of a tile each,
// which meet only where a row ends; in turn they start the bulk copies of the next tile, one copy per page and head.
// There is no warp for the copies alone: the unpacking is bound by the instructions the SM can issue, and four CTAs of
// four 128-register warps are all it holds (with a fifth warp it held three).  The page size is a template parameter,
// so that every shared-memory address is a constant off three per-thread bases.
// A row that one CTA scans whole is written there; a row cut between CTAs leaves at most two partial rows per CTA,
// merged by a second kernel that is launched behind the first one's tail.
// Measured: 32 requests up to 32768 positions, 32/8 heads, D 128, 64-position pages, 122-130 us a call (floor at the copy
// rate: 95.8); 24 up to 4096, 12/12 heads, D 64: 20 us (6.8).  No unit is full: 52 % of the issue slots at 16 warps an SM,
// the ALU pipe, which unpacks, 54 %, memory 64 %; the empty slots are latency (fixed-latency dependencies, shared memory).
#include "kv4.cuh"
#include "score_reference.cuh"

#include <cmath>

namespace i8tk {
namespace {

// Positions of a tile: about 18 KB of the cache.  A warp takes a quarter, 32 positions at a time.  (128 positions at
// head_dim 64 too: 16 requests of 16384, 12/12 heads, 60.7 us against 55.4.)
__host__ __device__ constexpr int tile_of(int D) { return D == 64 ? 256 : 128; }
constexpr int kWarps = 4;
constexpr int kScanThreads = kWarps * 32;
// P = p * s has to stay an fp16 number (below 2^16) and should use its range: a row's reference lies kTop log2 units
// below its largest score times the largest scale met so far, and moves when a product would run kSlack above that.
constexpr float kTop = 13.0f, kSlack = 2.0f;
constexpr int kLeastScale = -20;          // log2 of the scale assumed for values that have none (p itself stays below 2^35)
constexpr float kNoReference = 3e38f;       // negative reference of a row that has met nothing: 2^(-inf + 3e38) is still 0

template <int D, int NT, int W>             // NT: blocks of 8 query heads per key head; W: copies of the heads in a block
struct Kv4Cfg {
    static constexpr int G = D / 64;
    static constexpr int TILE = tile_of(D), TILE_BYTES = TILE * (D + D / 8);
    // Two stages: a third (32 requests, up to 32768 positions, 32/8 heads, D 128: 127 us a call waited for, against 134)
    // fills the SM's shared memory, and a call that follows at once loses more (153 us against 122).
    static constexpr int STAGES = 2;
    static constexpr int CTAS = NT == 2 ? 3 : 4;                  // per SM: 168 and 128 registers a thread
    static constexpr int ROW = D + 4;                             // floats of a partial row: acc[D], m, l, -, -
    static constexpr int OFF_BARS = STAGES * TILE_BYTES;
    static constexpr int SMEM = OFF_BARS + STAGES * 16;
    // where a row ends, the warps' rows of 8 columns meet in the stage just read
    static_assert(kWarps * 8 * ROW * 4 <= TILE_BYTES, "a stage holds the rows of the warps");
    static_assert(STAGES >= 2 && STAGES <= kWarps, "each of the first tiles has a warp of its own");
    static_assert((SMEM + 1024 + 128) * CTAS <= 227 * 1024, "shared memory of an SM");
};

constexpr uint32_t kEight = 0x00080008u, kEightHigh = 0x00800080u;      // the code 8 in both forms

constexpr uint32_t kNotedBadIndex = 1u, kNotedTimeout = 2u;

struct Kv4Args {
    const int8_t* Q;                        // rows of heads * D codes, q_stride apart
    const float* sQ;                        // rows of heads scales, sq_stride apart
    long long q_stride, sq_stride;
    const unsigned char* pool;
    const int* table;                       // [B][max_pages]
    const int* lens;                        // [B]
    __half* out;                            // [B][heads][D]
    int B, kv_heads, group, max_len, max_pages, num_pages;
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
template <int D>
__device__ __forceinline__ int row_tiles(const Kv4Args& a, int b) { return (row_len(a, b) + tile_of(D) - 1) / tile_of(D); }
// The first n CTAs have a run each, none of them empty: n is the grid or, with fewer tiles than that, their number.
// First tile of CTA c's run, and the CTA that a tile belongs to.
__device__ __forceinline__ int runs_of(long long total, int ctas) { return total < ctas ? (int)total : ctas; }
__device__ __forceinline__ long long run_start(long long total, int c, int n) { return total * c / n; }
__device__ __forceinline__ int run_owner(long long total, long long tile, int n) { return (int)(((tile + 1) * n - 1) / total); }

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_16816_from_zero(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <int W>
__device__ __forceinline__ void lds_words(const unsigned char* at, uint32_t (&w)[W]) {
    if constexpr (W == 1) w[0] = *reinterpret_cast<const uint32_t*>(at);
    if constexpr (W == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(at);
        w[0] = v.x, w[1] = v.y;
    }
    if constexpr (W == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(at);
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    }
}
__device__ __forceinline__ float2 pair_of(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// A row of the sequence: request, key head, tiles.
struct Row {
    int b, h, len, tiles;
};
template <int D>
__device__ __forceinline__ void load_row(const Kv4Args& a, Row& r) {
    r.len = row_len(a, r.b);
    r.tiles = (r.len + tile_of(D) - 1) / tile_of(D);
}
// the next row that has tiles; called only while tiles remain, the bound on b (and the length it then gives) is for
// lengths that changed under the kernel
template <int D>
__device__ __forceinline__ void next_row(const Kv4Args& a, Row& r) {
    if (++r.h < a.kv_heads) return;
    r.h = 0;
    while (r.b + 1 < a.B) {
        ++r.b;
        load_row<D>(a, r);
        if (r.tiles > 0) return;
    }
    r.tiles = 1 << 30, r.len = 0;
}

template <int D, int NT, int W, int PAGE>
__global__ void __launch_bounds__(kScanThreads, Kv4Cfg<D, NT, W>::CTAS)
kv4_scan_kernel(const Kv4Args a) {
    using Cfg = Kv4Cfg<D, NT, W>;
    constexpr int G = Cfg::G, ROW = Cfg::ROW;
    constexpr int HEADS = 8 / W;             // query heads of a block of columns
    constexpr int NU = W == 4 ? 1 : 2, NE = W == 1 ? 2 : 1;      // octets of 32 positions a lane has scores of: NU * NE
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int s_warp[kWarps];
    __shared__ int s_start[2];
    const uint32_t base = smem_u32(smem), bars = base + Cfg::OFF_BARS;
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
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
    for (int b = lo; b < hi; ++b) mine += row_tiles<D>(a, b);
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
    for (int w = 0; w < kWarps; ++w) {
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
            const int n = row_tiles<D>(a, b);
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
            at += row_tiles<D>(a, b);
        }
        if (threadIdx.x == 0) a.prefix[a.B] = sum;
    }
    if (threadIdx.x == 0) a.noted[blockIdx.x] = 0u;
    __syncthreads();
    if (run == 0) return;
    Row cur;
    cur.b = s_start[0];
    load_row<D>(a, cur);
    int tile;                                // of the row
    {
        const long long in = first - (long long)s_start[1] * a.kv_heads;
        cur.h = (int)(in / max(cur.tiles, 1));
        tile = (int)(in - (long long)cur.h * cur.tiles);
    }
    static_assert(kv4_block_bytes(PAGE, D) % D == 0 && Cfg::TILE_BYTES % D == 0, "rows pair up by one address bit");
    constexpr int BLOCK = kv4_block_bytes(PAGE, D), PAGES = Cfg::TILE / PAGE;  // pages of a tile: 1 to 16, a lane each

    // ---- copies: tile i of the run is brought by warp i % 4, a lane per page, STAGES - 1 tiles ahead ----
    auto look_up = [&](const Row& r, int t) {
        const int p = t * PAGES + lane;
        return lane < PAGES && p * PAGE < r.len ? __ldg(a.table + (long long)r.b * a.max_pages + p) : 0;
    };
    // tile t counted from the start of row `r`, which may lie rows behind it
    auto find = [&](Row& r, int& t) {
        while (t >= r.tiles) {
            t -= r.tiles;
            next_row<D>(a, r);
        }
    };
    auto issue = [&](const Row& r, int t, int id, int s) {       // tile t of row r, whose page ids the lanes hold, into stage s
        const int left = max(r.len - t * Cfg::TILE, 0);
        if ((unsigned)id >= (unsigned)a.num_pages) {                           // never followed
            id = 0;
            note(a, kNotedBadIndex, 1u);
        }
        if (lane == 0) mbar_expect_tx(full(s), (left >= Cfg::TILE ? PAGES : (left + PAGE - 1) / PAGE) * BLOCK);
        __syncwarp();
        if (lane < PAGES && lane * PAGE < left)
            bulk_g2s(base + s * Cfg::TILE_BYTES + lane * BLOCK, a.pool + ((long long)id * a.kv_heads + r.h) * BLOCK, BLOCK, full(s));
    };

    const int gid = lane >> 2, tig = lane & 3;
    const int row = gid ^ ((gid >> 1) & 1);                  // row gid of an operand holds this position of eight: the two
                                                             // lanes groups of a shared-memory phase then differ in parity
    const int vrow = (2 * tig) ^ (tig & 1);                  // the same order seen from the second product
    const int heads = a.kv_heads * a.group;
    // this lane's octet among the two of 16 positions (W >= 2), and its 16 of the 32 (W = 4); the copy its operand rows
    // of the second product belong to
    const int my_e = W == 2 ? tig >> 1 : W == 4 ? tig & 1 : 0, my_u = W == 4 ? tig >> 1 : 0, copy = gid / HEADS;

    uint32_t q[NT][G * 2][4];                                // per word of a key row: code pairs (0,4) (1,5)/16 (2,6) (3,7)/16
    f32x2 to_log2[NT], qz[NT][G], q8[NT][G];                 // heads 2 tig, 2 tig + 1
    float acc[NT][G][4][4], ones[NT][G][4];
    f32x2 neg[NT], l2[NT], w2[NT][G];                        // negative reference; sums of p and of p * centre
    float top, room;                                         // a power of two no value scale met is above; how far a score
                                                             // may be above the reference with it

    auto begin_row = [&]() {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int j = n * 8 + gid % HEADS;               // this lane's query head in the group
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
            neg[n] = pack2(kNoReference, kNoReference);
            l2[n] = pack2(0.f, 0.f);
        }
        top = 1.0f / (1 << -kLeastScale);
        room = kTop + kSlack - kLeastScale;
    };

    int s = 0;
    uint32_t phase = 0;
    if (warp < min(Cfg::STAGES - 1, run)) {
        Row r = cur;
        int t = tile + warp;
        find(r, t);
        issue(r, t, look_up(r, t), warp);
    }
    // this thread's rows: keys at row `row` of its 16, values at row vrow, both of the warp's first 16 positions
    constexpr int U = PAGE == 16 ? BLOCK : 16 * (D / 2), U_PAIRS = PAGE == 16 ? BLOCK : 16 * G * 4;     // to the next 16
    const int p0 = warp * (Cfg::TILE / kWarps), in_page = p0 % PAGE;
    const int warp_block = p0 / PAGE * BLOCK;
    int k_at = warp_block + (in_page + row) * (D / 2) + tig * (D / 8);
    int pair_at = warp_block + PAGE * D + (in_page + row + 8 * my_e) * (G * 4) + my_u * U_PAIRS;
    int v_at = warp_block + PAGE * (D / 2) + (in_page + vrow) * (D / 2) + gid * (G * 4);
    constexpr int PAIRS = PAGE * G * 4;                      // from the keys' pairs to the values'
    constexpr int SUB = PAGE >= 64 ? 32 * (D / 2) : 32 / PAGE * BLOCK, SUB_PAIRS = PAGE >= 64 ? 32 * G * 4 : 32 / PAGE * BLOCK;    // to the next 32
    auto next_stage = [&]() {
        const bool wrap = s == Cfg::STAGES - 1;
        const int to = wrap ? -(Cfg::STAGES - 1) * Cfg::TILE_BYTES : Cfg::TILE_BYTES;
        k_at += to, pair_at += to, v_at += to;
        phase ^= wrap ? 1u : 0u;
        s = wrap ? 0 : s + 1;
    };
    for (int i = 0; i < run;) {              // a piece of a row: to its end, or to the end of the run
        const int pieces = min(cur.tiles - tile, run - i), seg_first = tile;
        const bool row_ends = tile + pieces == cur.tiles, more = i + pieces < run;
        begin_row();
        int here = cur.len - tile * Cfg::TILE - p0;              // positions of this warp's quarter that exist
        int ahead_id = 0;                                        // page ids of this warp's next turn in this row
        for (int k = 0; k < pieces; ++k, ++i, here -= Cfg::TILE) {
            // ---- the tile STAGES - 1 ahead, into the stage the last one was read from ----
            if (((i + Cfg::STAGES - 1) & 3) == warp && i + Cfg::STAGES - 1 < run) {
                const int o = s == 0 ? Cfg::STAGES - 1 : s - 1;
                if (i > 0) {
                    const bool got = mbar_wait_bounded(empty(o), s == 0 ? phase ^ 1 : phase);
                    if (!__all_sync(0xffffffffu, got)) goto late;
                }
                int t = tile + k + Cfg::STAGES - 1;
                if (t < cur.tiles) {
                    issue(cur, t, k >= 4 ? ahead_id : look_up(cur, t), o);
                    ahead_id = look_up(cur, t + 4);              // (behind the row's end: nothing)
                } else {
                    Row r = cur;
                    find(r, t);
                    issue(r, t, look_up(r, t), o);
                }
            }
            {
                const bool got = mbar_try_wait(full(s), phase);
                if (!__all_sync(0xffffffffu, got)) {
                    const bool at_last = mbar_wait_bounded(full(s), phase);
                    if (!__all_sync(0xffffffffu, at_last)) goto late;
                }
            }
#pragma unroll 1
            for (int sub = 0, left = here; sub < Cfg::TILE / kWarps / 32 && left > 0; ++sub, left -= 32) {
                const int ks = k_at + sub * SUB, ps = pair_at + sub * SUB_PAIRS, vs = v_at + sub * SUB;
            // ---- scores of 2 x 16 positions ----
            f32x2 sc[NU][NE][NT];                            // [16 positions][row gid, gid + 8][8 columns]
            uint32_t vp[NU][NE][G];                          // the values' pairs of the same positions
            uint32_t wa[2][2 * G], wb[2][2 * G];
            float dot[2][NT][G][4];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                lds_words(smem + ks + u * U, wa[u]);
                lds_words(smem + ks + u * U + 8 * (D / 2), wb[u]);
            }
#pragma unroll
            for (int w = 0; w < 2 * G; ++w) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const uint32_t x = wa[u][w] >> (8 * half), y = wb[u][w] >> (8 * half);
                        const uint32_t a0 = x & 0x000f000fu, a1 = y & 0x000f000fu, a2 = x & 0x00f000f0u, a3 = y & 0x00f000f0u;
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            if (w < G && half == 0) mma_16816_from_zero(dot[u][n][w % G], a0, a1, a2, a3, q[n][w][0], q[n][w][1]);
                            else mma_16816(dot[u][n][w % G], a0, a1, a2, a3, q[n][w][2 * half], q[n][w][2 * half + 1]);
                        }
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < NU; ++u) {
#pragma unroll
                for (int e = 0; e < NE; ++e) {
                    uint32_t kp[G];
                    lds_words(smem + ps + u * U_PAIRS + 8 * e * (G * 4), kp);
                    lds_words(smem + ps + u * U_PAIRS + 8 * e * (G * 4) + PAIRS, vp[u][e]);
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const float2 sz = pair_of(kp[g]);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            f32x2 c = pack2(dot[u][n][g][2 * e], dot[u][n][g][2 * e + 1]);
                            if constexpr (W >= 2) {          // this lane's octet
                                if (my_e) c = pack2(dot[u][n][g][2], dot[u][n][g][3]);
                            }
                            if constexpr (W == 4) {
                                if (my_u) c = my_e ? pack2(dot[1][n][g][2], dot[1][n][g][3]) : pack2(dot[1][n][g][0], dot[1][n][g][1]);
                            }
                            const f32x2 t = fma2(c, to_log2[n], q8[n][g]);
                            // one factor for two heads: two instructions, where the packed form needs two moves for the pair
                            const float x = g == 0 ? sz.y * qz[n][g].x : fmaf(sz.y, qz[n][g].x, sc[u][e][n].x);
                            const float y = g == 0 ? sz.y * qz[n][g].y : fmaf(sz.y, qz[n][g].y, sc[u][e][n].y);
                            sc[u][e][n] = pack2(fmaf(sz.x, t.x, x), fmaf(sz.x, t.y, y));
                        }
                    }
                }
            }
            if (left < 32) {                                 // positions that do not exist: whatever the page holds there
#pragma unroll
                for (int u = 0; u < NU; ++u)
#pragma unroll
                    for (int e = 0; e < NE; ++e)
                        if ((u + my_u) * 16 + 8 * (e + my_e) + row >= left) {
#pragma unroll
                            for (int n = 0; n < NT; ++n) sc[u][e][n] = pack2(-INFINITY, -INFINITY);
#pragma unroll
                            for (int g = 0; g < G; ++g) vp[u][e][g] = 0u;
                        }
            }
            // ---- reference: moved only when a product would run ahead of it ----
            __half2 big = *reinterpret_cast<const __half2*>(&vp[0][0][0]);       // largest value scale, in the low half
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int e = 0; e < NE; ++e)
#pragma unroll
                    for (int g = 0; g < G; ++g) big = __hmax2(big, *reinterpret_cast<const __half2*>(&vp[u][e][g]));
            const float big_scale = __low2float(big);
            float over = -INFINITY;                          // the largest score above its reference
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int e = 0; e < NE; ++e)
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const f32x2 x = add2(sc[u][e][n], neg[n]);
                        over = max3(over, x.x, x.y);
                    }
            if (__any_sync(0xffffffffu, over > room || big_scale > top)) {
                const uint32_t top_bits = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(big_scale, top)));
                const int exponent = (int)((top_bits + 0x7fffffu) >> 23);                        // rounded up
                top = __int_as_float(exponent << 23);
                room = kTop + kSlack + 127.0f - (float)exponent;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    f32x2 mx = sc[0][0][n];
#pragma unroll
                    for (int u = 0; u < NU; ++u)
#pragma unroll
                        for (int e = 0; e < NE; ++e) mx = pack2(fmaxf(mx.x, sc[u][e][n].x), fmaxf(mx.y, sc[u][e][n].y));
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) {
                        mx.x = fmaxf(mx.x, __shfl_xor_sync(0xffffffffu, mx.x, o));
                        mx.y = fmaxf(mx.y, __shfl_xor_sync(0xffffffffu, mx.y, o));
                    }
                    // the reference goes up to kTop - (largest scale) below the largest score (to the score itself where
                    // that offset would be rounded away: p * s is then at most s), never down
                    const f32x2 to = pack2(fminf(neg[n].x, negative_reference(mx.x, room - kSlack)), fminf(neg[n].y, negative_reference(mx.y, room - kSlack)));
                    const f32x2 keep = pack2(ex2_approx(to.x - neg[n].x), ex2_approx(to.y - neg[n].y));
                    neg[n] = to;
                    l2[n] = mul2(l2[n], keep);
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        w2[n][g] = mul2(w2[n][g], keep);
                        ones[n][g][0] *= keep.x, ones[n][g][1] *= keep.y, ones[n][g][2] *= keep.x, ones[n][g][3] *= keep.y;
#pragma unroll
                        for (int t = 0; t < 4; ++t) acc[n][g][t][0] *= keep.x, acc[n][g][t][1] *= keep.y, acc[n][g][t][2] *= keep.x, acc[n][g][t][3] *= keep.y;
                    }
                }
            }
            // ---- probabilities, and the second product ----
            uint32_t turned[NU][NE][NT][G];                  // P with columns as rows
#pragma unroll
            for (int u = 0; u < NU; ++u) {
#pragma unroll
                for (int e = 0; e < NE; ++e) {
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
                            w2[n][g] = pack2(fmaf(p[n].x, sz.y, w2[n][g].x), fmaf(p[n].y, sz.y, w2[n][g].y));
                            turned[u][e][n][g] = transpose8x8(pack_half2(p[n].x * sz.x, p[n].y * sz.x));
                        }
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                uint32_t pb[NT][G][2];                       // an octet's P, in the columns of the copy that has it
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int g = 0; g < G; ++g)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            if constexpr (W == 1) pb[n][g][e] = turned[u][e][n][g];
                            else pb[n][g][e] = copy == (W == 2 ? e : 2 * u + e) ? turned[W == 4 ? 0 : u][0][n][g] : 0u;
                        }
                uint32_t v0[G], v1[G], v2[G], v3[G];
                // the odd position of the pair: blocks and stages are multiples of two rows
                lds_words(smem + vs + u * U, v0);
                lds_words(smem + (vs ^ (D / 2)) + u * U, v1);
                lds_words(smem + vs + u * U + 8 * (D / 2), v2);
                lds_words(smem + (vs ^ (D / 2)) + u * U + 8 * (D / 2), v3);
#pragma unroll
                for (int g = 0; g < G; ++g) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        mma_16816(ones[n][g], kEight, kEightHigh, kEight, kEightHigh, pb[n][g][0], pb[n][g][1]);
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
            if (k % (256 * kWarps / Cfg::TILE) == 0) {       // every 256 positions of the warp: the 8 leaves the sums
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int g = 0; g < G; ++g)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
#pragma unroll
                            for (int t = 0; t < 4; ++t) acc[n][g][t][i] -= ones[n][g][i];
                            ones[n][g][i] = 0.f;
                        }
            }
            if (k + 1 < pieces) {
                __syncwarp();
                if (lane == 0) mbar_arrive(empty(s));
                next_stage();
            }
        }
        {
            // ---- the rows of the four warps and of the copies become one, in the stage that all have read ----
            float* merge = reinterpret_cast<float*>(smem + s * Cfg::TILE_BYTES);
            const bool whole = seg_first == 0 && row_ends;
            float* part = a.parts + ((long long)blockIdx.x * 2 + (seg_first == 0 ? 1 : 0)) * a.group * ROW;
            __half* out = a.out + ((long long)cur.b * heads + (long long)cur.h * a.group) * D;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                __syncthreads();
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) {
                    l2[n].x += __shfl_xor_sync(0xffffffffu, l2[n].x, o), l2[n].y += __shfl_xor_sync(0xffffffffu, l2[n].y, o);
#pragma unroll
                    for (int g = 0; g < G; ++g)
                        w2[n][g].x += __shfl_xor_sync(0xffffffffu, w2[n][g].x, o), w2[n][g].y += __shfl_xor_sync(0xffffffffu, w2[n][g].y, o);
                }
                float* r0 = merge + (warp * 8 + 2 * tig) * ROW;      // columns 2 tig, 2 tig + 1
                float* r1 = r0 + ROW;
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const int d = 64 * g + 8 * gid;
#pragma unroll
                    for (int t = 0; t < 4; ++t) {            // rows gid: an even channel; rows gid + 8: the odd one, 16 times
                        r0[d + 2 * t] = fmaf(acc[n][g][t][0] - ones[n][g][0], 16777216.0f, w2[n][g].x);
                        r1[d + 2 * t] = fmaf(acc[n][g][t][1] - ones[n][g][1], 16777216.0f, w2[n][g].y);
                        r0[d + 2 * t + 1] = fmaf(acc[n][g][t][2] - ones[n][g][2], 1048576.0f, w2[n][g].x);
                        r1[d + 2 * t + 1] = fmaf(acc[n][g][t][3] - ones[n][g][3], 1048576.0f, w2[n][g].y);
                    }
                }
                if (gid == 0) {
                    r0[D] = -neg[n].x, r0[D + 1] = l2[n].x;
                    r1[D] = -neg[n].y, r1[D + 1] = l2[n].y;
                }
                __syncthreads();
                const int real = min(a.group - n * 8, HEADS);
                for (int e = threadIdx.x; e < real * (D / 4); e += kScanThreads) {
                    const int c = e / (D / 4), d = (e - c * (D / 4)) * 4, j = n * 8 + c;
                    const float* r = merge + c * ROW;        // row (warp, copy) of the head: 8 warp + HEADS copy further
                    float m = r[D];
#pragma unroll
                    for (int w = 1; w < kWarps * W; ++w) m = fmaxf(m, r[w * HEADS * ROW + D]);
                    float l = 0.f;
                    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int w = 0; w < kWarps * W; ++w) {
                        const float* rw = r + w * HEADS * ROW;
                        const float f = ex2_approx(rw[D] - m);       // (a row of NaN sums stays NaN under any factor)
                        const float4 x = *reinterpret_cast<const float4*>(rw + d);
                        l = fmaf(f, rw[D + 1], l);
                        o.x = fmaf(f, x.x, o.x), o.y = fmaf(f, x.y, o.y), o.z = fmaf(f, x.z, o.z), o.w = fmaf(f, x.w, o.w);
                    }
                    if (whole) {
                        const float inv = 1.0f / l;
                        *reinterpret_cast<uint2*>(out + (long long)j * D + d) = make_uint2(pack_half2(o.x * inv, o.y * inv), pack_half2(o.z * inv, o.w * inv));
                    } else {
                        *reinterpret_cast<float4*>(part + j * ROW + d) = o;
                        if (d == 0) part[j * ROW + D] = m, part[j * ROW + D + 1] = l;
                    }
                }
            }
            fence_proxy_async();                                 // before the next copy into this stage
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty(s));
        next_stage();
        if (more) next_row<D>(a, cur);
        tile = 0;
    }
    return;
late:                                        // a wait gave up: copies still in flight land before this warp leaves
    if (lane == 0) note(a, kNotedTimeout, 1u);
    for (int k = 0; k < Cfg::STAGES; ++k)
        for (uint32_t ph = 0; ph < 2; ++ph) mbar_wait_bounded(full(k), ph, 64u);
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
    float m = -kNoReference;
    for (int i = threadIdx.x; i < parts; i += 128) m = fmaxf(m, part_of(i)[D]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((threadIdx.x & 31) == 0) s_m[threadIdx.x >> 5] = m;
    __syncthreads();
    m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    const int k = threadIdx.x / LPR, d = (threadIdx.x % LPR) * 4;
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = k; i < parts; i += PER) {
        const float* p = part_of(i);
        const float4 x = *reinterpret_cast<const float4*>(p + d);
        const float2 ml = *reinterpret_cast<const float2*>(p + D);
        const float f = ex2_approx(ml.x - m);
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

int resident_ctas(int group) { return group <= 8 ? Kv4Cfg<128, 1, 1>::CTAS : Kv4Cfg<128, 2, 1>::CTAS; }

Kv4Layout kv4_layout(int B, int kv_heads, int group, int max_len, int D) {
    Kv4Layout y;
    const long long tiles = (long long)B * kv_heads * ((max_len + tile_of(D) - 1) / tile_of(D));
    const long long resident = (long long)sms() * resident_ctas(group);
    y.ctas = (int)(tiles < resident ? tiles : resident);
    y.prefix_off = 256;
    y.noted_off = y.prefix_off + round_up((size_t)(B + 1) * 4, 256);
    y.parts_off = y.noted_off + round_up((size_t)y.ctas * 4, 256);
    y.total = y.parts_off + round_up((size_t)y.ctas * 2 * group * (D + 4) * 4, 256);
    return y;
}

bool kv4_shape_ok(int B, int heads, int kv_heads, int max_len, int D) {
    return B > 0 && kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && heads / kv_heads <= 16 && max_len > 0 && (D == 64 || D == 128) &&
           (long long)B * kv_heads * ((max_len + tile_of(D) - 1) / tile_of(D)) < (1ll << 31) && (long long)B * kv_heads < (1ll << 31);
}

template <int D, int NT, int W, int PAGE>
int launch_kv4(const Kv4Args& a, int ctas, cudaStream_t st) {
    using Cfg = Kv4Cfg<D, NT, W>;
    static bool attr_done[64] = {false};
    int dev = 0;
    I8TK_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !attr_done[dev]) {
        I8TK_CUDA(cudaFuncSetAttribute(kv4_scan_kernel<D, NT, W, PAGE>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM));
        // the merge under the same split of L1 and shared memory: an SM changes it only when it is empty, and then the
        // two kernels do not overlap
        I8TK_CUDA(cudaFuncSetAttribute(kv4_scan_kernel<D, NT, W, PAGE>, cudaFuncAttributePreferredSharedMemoryCarveout, 100));
        I8TK_CUDA(cudaFuncSetAttribute(kv4_merge_kernel<D>, cudaFuncAttributePreferredSharedMemoryCarveout, 100));
        if (dev >= 0 && dev < 64) attr_done[dev] = true;
    }
    I8TK_CUDA(launch_after(kv4_scan_kernel<D, NT, W, PAGE>, dim3((unsigned)ctas), dim3(kScanThreads), Cfg::SMEM, st, a));
    I8TK_CUDA(launch_after(kv4_merge_kernel<D>, dim3((unsigned)(a.B * a.kv_heads), (unsigned)a.group), dim3(128), 0, st, a, ctas));
    return I8TK_OK;
}
template <int D, int NT, int W>
int launch_page(const Kv4Args& a, int page, int ctas, cudaStream_t st) {
    if (page == 16) return launch_kv4<D, NT, W, 16>(a, ctas, st);
    if (page == 32) return launch_kv4<D, NT, W, 32>(a, ctas, st);
    if (page == 64) return launch_kv4<D, NT, W, 64>(a, ctas, st);
    return launch_kv4<D, NT, W, 128>(a, ctas, st);
}
template <int D>
int launch_group(const Kv4Args& a, int page, int ctas, cudaStream_t st) {
    if (a.group <= 2) return launch_page<D, 1, 4>(a, page, ctas, st);
    if (a.group <= 4) return launch_page<D, 1, 2>(a, page, ctas, st);
    if (a.group <= 8) return launch_page<D, 1, 1>(a, page, ctas, st);
    return launch_page<D, 2, 1>(a, page, ctas, st);
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
    const Kv4Args a{Q, sQ, q_stride, sq_stride, static_cast<const unsigned char*>(pool), page_table, seq_lens,
                    static_cast<__half*>(out_f16), batch, kv_heads, group, max_seq_len, max_pages_per_seq, (int)num_pages,
                    1.4426950408889634f / sqrtf((float)head_dim), reinterpret_cast<uint32_t*>(ws),
                    reinterpret_cast<int*>(ws + y.prefix_off), reinterpret_cast<uint32_t*>(ws + y.noted_off), reinterpret_cast<float*>(ws + y.parts_off)};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return head_dim == 64 ? launch_group<64>(a, page_size, y.ctas, st) : launch_group<128>(a, page_size, y.ctas, st);
}
