// INT8 attention over packed sequences of different lengths, grouped heads, causal or not.
//
//   score[i][j] = (q_i . k_j) * sQ_i * sK_j / sqrt(D),  j in i's sequence (and j <= i when causal)
//   out_i       = sum_j softmax(score_i)_j * sV_j * v_j
//
// The tensor-core shape of prefill_attention.cu (Q.K^T as kind::i8 into tensor memory, P.V as kind::f16 with P read
// from tensor memory, lazy maximum), with the differences below.  head_dim 256 runs it as it is (six sequences up to 1111,
// 14/2 heads, not causal: 64-66 us); head_dim 64 and 128 run varlen_wide_kernel, which has its own comment:
//
// * A CTA's 128 query rows are floor(128/group) tokens of ALL the query heads that share a key head (row = token *
//   group + head).  K and V tiles are then read once for the group, and with a causal mask the part of the last tiles
//   that is computed and thrown away covers 128/group tokens instead of 128.  One three-dimensional TMA box brings
//   the query tile from the caller's [token][head][channel] layout; rows past the box are never stored.
// * Sequences are found on the device.  Sequence b owns the tile slots cu[b]/n + b .. cu[b+1]/n + b + 1 of n tokens
//   each -- at least as many as it needs, for any lengths -- so a CTA finds its work by a search and no plan runs
//   ahead; at most one slot per sequence and head is empty.
// * P carries the values' scales: P_ij = fp16(p_ij * sV_j * c), and V enters as its codes, exact in fp16.  c is the
//   power of two that brings the largest scale of the sequence and head to [2^6, 2^7), so P stays in range for any
//   scales.  Against fp16(V * sV) this leaves one rounding instead of two in the product, and what a MASKED position
//   holds cannot reach the result: p = 0 times a finite code.
// * A pre-pass lays V's codes out as fp16 [key head][slot of 64][D], with zeros behind each sequence's end, and the
//   keys' and values' scales as [key head][slot of 64] (coalesced for the softmax warps; in the caller's layout the
//   scales of a head are a token apart).  A value scale that is not finite becomes a NaN key scale there: rows that
//   see the position are NaN, rows that do not are untouched.
#include "score_reference.cuh"
#include "tcgen05.cuh"

#include <cmath>
#include <type_traits>

namespace i8tk {
namespace {

constexpr int kQT = 128;                 // query rows per CTA
constexpr int KT = 64;                   // key positions per tile, and per slot of the pre-pass
constexpr int HK = KT / 2;               // key positions of a tile per softmax thread
constexpr int kSoftmaxWarps = 8;         // two per TMEM lane quarter
constexpr int kThreads = (2 + kSoftmaxWarps) * 32;
constexpr int kRing = 3;
constexpr float kLazyStep = 8.0f;        // log2 units the true maximum may run ahead of the reference: p <= 2^8, P < 2^15

// head_dim 256 (64 and 128: WideCfg)
struct VarCfg {
    static constexpr int D = 256;
    static constexpr int QK_SLABS = D / 128;
    static constexpr int Q_SLAB = kQT * 128;
    static constexpr int K_SLAB = KT * 128;
    static constexpr int Q_BYTES = kQT * D;
    static constexpr int K_BYTES = KT * D;
    static constexpr int V_BYTES = KT * D * 2;
    static constexpr int V_SLAB = KT * 128;
    static constexpr int OFF_Q = 0;
    static constexpr int OFF_K = OFF_Q + Q_BYTES;
    static constexpr int OFF_V = OFF_K + kRing * K_BYTES;
    static constexpr int OFF_SCALES = OFF_V + kRing * V_BYTES;                 // 8 warps x 2 tiles x (sK[HK], sV[HK]) fp32
    static constexpr int OFF_XCH = OFF_SCALES + kSoftmaxWarps * 4 * HK * 4;    // [2][2 halves][128 rows] fp32
    static constexpr int OFF_BARS = OFF_XCH + 2 * 2 * kQT * 4;
    static constexpr int NUM_BARS = 24;
    static constexpr int SMEM_BYTES = 1024 + OFF_BARS + NUM_BARS * 8 + 16;
    static constexpr int TM_P = 2 * KT;                                        // behind two score tiles
    static constexpr int TM_O = 256;
    static constexpr int TMEM_COLS = 512;
    static_assert(TM_P + KT <= TM_O && TM_O + D <= TMEM_COLS, "tensor-memory layout");
    static_assert(SMEM_BYTES <= 227 * 1024, "shared memory of an SM");
};

enum Bar : int {
    B_QFULL = 0,
    B_KFULL = 1,      // [kRing]
    B_KEMPTY = 4,     // [kRing]
    B_SFULL = 7,      // [2]
    B_SEMPTY = 9,     // [2]
    B_PFULL = 11,     // [2]
    B_VFULL = 13,     // [kRing]
    B_VEMPTY = 16,    // [kRing]
    B_PVDONE = 19,    // [2]
};

struct Packed {
    const int* cu;               // [B + 1]
    int B, T, max_len, causal;
    int heads, kv_heads, group;
    int tokens;                  // query tokens per CTA: floor(128 / group)
    int slots;                   // of 64 positions in the pre-pass's arrays: T / 64 + B, and two behind the last
    const float* sQ;
    long long sq_stride;
    const float* sK;             // pre-pass: [kv_heads][slots * 64]
    const float* sV;
    const float* top;            // pre-pass: [kv_heads][slots] largest finite value scale of a slot
    __half* out;                 // [T][heads][D]
    float score_scale_log2;
    uint32_t* status;
    uint32_t* counter;           // work taken so far beyond a first piece per CTA (head_dim 64 and 128); the pre-pass
                                 // sets it to zero
};

// The sequence that owns slot `slot` of n-token slots, its first row and length, and the slot's place in it.  Values of
// cu are read inside [0, T], so a damaged table cannot lead outside the arrays.
struct Seq {
    int start, len, first_slot, local;
    int whole;                   // length before it is cut to max_len
};
__device__ __forceinline__ int cu_at(const int* cu, int i, int T) { return min(max(__ldg(cu + i), 0), T); }
__device__ __forceinline__ Seq sequence_of(int from, int to, int found, int max_len, int slot, int n) {
    Seq s;
    s.start = from;
    s.whole = max(to - from, 0);
    s.len = min(s.whole, max_len);
    s.first_slot = from / n + found;
    s.local = slot - s.first_slot;
    return s;
}
// One lane looks: seven probes a round, whose loads are on their way together.
__device__ __forceinline__ Seq find_sequence_alone(const int* cu, int B, int T, int max_len, int slot, int n) {
    int lo = 0, hi = B - 1;                  // largest b with cu[b] / n + b <= slot, or 0
    while (lo < hi) {
        const int step = (hi - lo + 8) >> 3;
        int from[7], run = 0;
#pragma unroll
        for (int k = 0; k < 7; ++k) from[k] = cu_at(cu, min(lo + (k + 1) * step, hi), T);
        bool below = true;
#pragma unroll
        for (int k = 0; k < 7; ++k) {        // the unbroken run of probes at or below the slot (a damaged table may break it)
            const int b = min(lo + (k + 1) * step, hi);
            below = below && from[k] < (long long)(slot - b + 1) * n;
            run += below ? 1 : 0;
        }
        lo = min(lo + run * step, hi);
        hi = run == 7 ? hi : min(lo + step - 1, hi);
    }
    return sequence_of(cu_at(cu, lo, T), cu_at(cu, lo + 1, T), lo, max_len, slot, n);
}
// A whole warp looks: 32 probes a round, so up to 32 sequences cost one load's latency, up to 1024 two.
__device__ __forceinline__ Seq find_sequence(const int* cu, int B, int T, int max_len, int slot, int n) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = B - 1;                  // largest b with cu[b] / n + b <= slot, or 0
    for (;;) {
        const int step = (hi - lo + 32) >> 5, b = min(lo + lane * step, hi);
        const int from = cu_at(cu, b, T), to = cu_at(cu, b + 1, T);
        const unsigned below = __ballot_sync(0xffffffffu, from / n + b <= slot);
        // the last probe of the unbroken run from lane 0 on (a damaged table may break it)
        const int run = below == 0xffffffffu ? 32 : __ffs((int)~below) - 1, at = max(run - 1, 0);
        if (step == 1) {
            return sequence_of(__shfl_sync(0xffffffffu, from, at), __shfl_sync(0xffffffffu, to, at), min(lo + at, hi), max_len, slot, n);
        }
        lo = min(lo + at * step, hi);
        hi = min(lo + step - 1, hi);
    }
}

__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Pre-pass, one CTA per (slot of 64 positions, key head).
template <int D>
__global__ void __launch_bounds__(128)
varlen_prepare_kernel(const int8_t* __restrict__ V, long long v_stride, const float* __restrict__ sK, long long sk_stride,
                      const float* __restrict__ sV, long long sv_stride, __half* __restrict__ V16, float* __restrict__ sKp,
                      float* __restrict__ sVp, float* __restrict__ top, Packed a) {
    __shared__ float s_top[2];
    pdl_wait();
    pdl_launch_dependents();
    const int slot = blockIdx.x, h = blockIdx.y;
    if (slot == 0 && h == 0 && threadIdx.x == 0) {
        clear_call_status(a.status);
        *a.counter = 0u;
    }
    const Seq s = find_sequence(a.cu, a.B, a.T, a.max_len, slot, KT);
    const int valid = s.local < 0 ? 0 : min(KT, s.len - s.local * KT);      // positions of the slot that exist
    const long long row0 = (long long)s.start + (long long)s.local * KT;
    const long long at = ((long long)h * a.slots + slot) * KT;
    constexpr int LPR = D / 16;                  // 16 codes per thread
    for (int e = threadIdx.x; e < KT * LPR; e += 128) {
        const int r = e / LPR, c = (e % LPR) * 16;
        uint4 w = make_uint4(0u, 0u, 0u, 0u);
        if (r < valid) w = *reinterpret_cast<const uint4*>(V + (row0 + r) * v_stride + h * D + c);
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
        uint32_t o[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {            // code + 128 in the low byte of a half of 1024: exact
            const uint32_t u = ww[k] ^ 0x80808080u;
            const uint32_t lo = prmt(u, 0x64646464u, 0x4140u), hi = prmt(u, 0x64646464u, 0x4342u);
            const __half2 bias = __floats2half2_rn(1152.f, 1152.f);
            const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&lo), bias), y = __hsub2(*reinterpret_cast<const __half2*>(&hi), bias);
            o[2 * k] = *reinterpret_cast<const uint32_t*>(&x);
            o[2 * k + 1] = *reinterpret_cast<const uint32_t*>(&y);
        }
        __half* dst = V16 + (at + r) * D + c;
        *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
        *reinterpret_cast<uint4*>(dst + 8) = make_uint4(o[4], o[5], o[6], o[7]);
    }
    if (threadIdx.x < KT) {
        const int r = threadIdx.x;
        float k = 0.f, v = 0.f;
        if (r < valid) {
            k = sK[(row0 + r) * sk_stride + h];
            v = sV[(row0 + r) * sv_stride + h];
            if (!(fabsf(v) <= 3.402823466e38f)) k = __int_as_float(0x7fc00000), v = 0.f;
        }
        sKp[at + r] = k;
        sVp[at + r] = v;
        float m = fabsf(v);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if ((r & 31) == 0) s_top[r >> 5] = m;
    }
    __syncthreads();
    if (threadIdx.x == 0) top[(long long)h * a.slots + slot] = fmaxf(s_top[0], s_top[1]);
    // rows that nothing is computed for: behind the cut of a longer sequence, and outside every sequence
    if (s.whole > s.len && s.local >= 0) {
        const int lo = max(s.len, s.local * KT), hi = min(s.whole, s.local * KT + KT), vecs = a.group * D / 8;
        for (int p = lo; p < hi; ++p) {
            uint4* row = reinterpret_cast<uint4*>(a.out + ((long long)(s.start + p) * a.heads + h * a.group) * D);
            for (int e = threadIdx.x; e < vecs; e += 128) row[e] = make_uint4(0u, 0u, 0u, 0u);
        }
    }
    const long long before = cu_at(a.cu, 0, a.T), rest = before + (a.T - cu_at(a.cu, a.B, a.T));
    const int vecs = a.heads * D / 8;
    for (long long r = (long long)slot * gridDim.y + h; r < rest; r += (long long)gridDim.x * gridDim.y) {
        uint4* row = reinterpret_cast<uint4*>(a.out + (r < before ? r : a.T - rest + r) * a.heads * D);
        for (int e = threadIdx.x; e < vecs; e += 128) row[e] = make_uint4(0u, 0u, 0u, 0u);
    }
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
        : "memory");
}

__global__ void __launch_bounds__(kThreads, 1)
varlen_attention_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                        const __grid_constant__ CUtensorMap tmV, const __grid_constant__ Packed a) {
    using Cfg = VarCfg;
    constexpr int D = Cfg::D;
    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw_s = smem_u32(smem_raw);
    const uint32_t base_s = (raw_s + 1023u) & ~1023u;       // swizzle patterns are functions of address bits
    unsigned char* base = smem_raw + (base_s - raw_s);
    const uint32_t bars = base_s + Cfg::OFF_BARS;
    auto bar = [&](int i) -> uint32_t { return bars + 8u * i; };
    const uint32_t tmem_slot = bars + Cfg::NUM_BARS * 8;
    volatile uint32_t* tmem_slot_p = reinterpret_cast<volatile uint32_t*>(base + Cfg::OFF_BARS + Cfg::NUM_BARS * 8);

    pdl_wait();
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    // the last slots first: with a causal mask the long rows of a sequence are its last
    const int hk = blockIdx.x % a.kv_heads;
    const int slot = (int)(gridDim.x - 1 - blockIdx.x) / a.kv_heads;
    const Seq s = find_sequence(a.cu, a.B, a.T, a.max_len, slot, a.tokens);
    const int tok0 = s.local * a.tokens;                    // first query token of this CTA in its sequence
    if (s.local < 0 || tok0 >= s.len) return;               // an empty slot: the whole CTA leaves
    const int kv_end = a.causal ? min(s.len, tok0 + a.tokens) : s.len;
    const int nt = (kv_end + KT - 1) / KT;
    const int all_visible = a.causal ? tok0 + 1 : s.len;    // positions that every row of the CTA sees
    const int kv_slot = s.start / KT + (s.first_slot - s.start / a.tokens);    // first slot of 64 of this sequence

    if (threadIdx.x == 0) {
        mbar_init(bar(B_QFULL), 1);
        for (int i = 0; i < kRing; ++i) {
            mbar_init(bar(B_KFULL + i), 1);
            mbar_init(bar(B_KEMPTY + i), 1);
            mbar_init(bar(B_VFULL + i), 1);
            mbar_init(bar(B_VEMPTY + i), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(B_SFULL + i), 1);
            mbar_init(bar(B_SEMPTY + i), kSoftmaxWarps);
            mbar_init(bar(B_PFULL + i), kSoftmaxWarps);
            mbar_init(bar(B_PVDONE + i), 1);
        }
        fence_mbar_init();
    }
    if (warp == 1) tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot_p;

    if (warp == 0) {
        // ================= TMA producers: K by one lane, V by another (they are freed by different products) =========
        if (lane == 0) {
            mbar_expect_tx(bar(B_QFULL), a.tokens * a.group * D);
#pragma unroll
            for (int sl = 0; sl < Cfg::QK_SLABS; ++sl)
                tma_load_3d(base_s + Cfg::OFF_Q + sl * Cfg::Q_SLAB, &tmQ, sl * 128, hk * a.group, s.start + tok0, bar(B_QFULL));
            for (int j = 0; j < nt; ++j) {
                const int st = j % kRing;
                if (!mbar_wait_spin_bounded(bar(B_KEMPTY + st), ((j / kRing) & 1) ^ 1)) {
                    note_timeout(a.status);
                    break;
                }
                mbar_expect_tx(bar(B_KFULL + st), Cfg::K_BYTES);
#pragma unroll
                for (int sl = 0; sl < Cfg::QK_SLABS; ++sl)
                    tma_load_3d(base_s + Cfg::OFF_K + st * Cfg::K_BYTES + sl * Cfg::K_SLAB, &tmK, sl * 128, hk, s.start + j * KT,
                                bar(B_KFULL + st));
            }
        } else if (lane == 1) {
            const int row0 = (hk * a.slots + kv_slot) * KT;
            for (int j = 0; j < nt; ++j) {
                const int st = j % kRing;
                if (!mbar_wait_spin_bounded(bar(B_VEMPTY + st), ((j / kRing) & 1) ^ 1)) {
                    note_timeout(a.status);
                    break;
                }
                mbar_expect_tx(bar(B_VFULL + st), Cfg::V_BYTES);
#pragma unroll
                for (int sl = 0; sl < D / 64; ++sl)
                    tma_load_2d(base_s + Cfg::OFF_V + st * Cfg::V_BYTES + sl * Cfg::V_SLAB, &tmV, sl * 128, row0 + j * KT,
                                bar(B_VFULL + st));
            }
        }
    } else if (warp == 1) {
        // ================= MMA issuer =================
        if (elect_one()) {
            constexpr uint32_t idesc_qk = idesc_i8(kQT, KT);
            constexpr uint32_t idesc_pv = idesc_f16(kQT, D, true);
            bool ok = mbar_wait_spin_bounded(bar(B_QFULL), 0);
            auto issue_pv = [&](int t) -> bool {
                if (!mbar_wait_spin_bounded(bar(B_PFULL + (t & 1)), (t >> 1) & 1)) return false;
                const int vs = t % kRing;
                if (!mbar_wait_spin_bounded(bar(B_VFULL + vs), (t / kRing) & 1)) return false;
                tc_fence_after();
                const uint64_t db0 = smem_desc_sw128_mn(base_s + Cfg::OFF_V + vs * Cfg::V_BYTES, Cfg::V_SLAB);
#pragma unroll
                for (int i = 0; i < KT / 16; ++i)
                    mma_f16_ta(tmem_base + Cfg::TM_O, tmem_base + Cfg::TM_P + (t & 1) * (KT / 2) + i * 8, db0 + (uint64_t)(128 * i),
                               idesc_pv, (t | i) != 0);
                tc_commit(bar(B_VEMPTY + vs));
                tc_commit(bar(B_PVDONE + (t & 1)));
                return true;
            };
            // Q.K^T runs two tiles ahead of P.V (the softmax warps convert tile j + 1 while they exponentiate tile j)
            for (int j = 0; j < nt + 2 && ok; ++j) {
                if (j < nt) {
                    const int st = j & 1, kst = j % kRing;
                    if (!mbar_wait_spin_bounded(bar(B_KFULL + kst), (j / kRing) & 1) ||
                        !mbar_wait_spin_bounded(bar(B_SEMPTY + st), ((j >> 1) & 1) ^ 1)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t ks = base_s + Cfg::OFF_K + kst * Cfg::K_BYTES;
#pragma unroll
                    for (int k = 0; k < D / 32; ++k) {
                        const uint32_t qa = base_s + Cfg::OFF_Q + (k / 4) * Cfg::Q_SLAB;
                        const uint32_t ka = ks + (k / 4) * Cfg::K_SLAB;
                        mma_i8(tmem_base + st * KT, smem_desc_sw128(qa) + 2 * (k % 4), smem_desc_sw128(ka) + 2 * (k % 4), idesc_qk, k != 0);
                    }
                    tc_commit(bar(B_KEMPTY + kst));
                    tc_commit(bar(B_SFULL + st));
                }
                if (j >= 2) ok = issue_pv(j - 2);
            }
            if (!ok) note_timeout(a.status);
        }
    } else {
        // ================= softmax: half a query row (32 of 64 positions of every tile) per thread =================
        const int sw = warp - 2;
        const int q = warp & 3;                          // TMEM lane quarter of this warp
        const int half = sw >> 2;
        const int r = q * 32 + lane;                     // row of the tile
        const int tok = tok0 + r / a.group;              // its token in the sequence, and its query head
        const int head = hk * a.group + r % a.group;
        const bool stored = r < a.tokens * a.group && tok < s.len;
        float* wsc = reinterpret_cast<float*>(base + Cfg::OFF_SCALES) + sw * (4 * HK);   // [tile & 1]{sK[HK], sV[HK]}
        float* xch = reinterpret_cast<float*>(base + Cfg::OFF_XCH);                      // [2][half][row]
        float qscale = stored ? a.sQ[(long long)(s.start + tok) * a.sq_stride + head] * a.score_scale_log2 : 0.f;
        if (qscale == 0.f) qscale = 1e-30f;              // a removed position (-inf) stays removed under a scale of zero
        const int visible = a.causal ? min(s.len, tok + 1) : s.len;      // positions that this row sees
        const uint32_t lane_addr = tmem_base + ((uint32_t)(q * 32) << 16);
        constexpr uint32_t kMagicI = 0x4B400000u;        // 1.5 * 2^23: |q.k| < 2^22 converts by an add and a subtract
        const f32x2 nmagic2 = pack2(-12582912.f, -12582912.f);
        const long long sc0 = ((long long)hk * a.slots + kv_slot) * KT + half * HK + lane;
        ScoreReference ref{INFINITY, 0.f, false};        // none yet: any score is ahead of it
        float nm = 0.f;                                  // ref.nm once there is one
        bool far_rows = false;                           // some row of the warp has a far reference
        f32x2 l2 = pack2(0.f, 0.f);
        bool ok = true;

        // the power of two c that brings the largest value scale of the sequence to [2^6, 2^7)
        float most = 0.f;
        for (int j = lane; j < nt; j += 32) most = fmaxf(most, a.top[(long long)hk * a.slots + kv_slot + j]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        const int e2 = min(120, max(-120, 6 - ((int)(__float_as_uint(most) >> 23) - 127)));
        const float c_up = __uint_as_float((uint32_t)(127 + e2) << 23), c_down = __uint_as_float((uint32_t)(127 - e2) << 23);

        float pk, pv;                                    // scales of this warp's positions, fetched ahead of their tile
        auto prefetch = [&](int j) {
            asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(pk) : "l"(a.sK + sc0 + j * KT));
            asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(pv) : "l"(a.sV + sc0 + j * KT));
        };
        auto commit_scales = [&](int j) {
            float* w = wsc + (j & 1) * (2 * HK);
            w[lane] = pk;
            w[HK + lane] = pv * c_up;
            __syncwarp();
        };
        // y = (q.k) * sK for 8 columns of a score block held in registers, and their maximum
        auto convert8 = [&](const uint32_t* sr8, const float* k8, f32x2* y4, float& mx) {
            const float4 ka = *reinterpret_cast<const float4*>(k8);
            const float4 kb = *reinterpret_cast<const float4*>(k8 + 4);
            const f32x2 t01 = add2(pack2(__uint_as_float(sr8[0] + kMagicI), __uint_as_float(sr8[1] + kMagicI)), nmagic2);
            const f32x2 t23 = add2(pack2(__uint_as_float(sr8[2] + kMagicI), __uint_as_float(sr8[3] + kMagicI)), nmagic2);
            const f32x2 t45 = add2(pack2(__uint_as_float(sr8[4] + kMagicI), __uint_as_float(sr8[5] + kMagicI)), nmagic2);
            const f32x2 t67 = add2(pack2(__uint_as_float(sr8[6] + kMagicI), __uint_as_float(sr8[7] + kMagicI)), nmagic2);
            y4[0] = mul2(t01, pack2(ka.x, ka.y));
            y4[1] = mul2(t23, pack2(ka.z, ka.w));
            y4[2] = mul2(t45, pack2(kb.x, kb.y));
            y4[3] = mul2(t67, pack2(kb.z, kb.w));
            mx = max3(max3(mx, y4[0].x, y4[0].y), max3(y4[1].x, y4[1].y, y4[2].x), fmaxf(y4[2].y, fmaxf(y4[3].x, y4[3].y)));
        };
        // a tile that some row does not see whole: this row's positions from `visible` on are removed, whatever was there
        auto mask_tile = [&](f32x2* yy, float& mx, int j) {
            const int lim = visible - j * KT - half * HK;
            mx = -INFINITY;
#pragma unroll
            for (int e = 0; e < HK / 2; ++e) {
                if (2 * e >= lim) yy[e].x = -INFINITY;
                if (2 * e + 1 >= lim) yy[e].y = -INFINITY;
                mx = fmaxf(mx, fmaxf(yy[e].x, yy[e].y));
            }
        };
        // p = 2^(y*qs + nm) for 8 columns; p * sV * c leaves as four fp16 pairs for this row's lane of the P tile
        auto exp8 = [&](const f32x2* y4, const float* v8, f32x2 qs2, f32x2 nm2, uint32_t dst) {
            const float4 va = *reinterpret_cast<const float4*>(v8);
            const float4 vb = *reinterpret_cast<const float4*>(v8 + 4);
            const f32x2 x0 = fma2(y4[0], qs2, nm2), x1 = fma2(y4[1], qs2, nm2);
            const f32x2 x2 = fma2(y4[2], qs2, nm2), x3 = fma2(y4[3], qs2, nm2);
            const f32x2 p0 = pack2(ex2_approx(x0.x), ex2_approx(x0.y)), p1 = pack2(ex2_approx(x1.x), ex2_approx(x1.y));
            const f32x2 p2 = pack2(ex2_approx(x2.x), ex2_approx(x2.y)), p3 = pack2(ex2_approx(x3.x), ex2_approx(x3.y));
            l2 = add2(l2, add2(add2(p0, p1), add2(p2, p3)));
            const f32x2 s0 = mul2(p0, pack2(va.x, va.y)), s1 = mul2(p1, pack2(va.z, va.w));
            const f32x2 s2 = mul2(p2, pack2(vb.x, vb.y)), s3 = mul2(p3, pack2(vb.z, vb.w));
            tmem_st4(dst, pack_h2(s0.x, s0.y), pack_h2(s1.x, s1.y), pack_h2(s2.x, s2.y), pack_h2(s3.x, s3.y));
        };

        // ---- prologue: scores of tile 0 into registers ----
        f32x2 y[HK / 2];
        float mx = -INFINITY;
        prefetch(0);
        commit_scales(0);
        if (nt > 1) prefetch(1);
        {
            const bool got = mbar_wait_spin_bounded(bar(B_SFULL), 0);
            ok = __all_sync(0xffffffffu, got);
            if (ok) {
                tc_fence_after();
                uint32_t sr[2][16];
                const uint32_t s_addr = lane_addr + half * HK;
                tmem_ld16(s_addr, sr[0]);
#pragma unroll
                for (int cc = 0; cc < HK / 16; ++cc) {
                    tmem_ld_wait(sr[cc & 1]);
                    if (cc < HK / 16 - 1) tmem_ld16(s_addr + (cc + 1) * 16, sr[(cc + 1) & 1]);
                    convert8(&sr[cc & 1][0], wsc + cc * 16, &y[cc * 8], mx);
                    convert8(&sr[cc & 1][8], wsc + cc * 16 + 8, &y[cc * 8 + 4], mx);
                }
                if (KT > all_visible) mask_tile(y, mx, 0);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(B_SEMPTY));
            }
        }

        for (int j = 0; j < nt && ok; ++j) {
            const int st = j & 1;
            const bool has_next = j + 1 < nt;
            // ---- row maximum across the two halves ----
            xch[(st * 2 + half) * kQT + r] = mx;
            asm volatile("bar.sync %0, 64;" ::"r"(1 + q) : "memory");
            mx = fmaxf(mx, xch[(st * 2 + (half ^ 1)) * kQT + r]);

            const bool move = fmaf(mx, qscale, ref.nm) + ref.rest > kLazyStep;
            const bool warp_moves = __any_sync(0xffffffffu, move);
            float corr = 1.0f;
            if (warp_moves) {
                if (move) {
                    corr = ex2_approx(ref.move_to(mx, qscale, 0.f));
                    nm = ref.nm;
                    l2 = mul2(l2, pack2(corr, corr));
                }
                far_rows = __any_sync(0xffffffffu, ref.far);
            }

            // ---- this tile's P buffer is free once PV of tile j-2 retired; the accumulator is touched only when a
            // maximum moved, and then PV of tile j-1 must have retired too ----
            if (j >= 2) {
                const bool got2 = mbar_wait_spin_bounded(bar(B_PVDONE + st), ((j - 2) >> 1) & 1);
                if (!__all_sync(0xffffffffu, got2)) { ok = false; break; }
            }
            if (j > 0 && warp_moves) {
                const bool got3 = mbar_wait_spin_bounded(bar(B_PVDONE + (st ^ 1)), ((j - 1) >> 1) & 1);
                if (!__all_sync(0xffffffffu, got3)) { ok = false; break; }
                tc_fence_after();
                uint32_t o[32];
#pragma unroll 1
                for (int cc = 0; cc < D / 64; ++cc) {
                    const uint32_t oa = lane_addr + Cfg::TM_O + half * (D / 2) + cc * 32;
                    tmem_ld32(oa, o);
                    tmem_ld_wait(o);
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
                    tmem_st32(oa, o);
                }
                tmem_st_wait();
            }
            // ---- exponentials of this tile interleaved with the conversion of the NEXT tile's scores ----
            const uint32_t prow = lane_addr + Cfg::TM_P + st * (KT / 2) + half * (HK / 2);
            f32x2 qs2 = pack2(qscale, qscale), nm2 = pack2(nm, nm);
            if (far_rows) {          // the remainder of a far reference: the exponents are made here
                const f32x2 rest2 = pack2(ref.rest, ref.rest);
#pragma unroll
                for (int e = 0; e < HK / 2; ++e) y[e] = add2(fma2(y[e], qs2, nm2), rest2);
                qs2 = pack2(1.f, 1.f), nm2 = pack2(0.f, 0.f);
            }
            const float* vsc = wsc + st * (2 * HK) + HK;
            mx = -INFINITY;
            if (has_next) {
                commit_scales(j + 1);
                if (j + 2 < nt) prefetch(j + 2);
                const int sb1 = st ^ 1;
                const bool got = mbar_wait_spin_bounded(bar(B_SFULL + sb1), ((j + 1) >> 1) & 1);
                if (!__all_sync(0xffffffffu, got)) { ok = false; break; }
                tc_fence_after();
                const float* ksc = wsc + (st ^ 1) * (2 * HK);
                const uint32_t s_addr = lane_addr + sb1 * KT + half * HK;
                uint32_t sr[2][16];
                tmem_ld16(s_addr, sr[0]);
#pragma unroll
                for (int cc = 0; cc < HK / 16; ++cc) {
                    tmem_ld_wait(sr[cc & 1]);
                    if (cc < HK / 16 - 1) tmem_ld16(s_addr + (cc + 1) * 16, sr[(cc + 1) & 1]);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int c = cc * 2 + h;
                        exp8(&y[c * 4], vsc + c * 8, qs2, nm2, prow + c * 4);
                        convert8(&sr[cc & 1][h * 8], ksc + c * 8, &y[c * 4], mx);
                    }
                }
                if ((j + 2) * KT > all_visible) mask_tile(y, mx, j + 1);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(B_SEMPTY + sb1));
            } else {
#pragma unroll
                for (int c = 0; c < HK / 8; ++c) exp8(&y[c * 4], vsc + c * 8, qs2, nm2, prow + c * 4);
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(B_PFULL + st));
        }
        // ---- epilogue: O / (l c) -> fp16, each thread its half of the output columns ----
        if (ok) {
            const bool got = mbar_wait_spin_bounded(bar(B_PVDONE + ((nt - 1) & 1)), ((nt - 1) >> 1) & 1);
            ok = __all_sync(0xffffffffu, got);
        }
        if (ok) {
            tc_fence_after();
            float l = l2.x + l2.y;
            // the buffer of the tile before the last: a warp still reading the last tile's maxima is not overwritten
            float* fin = xch + (nt & 1) * 2 * kQT;
            fin[half * kQT + r] = l;
            asm volatile("bar.sync %0, 64;" ::"r"(1 + q) : "memory");
            l += fin[(half ^ 1) * kQT + r];
            const float inv = 1.0f / l * c_down;
            __half* orow = a.out + ((long long)(s.start + tok) * a.heads + head) * D + half * (D / 2);
            uint32_t o[32];
#pragma unroll 1
            for (int cc = 0; cc < D / 64; ++cc) {
                tmem_ld32(lane_addr + Cfg::TM_O + half * (D / 2) + cc * 32, o);
                tmem_ld_wait(o);
                uint32_t hp[16];
#pragma unroll
                for (int i = 0; i < 32; i += 2)
                    hp[i >> 1] = pack_h2(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv);
                if (stored) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        *reinterpret_cast<uint4*>(orow + cc * 32 + k * 8) =
                            make_uint4(hp[4 * k], hp[4 * k + 1], hp[4 * k + 2], hp[4 * k + 3]);
                }
            }
        } else if (lane == 0) {
            note_timeout(a.status);
        }
    }

    // common exit: every role ends here, then the allocating warp frees tensor memory
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
    }
}

// ---- head_dim 64 and 128: two query tiles per CTA, a thread per row -------------------------------------------
// One persistent CTA per SM holds two query tiles (A and B, 128 rows each) against the same key tiles of 128
// positions.  Each tile has its own score block and accumulator in tensor memory and its own four softmax warps, a
// thread per row: no row is shared between threads, so nothing is exchanged, and what a tile costs besides its scores
// (barriers, waits, the check of the maximum) is paid once per 128 scores of a thread.  While the softmax of one tile
// runs, the tensor core works for the other.  P overwrites the scores it came from: Q.K^T of the next key tile follows
// P.V in the order of the one thread that issues both.
// The exponentials are taken against the reference of the tiles before, without looking for the maximum first; the
// maximum is found on the way, and only where it runs more than kLazyStep ahead (the scores are still there) is the
// reference moved, the accumulator rescaled and the tile done again, once: then no score is ahead by more than the
// rounding of the reference.  Where that rounding would matter, far_tile() does the tile.  The first reference of a row
// comes from its first 32 scores.
// The pairs of tiles are taken from a counter, long rows first, by the thread that starts the loads, which runs ahead
// into the next pair while the last one is finished.
// (8192 tokens causal, 32/8 heads, D 128: 519-547 us, 1.02 PFLOP/s at 540; with prefill_attention.cu's shape 622.  Two score blocks of
// 64 positions per query tile, Q.K^T a tile ahead: 592; halves of 64 with an issuing thread for each query tile: 585.)
constexpr int kWideThreads = 12 * 32;    // 2 x 4 softmax warps, loads, MMA, and two that fill their warpgroup
// Registers per thread: 168 at launch; the warpgroup of loads and MMA hands most of its own to the softmax warpgroups
// (2 * 128 * 224 + 128 * 56 = 384 * 168).
constexpr int kSoftmaxRegs = 224, kOtherRegs = 56;
static_assert(256 * kSoftmaxRegs + 128 * kOtherRegs <= kWideThreads * 168, "more registers than the block was launched with");
constexpr int kWideKT = 128;
constexpr int kScaleRing = 4;

template <int D>
struct WideCfg {
    static constexpr int Q_BYTES = kQT * D;                                     // one query tile, one swizzled slab
    static constexpr int K_BYTES = kWideKT * D;
    static constexpr int V_BYTES = kWideKT * D * 2;
    static constexpr int V_SLAB = kWideKT * 128;
    static constexpr int OFF_Q = 0;                                             // [2 pairs][A, B]
    static constexpr int OFF_K = OFF_Q + 4 * Q_BYTES;
    static constexpr int OFF_V = OFF_K + kRing * K_BYTES;
    static constexpr int OFF_SCALES = OFF_V + kRing * V_BYTES;                  // [kScaleRing]{sK[128], sV[128]}
    static constexpr int OFF_BARS = OFF_SCALES + kScaleRing * 2 * kWideKT * 4;
    static constexpr int NUM_BARS = 40;
    static constexpr int SMEM_BYTES = 1024 + OFF_BARS + NUM_BARS * 8 + 16;
    static constexpr int TM_S = 0;                                              // A, B: 128 columns each; P in the first 64
    static constexpr int TM_O = 256;                                            // A, B: D columns each
    static_assert(SMEM_BYTES + 1024 <= 227 * 1024, "shared memory of an SM");
};
enum WideBar : int {
    W_WFULL = 0,      // [2]
    W_WEMPTY = 2,     // [2]
    W_QFULL = 4,      // [2]
    W_QEMPTY = 6,     // [2]
    W_KFULL = 8,      // [kRing]
    W_KEMPTY = 11,    // [kRing]
    W_VFULL = 14,     // [kRing]
    W_VEMPTY = 17,    // [kRing]
    W_CFULL = 20,     // [kScaleRing]
    W_CEMPTY = 24,    // [kScaleRing]
    W_SFULL = 28,     // [A, B]
    W_PFULL = 30,     // [A, B]
    W_ODONE = 32,     // [A, B]
    W_OEMPTY = 34,    // [A, B]
};
struct WideWork {
    int start, len, tok0, hk, kv_slot, nt_a, nt_b, pad;      // nt_a < 0: no more work
};

// A tile of which some row's scores are too far out for a reference of one fp32 number: its largest score first, then the
// reference and what it changes, then the probabilities with the reference's remainder, four words of P over columns that
// have been read.  In a function of its own, so that the common way keeps its registers; the steps and their order are
// the same, so the other rows of the warp get the bits they get there.  Returns the row's reference and sum.  kFarMark
// stands for a far reference, or for none yet, that is in *kept: against it any score that the row sees is ahead, so the
// row's next tile comes here as well.
constexpr float kFarMark = 3.402823466e38f;
template <int D>
__device__ __noinline__ float2 far_tile(uint32_t s_addr, uint32_t o_addr, const float* sk, int lim, float qscale, float lift, float nm, float l,
                                        bool first, ScoreReference* kept) {
    auto scores8 = [&](int c, float (&y)[8]) {
        uint32_t sr[8];
        tmem_ld8(s_addr + c, sr);
        tmem_ld_wait(sr);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = c + e < lim ? (float)(int)sr[e] * sk[c + e] : -INFINITY;
    };
    float top = -INFINITY, y[8];
#pragma unroll 1
    for (int c = 0; c < kWideKT; c += 8) {
        scores8(c, y);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, y[e]);
    }
    ScoreReference ref = nm == kFarMark ? *kept : ScoreReference{nm, 0.f, false};
    float corr = 1.0f;
    if (ref.exponent(top, qscale, lift) > lift + kLazyStep) corr = ex2_approx(ref.move_to(top, qscale, lift));
    *kept = ref;
    const bool mark = ref.far || ref.nm == INFINITY;
    if (ref.nm == INFINITY) ref.nm = lift;           // no score yet: no probability either
    if (!first) {
        l *= corr;
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tmem_ld16(o_addr + c, o);
            tmem_ld_wait(o);
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
            tmem_st16(o_addr + c, o);
        }
    }
    const float* sv = sk + kWideKT;
    f32x2 sum2 = pack2(0.f, 0.f);
#pragma unroll 1
    for (int c = 0; c < kWideKT; c += 8) {
        scores8(c, y);
        f32x2 p[4];
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            p[e] = pack2(ex2_approx(ref.exponent(y[2 * e], qscale, lift)), ex2_approx(ref.exponent(y[2 * e + 1], qscale, lift)));
            w[e] = pack_h2(p[e].x * sv[c + 2 * e], p[e].y * sv[c + 2 * e + 1]);
        }
        sum2 = add2(sum2, add2(add2(p[0], p[1]), add2(p[2], p[3])));
        tmem_st4(s_addr + c / 2, w[0], w[1], w[2], w[3]);
    }
    return make_float2(mark ? kFarMark : ref.nm, l + (sum2.x + sum2.y));
}

template <int D>
__global__ void __launch_bounds__(kWideThreads, 1)
varlen_wide_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                   const __grid_constant__ CUtensorMap tmV, const __grid_constant__ Packed a) {
    using Cfg = WideCfg<D>;
    extern __shared__ unsigned char smem_raw[];
    __shared__ WideWork work[2];
    __shared__ ScoreReference far_refs[256];                 // of a softmax thread
    const uint32_t raw_s = smem_u32(smem_raw);
    const uint32_t base_s = (raw_s + 1023u) & ~1023u;       // swizzle patterns are functions of address bits
    unsigned char* base = smem_raw + (base_s - raw_s);
    const uint32_t bars = base_s + Cfg::OFF_BARS;
    auto bar = [&](int i) -> uint32_t { return bars + 8u * i; };
    const uint32_t tmem_slot = bars + Cfg::NUM_BARS * 8;
    volatile uint32_t* tmem_slot_p = reinterpret_cast<volatile uint32_t*>(base + Cfg::OFF_BARS + Cfg::NUM_BARS * 8);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(W_WFULL + i), 1);
            mbar_init(bar(W_WEMPTY + i), 9);
            mbar_init(bar(W_QFULL + i), 1);
            mbar_init(bar(W_QEMPTY + i), 1);
            mbar_init(bar(W_SFULL + i), 1);
            mbar_init(bar(W_PFULL + i), 4);
            mbar_init(bar(W_ODONE + i), 1);
            mbar_init(bar(W_OEMPTY + i), 4);
        }
        for (int i = 0; i < kRing; ++i) {
            mbar_init(bar(W_KFULL + i), 1);
            mbar_init(bar(W_KEMPTY + i), 1);
            mbar_init(bar(W_VFULL + i), 1);
            mbar_init(bar(W_VEMPTY + i), 1);
        }
        for (int i = 0; i < kScaleRing; ++i) {
            mbar_init(bar(W_CFULL + i), 1);
            mbar_init(bar(W_CEMPTY + i), 8);
        }
        fence_mbar_init();
    }
    if (warp == 9) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot_p;
    pdl_wait();
    pdl_launch_dependents();
    const int two = 2 * a.tokens;                            // query tokens of a pair of tiles

    // (each split in its own branch: where the two meet, the compiler has the smaller one)
    if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 8) {
        // ================= work and loads, by one lane =================
        // A choice with two sides, timed in turn.  With the whole warp searching (find_sequence) 16 prompts up to 2048 tokens
        // take 309 us instead of 299.5, 64 up to 1000 425 instead of 410, eight of 4096 at D 64 352 instead of 338, one of
        // 8192 at D 128 538 instead of 530; 700 up to 60 tokens, 16/4 heads, 117 instead of 123.  One lane that bisects:
        // 296, 404, 336, 530 and 134; fifteen probes a round: 305, 423, 342, 543 and 149.
        const int slots = a.T / two + a.B, items = slots * a.kv_heads;
        int t = 0;                                           // key tiles loaded so far
        int next = blockIdx.x;                               // the first of a CTA by its number, the others from the counter
        WideWork x{};
        // this pair to the other roles, then its queries, keys and values; false when a wait gave up
        auto load = [&](int w) -> bool {
            const int ws = w & 1;
            const uint32_t round = (uint32_t)(w >> 1) & 1u;
            if (!mbar_wait_bounded(bar(W_WEMPTY + ws), round ^ 1u)) return false;
            work[ws] = x;
            mbar_arrive(bar(W_WFULL + ws));
            if (x.nt_a < 0) return true;
            if (!mbar_wait_bounded(bar(W_QEMPTY + ws), round ^ 1u)) return false;
            const int q_rows = a.tokens * a.group * D, q_at = base_s + Cfg::OFF_Q + ws * 2 * Cfg::Q_BYTES;
            mbar_expect_tx(bar(W_QFULL + ws), x.nt_b > 0 ? 2 * q_rows : q_rows);
            tma_load_3d(q_at, &tmQ, 0, x.hk * a.group, x.start + x.tok0, bar(W_QFULL + ws));
            if (x.nt_b > 0) tma_load_3d(q_at + Cfg::Q_BYTES, &tmQ, 0, x.hk * a.group, x.start + x.tok0 + a.tokens, bar(W_QFULL + ws));
            const int nt = max(x.nt_a, x.nt_b);
            const long long sc0 = ((long long)x.hk * a.slots + x.kv_slot) * KT;
            for (int j = 0; j < nt; ++j, ++t) {
                const int st = t % kRing, cs = t % kScaleRing;
                const uint32_t r = ((uint32_t)(t / kRing) & 1u) ^ 1u, cr = ((uint32_t)(t / kScaleRing) & 1u) ^ 1u;
                if (!mbar_wait_bounded(bar(W_KEMPTY + st), r) || !mbar_wait_bounded(bar(W_CEMPTY + cs), cr)) return false;
                mbar_expect_tx(bar(W_KFULL + st), Cfg::K_BYTES);
                tma_load_3d(base_s + Cfg::OFF_K + st * Cfg::K_BYTES, &tmK, 0, x.hk, x.start + j * kWideKT, bar(W_KFULL + st));
                mbar_expect_tx(bar(W_CFULL + cs), 2 * kWideKT * 4);
                const uint32_t c_at = base_s + Cfg::OFF_SCALES + cs * (2 * kWideKT * 4);
                bulk_g2s(c_at, a.sK + sc0 + j * kWideKT, kWideKT * 4, bar(W_CFULL + cs));
                bulk_g2s(c_at + kWideKT * 4, a.sV + sc0 + j * kWideKT, kWideKT * 4, bar(W_CFULL + cs));
                if (!mbar_wait_bounded(bar(W_VEMPTY + st), r)) return false;
                mbar_expect_tx(bar(W_VFULL + st), Cfg::V_BYTES);
#pragma unroll
                for (int sl = 0; sl < D / 64; ++sl)
                    tma_load_2d(base_s + Cfg::OFF_V + st * Cfg::V_BYTES + sl * Cfg::V_SLAB, &tmV, sl * 128, (int)(sc0 + j * kWideKT),
                                bar(W_VFULL + st));
            }
            return true;
        };
        bool ok = lane == 0;
        for (int w = 0; ok; ++w) {
            x.nt_a = -1;
            while (next < items && x.nt_a < 0) {             // to a slot that has rows
                const int item = next;
                next = (int)(gridDim.x + atomicAdd(a.counter, 1u));
                x.hk = item % a.kv_heads;
                const Seq s = find_sequence_alone(a.cu, a.B, a.T, a.max_len, slots - 1 - item / a.kv_heads, two);
                x.start = s.start, x.len = s.len, x.tok0 = s.local * two;
                if (s.local < 0 || x.tok0 >= s.len) continue;
                x.kv_slot = s.start / KT + (s.first_slot - s.start / two);
                auto tiles = [&](int tok) {                  // key tiles of the query tile that begins at this token
                    return tok >= s.len ? 0 : ((a.causal ? min(s.len, tok + a.tokens) : s.len) + kWideKT - 1) / kWideKT;
                };
                x.nt_a = tiles(x.tok0), x.nt_b = tiles(x.tok0 + a.tokens);
            }
            ok = load(w);
            if (!ok) {                                       // copies in flight land before the block lets go of its memory
                note_timeout(a.status);
                for (int i = 0; i < kRing; ++i)
                    for (uint32_t ph = 0; ph < 2; ++ph)
                        mbar_wait_bounded(bar(W_KFULL + i), ph, 64u), mbar_wait_bounded(bar(W_VFULL + i), ph, 64u);
            }
            if (x.nt_a < 0) break;
        }
    } else if (warp == 9) {
        // ================= MMA issuer =================
        if (elect_one()) {
            constexpr uint32_t idesc_qk = idesc_i8(kQT, kWideKT);
            constexpr uint32_t idesc_pv = idesc_f16(kQT, D, true);
            int t0 = 0;                                      // key tiles of the pairs before
            uint32_t n_p[2] = {0u, 0u}, n_o[2] = {0u, 0u};   // softmax tiles and accumulators waited for
            // the next pair's sizes, its queries and its first keys: false when a wait gave up
            auto take = [&](int w, int first, int (&nt)[2]) -> bool {
                const int ws = w & 1;
                const uint32_t round = (uint32_t)(w >> 1) & 1u;
                if (!mbar_wait_spin_bounded(bar(W_WFULL + ws), round)) return false;
                nt[0] = work[ws].nt_a, nt[1] = work[ws].nt_b;
                mbar_arrive(bar(W_WEMPTY + ws));
                return nt[0] < 0 || (mbar_wait_spin_bounded(bar(W_QFULL + ws), round) &&
                                     mbar_wait_spin_bounded(bar(W_KFULL + first % kRing), (uint32_t)(first / kRing) & 1u));
            };
            auto qk = [&](int ws, int x, int t) {            // scores of tile x of pair slot ws against key tile t
                tc_fence_after();
                const uint32_t qa = base_s + Cfg::OFF_Q + (ws * 2 + x) * Cfg::Q_BYTES;
                const uint32_t ka = base_s + Cfg::OFF_K + (t % kRing) * Cfg::K_BYTES;
                const uint64_t da = D == 128 ? smem_desc_sw128(qa) : smem_desc_sw64(qa);
                const uint64_t db = D == 128 ? smem_desc_sw128(ka) : smem_desc_sw64(ka);
#pragma unroll
                for (int k = 0; k < D / 32; ++k) mma_i8(tmem_base + Cfg::TM_S + x * 128, da + 2 * k, db + 2 * k, idesc_qk, k != 0);
                tc_commit(bar(W_SFULL + x));
            };
            int cur[2] = {-1, -1}, then[2] = {-1, -1};       // key tiles of A and B, of this pair and of the next
            bool ok = take(0, 0, cur);
            if (ok && cur[0] > 0) {
                qk(0, 0, 0);
                if (cur[1] > 0) qk(0, 1, 0);
                tc_commit(bar(W_KEMPTY));
            }
            for (int w = 0; ok && cur[0] > 0; ++w) {
                const int ws = w & 1, nt = max(cur[0], cur[1]);
                // A's and B's turn at key tile j: P.V of j, then Q.K^T of j + 1 -- behind the last tile, of the next pair's
                // first -- into the scores' place
                for (int j = 0; j < nt; ++j) {
                    const bool last = j + 1 == nt;
                    const int kt = t0 + j + 1, vt = t0 + j;
                    ok = (last ? take(w + 1, kt, then) : mbar_wait_spin_bounded(bar(W_KFULL + kt % kRing), (uint32_t)(kt / kRing) & 1u)) &&
                         mbar_wait_spin_bounded(bar(W_VFULL + vt % kRing), (uint32_t)(vt / kRing) & 1u);
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        if (ok && j < cur[x]) {
                            ok = mbar_wait_spin_bounded(bar(W_PFULL + x), n_p[x] & 1u);
                            ++n_p[x];
                            if (ok && j == 0) {              // the accumulator of the pair before has been read
                                ok = mbar_wait_spin_bounded(bar(W_OEMPTY + x), (n_o[x] & 1u) ^ 1u);
                                ++n_o[x];
                            }
                            if (!ok) break;
                            tc_fence_after();
                            const uint64_t db0 = smem_desc_sw128_mn(base_s + Cfg::OFF_V + (vt % kRing) * Cfg::V_BYTES, Cfg::V_SLAB);
#pragma unroll
                            for (int i = 0; i < kWideKT / 16; ++i)
                                mma_f16_ta(tmem_base + Cfg::TM_O + x * D, tmem_base + Cfg::TM_S + x * 128 + i * 8, db0 + (uint64_t)(128 * i),
                                           idesc_pv, (j | i) != 0);
                            if (j + 1 == cur[x]) tc_commit(bar(W_ODONE + x));
                        }
                        if (ok && (last ? then[x] > 0 : j + 1 < cur[x])) qk(last ? ws ^ 1 : ws, x, kt);
                    }
                    if (!ok) break;
                    if (!last || then[0] > 0) tc_commit(bar(W_KEMPTY + kt % kRing));
                    tc_commit(bar(W_VEMPTY + vt % kRing));
                }
                if (!ok) break;
                tc_commit(bar(W_QEMPTY + ws));
                t0 += nt;
                cur[0] = then[0], cur[1] = then[1];
            }
            if (!ok) note_timeout(a.status);
        }
    }
    } else {
        // ================= softmax: a query row per thread =================
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        const int x = warp >> 2;                             // tile A or B
        const int r = (warp & 3) * 32 + lane;                // row of the tile; the warp's quarter of the lanes of tensor memory
        const uint32_t lane_addr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t s_addr = lane_addr + Cfg::TM_S + x * 128, o_addr = lane_addr + Cfg::TM_O + x * D;
        constexpr uint32_t kMagicI = 0x4B400000u;            // 1.5 * 2^23: |q.k| < 2^22 converts by an add and a subtract
        const f32x2 nmagic2 = pack2(-12582912.f, -12582912.f);
        bool ok = true;
        int t0 = 0;
        uint32_t n_s = 0u, n_o = 0u;                         // score blocks and accumulators waited for
        for (int w = 0; ok; ++w) {
            const int ws = w & 1;
            const uint32_t round = (uint32_t)(w >> 1) & 1u;
            ok = __all_sync(0xffffffffu, mbar_wait_spin_bounded(bar(W_WFULL + ws), round));
            if (!ok) break;
            const WideWork job = work[ws];
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(W_WEMPTY + ws));
            if (job.nt_a < 0) break;
            const int nt = max(job.nt_a, job.nt_b), mine = x == 0 ? job.nt_a : job.nt_b;
            const int first_tok = job.tok0 + x * a.tokens;
            const int tok = first_tok + r / a.group, head = job.hk * a.group + r % a.group;
            const bool stored = r < a.tokens * a.group && tok < job.len;
            float qscale = stored ? a.sQ[(long long)(job.start + tok) * a.sq_stride + head] * a.score_scale_log2 : 0.f;
            if (qscale == 0.f) qscale = 1e-30f;              // a removed position (-inf) stays removed under a scale of zero
            const f32x2 qs2 = pack2(qscale, qscale);
            const int visible = a.causal ? min(job.len, tok + 1) : job.len;             // positions that this row sees
            const int all_visible = a.causal ? first_tok + 1 : job.len;                 // that every row of the tile sees
            const int any_visible = a.causal ? min(job.len, first_tok + a.tokens) : job.len;   // that some row of it sees
            // the power of two that brings the largest value scale of the sequence to [2^6, 2^7), as an addend of the
            // exponent: it cancels against the sum of the probabilities
            float most = 0.f;
            const int top_slots = (any_visible + KT - 1) / KT;
            for (int j = lane; j < top_slots && mine > 0; j += 32) most = fmaxf(most, a.top[(long long)job.hk * a.slots + job.kv_slot + j]);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            const float lift = (float)min(100, max(-100, 6 - ((int)(__float_as_uint(most) >> 23) - 127)));

            float nm = 0.f;                                  // the row's reference (ScoreReference), or kFarMark: it is in far_refs
            float l = 0.f;
            for (int j = 0; j < nt; ++j) {
                const int cs = (t0 + j) % kScaleRing;
                ok = __all_sync(0xffffffffu, mbar_wait_spin_bounded(bar(W_CFULL + cs), (uint32_t)((t0 + j) / kScaleRing) & 1u));
                if (!ok) break;
                if (j < mine) {
                    ok = __all_sync(0xffffffffu, mbar_wait_spin_bounded(bar(W_SFULL + x), n_s & 1u));
                    if (!ok) break;
                    ++n_s;
                    tc_fence_after();
                    const float* sk = reinterpret_cast<const float*>(base + Cfg::OFF_SCALES) + cs * (2 * kWideKT);
                    const float* sv = sk + kWideKT;
                    const int lim = visible - j * kWideKT;               // columns of this tile that the row sees
                    const bool edge = (j + 1) * kWideKT > all_visible;   // (the same for the whole tile)
                    const int tile_lim = any_visible - j * kWideKT;      // columns that some row of the tile sees
                    // y = (q.k) * sK for 8 columns; columns the row does not see are removed, whatever was there
                    auto scores8 = [&](auto at_edge, const uint32_t* sr8, int c, f32x2* y4) {
                        const float4 ka = *reinterpret_cast<const float4*>(sk + c), kb = *reinterpret_cast<const float4*>(sk + c + 4);
                        const f32x2 t01 = add2(pack2(__uint_as_float(sr8[0] + kMagicI), __uint_as_float(sr8[1] + kMagicI)), nmagic2);
                        const f32x2 t23 = add2(pack2(__uint_as_float(sr8[2] + kMagicI), __uint_as_float(sr8[3] + kMagicI)), nmagic2);
                        const f32x2 t45 = add2(pack2(__uint_as_float(sr8[4] + kMagicI), __uint_as_float(sr8[5] + kMagicI)), nmagic2);
                        const f32x2 t67 = add2(pack2(__uint_as_float(sr8[6] + kMagicI), __uint_as_float(sr8[7] + kMagicI)), nmagic2);
                        y4[0] = mul2(t01, pack2(ka.x, ka.y));
                        y4[1] = mul2(t23, pack2(ka.z, ka.w));
                        y4[2] = mul2(t45, pack2(kb.x, kb.y));
                        y4[3] = mul2(t67, pack2(kb.z, kb.w));
                        if constexpr (decltype(at_edge)::value) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                if (c + 2 * e >= lim) y4[e].x = -INFINITY;
                                if (c + 2 * e + 1 >= lim) y4[e].y = -INFINITY;
                            }
                        }
                    };
                    if (j == 0) {                            // the first reference: largest of the first 32 scores
                        uint32_t sr[32];
                        float m0 = -INFINITY;
                        tmem_ld32(s_addr, sr);
                        tmem_ld_wait(sr);
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            f32x2 y4[4];
                            scores8(std::true_type{}, &sr[8 * g], 8 * g, y4);
#pragma unroll
                            for (int e = 0; e < 4; ++e) m0 = max3(m0, y4[e].x, y4[e].y);
                        }
                        nm = lift - m0 * qscale;
                        if (!(fabsf(nm) < kFarScore)) nm = kFarMark, far_refs[threadIdx.x] = ScoreReference{INFINITY, 0.f, false};
                    }
                    uint32_t P[64];
                    f32x2 sum2;
                    float mx;
                    auto pass = [&](auto at_edge, auto chunks) {         // of 16 columns; the others have no probability
                        constexpr int CHUNKS = decltype(chunks)::value;
                        const f32x2 nm2 = pack2(nm, nm);
                        sum2 = pack2(0.f, 0.f);
                        mx = -INFINITY;
                        uint32_t sr[2][16];
                        tmem_ld16(s_addr, sr[0]);
#pragma unroll
                        for (int c = 0; c < CHUNKS; ++c) {
                            tmem_ld_wait(sr[c & 1]);
                            if (c < CHUNKS - 1) tmem_ld16(s_addr + (c + 1) * 16, sr[(c + 1) & 1]);
#pragma unroll
                            for (int g = 0; g < 2; ++g) {
                                const int col = c * 16 + g * 8;
                                f32x2 y4[4];
                                scores8(at_edge, &sr[c & 1][8 * g], col, y4);
                                const float4 va = *reinterpret_cast<const float4*>(sv + col), vb = *reinterpret_cast<const float4*>(sv + col + 4);
                                const f32x2 x0 = fma2(y4[0], qs2, nm2), x1 = fma2(y4[1], qs2, nm2);
                                const f32x2 x2 = fma2(y4[2], qs2, nm2), x3 = fma2(y4[3], qs2, nm2);
                                mx = max3(max3(mx, x0.x, x0.y), max3(x1.x, x1.y, x2.x), fmaxf(x2.y, fmaxf(x3.x, x3.y)));
                                const f32x2 p0 = pack2(ex2_approx(x0.x), ex2_approx(x0.y)), p1 = pack2(ex2_approx(x1.x), ex2_approx(x1.y));
                                const f32x2 p2 = pack2(ex2_approx(x2.x), ex2_approx(x2.y)), p3 = pack2(ex2_approx(x3.x), ex2_approx(x3.y));
                                sum2 = add2(sum2, add2(add2(p0, p1), add2(p2, p3)));
                                const f32x2 s0 = mul2(p0, pack2(va.x, va.y)), s1 = mul2(p1, pack2(va.z, va.w));
                                const f32x2 s2 = mul2(p2, pack2(vb.x, vb.y)), s3 = mul2(p3, pack2(vb.z, vb.w));
                                P[col / 2] = pack_h2(s0.x, s0.y), P[col / 2 + 1] = pack_h2(s1.x, s1.y);
                                P[col / 2 + 2] = pack_h2(s2.x, s2.y), P[col / 2 + 3] = pack_h2(s3.x, s3.y);
                            }
                        }
#pragma unroll
                        for (int i = CHUNKS * 8; i < 64; ++i) P[i] = 0u;
                    };
                    int turn = 0;
#pragma unroll 1
                    for (;; turn = 1) {
                        // a last tile that no row sees the second half of costs half (sixteen prompts up to 2048, 32/8 heads:
                        // 304 -> 295 us; at head_dim 64 the third form does not fit the registers: 482 -> 507 us for eight
                        // sequences of 4096, 8 heads)
                        if (!edge) pass(std::false_type{}, std::integral_constant<int, 8>{});
                        else if (D == 64 || tile_lim > 64) pass(std::true_type{}, std::integral_constant<int, 8>{});
                        else pass(std::true_type{}, std::integral_constant<int, 4>{});
                        const bool ahead = mx > lift + kLazyStep;
                        if (turn | !__any_sync(0xffffffffu, ahead)) break;
                        // the reference moves to this tile's maximum, and the tile is done again, once; P.V of the tile before
                        // has retired (its commit came before that of these scores)
                        const float to = ahead ? nm - (mx - lift) : nm;
                        if (__any_sync(0xffffffffu, nm == kFarMark || fabsf(to) >= kFarScore)) {
                            const float2 r = far_tile<D>(s_addr, o_addr, sk, lim, qscale, lift, nm, l, j == 0, far_refs + threadIdx.x);
                            nm = r.x, l = r.y;
                            goto stored;
                        }
                        const float corr = ex2_approx(to - nm);
                        nm = to;
                        l *= corr;
                        if (j > 0) {
                            uint32_t o[32];
#pragma unroll 1
                            for (int cc = 0; cc < D / 32; ++cc) {
                                tmem_ld32(o_addr + cc * 32, o);
                                tmem_ld_wait(o);
#pragma unroll
                                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
                                tmem_st32(o_addr + cc * 32, o);
                            }
                        }
                    }
                    l += sum2.x + sum2.y;
                    tmem_st32(s_addr, *reinterpret_cast<uint32_t(*)[32]>(&P[0]));
                    tmem_st32(s_addr + 32, *reinterpret_cast<uint32_t(*)[32]>(&P[32]));
                stored:
                    tmem_st_wait();
                    tc_fence_before();
                }
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(bar(W_CEMPTY + cs));
                    if (j < mine) mbar_arrive(bar(W_PFULL + x));
                }
            }
            t0 += nt;
            // ---- epilogue: O / l -> fp16 ----
            if (ok && mine > 0) {
                ok = __all_sync(0xffffffffu, mbar_wait_spin_bounded(bar(W_ODONE + x), n_o & 1u));
                if (!ok) break;
                ++n_o;
                tc_fence_after();
                const float inv = 1.0f / l;
                __half* orow = a.out + ((long long)(job.start + tok) * a.heads + head) * D;
#pragma unroll 1
                for (int cc = 0; cc < D / 32; ++cc) {
                    uint32_t o[32];
                    tmem_ld32(o_addr + cc * 32, o);
                    tmem_ld_wait(o);
                    if (stored) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            *reinterpret_cast<uint4*>(orow + cc * 32 + k * 8) =
                                make_uint4(pack_h2(__uint_as_float(o[8 * k]) * inv, __uint_as_float(o[8 * k + 1]) * inv),
                                           pack_h2(__uint_as_float(o[8 * k + 2]) * inv, __uint_as_float(o[8 * k + 3]) * inv),
                                           pack_h2(__uint_as_float(o[8 * k + 4]) * inv, __uint_as_float(o[8 * k + 5]) * inv),
                                           pack_h2(__uint_as_float(o[8 * k + 6]) * inv, __uint_as_float(o[8 * k + 7]) * inv));
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(W_OEMPTY + x));
            }
        }
        if (!ok && lane == 0) note_timeout(a.status);
    }

    // common exit: every role ends here, then the allocating warp frees tensor memory
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
}

// ---- host ----------------------------------------------------------------------------------------------
// [rows][heads][D] bytes with `stride` bytes between rows: boxes of box_rows x box_heads x box_bytes
int encode_heads(CUtensorMap* map, const void* ptr, unsigned long long rows, unsigned heads, unsigned D, unsigned long long stride,
                 unsigned box_rows, unsigned box_heads, unsigned box_bytes, CUtensorMapSwizzle swizzle) {
    EncodeTiledFn fn = encode_fn();
    if (fn == nullptr) return -1;
    const cuuint64_t dims[3] = {D, heads, rows};
    const cuuint64_t strides[2] = {D, stride};
    const cuuint32_t box[3] = {box_bytes, box_heads, box_rows};
    const cuuint32_t estr[3] = {1, 1, 1};
    return (int)fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(ptr), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

struct VarLayout {
    int slots;
    size_t sk_off, sv_off, top_off, v_off, total;
};
VarLayout var_layout(long long T, long long B, int kv_heads, int D) {
    VarLayout y;
    y.slots = (int)(T / KT + B + 2);
    const size_t rows = (size_t)kv_heads * y.slots * KT;
    y.sk_off = 256;
    y.sv_off = y.sk_off + round_up(rows * 4, 256);
    y.top_off = y.sv_off + round_up(rows * 4, 256);
    y.v_off = y.top_off + round_up(rows / KT * 4, 256);
    y.total = y.v_off + round_up(rows * D * 2, 256);
    return y;
}
bool var_shape_ok(long long T, long long B, int heads, int kv_heads, int D) {
    if (T <= 0 || B <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || heads / kv_heads > 64 || (D != 64 && D != 128 && D != 256))
        return false;
    const int tokens = kQT / (heads / kv_heads);
    return T < (1ll << 30) && B < (1ll << 28) && kv_heads <= 65535 && (T / KT + B + 2) * kv_heads * KT < (1ll << 31) &&
           (T / tokens + B + 1) * kv_heads < (1ll << 31);
}

template <int D>
int launch_varlen(const int8_t* Q, long long q_stride, const int8_t* K, long long k_stride, const int8_t* V, long long v_stride,
                  const float* sK, long long sk_stride, const float* sV, long long sv_stride, Packed a, unsigned char* ws,
                  cudaStream_t st) {
    constexpr bool kWide = D <= 128;
    constexpr int KEYS = kWide ? kWideKT : KT;               // positions of a key tile
    constexpr int ROW = D < 128 ? D : 128;
    static int sms[64] = {0};
    int dev = 0;
    I8TK_CUDA(cudaGetDevice(&dev));
    I8TK_REQUIRE(dev >= 0 && dev < 64, I8TK_ERR_UNSUPPORTED, "device %d", dev);
    if (sms[dev] == 0) {
        int n = 0;
        I8TK_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
        if constexpr (kWide)
            I8TK_CUDA(cudaFuncSetAttribute(varlen_wide_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, WideCfg<D>::SMEM_BYTES));
        else
            I8TK_CUDA(cudaFuncSetAttribute(varlen_attention_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, VarCfg::SMEM_BYTES));
        sms[dev] = n;
    }
    const VarLayout y = var_layout(a.T, a.B, a.kv_heads, D);
    float* sKp = reinterpret_cast<float*>(ws + y.sk_off);
    float* sVp = reinterpret_cast<float*>(ws + y.sv_off);
    float* top = reinterpret_cast<float*>(ws + y.top_off);
    __half* V16 = reinterpret_cast<__half*>(ws + y.v_off);
    a.slots = y.slots;
    a.sK = sKp, a.sV = sVp, a.top = top;

    const CUtensorMapSwizzle sw = (D >= 128) ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    CUtensorMap tmQ, tmK, tmV;
    int rc = encode_heads(&tmQ, Q, a.T, a.heads, D, q_stride, a.tokens, a.group, ROW, sw);
    I8TK_REQUIRE(rc == 0, I8TK_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", rc);
    rc = encode_heads(&tmK, K, a.T, a.kv_heads, D, k_stride, KEYS, 1, ROW, sw);
    I8TK_REQUIRE(rc == 0, I8TK_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", rc);
    rc = encode_map_2d_u8(&tmV, V16, (unsigned long long)a.kv_heads * a.slots * KT, 2ull * D, KEYS, 128, CU_TENSOR_MAP_SWIZZLE_128B);
    I8TK_REQUIRE(rc == 0, I8TK_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", rc);

    I8TK_CUDA(launch_after(varlen_prepare_kernel<D>, dim3((unsigned)a.slots, (unsigned)a.kv_heads), dim3(128), 0, st, V, v_stride, sK,
                           sk_stride, sV, sv_stride, V16, sKp, sVp, top, a));
    if constexpr (kWide) {
        const long long items = (a.T / (2 * a.tokens) + a.B) * (long long)a.kv_heads;
        I8TK_CUDA(launch_after(varlen_wide_kernel<D>, dim3((unsigned)(items < sms[dev] ? items : sms[dev])), dim3(kWideThreads),
                               WideCfg<D>::SMEM_BYTES, st, tmQ, tmK, tmV, a));
    } else {
        const unsigned ctas = (unsigned)((a.T / a.tokens + a.B) * (long long)a.kv_heads);
        I8TK_CUDA(launch_after(varlen_attention_kernel, dim3(ctas), dim3(kThreads), VarCfg::SMEM_BYTES, st, tmQ, tmK, tmV, a));
    }
    return I8TK_OK;
}

}  // namespace
}  // namespace i8tk

using namespace i8tk;

extern "C" size_t i8tk_attention_varlen_workspace_bytes(int64_t tokens, int batch, int heads, int kv_heads, int head_dim) {
    if (!var_shape_ok(tokens, batch, heads, kv_heads, head_dim)) return 0;
    return var_layout(tokens, batch, kv_heads, head_dim).total;
}

extern "C" int i8tk_attention_varlen(const int8_t* Q, int64_t q_stride, const int8_t* K, int64_t k_stride, const int8_t* V,
                                     int64_t v_stride, const float* sQ, int64_t sq_stride, const float* sK, int64_t sk_stride,
                                     const float* sV, int64_t sv_stride, const int32_t* cu_seqlens, void* out_f16, int64_t tokens,
                                     int batch, int max_seqlen, int heads, int kv_heads, int head_dim, int causal, void* workspace,
                                     size_t workspace_bytes, i8tk_stream_t stream) {
    I8TK_REQUIRE(Q && K && V && sQ && sK && sV && cu_seqlens && out_f16, I8TK_ERR_INVALID_ARGUMENT, "null pointer argument");
    I8TK_REQUIRE(tokens > 0 && batch > 0 && max_seqlen > 0 && heads > 0 && kv_heads > 0, I8TK_ERR_INVALID_ARGUMENT, "sizes must be positive");
    I8TK_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, I8TK_ERR_UNSUPPORTED, "head_dim must be 64, 128 or 256 (got %d)",
                 head_dim);
    I8TK_REQUIRE(heads % kv_heads == 0 && heads / kv_heads <= 64, I8TK_ERR_UNSUPPORTED,
                 "heads must be a multiple of kv_heads, at most 64 times as many");
    I8TK_REQUIRE(var_shape_ok(tokens, batch, heads, kv_heads, head_dim), I8TK_ERR_UNSUPPORTED, "shape too large");
    const int64_t qrow = (int64_t)heads * head_dim, krow = (int64_t)kv_heads * head_dim;
    I8TK_REQUIRE(q_stride >= qrow && k_stride >= krow && v_stride >= krow && q_stride % 16 == 0 && k_stride % 16 == 0 && v_stride % 16 == 0 &&
                     q_stride < (1ll << 39) && k_stride < (1ll << 39) && v_stride < (1ll << 39),
                 I8TK_ERR_INVALID_ARGUMENT, "token strides must cover a token's heads and be multiples of 16");
    I8TK_REQUIRE(sq_stride >= heads && sk_stride >= kv_heads && sv_stride >= kv_heads, I8TK_ERR_INVALID_ARGUMENT,
                 "scale strides must cover a token's heads");
    I8TK_REQUIRE(aligned_to(Q, 16) && aligned_to(K, 16) && aligned_to(V, 16) && aligned_to(out_f16, 16), I8TK_ERR_ALIGNMENT,
                 "Q, K, V and out must be 16-byte aligned");
    const VarLayout y = var_layout(tokens, batch, kv_heads, head_dim);
    I8TK_REQUIRE(workspace != nullptr && workspace_bytes >= y.total, I8TK_ERR_WORKSPACE,
                 "attention workspace too small: need %zu bytes, got %zu", y.total, workspace_bytes);
    I8TK_REQUIRE(aligned_to(workspace, 256), I8TK_ERR_ALIGNMENT, "workspace must be 256-byte aligned");
    const int group = heads / kv_heads;
    Packed a{cu_seqlens, batch, (int)tokens, max_seqlen, causal ? 1 : 0, heads, kv_heads, group, kQT / group, 0, sQ, sq_stride,
             nullptr, nullptr, nullptr, static_cast<__half*>(out_f16), 1.4426950408889634f / sqrtf((float)head_dim),
             static_cast<uint32_t*>(workspace), static_cast<uint32_t*>(workspace) + 2};
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (head_dim == 64) return launch_varlen<64>(Q, q_stride, K, k_stride, V, v_stride, sK, sk_stride, sV, sv_stride, a, ws, st);
    if (head_dim == 128) return launch_varlen<128>(Q, q_stride, K, k_stride, V, v_stride, sK, sk_stride, sV, sv_stride, a, ws, st);
    return launch_varlen<256>(Q, q_stride, K, k_stride, V, v_stride, sK, sk_stride, sV, sv_stride, a, ws, st);
}
