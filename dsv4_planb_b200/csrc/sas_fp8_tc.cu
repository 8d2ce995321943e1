// sm_100a tensor-core attention over the 8-bit cache: bf16 queries, D_qk 512 or 576, D_v 512, up to
// 128 heads.
//
// The keys stay e4m3 from HBM to the MMA (kind::f8f6f4).  What multiplies them is split exactly into
// two e4m3 terms: a bf16 value has 8 significant bits, and x = hi + lo with hi = e4m3(x) leaves a lo
// of 4 bits.  Queries are scaled per row by a power of two that brings the largest element to
// [128, 256): elements down to 2^-10 of it split without error, smaller ones are off by at most 2^-10
// (2^-17 of the largest).  Softmax weights, at most 431 by their scale, lose 2^-9 relative (bf16 would
// lose 2^-8) and 2^-10 where lo is subnormal.  So one product costs two e4m3 MMAs, which is the time
// of one bf16 MMA, at half the bytes gathered.
//
// A key's scale s_j multiplies its score and its value.  With t_ij = scale q_i k_j in log2 units, the
// weight of value row j (its codes) is 2^(t_ij) s_j, so the running maximum is taken over
// x_ij = t_ij + log2 s_j, P_ij = 2^(x_ij - m_i + 5.75) goes to the MMA, and the softmax's denominator
// adds P_ij / s_j.  The sink joins at the end.
//
// A unit of work (a token, or a piece of one) goes to a cluster of two CTAs on two SMs that split it
// by role, because O alone (128 heads x 512 fp32) fills one SM's tensor memory:
//
//   CTA 0 ("score")                              CTA 1 ("output")
//   TMEM: Q hi / lo of 512 dims (256 columns),   TMEM: O (128 x 512 fp32)
//         S (2 x 128 columns); the Q of dims
//         512 .. 575 lies in shared memory
//   4 warps gather 128 key rows per tile (TMA    4 warps gather the first 512 bytes of the rows
//           tile::gather4, 128-byte swizzle)
//   1 warp  S = Q K^T: 2 MMAs (hi, lo) of M 128, 1 warp  O += P V: 2 (hi, lo) per 32 keys and 128
//           N 128, K 32 per 32 dims                      value dims; V is the N-major B operand, the
//                                                        same bytes in the same swizzle as K
//   8 warps split Q; softmax (two threads per    8 warps rescale O where a maximum rose; epilogue
//           head, 64 keys each); P and factors
//           go to CTA 1 (st.async)
//
// Tiles hold 128 keys because an MMA of N 64 takes nearly as long as one of N 128 (58 and 70 cycles).
// The ring of the gather holds slabs (128 rows x 128 dims), each released as soon as its MMAs have
// read it.  The maximum follows a rise of more than 2^3 only (P <= 2^8.75, the e4m3 range): with 128
// heads some maximum rises in nearly every tile, and a rescale of O (512 columns read and written)
// takes longer than the tile's MMAs.  The largest weight is then at least 2^5.75, and the 2^-10 that a
// weight can be off by where its lo is subnormal are 2^-15.75 of it.  The softmax reads S twice from TMEM in short loops: unrolled
// over 64 keys it was bound by instruction fetch (3.7 times the cycles of the same code alone).
//
// Keys of a token: first positions, then the window, padded to a multiple of 4, then the compressed
// rows, so that the four rows of one gather come from one pool.  Slots without a key carry weight 0
// (log2 s = -inf); rows of unmapped blocks are gathered from one past the pool, which reads zeros.
//
// Every wait is bounded (sas_tc_sync.cuh): a timeout sets SAS_STATUS_WAIT_TIMEOUT and every role falls
// through to the teardown, which frees TMEM after a cluster barrier.

#include <cuda.h>

#include <algorithm>
#include <atomic>

#include "sas_fp8_attn.cuh"
#include "sas_tc_ptx.cuh"
#include "sas_tc_sync.cuh"

namespace {

using namespace sas_ptx;
using namespace sas_tc;
using namespace sas_fp8;

constexpr int kBK = 128;             // keys per tile
constexpr int kUnit = kBK * 128;     // ring unit: 128 dims of a tile's rows, or 64 bf16 dims of 128 query rows
constexpr int kKUnits = 12, kVUnits = 7, kPStages = 2;
constexpr int kDv = 512, kVSlabs = kDv / 128, kQChunks = 8;
constexpr int kSoftWarps = 8, kMmaWarp = 8, kProdWarp0 = 9, kProdWarps = 4;
constexpr int kThreads = 32 * (kProdWarp0 + kProdWarps);
constexpr uint32_t kReaders = 2 * (kSoftWarps + 1 + kProdWarps) - 1;  // of the unit queue: every warp but its writer
constexpr int kTmemCols = 512, kTmemS = 256;
constexpr int kConsts = 8;           // ring of per-tile key constants; the gather is at most 5 tiles ahead
constexpr float kTop = 8.75f;        // log2 of the largest P: 431, within e4m3's 448
constexpr float kRise = 3.f;         // log2 of the rise of a maximum that is left to P
constexpr int kMaxPieces = 64;

// P message: per head 128 hi codes (a 128-byte row, SW128), then the lo codes the same way, then alpha
// and the unit's final factor per head.
constexpr int kMsgLo = 128 * 128, kMsgStats = 2 * kMsgLo, kMsgBytes = kMsgStats + 1024;
constexpr uint32_t kMsgTx = 128 * (256 + 8);

struct KeyConst {
    float s[kBK];   // scale; 0: a zero row or no key
    float ls[kBK];  // log2 s; -60 for zero rows (their values do not count), -inf: no key
    float r[kBK];   // 1 / s (2^60 for zero rows, 0: no key)
};

struct Hdr {
    uint64_t full[kKUnits], empty[kKUnits], s_full[2], s_free[2], q_raw, q_full, p_empty[kPStages], c_full[kConsts];
    uint64_t p_full[kPStages], o_full, o_empty, rs_req, rs_done, pv_done, fin_ready;
    uint64_t tq_full[kTq], tq_empty[kTq];
    volatile int tq[kTq];
    uint32_t tmem_base;
    volatile int abort;
    int rs_stage;
    float fin[128];       // per head: factor of O at the end of the unit
    float pair[2][2][128];  // what the two threads of a head tell each other, two exchanges
};
constexpr int kHdr = 4 * 1024;
static_assert(sizeof(Hdr) <= kHdr && kVUnits <= kKUnits, "header");
constexpr int kConstOff = kHdr;
constexpr int kQRope = kConstOff + kConsts * (int)sizeof(KeyConst);  // [128 rows][64 hi | 64 lo codes], SW128
constexpr int kScoreRing = kQRope + 128 * 128;
constexpr int kScoreSmem = kScoreRing + kKUnits * kUnit;
constexpr int kOutRing = kHdr;
constexpr int kOutMsgs = kOutRing + kVUnits * kUnit;
constexpr int kOutStage = kOutMsgs + kPStages * kMsgBytes;  // epilogue staging: 64 columns of 32 heads per warp
constexpr int kWarpSlab = 32 * 128;
constexpr int kOutSmem = kOutStage + kSoftWarps * kWarpSlab;
constexpr int kSmemBytes = (kScoreSmem > kOutSmem ? kScoreSmem : kOutSmem) + 1024;  // + alignment slack
static_assert(kQRope % 1024 == 0 && kScoreRing % 1024 == 0 && kOutRing % 1024 == 0 && kOutMsgs % 1024 == 0 &&
              kMsgBytes % 1024 == 0 && kOutStage % 1024 == 0, "128B-swizzled tiles are 1 KiB aligned");
static_assert(kSmemBytes <= 232448, "shared memory");

struct TcArgs : Args {
    uint32_t *status;
    int ori_rows, cmp_rows;  // rows of each pool: the index one past the end reads zeros
    int U, P, M;             // units; pieces per token, tiles per piece (P = 1: whole tokens)
    float *part_o, *part_s;
};

__device__ __forceinline__ void mma8_ts(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n\t}" ::"r"(d),
        "r"(a_tmem), "l"(b), "r"(idesc), "r"(acc), "r"(0u), "r"(0u), "r"(0u), "r"(0u)
        : "memory");
}
__device__ __forceinline__ void mma8_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0u), "r"(0u), "r"(0u), "r"(0u)
        : "memory");
}
// Instruction descriptor of kind::f8f6f4, both operands e4m3 (format 0), fp32 accumulation; b_mn: B is
// N-major.
__host__ __device__ constexpr uint32_t idesc_e4m3(uint32_t m, uint32_t n, uint32_t b_mn) {
    return (1u << 4) | (b_mn << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
__device__ __forceinline__ void st_async_v2(uint32_t addr, uint32_t a, uint32_t b, uint32_t cluster_bar) {
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];" ::"r"(addr), "r"(a),
                 "r"(b), "r"(cluster_bar)
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

struct Item {
    int32_t rec[TR_INTS];
    int t, piece, np, n4, ntiles, j0, j1;  // tiles [j0, j1) of token t; slots below n4 belong to the window's pool
    bool skip;                             // a piece past the token's last tile
};

__device__ __forceinline__ Item load_unit(const TcArgs &p, int u) {
    Item it;
    it.piece = u / p.T;
    it.t = u - it.piece * p.T;
    const int4 *r = reinterpret_cast<const int4 *>(p.rec + (int64_t)it.t * TR_INTS);
    const int4 a = r[0], b = r[1];
    it.rec[TR_B] = a.x;
    it.rec[TR_LEFT] = a.y;
    it.rec[TR_FIRST] = a.z;
    it.rec[TR_NORI] = a.w;
    it.rec[TR_NCMP] = b.x;
    it.rec[TR_VALID] = b.y;
    it.n4 = (a.w + 3) & ~3;
    it.ntiles = b.y && a.w + b.x > 0 ? (it.n4 + b.x + kBK - 1) / kBK : 0;
    it.np = p.P > 1 && it.ntiles > p.M ? min((it.ntiles + p.M - 1) / p.M, p.P) : 1;
    it.skip = it.piece >= it.np;
    it.j0 = it.np > 1 ? it.piece * p.M : 0;
    it.j1 = it.np > 1 && it.piece < it.np - 1 ? it.j0 + p.M : it.ntiles;  // the last piece takes the rest
    return it;
}

// Row lookup of key slot i in three steps, each a tile ahead of the next so that their loads hide
// behind the copies: the table entry (or the resolved row), the physical row, its block's scale.
__device__ __forceinline__ int32_t key_fetch(const TcArgs &p, const Item &it, int i) {
    const int32_t *table = p.ori_bt;
    int slot = i, bs = p.ori_bs, len = p.ori_table_len;
    if (i < it.n4) {
        if (i >= it.rec[TR_NORI]) return -1;
        slot = ori_position(it.rec, i);
    } else {
        slot = i - it.n4;
        if (slot >= it.rec[TR_NCMP]) return -1;
        if (p.scenario == 3) return __ldg(p.rows + (int64_t)it.t * p.K + slot);
        table = p.cmp_bt, bs = p.cmp_bs, len = p.cmp_table_len;
    }
    const int blk = slot / bs;
    return blk < len ? __ldg(table + (int64_t)it.rec[TR_B] * len + blk) : -2;
}

struct Key {
    int32_t row;  // physical row, or -1: zeros
    float s;      // its block's scale (loaded), 1 without a row
    bool live;    // the slot holds a key
};

__device__ __forceinline__ Key key_row(const TcArgs &p, const Item &it, int i, int32_t fetched, uint32_t &bits) {
    Key key{-1, 1.f, false};
    const bool win = i < it.n4;
    const int slot = win ? i : i - it.n4;
    key.live = slot < (win ? it.rec[TR_NORI] : it.rec[TR_NCMP]);
    if (!key.live) return key;
    const int bs = win ? p.ori_bs : p.cmp_bs;
    int blk = fetched;
    if (!win && p.scenario == 3) {
        if (fetched < 0) return key;
        key.row = fetched;
        blk = fetched / bs;
    } else {
        if (fetched < -1 || fetched >= (win ? p.ori_block_num : p.cmp_block_num)) bits |= SAS_STATUS_BAD_BLOCK;
        else if (fetched >= 0) key.row = fetched * bs + (win ? ori_position(it.rec, slot) : slot) % bs;
        if (key.row < 0) return key;
    }
    key.s = __ldg((win ? p.ori_scale : p.cmp_scale) + blk);
    return key;
}

// The gather warps.  Each takes 32 of a tile's 128 key slots (a lane per slot) and copies its rows slab
// by slab with TMA tile::gather4 (4 rows x 128 bytes): row r of a unit at r * 128, its 16-byte granules
// permuted by r % 8, the MMA's 128-byte swizzle.  The slab behind D_qk 512 reads 64 bytes past the
// row's end as zeros.  A unit's full barrier counts the four warps, each of which announces its own
// 4 KiB first.  The warps share nothing else.
template <bool kScore>
__device__ void producer(const TcArgs &p, const Sync &sy, const CUtensorMap *ori_map, const CUtensorMap *cmp_map,
                         const CUtensorMap *q_map, uint8_t *ring, Hdr *hd, KeyConst *consts) {
    constexpr uint32_t kUnits = kScore ? kKUnits : kVUnits;
    const int w = (threadIdx.x >> 5) - kProdWarp0, lane = threadIdx.x & 31, key_at = w * 32 + lane;
    const int slabs = kScore ? (p.Dq + 127) / 128 : kVSlabs;
    const bool writer = kScore && w == 0;
    const uint32_t dst0 = smem_u32(ring) + w * 4096;
    uint32_t at = 0, phase = 1, tiles = 0, bits = 0;  // unit of the ring, and the parity its empty barrier is waited on
    int pend = -1;
    auto next = [&] {
        if (++at == kUnits) {
            at = 0;
            phase ^= 1;
        }
    };
    for (uint32_t k = 0;; ++k) {
        int u = -1;
        if (!(writer ? tq_publish(p, sy, k, pend, u) : tq_read(p, sy, kScore ? 0 : 1, k, u))) return;
        if (u < 0) break;
        const Item it = load_unit(p, u);
        if (it.skip || it.j1 <= it.j0) continue;
        const int end = it.j1 * kBK;
        int i = it.j0 * kBK + key_at;
        const int32_t f0 = key_fetch(p, it, i);
        int32_t fetched = i + kBK < end ? key_fetch(p, it, i + kBK) : -1;
        Key key = key_row(p, it, i, f0, bits);
        if constexpr (kScore) {
            // raw Q of the token, 64 of its first 512 dims per unit: this warp's 32 head rows
            for (int c = 0; c < kQChunks; ++c, next()) {
                if (!wait_warp(sy, smem_u32(&hd->empty[at]), phase)) return;
                if (lane == 0) {
                    const uint32_t fb = smem_u32(&hd->full[at]);
                    if (w * 32 < p.N1) {
                        mbar_arrive_expect_tx(fb, 4096);
                        tma_load_2d(dst0 + at * kUnit, q_map, c * 64, it.t * p.N1 + w * 32, fb);
                    } else {
                        mbar_arrive(fb);  // rows of no head: whatever lies there
                    }
                }
            }
        }
        for (int j = it.j0; j < it.j1; ++j, i += kBK, ++tiles) {
            if (key.row >= 0 && !scale_ok(key.s)) {
                bits |= SAS_STATUS_BAD_SCALE;
                key.row = -1;
            }
            if constexpr (kScore) {
                KeyConst &c = consts[tiles % kConsts];
                const bool row = key.row >= 0;
                c.s[key_at] = row ? key.s : 0.f;
                c.ls[key_at] = row ? log2f(key.s) : key.live ? -60.f : -INFINITY;
                c.r[key_at] = row ? 1.f / key.s : key.live ? kScaleMax : 0.f;
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(smem_u32(&hd->c_full[tiles % kConsts]));
                    if (writer && j == (it.j1 - it.j0 > 1 ? it.j1 - 2 : it.j0))
                        pend = (int)ncluster_x() + atomicAdd(p.counter, 1);
                }
            }
            // lane q < 8 copies the rows of lanes 4 q .. 4 q + 3
            const bool win = j * kBK + w * 32 + (lane & 7) * 4 < it.n4;
            const CUtensorMap *map = win ? ori_map : cmp_map;
            const int32_t oob = win ? p.ori_rows : p.cmp_rows;
            int32_t r[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int32_t v = __shfl_sync(0xffffffffu, key.row, (lane & 7) * 4 + e);
                r[e] = v >= 0 ? v : oob;
            }
            const int32_t f = fetched;
            for (int c = 0; c < slabs; ++c, next()) {
                if (!wait_warp(sy, smem_u32(&hd->empty[at]), phase)) return;
                const uint32_t fb = smem_u32(&hd->full[at]);
                if (lane == 0) mbar_arrive_expect_tx(fb, 4096);
                __syncwarp();
                if (lane < 8) tma_gather4(dst0 + at * kUnit + lane * 512, map, c * 128, r[0], r[1], r[2], r[3], fb);
                if (c == 0) {  // the next tile's lookups, behind the copies
                    key = Key{-1, 1.f, false};
                    if (i + kBK < end) key = key_row(p, it, i + kBK, f, bits);
                    fetched = i + 2 * kBK < end ? key_fetch(p, it, i + 2 * kBK) : -1;
                }
            }
        }
    }
    if (bits) sas::set_status(p.status, bits);
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}

// Two fp32 values (at most 448) as two pairs of e4m3 codes, hi + lo.  fp16 holds hi and the difference
// exactly; the value itself is first rounded to fp16 (2^-12 relative).
__device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
    const __half2 x = __floats2half2_rn(a, b);
    uint16_t h, l;
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(h) : "r"(*reinterpret_cast<const uint32_t *>(&x)));
    const uint32_t back = e4m3x2_to_half2(h);
    const __half2 d = __hsub2(x, *reinterpret_cast<const __half2 *>(&back));
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(l) : "r"(*reinterpret_cast<const uint32_t *>(&d)));
    hi = h;
    lo = l;
}

// What the other thread of a head says (x: what this one says).  Exchanges alternate between two
// buffers, so one barrier of the two warps each is enough: a buffer is written again only past the
// next exchange's barrier, which the partner reaches after it has read.
__device__ __forceinline__ float exchange(float (*pair)[2][128], uint32_t &n, float x) {
    const int g = threadIdx.x >> 7, h = threadIdx.x & 127;
    float (*buf)[128] = pair[n++ & 1];
    buf[g][h] = x;
    asm volatile("bar.sync %0, 64;" ::"r"(1 + (h >> 5)) : "memory");
    return buf[g ^ 1][h];
}

__device__ __forceinline__ void note_max(uint32_t v, float &amax, bool &odd) {
    const float2 f = sas::DT<__nv_bfloat16>::to_f2(v);
    amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
    odd |= f.x - f.x != 0.f || f.y - f.y != 0.f;
}

__device__ __forceinline__ void split4(uint32_t a, uint32_t b, float f, uint32_t &hi, uint32_t &lo) {
    const float2 x = sas::DT<__nv_bfloat16>::to_f2(a), y = sas::DT<__nv_bfloat16>::to_f2(b);
    uint32_t h0, l0, h1, l1;
    split2(x.x * f, x.y * f, h0, l0);
    split2(y.x * f, y.y * f, h1, l1);
    hi = h0 | (h1 << 16);
    lo = l0 | (l1 << 16);
}

// Q of head row h into hi and lo codes.  Dims below 512, raw bf16 in TMEM columns [0, 256): chunk c of
// 64 dims keeps its 32 columns, hi codes in the first 16 and lo codes in the last 16.  Dims 512 .. 575
// (rope, this thread's 32 of them) go to shared memory.  The row's two threads take half each and
// agree on the largest element.  Returns the row's power-of-two factor f (q f = hi + lo), NaN for a row
// that holds an infinity or NaN.
__device__ float split_q(uint32_t trow, int warp, int h, const uint4 *rope, uint32_t rope_row, float (*pair)[2][128],
                         uint32_t &xc) {
    const int g = warp >> 2;
    uint32_t rp[16];
    if (rope) {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const uint4 x = __ldg(rope + g * 4 + v);
            rp[4 * v] = x.x, rp[4 * v + 1] = x.y, rp[4 * v + 2] = x.z, rp[4 * v + 3] = x.w;
        }
    }
    float amax = 0.f;
    bool odd = false;
#pragma unroll 1
    for (int c = 4 * g; c < 4 * g + 4; ++c) {
        uint32_t r[32];
        tmem_ld32(trow + c * 32, r);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) note_max(r[i], amax, odd);
    }
    if (rope) {
#pragma unroll
        for (int i = 0; i < 16; ++i) note_max(rp[i], amax, odd);
    }
    if (odd) amax = INFINITY;
    amax = fmaxf(amax, exchange(pair, xc, amax));
    // largest element to [128, 256); rows of zeros and of the smallest subnormals: f = 2^126
    const int e = (int)(__float_as_uint(amax) >> 23) - 127;
    const float f = amax == INFINITY ? NAN : __uint_as_float((uint32_t)(min(126, 7 - e) + 127) << 23);
#pragma unroll 1
    for (int c = 4 * g; c < 4 * g + 4; ++c) {
        uint32_t r[32], hi[16], lo[16];
        tmem_ld32(trow + c * 32, r);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) split4(r[2 * i], r[2 * i + 1], f, hi[i], lo[i]);
        tmem_st16(trow + c * 32, hi);
        tmem_st16(trow + c * 32 + 16, lo);
    }
    if (rope) {
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) split4(rp[2 * i], rp[2 * i + 1], f, hi[i], lo[i]);
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            st_shared_v4(rope_row + (((2 * g + v) ^ (h & 7)) << 4), hi[4 * v], hi[4 * v + 1], hi[4 * v + 2], hi[4 * v + 3]);
            st_shared_v4(rope_row + (((4 + 2 * g + v) ^ (h & 7)) << 4), lo[4 * v], lo[4 * v + 1], lo[4 * v + 2], lo[4 * v + 3]);
        }
        fence_proxy_async_smem();
    }
    tc_wait_st();
    return f;
}

__global__ void __launch_bounds__(kThreads, 1)
    fp8_tc_kernel(const TcArgs p, const __grid_constant__ CUtensorMap ori_map, const __grid_constant__ CUtensorMap cmp_map,
                  const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap out_map) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    Hdr *hd = reinterpret_cast<Hdr *>(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();

    if (threadIdx.x == 0) {
        auto init = [](uint64_t *b, int n, uint32_t count) {
            for (int i = 0; i < n; ++i) mbar_init(smem_u32(b + i), count);
        };
        init(hd->full, kKUnits, kProdWarps);
        init(hd->empty, kKUnits, 1);
        init(hd->s_full, 2, 1);
        init(hd->s_free, 2, kSoftWarps);
        init(&hd->q_raw, 1, 1);
        init(&hd->q_full, 1, kSoftWarps);
        init(hd->p_empty, kPStages, 1);
        init(hd->c_full, kConsts, kProdWarps);
        init(hd->p_full, kPStages, 1);
        init(&hd->o_full, 1, 1);
        init(&hd->o_empty, 1, kSoftWarps);
        init(&hd->rs_req, 1, 1);
        init(&hd->rs_done, 1, kSoftWarps);
        init(&hd->pv_done, 1, 1);
        init(&hd->fin_ready, 1, 1);
        init(hd->tq_full, kTq, 1);
        init(hd->tq_empty, kTq, kReaders);
        hd->abort = 0;
        hd->rs_stage = 0;
        // the output CTA expects the first message of each P stage (st.async complete_tx)
        if (rank == 1)
            for (int i = 0; i < kPStages; ++i) mbar_arrive_expect_tx(smem_u32(&hd->p_full[i]), kMsgTx);
        mbar_fence_init();
    }
    if (warp == kMmaWarp) {
        tmem_alloc(smem_u32(&hd->tmem_base), kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // both CTAs' barriers are initialised before any remote arrive
    tc_fence_after();
    // a programmatic dependent of the resolve kernel: its records are visible after this wait
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (p.P > 1) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t tmem = hd->tmem_base;
    Sync sy{&hd->abort, p.status, map_to_cta(smem_u32((const void *)&hd->abort), rank ^ 1u), hd->tq_full, hd->tq_empty,
            hd->tq};

    if (rank == 0) {
        // ======================= score CTA =======================
        uint8_t *ring = smem + kScoreRing;
        KeyConst *consts = reinterpret_cast<KeyConst *>(smem + kConstOff);
        if (warp >= kProdWarp0) {
            producer<true>(p, sy, &ori_map, &cmp_map, &q_map, ring, hd, consts);
        } else if (warp == kMmaWarp) {
            constexpr uint32_t idesc = idesc_e4m3(128, kBK, 0);
            const int slabs = (p.Dq + 127) / 128;
            uint32_t at = 0, phase = 0, sc = 0, qc = 0;
            auto next = [&] {
                if (++at == kKUnits) {
                    at = 0;
                    phase ^= 1;
                }
            };
            for (uint32_t k = 0;; ++k) {
                int u;
                if (!tq_read(p, sy, rank, k, u)) goto done;
                if (u < 0) break;
                const Item it = load_unit(p, u);
                if (it.skip || it.j1 <= it.j0) continue;
                // raw Q -> TMEM, once the previous unit's last product has read the old one
                if (sc > 0 && !wait_warp(sy, smem_u32(&hd->s_full[(sc - 1) & 1]), ((sc - 1) >> 1) & 1)) goto done;
                for (int c = 0; c < kQChunks; ++c, next()) {
                    if (!wait_warp(sy, smem_u32(&hd->full[at]), phase)) goto done;
                    tc_fence_after();
                    if (lane == 0) {
                        const uint64_t d = sdesc_sw128(smem_u32(ring) + at * kUnit, 16, 1024);
                        for (int kq = 0; kq < 4; ++kq) tmem_cp_128x256b(tmem + (c * 4 + kq) * 8, d + 2 * kq);
                        tc_commit(smem_u32(&hd->empty[at]));
                        if (c == kQChunks - 1) tc_commit(smem_u32(&hd->q_raw));
                    }
                    __syncwarp();
                }
                if (!wait_warp(sy, smem_u32(&hd->q_full), qc & 1)) goto done;
                ++qc;
                for (int j = it.j0; j < it.j1; ++j, ++sc) {
                    const int sb = sc & 1;
                    const uint32_t d = tmem + kTmemS + sb * kBK;
                    if (!wait_warp(sy, smem_u32(&hd->s_free[sb]), ((sc >> 1) & 1) ^ 1)) goto done;
                    for (int c = 0; c < slabs; ++c, next()) {
                        if (!wait_warp(sy, smem_u32(&hd->full[at]), phase)) goto done;
                        tc_fence_after();
                        if (lane == 0) {
                            const uint64_t b = sdesc_sw128(smem_u32(ring) + at * kUnit, 16, 1024);
                            if (c < kQChunks / 2) {
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const uint32_t a = tmem + c * 64 + (i >> 1) * 32 + (i & 1) * 8;
                                    mma8_ts(d, a, b + 2 * i, idesc, c + i > 0 ? 1u : 0u);
                                    mma8_ts(d, a + 16, b + 2 * i, idesc, 1u);
                                }
                            } else {
                                const uint64_t a = sdesc_sw128(smem_u32(smem + kQRope), 16, 1024);
#pragma unroll
                                for (int i = 0; i < 2; ++i) {
                                    mma8_ss(d, a + 2 * i, b + 2 * i, idesc, 1u);
                                    mma8_ss(d, a + 4 + 2 * i, b + 2 * i, idesc, 1u);
                                }
                            }
                            tc_commit(smem_u32(&hd->empty[at]));
                            if (c == slabs - 1) tc_commit(smem_u32(&hd->s_full[sb]));
                        }
                        __syncwarp();
                    }
                }
            }
        } else {
            const int g = warp >> 2, h = threadIdx.x & 127;  // head row, and which half of the keys
            const bool head = h < p.N1;
            const uint32_t trow = tmem + ((uint32_t)((warp & 3) * 32) << 16);
            const uint32_t msg0 = map_to_cta(smem_u32(smem + kOutMsgs), 1);
            const uint32_t pfull0 = map_to_cta(smem_u32(&hd->p_full[0]), 1);
            const float sink = head && p.sinks ? p.sinks[h] : -INFINITY;
            uint32_t sc = 0, qc = 0, xc = 0;
            for (uint32_t k = 0;; ++k) {
                int u;
                if (!tq_read(p, sy, rank, k, u)) goto done;
                if (u < 0) break;
                const Item it = load_unit(p, u);
                if (it.skip) continue;
                if (it.ntiles == 0) {
                    if (p.lse && head && g == 0) p.lse[(int64_t)it.t * p.N1 + h] = it.rec[TR_VALID] ? sink : 0.f;
                    continue;
                }
                if (!wait_warp(sy, smem_u32(&hd->q_raw), qc & 1)) goto done;
                ++qc;
                tc_fence_after();
                const uint4 *rope = reinterpret_cast<const uint4 *>(
                    reinterpret_cast<const uint16_t *>(p.q) + ((int64_t)it.t * p.N1 + (head ? h : 0)) * p.Dq + 512);
                const float rq = p.scale_log2 / split_q(trow, warp, h, p.Dq > 512 ? rope : nullptr,
                                                        smem_u32(smem + kQRope) + h * 128, hd->pair, xc);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&hd->q_full));
                float m = -INFINITY, l = 0.f;  // l: of this thread's keys
                for (int j = it.j0; j < it.j1; ++j, ++sc) {
                    const int sb = sc & 1;
                    if (!wait_warp(sy, smem_u32(&hd->c_full[sc % kConsts]), (sc / kConsts) & 1)) goto done;
                    if (!wait_warp(sy, smem_u32(&hd->s_full[sb]), (sc >> 1) & 1)) goto done;
                    tc_fence_after();
                    const uint32_t s_at = trow + kTmemS + sb * kBK + g * 64;
                    const KeyConst &c = consts[sc % kConsts];
                    float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
                    for (int i0 = 0; i0 < 64; i0 += 32) {
                        uint32_t sr[32];
                        tmem_ld32(s_at + i0, sr);
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const float4 s4 = *reinterpret_cast<const float4 *>(&c.s[g * 64 + i0 + i]);
                            const float4 l4 = *reinterpret_cast<const float4 *>(&c.ls[g * 64 + i0 + i]);
                            mx4[0] = fmaxf(mx4[0], fmaf(__uint_as_float(sr[i]) * rq, s4.x, l4.x));
                            mx4[1] = fmaxf(mx4[1], fmaf(__uint_as_float(sr[i + 1]) * rq, s4.y, l4.y));
                            mx4[2] = fmaxf(mx4[2], fmaf(__uint_as_float(sr[i + 2]) * rq, s4.z, l4.z));
                            mx4[3] = fmaxf(mx4[3], fmaf(__uint_as_float(sr[i + 3]) * rq, s4.w, l4.w));
                        }
                    }
                    float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
                    mx = fmaxf(mx, exchange(hd->pair, xc, mx));
                    float alpha = 1.f;
                    if (j == it.j0) {
                        m = mx;
                    } else if (mx > m + kRise) {
                        alpha = exp2f(m - mx);
                        l *= alpha;
                        m = mx;
                    }
                    const float mb = m - (kTop - kRise);
                    const int ps = sc % kPStages;
                    if (!wait_warp(sy, smem_u32(&hd->p_empty[ps]), ((sc / kPStages) & 1) ^ 1, true)) goto done;
                    const uint32_t msg = msg0 + ps * kMsgBytes, pbar = pfull0 + ps * 8, prow = msg + h * 128;
                    float sum4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
                    for (int i0 = 0; i0 < 64; i0 += 32) {
                        uint32_t sr[32], hi[8], lo[8];
                        tmem_ld32(s_at + i0, sr);
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const float4 s4 = *reinterpret_cast<const float4 *>(&c.s[g * 64 + i0 + i]);
                            const float4 l4 = *reinterpret_cast<const float4 *>(&c.ls[g * 64 + i0 + i]);
                            const float4 r4 = *reinterpret_cast<const float4 *>(&c.r[g * 64 + i0 + i]);
                            const float p0 = ex2_approx(fmaf(__uint_as_float(sr[i]) * rq, s4.x, l4.x) - mb);
                            const float p1 = ex2_approx(fmaf(__uint_as_float(sr[i + 1]) * rq, s4.y, l4.y) - mb);
                            const float p2 = ex2_approx(fmaf(__uint_as_float(sr[i + 2]) * rq, s4.z, l4.z) - mb);
                            const float p3 = ex2_approx(fmaf(__uint_as_float(sr[i + 3]) * rq, s4.w, l4.w) - mb);
                            sum4[0] = fmaf(p0, r4.x, sum4[0]);
                            sum4[1] = fmaf(p1, r4.y, sum4[1]);
                            sum4[2] = fmaf(p2, r4.z, sum4[2]);
                            sum4[3] = fmaf(p3, r4.w, sum4[3]);
                            uint32_t h0, l0, h1, l1;
                            split2(p0, p1, h0, l0);
                            split2(p2, p3, h1, l1);
                            hi[i >> 2] = h0 | (h1 << 16);
                            lo[i >> 2] = l0 | (l1 << 16);
                        }
#pragma unroll
                        for (int v = 0; v < 2; ++v) {
                            const uint32_t at = prow + (((g * 4 + (i0 >> 4) + v) ^ (h & 7)) << 4);
                            st_async_v4(at, hi[4 * v], hi[4 * v + 1], hi[4 * v + 2], hi[4 * v + 3], pbar);
                            st_async_v4(at + kMsgLo, lo[4 * v], lo[4 * v + 1], lo[4 * v + 2], lo[4 * v + 3], pbar);
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&hd->s_free[sb]));
                    l += (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
                    float fin = 0.f;
                    if (j == it.j1 - 1) {
                        const float total = l + exchange(hd->pair, xc, l), own = mb + log2f(total);
                        fin = 1.f / total;
                        if (it.np == 1) {
                            const float lse2 = log2_add(own, sink * 1.4426950408889634f);
                            fin *= exp2f(own - lse2);
                            if (p.lse && head && g == 0) p.lse[(int64_t)it.t * p.N1 + h] = lse2 * 0.6931471805599453f;
                        } else if (head && g == 0) {
                            p.part_s[((int64_t)it.t * p.P + it.piece) * p.N1 + h] = own;
                        }
                    }
                    if (g == 0) st_async_v2(msg + kMsgStats + h * 8, __float_as_uint(head ? alpha : 1.f), __float_as_uint(fin), pbar);
                }
            }
            // every P stage must be handed back before this CTA may exit
            for (int s2 = 0; s2 < kPStages; ++s2) {
                if ((int)sc > s2) {
                    const uint32_t n = (sc - s2 + kPStages - 1) / kPStages;
                    if (!wait_warp(sy, smem_u32(&hd->p_empty[s2]), (n - 1) & 1, true)) goto done;
                }
            }
        }
    } else {
        // ======================= output CTA =======================
        uint8_t *ring = smem + kOutRing, *msgs = smem + kOutMsgs;
        if (warp >= kProdWarp0) {
            producer<false>(p, sy, &ori_map, &cmp_map, nullptr, ring, hd, nullptr);
        } else if (warp == kMmaWarp) {
            constexpr uint32_t idesc = idesc_e4m3(128, 128, 1);
            uint32_t at = 0, phase = 0, pc = 0, oc = 0, pvc = 0, rsc = 0;
            for (uint32_t k = 0;; ++k) {
                int u;
                if (!tq_read(p, sy, rank, k, u)) goto done;
                if (u < 0) break;
                const Item it = load_unit(p, u);
                if (it.skip || it.j1 <= it.j0) continue;
                if (!wait_warp(sy, smem_u32(&hd->o_empty), (oc & 1) ^ 1)) goto done;
                ++oc;
                for (int j = it.j0; j < it.j1; ++j, ++pc) {
                    const int ps = pc % kPStages;
                    if (!wait_warp(sy, smem_u32(&hd->p_full[ps]), (pc / kPStages) & 1, true)) goto done;
                    if (lane == 0) mbar_arrive_expect_tx(smem_u32(&hd->p_full[ps]), kMsgTx);  // the next message
                    const uint8_t *msg = msgs + ps * kMsgBytes;
                    const float2 *stat = reinterpret_cast<const float2 *>(msg + kMsgStats);
                    bool need = false;
                    for (int i = lane; i < 128; i += 32) need |= stat[i].x != 1.f;
                    if (__any_sync(0xffffffffu, need) && j > it.j0) {
                        // every PV product so far, then warps 0-7 scale the rows
                        if (lane == 0) tc_commit(smem_u32(&hd->pv_done));
                        __syncwarp();
                        if (!wait_warp(sy, smem_u32(&hd->pv_done), pvc & 1)) goto done;
                        ++pvc;
                        if (lane == 0) {
                            hd->rs_stage = ps;
                            mbar_arrive(smem_u32(&hd->rs_req));
                        }
                        __syncwarp();
                        if (!wait_warp(sy, smem_u32(&hd->rs_done), rsc & 1)) goto done;
                        ++rsc;
                    }
                    const bool last = j == it.j1 - 1;
                    if (last) {
                        for (int i = lane; i < 128; i += 32) hd->fin[i] = stat[i].y;
                        __syncwarp();
                        if (lane == 0) {
                            __threadfence_block();
                            mbar_arrive(smem_u32(&hd->fin_ready));
                        }
                    }
                    fence_proxy_async_smem();
                    const uint64_t a = sdesc_sw128(smem_u32(msg), 16, 1024);
                    for (int c = 0; c < kVSlabs; ++c) {
                        if (!wait_warp(sy, smem_u32(&hd->full[at]), phase)) goto done;
                        tc_fence_after();
                        if (lane == 0) {
                            const uint64_t b = sdesc_sw128(smem_u32(ring) + at * kUnit, kUnit, 1024);
                            const uint32_t d = tmem + c * 128;
#pragma unroll
                            for (int i = 0; i < kBK / 32; ++i) {
                                mma8_ss(d, a + 2 * i, b + 256 * i, idesc, (j > it.j0 || i > 0) ? 1u : 0u);
                                mma8_ss(d, a + kMsgLo / 16 + 2 * i, b + 256 * i, idesc, 1u);
                            }
                            tc_commit(smem_u32(&hd->empty[at]));
                            if (c == kVSlabs - 1) {
                                tc_commit_mc(smem_u32(&hd->p_empty[ps]), (uint16_t)1);
                                if (last) tc_commit(smem_u32(&hd->o_full));
                            }
                        }
                        __syncwarp();
                        if (++at == kVUnits) {
                            at = 0;
                            phase ^= 1;
                        }
                    }
                }
            }
        } else {
            const int g = warp >> 2, h = threadIdx.x & 127;  // head row, and which half of the columns
            const bool head = h < p.N1;
            const uint32_t trow = tmem + ((uint32_t)((warp & 3) * 32) << 16) + g * (kDv / 2);
            uint32_t ofc = 0, rsc = 0, frc = 0;
            for (uint32_t k = 0;; ++k) {
                int u;
                if (!tq_read(p, sy, rank, k, u)) goto done;
                if (u < 0) break;
                const Item it = load_unit(p, u);
                if (it.skip) continue;
                __nv_bfloat16 *orow = reinterpret_cast<__nv_bfloat16 *>(p.out) +
                                      ((int64_t)it.t * p.N1 + (head ? h : 0)) * kDv + g * (kDv / 2);
                if (it.ntiles == 0) {
                    if (head)
                        for (int d = 0; d < kDv / 2; d += 8) *reinterpret_cast<uint4 *>(orow + d) = make_uint4(0, 0, 0, 0);
                    continue;
                }
                // serve rescale requests until the unit's O is complete
                uint64_t t0 = 0;
                for (uint32_t spin = 0;; ++spin) {
                    if (poll_warp(smem_u32(&hd->rs_req), rsc & 1)) {
                        ++rsc;
                        tc_fence_after();
                        const float a = reinterpret_cast<const float2 *>(msgs + hd->rs_stage * kMsgBytes + kMsgStats)[h].x;
                        if (__any_sync(0xffffffffu, a != 1.f)) {
                            // two 32-column loads in flight per wait: TMEM latency bounds the loop
#pragma unroll 1
                            for (int c = 0; c < kDv / 2; c += 64) {
                                uint32_t r0[32], r1[32];
                                tmem_ld32(trow + c, r0);
                                tmem_ld32(trow + c + 32, r1);
                                tc_wait_ld();
#pragma unroll
                                for (int i = 0; i < 32; ++i) {
                                    r0[i] = __float_as_uint(__uint_as_float(r0[i]) * a);
                                    r1[i] = __float_as_uint(__uint_as_float(r1[i]) * a);
                                }
                                tmem_st32(trow + c, r0);
                                tmem_st32(trow + c + 32, r1);
                            }
                            tc_wait_st();
                        }
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(smem_u32(&hd->rs_done));
                        t0 = 0;
                        continue;
                    }
                    if (poll_warp(smem_u32(&hd->o_full), ofc & 1)) break;
                    if ((spin & 15u) == 15u) {
                        if (hd->abort) goto done;
                        const uint64_t now = globaltimer();
                        if (t0 == 0) t0 = now;
                        else if (now - t0 > kTimeoutNs) {
                            raise_abort(sy, SAS_STATUS_WAIT_TIMEOUT);
                            goto done;
                        }
                    }
                }
                ++ofc;
                if (!wait_warp(sy, smem_u32(&hd->fin_ready), frc & 1)) goto done;
                ++frc;
                tc_fence_after();
                const float fin = hd->fin[h];
                if (it.np == 1 && p.N1 % 32 == 0) {
                    // 64 columns at a time: each warp stages its 32 head rows (128-byte swizzled) and writes
                    // them with one TMA store
                    if ((warp & 3) * 32 < p.N1) {
                        const uint32_t buf = smem_u32(smem + kOutStage) + warp * kWarpSlab;
#pragma unroll 1
                        for (int sl = 0; sl < kDv / 2 / 64; ++sl) {
                            uint32_t r0[32], r1[32];
                            tmem_ld32(trow + sl * 64, r0);
                            tmem_ld32(trow + sl * 64 + 32, r1);
                            if (lane == 0) bulk_wait_read<0>();  // the last store has read buf
                            __syncwarp();
                            tc_wait_ld();
#pragma unroll
                            for (int cc = 0; cc < 8; ++cc) {
                                uint32_t w[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const int i = 8 * (cc & 3) + 2 * e;
                                    w[e] = pack_bf16(__uint_as_float(cc < 4 ? r0[i] : r1[i]) * fin,
                                                     __uint_as_float(cc < 4 ? r0[i + 1] : r1[i + 1]) * fin);
                                }
                                st_shared_v4(buf + lane * 128 + ((cc ^ (lane & 7)) << 4), w[0], w[1], w[2], w[3]);
                            }
                            fence_proxy_async_smem();
                            __syncwarp();
                            if (lane == 0) {
                                tma_store_2d(&out_map, buf, g * (kDv / 2) + sl * 64, it.t * p.N1 + (warp & 3) * 32);
                                bulk_commit();
                            }
                        }
                    }
                } else {
                    // other head counts, and pieces (fp32, normalised within the piece)
                    float *po = p.part_o + (((int64_t)it.t * p.P + it.piece) * p.N1 + (head ? h : 0)) * kDv + g * (kDv / 2);
#pragma unroll 1
                    for (int c = 0; c < kDv / 2; c += 32) {
                        uint32_t r[32];
                        tmem_ld32(trow + c, r);
                        tc_wait_ld();
                        float x[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(r[i]) * fin;
                        if (head && it.np > 1) {
                            float4 *d = reinterpret_cast<float4 *>(po + c);
#pragma unroll
                            for (int i = 0; i < 8; ++i) d[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
                        } else if (head) {
                            uint4 *d = reinterpret_cast<uint4 *>(orow + c);
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                d[i] = make_uint4(pack_bf16(x[8 * i], x[8 * i + 1]), pack_bf16(x[8 * i + 2], x[8 * i + 3]),
                                                  pack_bf16(x[8 * i + 4], x[8 * i + 5]), pack_bf16(x[8 * i + 6], x[8 * i + 7]));
                        }
                        __syncwarp();  // the next load is warp-wide
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&hd->o_empty));
            }
        }
    }
done:
    __syncwarp();
    if (hd->abort) {
        // let in-flight TMA / MMA work land before the shared memory goes away
        const uint64_t t0 = globaltimer();
        while (globaltimer() - t0 < 20000000ull) {
        }
    }
    if (rank == 1 && warp < kSoftWarps && lane == 0) bulk_wait_all();  // each epilogue warp's stores have landed
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    if (warp == kMmaWarp) tmem_dealloc(tmem, kTmemCols);
}

// Pieces of split tokens, and the sink: out = sum_i 2^(own_i - lse2) o_i with o_i normalised within its
// piece and own_i the log2 of the piece's weight sum; lse2 = log2 (sum_i 2^own_i + 2^sink2).
// Block (t, h), thread = 4 columns.
__global__ void __launch_bounds__(kDv / 4) fp8_combine_kernel(const TcArgs p) {
    __shared__ float w_s[kMaxPieces];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int t = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
    const int np = load_unit(p, t).np;
    if (np == 1) return;  // written by the attention kernel
    const int64_t s0 = (int64_t)t * p.P;
    const float own = tid < np ? __ldcg(p.part_s + (s0 + tid) * p.N1 + h) : -INFINITY;
    if (tid < kMaxPieces) w_s[tid] = own;
    __syncthreads();
    float lse2 = p.sinks ? p.sinks[h] * 1.4426950408889634f : -INFINITY;
    for (int i = 0; i < np; ++i) lse2 = log2_add(lse2, w_s[i]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    const float4 *po = reinterpret_cast<const float4 *>(p.part_o + (s0 * p.N1 + h) * kDv) + tid;
    const int64_t stride = (int64_t)p.N1 * kDv / 4;
#pragma unroll 8
    for (int i = 0; i < np; ++i) {
        const float4 o = __ldcg(po + i * stride);
        const float w = exp2f(w_s[i] - lse2);
        acc.x = fmaf(w, o.x, acc.x);
        acc.y = fmaf(w, o.y, acc.y);
        acc.z = fmaf(w, o.z, acc.z);
        acc.w = fmaf(w, o.w, acc.w);
    }
    uint2 *out = reinterpret_cast<uint2 *>(reinterpret_cast<__nv_bfloat16 *>(p.out) + ((int64_t)t * p.N1 + h) * kDv) + tid;
    *out = make_uint2(pack_bf16(acc.x, acc.y), pack_bf16(acc.z, acc.w));
    if (p.lse && tid == 0) p.lse[(int64_t)t * p.N1 + h] = lse2 * 0.6931471805599453f;
}

// Tensor map over [rows][D] elements with 128-byte swizzle, boxes of 128 bytes x box_rows.
int make_map(CUtensorMap *map, const void *base, int64_t rows, int D, bool bf16, uint32_t box_rows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return SAS_ERR_CUDA;
    if (rows >= INT32_MAX) return SAS_ERR_UNSUPPORTED;
    cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)D * (bf16 ? 2 : 1)};
    cuuint32_t box[2] = {bf16 ? 64u : 128u, box_rows};
    cuuint32_t estr[2] = {1, 1};
    const CUresult r = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2,
                          const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? SAS_OK : SAS_ERR_CUDA;
}

constexpr int kClusters = 74;  // 148 SMs / 2
constexpr int kMinPieceTiles = 2;
constexpr int64_t kMaxPartialBytes = int64_t(1) << 30;

struct Plan {
    int P, M;
};

// Pieces per token: the lengths are on the device, so the plan goes by the most tiles a token can have.
Plan plan(const SasFp8Args &a) {
    Plan pl{1, 0};
    if (a.num_tokens <= 0 || 2 * (int64_t)a.num_tokens > kClusters) return pl;
    const int64_t win = std::min<int64_t>((int64_t)a.ori_win_left + 1 + a.ori_first, (int64_t)a.ori_table_len * a.ori_block_size);
    const int64_t cmp = a.scenario == 3 ? a.topk : a.scenario == 2 ? (int64_t)a.cmp_table_len * a.cmp_block_size : 0;
    const int64_t est = (win + 3 + cmp + kBK - 1) / kBK;
    int64_t P = std::min<int64_t>(kClusters / a.num_tokens, (est + kMinPieceTiles - 1) / kMinPieceTiles);
    P = std::min<int64_t>(P, kMaxPieces);
    if (P <= 1) return pl;
    pl.M = (int)((est + P - 1) / P);
    pl.P = (int)((est + pl.M - 1) / pl.M);
    const int64_t bytes = (int64_t)a.num_tokens * pl.P * a.num_heads * kDv * 4;
    return pl.P > 1 && bytes <= kMaxPartialBytes ? pl : Plan{1, 0};
}

} // namespace

namespace sas_host {

bool fp8_tc_supported(const SasFp8Args &a) {
    return a.dtype == SAS_DTYPE_BF16 && a.num_heads <= 128 && (a.head_dim == 512 || a.head_dim == 576) && a.v_head_dim == kDv &&
           (int64_t)a.num_tokens * a.num_heads < INT32_MAX;
}

size_t fp8_tc_pieces(const SasFp8Args &a) { return (size_t)plan(a).P; }

int launch_fp8_tc(const SasFp8Args &a, const Args &args, const Layout &L, char *ws, cudaStream_t s) {
    TcArgs p;
    static_cast<Args &>(p) = args;
    const Plan pl = plan(a);
    p.status = reinterpret_cast<uint32_t *>(p.rec + TR_STATUS);  // record 0 carries what no token is known for
    p.ori_rows = a.ori_block_num * a.ori_block_size;
    p.cmp_rows = a.scenario >= 2 ? a.cmp_block_num * a.cmp_block_size : p.ori_rows;
    p.P = pl.P;
    p.M = pl.M;
    if ((int64_t)a.num_tokens * pl.P >= INT32_MAX) return SAS_ERR_UNSUPPORTED;
    p.U = a.num_tokens * pl.P;
    p.part_o = reinterpret_cast<float *>(ws + L.part_o);
    p.part_s = reinterpret_cast<float *>(ws + L.part_s);
    CUtensorMap ori_map, cmp_map, q_map, out_map;
    int rc = make_map(&ori_map, p.ori, p.ori_rows, p.Dq, false, 1);
    if (!rc) rc = make_map(&cmp_map, a.scenario >= 2 ? p.cmp : p.ori, p.cmp_rows, p.Dq, false, 1);
    if (!rc) rc = make_map(&q_map, p.q, (int64_t)p.T * p.N1, p.Dq, true, 32);
    if (!rc) rc = make_map(&out_map, p.out, (int64_t)p.T * p.N1, kDv, true, 32);
    if (rc) return rc;
    int dev = 0;
    if (check_cuda(cudaGetDevice(&dev))) return SAS_ERR_CUDA;
    if (dev < 0 || dev >= sas::kMaxDevices) return SAS_ERR_UNSUPPORTED;
    static sas::DeviceOnce attr_done[sas::kMaxDevices];
    static std::atomic<int> num_sms[sas::kMaxDevices] = {};
    rc = attr_done[dev].run(1u, [&] {
        return check_cuda(cudaFuncSetAttribute(fp8_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
    });
    if (rc) return rc;
    int sms = num_sms[dev].load(std::memory_order_relaxed);
    if (!sms) {
        if (check_cuda(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev))) return SAS_ERR_CUDA;
        num_sms[dev].store(sms, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * std::max(1, std::min(p.U, sms / 2)), 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = kSmemBytes;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    if (check_cuda(cudaLaunchKernelEx(&cfg, fp8_tc_kernel, p, ori_map, cmp_map, q_map, out_map))) return SAS_ERR_CUDA;
    if (p.P > 1) {
        cudaLaunchConfig_t cc = {};
        cc.gridDim = dim3(a.num_tokens, a.num_heads, 1);
        cc.blockDim = dim3(kDv / 4, 1, 1);
        cc.stream = s;
        cc.attrs = &attr[1];
        cc.numAttrs = 1;
        if (check_cuda(cudaLaunchKernelEx(&cc, fp8_combine_kernel, p))) return SAS_ERR_CUDA;
    }
    return SAS_OK;
}

} // namespace sas_host
