// sm_100a tensor-core attention over the 8-bit cache: bf16 queries, D_qk 512 or 576, D_v 512, up to
// 128 heads.
//
// The keys stay e4m3 from HBM to the MMA (kind::f8f6f4).  What multiplies them is split into 8-bit
// terms.  Queries: two e4m3 terms, since a bf16 value has 8 significant bits and x = hi + lo with
// hi = e4m3(x) leaves a lo of 4 bits.  They are scaled per row by a power of two that brings the largest
// element to [128, 256): elements down to 2^-10 of it split without error, smaller ones are off by at most
// 2^-10 (2^-17 of the largest).  Softmax weights, at most 431 by their scale and rounded to fp16 (2^-11):
// hi in e4m3, then two e5m2 terms, which reach 2^-16 where hi has no bits left.  hi leaves at most 2^-4 of
// a weight's power of two (2^-10 where it is subnormal), and each e5m2 term cuts three bits off what is left:
// 2^-10 of a weight, or 2^-16 of a scale in which the row's largest weight is 2^6 or more.  Two e4m3 terms, whose
// smallest step is 2^-9, took 5 to 8 % less time (1.06 ms instead of 1.14 for 2048 tokens, 67.7 us instead of 71.6
// for 64; the products of V in the output CTA are 18 MMAs a tile instead of 12), but lost every weight below
// 2^-16 of the largest: 3 to 50 % of the output where one key with a small value holds 80 to 99 % of a row.
// One e5m2 term behind hi takes no more time than that, but loses 2^-8 of a weight where two e4m3 terms lose 2^-9.
// A QK product costs two 8-bit MMAs, the time of one bf16 MMA, at half the bytes gathered.
//
// A key's scale s_j multiplies its score and its value.  With t_ij = scale q_i k_j in log2 units, the
// weight of value row j (its codes) is 2^(t_ij) s_j = 2^(x_ij) with x_ij = t_ij + log2 s_j.  The running
// maximum m_i is taken over x_ij, P_ij = 2^(x_ij - m_i + 6) goes to the MMA and e_ij = P_ij / s_j adds to the
// softmax's denominator.  (P as e s with e = 2^(t - m + 6) saves a constant per key, 0.7 % of a prefill's time, but
// scores of 2^24 and more, which scales of 2^20 bring with them, have no digits left for log2 s, and P
// overflows.)  The sink joins at the end.
//
// A unit of work (a token, or a piece of one) goes to a cluster of two CTAs on two SMs that split it
// by role, because O alone (128 heads x 512 fp32) fills one SM's tensor memory:
//
//   CTA 0 ("score")                              CTA 1 ("output")
//   TMEM: Q hi / lo (D_qk / 2 columns),          TMEM: O (128 x 512 fp32)
//         S (2 x 96 columns)
//   4 warps gather 96 key rows per tile          4 warps gather the first 512 bytes of the rows
//           (cp.async into the MMA's swizzle)
//   1 warp  S = Q K^T: 2 MMAs (hi, lo) of M 128, 1 warp  O += P V: 3 per 32 keys and 256 value dims; V is the
//           N 96, K 32 per 32 dims                       N-major B operand, the same bytes in the same
//                                                        swizzle as K
//   8 warps split Q; softmax (thread = head;     8 warps split P (thread = head; warps 0-3 the even
//           warps 0-3 take the even tiles,               tiles, 4-7 the odd ones); rescale O where a
//           4-7 the odd ones); P in fp16 and             maximum rose; epilogue
//           factors go to CTA 1 by bulk copies   1 warp  acknowledges messages
//
// What the pieces measured on B200, each alone, and what follows from it:
//   - An MMA of N 64 takes 58 cycles, as one of N 96; N 128 takes 70-83.  96 keys leave room in TMEM for
//     all of Q beside two S.
//   - TMA tile::gather4 takes 24 cycles for 4 x 128 bytes wherever the rows lie (37 GB/s per SM);
//     16-byte cp.async reaches 56 bytes per cycle from L2 (110 GB/s), and the HBM's rate over all SMs.
//   - st.async to the other SM moves 12 bytes per cycle and holds the issuing warps meanwhile; a tile's
//     P is 24 KiB.  Bulk copies from a staging buffer run beside the next tile's softmax.
//   - With 128 heads some maximum rises in most tiles.  It is followed only past 2^2.75 (P <= 2^8.75, the
//     e4m3 range; the largest weight is then at least 2^6, and what a small weight is off by 2^-22 of it; 2^0.75
//     would take 2 % more time), and O is rescaled 256 columns at a time, each as soon as the last tile's
//     product of these columns is complete.
//
// Whole calls: 64 tokens of 2176 keys, 128 heads of 576 dims: 70 us (38.8 GFLOP, 98.6 MB); 2048 such
// tokens: 1.14 ms, 870 TFLOP/s, and 1.32 ms once the card is at its power limit (1.7 GHz).  A tile takes
// about 3000 cycles of a prefill (2800 with two terms per weight, where these were taken): 1960 of QK issue, the
// rest mostly waits for an S to come back: the two passes of the softmax are 1370 and 2140 cycles, so that
// QK and softmax of two tiles, which share an S buffer, take 5700, and a third S has no room.  The gather
// warps are busy for 2650; the 18 products of the output CTA take 2700.  Left out for timing, of 1178 us: the
// rescale of O 2 %, V's copies 2 %, both 3.5 %, then the third product nothing; the third product alone takes
// 2 to 8 % of the decode steps.  A unit adds 6500 cycles for the split of Q
// (conversions and byte shuffles at half and quarter rate), and the first tile 8 us of latency.  What did
// not help: 6 gather warps, or a warp of its own for the row lookups (they take the softmax's issue slots,
// 3 and 4 % slower); a tile taken in the last tile's frame and redone where that does not hold (some of 128
// heads mostly rises, 20 %); TMEM loads a step ahead or of 32 columns (0 to 5 %: longer loops; the roles of an
// SM share its instruction caches); a staging of 8 boxes, or rows of 128 bytes, in the epilogue; the next
// tile's weights split before the rescale (2 %); V's ring in halves of a tile (5 %).
//
// Keys of a token: first positions, then the window, then the compressed rows.  Slots without a key
// carry weight 0 (log2 s = -inf); they and rows of unmapped blocks are filled with zeros.
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

constexpr int kBK = 96;              // keys per tile
constexpr int kSlab = kBK * 128;     // 128 dims of a tile's rows
constexpr int kStages = 3, kVStages = 2;  // of the two CTAs' rings
constexpr int kDv = 512, kVSlabs = kDv / 128;
constexpr int kVStage = kVSlabs * kSlab, kKStage = kVStage + kBK * 64;  // K: dims 512 .. 575 as 64-byte rows behind
constexpr int kQChunk = 128 * 128, kQPerStage = 3;  // raw Q: 64 bf16 dims of 128 heads; chunks per stage of the K ring
constexpr int kQStages = (576 / 64 + kQPerStage - 1) / kQPerStage;
static_assert((512 / 64 + kQPerStage - 1) / kQPerStage == kQStages, "the last stage is the same one");
constexpr int kSoftWarps = 8, kMmaWarp = 8, kProdWarp0 = 9, kProdWarps = 4;
constexpr int kRows = kBK / kProdWarps;
static_assert(kRows % 8 == 0 && kProdWarps == 4, "whole swizzle periods, 32 heads of Q a warp");
// The output CTA's warp that gives the staging of messages back as they arrive.  Done by the warps that split them, after
// their last rescale, it held the score CTA up: 64 tokens took 73 us instead of 71.6, 256 mixed requests 123 instead of 120.
constexpr int kAckWarp = kProdWarp0 + kProdWarps;
constexpr int kThreads = 32 * (kAckWarp + 1);
constexpr uint32_t kReaders = 2 * kAckWarp;  // of the unit queue: every warp but its writer and the score CTA's last
constexpr int kTmemCols = 512, kTmemS = 320;
// Ring of per-tile key constants.  Those of tile n are written once its stage is free: the scores of tile n - 3 are
// complete, so that their buffer had been given back by tile n - 5, and the other one by tile n - 6 before.
constexpr int kConsts = 6;
constexpr float kTop = 8.75f;        // log2 of the largest P: 431, within e4m3's 448
constexpr float kRise = 2.75f;       // log2 of the rise of a maximum that is left to P
constexpr int kMaxPieces = 64;

// P message: per head 96 weights in fp16, 64 in a 128-byte row (SW128) and 32 in a 64-byte row (SW64), then
// {alpha, the unit's final factor}.  The 32 heads of a warp are contiguous in each part.  The output CTA
// puts codes in the weights' place, per 32 keys 32 hi and 32 mid; lo goes to a buffer of its own.
constexpr int kMsgLo = 128 * 128, kMsgStats = kMsgLo + 128 * 64, kMsgBytes = kMsgStats + 1024;

// Messages under way.  A slot is held from its copy's start over the split to the end of its product: with two of them
// 64 tokens take 4 % more time, with four as much as with three.
constexpr int kSlots = 3;

struct KeyConst {
    float s[kBK];    // scale; 0: a zero row
    float ls[kBK];   // log2 s; -60 for zero rows (their values do not count), -inf: no key
    float inv[kBK];  // 2^-ls; 0: no key
};

struct Hdr {
    uint64_t full[kStages], empty[kStages], s_full[2], s_free[2], q_raw[kQStages], q_full, c_full[kConsts];
    uint64_t x_bar[4][2], m_bar[4][2], l_bar[4];  // of the two warps that share 32 heads
    uint64_t p_full[kSlots], p_ready[kSlots], p_empty[kSlots], p_sent[2], o_full, o_empty, rs_done[2], pv_done[2][kSlots];
    uint64_t tq_full[kTq], tq_empty[kTq];
    volatile int tq[kTq];
    uint32_t tmem_base;
    volatile int abort;
    float amax[2][128], m[2][128], l[2][2][128];
};
constexpr int kHdr = 5 * 1024;
static_assert(sizeof(Hdr) <= kHdr, "header");
constexpr int kConstOff = kHdr;
constexpr int kScoreMsgs = (kConstOff + kConsts * (int)sizeof(KeyConst) + 1023) / 1024 * 1024;
constexpr int kScoreRing = kScoreMsgs + 2 * kMsgBytes;
constexpr int kScoreSmem = kScoreRing + kStages * kKStage;
constexpr int kOutRing = 1024;  // behind the barriers: the rest of the header is the score CTA's
static_assert(offsetof(Hdr, amax) <= kOutRing, "barriers of the output CTA");
constexpr int kOutMsgs = kOutRing + kVStages * kVStage;
// Third terms of a slot's weights: per 8 heads three blocks of 32 keys, each 8 rows of 32 bytes (SW32).  (Two buffers for
// even and odd tiles, which a split waits for, leave room for a second staging buffer per warp: 2 % slower.)
constexpr int kThirdBytes = 128 / 8 * 3 * 256;
constexpr int kOutThirds = kOutMsgs + kSlots * kMsgBytes;
constexpr int kOutStage = kOutThirds + kSlots * kThirdBytes;  // epilogue staging: 64 bytes of 32 heads per warp
constexpr int kWarpSlab = 32 * 64;
constexpr int kOutSmem = kOutStage + kSoftWarps * kWarpSlab;
constexpr int kSmemBytes = (kScoreSmem > kOutSmem ? kScoreSmem : kOutSmem) + 1024;  // + alignment slack
static_assert(kScoreMsgs % 1024 == 0 && kScoreRing % 1024 == 0 && kKStage % 1024 == 0 && kOutRing % 1024 == 0 &&
              kOutMsgs % 1024 == 0 && kMsgBytes % 1024 == 0 && kOutStage % 1024 == 0 && kThirdBytes % 1024 == 0, "swizzled tiles are 1 KiB aligned");
static_assert(kQPerStage * kQChunk <= kKStage && kSmemBytes <= 232448, "shared memory");

// n / d for 0 <= n < 2^31 as a multiplication: 2^(32 + s) <= m d < 2^(32 + s) + 2^(s + 1) with 2^s < d <= 2^(s + 1)
// makes the quotient exact; d = 1 has no such m.
struct Div {
    uint32_t d, m, s;
};
__device__ __forceinline__ int div(int n, const Div &v) { return v.d == 1 ? n : (int)(__umulhi((uint32_t)n, v.m) >> v.s); }
Div make_div(uint32_t d) {
    Div v{d, 0, 0};
    if (d == 1) return v;
    while ((2ull << v.s) < d) ++v.s;
    v.m = (uint32_t)(((1ull << (32 + v.s)) + d - 1) / d);
    return v;
}

struct TcArgs : Args {
    Div ori_div, cmp_div;    // by the block sizes
    uint32_t *status;
    int U, P, M;             // units; pieces per token, tiles per piece (P = 1: whole tokens)
    int NP;                  // rows of a slot of part_o: N1 rounded up to 32
    float *part_o, *part_s;
};

__device__ __forceinline__ void mma8_ts(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a_tmem), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma8_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
// Instruction descriptor of kind::f8f6f4, A e4m3 (format 0) or e5m2 (1), B e4m3, fp32 accumulation; b_mn: B is
// N-major.
__host__ __device__ constexpr uint32_t idesc_f8(uint32_t m, uint32_t n, uint32_t b_mn, uint32_t a_e5m2) {
    return (1u << 4) | (a_e5m2 << 7) | (b_mn << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// wait_warp with its polling loop out of line: the roles' loops share the instruction caches, and the
// first try (which suspends the warp for a while) mostly succeeds.
__device__ __noinline__ bool wait_long(const Sync &s, uint32_t bar, uint32_t parity, bool cluster_scope) {
    return wait_warp(s, bar, parity, cluster_scope);
}
__device__ __forceinline__ bool wait_on(const Sync &s, uint32_t bar, uint32_t parity, bool cluster_scope = false) {
    const bool done = cluster_scope ? mbar_try_cluster(bar, parity) : mbar_try(bar, parity);
    return __all_sync(0xffffffffu, done) || wait_long(s, bar, parity, cluster_scope);
}

// Whether some row of O is to be rescaled before the message's product: the sign bits of the four warps' first
// factors (bits, because a factor may be -0: a maximum that rose by 2^150 leaves nothing of what came before).
__device__ __forceinline__ bool some_alpha(const uint8_t *msg) {
    return __any_sync(0xffffffffu, reinterpret_cast<const int2 *>(msg + kMsgStats)[(threadIdx.x & 3) * 32].x < 0);
}

// One lane of the warp, the same one each time.  The compiler takes what it runs as warp-uniform: with
// `lane == 0` in its place an MMA of N 96 issued every 53 cycles instead of 48.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

struct Item {
    int32_t rec[TR_INTS];
    int t, piece, np, ntiles, j0, j1;  // tiles [j0, j1) of token t
    bool skip;                         // a piece past the token's last tile
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
    it.ntiles = b.y ? (a.w + b.x + kBK - 1) / kBK : 0;
    it.np = p.P > 1 && it.ntiles > p.M ? min((it.ntiles + p.M - 1) / p.M, p.P) : 1;
    it.skip = it.piece >= it.np;
    it.j0 = it.np > 1 ? it.piece * p.M : 0;
    it.j1 = it.np > 1 && it.piece < it.np - 1 ? it.j0 + p.M : it.ntiles;  // the last piece takes the rest
    return it;
}

// Row lookup of key slot i in three steps, each a tile ahead of the next so that their loads hide
// behind the copies: the table entry (or the resolved row), the physical row, its block's scale.
__device__ __forceinline__ int32_t key_fetch(const TcArgs &p, const Item &it, int i) {
    const bool win = i < it.rec[TR_NORI];
    const int slot = win ? ori_position(it.rec, i) : i - it.rec[TR_NORI];
    if (!win && slot >= it.rec[TR_NCMP]) return -1;
    if (!win && p.scenario == 3) return __ldg(p.rows + (int64_t)it.t * p.K + slot);
    const int blk = div(slot, win ? p.ori_div : p.cmp_div), len = win ? p.ori_table_len : p.cmp_table_len;
    return blk < len ? __ldg((win ? p.ori_bt : p.cmp_bt) + (int64_t)it.rec[TR_B] * len + blk) : -2;
}

struct Key {
    const uint8_t *row;  // nullptr: zeros
    float s;             // its block's scale (loaded), 1 without a row
    bool live;           // the slot holds a key
};

__device__ __forceinline__ Key key_row(const TcArgs &p, const Item &it, int i, int32_t fetched, uint32_t &bits) {
    Key key{nullptr, 1.f, false};
    const bool win = i < it.rec[TR_NORI];
    const int slot = win ? ori_position(it.rec, i) : i - it.rec[TR_NORI];
    key.live = win || slot < it.rec[TR_NCMP];
    if (!key.live) return key;
    const Div &d = win ? p.ori_div : p.cmp_div;
    int row, blk;
    if (!win && p.scenario == 3) {
        row = fetched;
        blk = div(max(row, 0), d);
    } else {
        blk = fetched;
        const bool bad = blk < -1 || blk >= (win ? p.ori_block_num : p.cmp_block_num);
        if (bad) bits |= SAS_STATUS_BAD_BLOCK;
        row = bad || blk < 0 ? -1 : blk * (int)d.d + (slot - div(slot, d) * (int)d.d);
    }
    if (row < 0) return key;
    key.row = (win ? p.ori : p.cmp) + (int64_t)row * p.Dq;
    key.s = __ldg((win ? p.ori_scale : p.cmp_scale) + blk);
    return key;
}

// The kernel is a programmatic dependent of the resolve kernel: its records are visible after this wait.
__device__ __forceinline__ void wait_resolved() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, uint32_t bytes) {  // bytes 0: zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// The gather warps.  Each takes 24 of a tile's 96 key slots (a lane per slot) and copies their rows with
// 16-byte cp.async: an instruction moves 128 bytes of 4 rows (row r of a slab at r * 128, granule g at
// g ^ r % 8: the MMA's 128-byte swizzle); dims 512 .. 575 go to 64-byte rows (granule g at g ^ r / 2 % 4:
// the 64-byte swizzle), 8 rows per instruction.  Row addresses go from lane to lane once per 4 rows.  A
// stage's full barrier counts the threads; each arrives when its copies have landed.  The warps share
// nothing else.
template <bool kScore>
__device__ void producer(const TcArgs &p, const Sync &sy, const CUtensorMap *q_map, uint8_t *ring, Hdr *hd,
                         KeyConst *consts) {
    constexpr uint32_t kStageBytes = kScore ? kKStage : kVStage, kRing = kScore ? kStages : kVStages;
    const int w = (threadIdx.x >> 5) - kProdWarp0, lane = threadIdx.x & 31;
    const bool holds = lane < kRows;
    const int key_at = w * kRows + (holds ? lane : 0);
    const bool writer = kScore && w == 0;
    const bool tail = kScore && p.Dq > 512;
    const uint32_t ring_at = smem_u32(ring);
    // this lane's granule lane % 8 of row 4 k + lane / 8: offsets for even k, and what odd k change
    const uint32_t dst0 = w * kRows * 128 + (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) << 4);
    const uint32_t src_off = (lane & 7) * 16;
    uint32_t st = 0, phase = 1, tiles = 0, bits = 0;  // stage, and the parity its empty barrier is waited on
    int pend = -1;
    auto next = [&] {
        if (++st == kRing) {
            st = 0;
            phase ^= 1;
        }
    };
    // raw Q of a token, three chunks of 64 dims per stage, 32 head rows per warp by TMA
    auto load_q = [&](int t) {
        const int chunks = p.Dq / 64;
        for (int c = 0; c < chunks; c += kQPerStage, next()) {
            if (!wait_on(sy, smem_u32(&hd->empty[st]), phase)) return false;
            const uint32_t fb = smem_u32(&hd->full[st]);
            if (lane == 0 && w * 32 < p.N1) {
                const int n = min(kQPerStage, chunks - c);
                mbar_arrive_expect_tx(fb, n * 4096);
                for (int e = 0; e < n; ++e)
                    tma_load_2d(ring_at + st * kStageBytes + e * kQChunk + w * 4096, q_map, (c + e) * 64, t * p.N1 + w * 32,
                                fb);
            } else {
                mbar_arrive(fb);  // rows of no head: whatever lies there
            }
        }
        return true;
    };
    for (uint32_t k = 0;; ++k) {
        int u = -1;
        if (!(writer ? tq_publish(p, sy, k, pend, u) : tq_read(p, sy, kScore ? 0 : 1, k, u))) return;
        if (u < 0) break;
        // q is older than the resolve kernel: the first unit's is loaded and split beside it, whatever the unit holds
        if (kScore && k == 0 && !load_q(u % p.T)) return;
        if (k == 0) wait_resolved();
        const Item it = load_unit(p, u);
        if (it.skip || it.j1 <= it.j0) continue;
        const int end = it.j1 * kBK;
        int i = it.j0 * kBK + key_at;
        const int32_t f0 = key_fetch(p, it, i);
        int32_t fetched = i + kBK < end ? key_fetch(p, it, i + kBK) : -1;
        if (kScore && k > 0 && !load_q(it.t)) return;
        Key key = key_row(p, it, i, f0, bits);  // behind Q's loads, which need no lookup
        for (int j = it.j0; j < it.j1; ++j, i += kBK, ++tiles, next()) {
            if (key.row != nullptr && !scale_ok(key.s)) {
                bits |= SAS_STATUS_BAD_SCALE;
                key.row = nullptr;
            }
            if (!wait_on(sy, smem_u32(&hd->empty[st]), phase)) return;
            const uint32_t base = ring_at + st * kStageBytes;
            const uint64_t mine = reinterpret_cast<uint64_t>(key.row);
#pragma unroll 1  // short code: the roles of an SM share its instruction caches
            for (int k4 = 0; k4 < kRows / 4; ++k4) {
                const uint64_t a = __shfl_sync(0xffffffffu, mine, 4 * k4 + (lane >> 3));
                const uint8_t *src = reinterpret_cast<const uint8_t *>(a ? a : reinterpret_cast<uint64_t>(p.ori)) + src_off;
                const uint32_t n = a ? 16 : 0, dst = base + (dst0 ^ ((k4 & 1) << 6)) + k4 * 512;
#pragma unroll
                for (int c = 0; c < kVSlabs; ++c) cp_async16(dst + c * kSlab, src + c * 128, n);
            }
            if (tail) {
#pragma unroll 1
                for (int r0 = 0; r0 < kRows; r0 += 8) {
                    const int r = r0 + (lane >> 2);
                    const uint64_t a = __shfl_sync(0xffffffffu, mine, r);
                    cp_async16(base + kVStage + (w * kRows + r) * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4),
                               a ? reinterpret_cast<const uint8_t *>(a) + 512 + (lane & 3) * 16 : p.ori, a ? 16 : 0);
                }
            }
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&hd->full[st])) : "memory");
            if constexpr (kScore) {
                KeyConst &c = consts[tiles % kConsts];
                const bool row = key.row != nullptr;
                if (holds) {  // the copies wait for this: approximations, off by 2^-22 (a weight is off by 2^-11 as it is)
                    const float ls = row ? __log2f(key.s) : -60.f;
                    c.s[key_at] = row ? key.s : key.live ? 0.f : 1.f;
                    c.ls[key_at] = key.live ? ls : -INFINITY;
                    c.inv[key_at] = key.live ? ex2_approx(-ls) : 0.f;
                }
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(smem_u32(&hd->c_full[tiles % kConsts]));
                    if (writer && j == (it.j1 - it.j0 > 1 ? it.j1 - 2 : it.j0))
                        pend = (int)ncluster_x() + atomicAdd(p.counter, 1);
                }
            }
            key = Key{nullptr, 1.f, false};  // the next tile's lookups, behind the copies
            if (i + kBK < end) key = key_row(p, it, i + kBK, fetched, bits);
            fetched = i + 2 * kBK < end ? key_fetch(p, it, i + 2 * kBK) : -1;
        }
    }
    // the copies' barriers are shared memory of this CTA: none may land after it has exited
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (bits) sas::set_status(p.status, bits);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// To fp16, a in the low half: nearest even, saturating; NaN stays NaN.
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
    uint32_t r;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}

// Two fp16 values (at most 448) as pairs of e4m3 codes, hi + lo, in 16 bits each.  Differences of a value and its
// code are exact in fp16.
__device__ __forceinline__ uint32_t to_e4m3(uint32_t x) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ uint32_t less(uint32_t x, uint32_t y) {  // halves of x minus halves of y
    const __half2 d = __hsub2(*reinterpret_cast<const __half2 *>(&x), *reinterpret_cast<const __half2 *>(&y));
    return *reinterpret_cast<const uint32_t *>(&d);
}
// Four fp16 values into four hi and four lo codes, both e4m3.
__device__ __forceinline__ void split4h(uint32_t a, uint32_t b, uint32_t &hi, uint32_t &lo) {
    const uint32_t h0 = to_e4m3(a), h1 = to_e4m3(b);
    lo = to_e4m3(less(a, e4m3x2_to_half2(h0))) | (to_e4m3(less(b, e4m3x2_to_half2(h1))) << 16);
    hi = h0 | (h1 << 16);
}
// Four fp16 values as hi (e4m3) + mid + lo (e5m2).  An fp16 value's upper byte is its e5m2 code, cut towards zero, so
// that mid and lo take no conversions.
__device__ __forceinline__ void split4w(uint32_t a, uint32_t b, uint32_t &hi, uint32_t &mid, uint32_t &lo) {
    const uint32_t h0 = to_e4m3(a), h1 = to_e4m3(b);
    const uint32_t r0 = less(a, e4m3x2_to_half2(h0)), r1 = less(b, e4m3x2_to_half2(h1));
    hi = __byte_perm(h0, h1, 0x5410);
    mid = __byte_perm(r0, r1, 0x7531);
    lo = __byte_perm(less(r0, r0 & 0xff00ff00u), less(r1, r1 & 0xff00ff00u), 0x7531);
}

// Four bf16 values times f into four hi and four lo codes.
__device__ __forceinline__ void split4(uint32_t a, uint32_t b, float f, uint32_t &hi, uint32_t &lo) {
    const float2 x = sas::DT<__nv_bfloat16>::to_f2(a), y = sas::DT<__nv_bfloat16>::to_f2(b);
    split4h(pack_half(x.x * f, x.y * f), pack_half(y.x * f, y.y * f), hi, lo);
}

// Q of head row h, raw bf16 in TMEM columns [0, D_qk / 2), into hi and lo codes in place: chunk c of 64
// dims keeps its 32 columns, hi codes in the first 16 and lo codes in the last 16.  The row's two
// threads (warp and warp ^ 4) take every other chunk and agree on the largest element.  Returns the
// row's power-of-two factor f (q f = hi + lo), NaN for a row that holds an infinity or NaN; false in
// `ok` on abort.
__device__ float split_q(const Sync &sy, Hdr *hd, uint32_t trow, int chunks, uint32_t parity, bool &ok) {
    const int warp = threadIdx.x >> 5, g = warp >> 2, h = threadIdx.x & 127;
    __nv_bfloat162 top = __floats2bfloat162_rn(0.f, 0.f);
#pragma unroll 1
    for (int c = g; c < chunks; c += 2) {  // as the chunks come
        uint32_t r[32];
        ok = wait_on(sy, smem_u32(&hd->q_raw[c / kQPerStage]), parity);
        if (!ok) return 0.f;
        tc_fence_after();
        tmem_ld32(trow + c * 32, r);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) top = __hmax2_nan(top, __habs2(*reinterpret_cast<__nv_bfloat162 *>(&r[i])));
    }
    const float2 t2 = __bfloat1622float2(top);
    float amax = t2.x + t2.y != t2.x + t2.y ? INFINITY : fmaxf(t2.x, t2.y);
    hd->amax[g][h] = amax;
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(smem_u32(&hd->x_bar[warp & 3][g]));
    ok = wait_on(sy, smem_u32(&hd->x_bar[warp & 3][g ^ 1]), parity);
    amax = fmaxf(amax, hd->amax[g ^ 1][h]);
    // largest element to [128, 256); rows of zeros and of the smallest subnormals: f = 2^126
    const int e = (int)(__float_as_uint(amax) >> 23) - 127;
    const float f = amax == INFINITY ? NAN : __uint_as_float((uint32_t)(min(126, 7 - e) + 127) << 23);
#pragma unroll 1
    for (int c = g; c < chunks; c += 2) {
        uint32_t r[32], hi[16], lo[16];
        tmem_ld32(trow + c * 32, r);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) split4(r[2 * i], r[2 * i + 1], f, hi[i], lo[i]);
        tmem_st16(trow + c * 32, hi);
        tmem_st16(trow + c * 32 + 16, lo);
    }
    tc_wait_st();
    return f;
}

// Two fp32 operations per instruction.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// Bulk copy of this CTA's shared memory to the cluster peer's, completing bytes on the peer's mbarrier.
__device__ __forceinline__ void bulk_to_peer(uint32_t dst, uint32_t src, uint32_t bytes, uint32_t cluster_bar) {
    asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "r"(src), "r"(bytes), "r"(cluster_bar)
                 : "memory");
}

// Shared-memory matrix descriptors, K-major rows of 64 or 32 bytes, 64- or 32-byte swizzle; sbo: bytes between groups
// of 8 rows.
__device__ __forceinline__ uint64_t sdesc_sw64(uint32_t saddr, uint32_t sbo) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)1 << 16 | (uint64_t)(sbo >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)4 << 61;
}
__device__ __forceinline__ uint64_t sdesc_sw32(uint32_t saddr, uint32_t sbo) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)1 << 16 | (uint64_t)(sbo >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)6 << 61;
}

__global__ void __launch_bounds__(kThreads, 1)
    fp8_tc_kernel(const TcArgs p, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap out_map,
                  const __grid_constant__ CUtensorMap part_map) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    Hdr *hd = reinterpret_cast<Hdr *>(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int quads = (p.N1 + 31) / 32;  // of 32 heads, a softmax warp's share
    const uint32_t msg_bytes = quads * (kMsgBytes / 4);

    if (threadIdx.x == 0) {
        auto init = [](uint64_t *b, int n, uint32_t count) {
            for (int i = 0; i < n; ++i) mbar_init(smem_u32(b + i), count);
        };
        init(hd->full, kStages, 32 * kProdWarps);
        init(hd->empty, kStages, 1);
        init(hd->s_full, 2, 1);
        init(hd->s_free, 2, 4);
        init(hd->q_raw, kQStages, 1);
        init(&hd->q_full, 1, kSoftWarps);
        init(hd->c_full, kConsts, kProdWarps);
        init(&hd->x_bar[0][0], 8, 1);
        init(&hd->m_bar[0][0], 8, 1);
        init(hd->l_bar, 4, 1);
        init(hd->p_full, kSlots, 1);
        init(hd->p_empty, kSlots, 1);
        init(hd->p_sent, 2, 1);
        init(hd->p_ready, kSlots, kSoftWarps);
        init(&hd->o_full, 1, 1);
        init(&hd->o_empty, 1, kSoftWarps);
        init(hd->rs_done, 2, kSoftWarps);
        init(&hd->pv_done[0][0], 2 * kSlots, 1);
        init(hd->tq_full, kTq, 1);
        init(hd->tq_empty, kTq, kReaders);
        hd->abort = 0;
        // the output CTA expects the first message of each P slot (bulk copies complete it)
        if (rank == 1)
            for (int i = 0; i < kSlots; ++i) mbar_arrive_expect_tx(smem_u32(&hd->p_full[i]), msg_bytes);
        mbar_fence_init();
    }
    if (rank == 1)  // factors of heads that no message brings
        for (int i = threadIdx.x; i < kSlots * 128; i += kThreads)
            if ((i & 127) >= quads * 32)
                reinterpret_cast<float2 *>(smem + kOutMsgs + (i >> 7) * kMsgBytes + kMsgStats)[i & 127] = make_float2(1.f, 0.f);
    if (warp == kMmaWarp) {
        tmem_alloc(smem_u32(&hd->tmem_base), kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // both CTAs' barriers are initialised before any remote arrive
    tc_fence_after();
    if (rank == 1 && (warp < kProdWarp0 || warp == kAckWarp)) wait_resolved();  // the others wait when they need a record
    if (p.P > 1) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t tmem = hd->tmem_base;
    Sync sy{&hd->abort, p.status, map_to_cta(smem_u32((const void *)&hd->abort), rank ^ 1u), hd->tq_full, hd->tq_empty,
            hd->tq};

    if (rank == 0) {
        // ======================= score CTA =======================
        uint8_t *ring = smem + kScoreRing;
        KeyConst *consts = reinterpret_cast<KeyConst *>(smem + kConstOff);
        if (warp == kAckWarp) {
            // nothing to do in this CTA
        } else if (warp >= kProdWarp0) {
            producer<true>(p, sy, &q_map, ring, hd, consts);
        } else if (warp == kMmaWarp) {
            constexpr uint32_t idesc = idesc_f8(128, kBK, 0, 0);
            const int chunks = p.Dq / 64;
            uint32_t st = 0, phase = 0, sc = 0, qc = 0;
            auto next = [&] {
                if (++st == kStages) {
                    st = 0;
                    phase ^= 1;
                }
            };
            for (uint32_t k = 0;; ++k) {
                int u;
                if (!tq_read(p, sy, rank, k, u)) goto done;
                if (u < 0) break;
                Item it;
                auto open = [&] {
                    it = load_unit(p, u);
                    return !it.skip && it.j1 > it.j0;
                };
                if (k > 0 && !open()) continue;
                // raw Q -> TMEM, once the previous unit's last product has read the old one
                if (sc > 0 && !wait_on(sy, smem_u32(&hd->s_full[(sc - 1) & 1]), ((sc - 1) >> 1) & 1)) goto done;
                for (int c = 0; c < chunks; c += kQPerStage, next()) {
                    if (!wait_on(sy, smem_u32(&hd->full[st]), phase)) goto done;
                    tc_fence_after();
                    if (elect_one()) {
                        for (int e = 0; e < kQPerStage && c + e < chunks; ++e) {
                            const uint64_t d = sdesc_sw128(smem_u32(ring) + st * kKStage + e * kQChunk, 16, 1024);
                            for (int kq = 0; kq < 4; ++kq) tmem_cp_128x256b(tmem + ((c + e) * 4 + kq) * 8, d + 2 * kq);
                        }
                        tc_commit(smem_u32(&hd->empty[st]));
                        tc_commit(smem_u32(&hd->q_raw[c / kQPerStage]));
                    }
                    __syncwarp();
                }
                if (!wait_on(sy, smem_u32(&hd->q_full), qc & 1)) goto done;
                ++qc;
                if (k == 0) {
                    wait_resolved();
                    if (!open()) continue;
                }
                for (int j = it.j0; j < it.j1; ++j, ++sc, next()) {
                    const int sb = sc & 1;
                    const uint32_t d = tmem + kTmemS + sb * kBK;
                    if (!wait_on(sy, smem_u32(&hd->s_free[sb]), ((sc >> 1) & 1) ^ 1)) goto done;
                    if (!wait_on(sy, smem_u32(&hd->full[st]), phase)) goto done;
                    tc_fence_after();
                    fence_proxy_async_smem();  // the rows were written by cp.async
                    if (elect_one()) {
                        const uint32_t base = smem_u32(ring) + st * kKStage;
                        const uint64_t b0 = sdesc_sw128(base, 16, 1024);
#pragma unroll
                        for (int c = 0; c < kVSlabs; ++c) {
                            const uint64_t b = b0 + c * (kSlab / 16);
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint32_t a = tmem + c * 64 + (i >> 1) * 32 + (i & 1) * 8;
                                mma8_ts(d, a, b + 2 * i, idesc, c + i > 0 ? 1u : 0u);
                                mma8_ts(d, a + 16, b + 2 * i, idesc, 1u);
                            }
                        }
                        if (chunks > 8) {
                            const uint64_t b = sdesc_sw64(base + kVStage, 512);
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                mma8_ts(d, tmem + 256 + i * 8, b + 2 * i, idesc, 1u);
                                mma8_ts(d, tmem + 256 + 16 + i * 8, b + 2 * i, idesc, 1u);
                            }
                        }
                        tc_commit(smem_u32(&hd->empty[st]));
                        tc_commit(smem_u32(&hd->s_full[sb]));
                    }
                    __syncwarp();
                }
            }
        } else {
            const int g = warp >> 2, h = threadIdx.x & 127;  // tile parity, head row
            const bool head = h < p.N1;
            const uint32_t trow = tmem + ((uint32_t)((warp & 3) * 32) << 16);
            const uint32_t s_at = trow + kTmemS + g * kBK;
            uint8_t *stage = smem + kScoreMsgs + g * kMsgBytes;
            const uint32_t row1 = smem_u32(stage) + h * 128, row2 = smem_u32(stage) + kMsgLo + h * 64;
            const uint32_t sw1 = (h & 7) << 4, sw2 = ((h >> 1) & 3) << 4;
            const uint32_t peer_msgs = map_to_cta(smem_u32(smem + kOutMsgs), 1), peer_full0 = map_to_cta(smem_u32(hd->p_full), 1);
            const float sink = head && p.sinks ? p.sinks[h] : -INFINITY;
            // a warp without heads: its rows of Q, S and P hold whatever lies there, and reach no other row (16 heads,
            // 11 tiles: 6 % less time than with all warps at work)
            const bool idle = (warp & 3) >= quads;
            uint32_t sc0 = 0, qc = 0, lc = 0, mine = 0;  // the unit's first tile; units; units of two tiles or more; own tiles
            for (uint32_t k = 0;; ++k) {
                int u;
                if (!tq_read(p, sy, rank, k, u)) goto done;
                if (u < 0) break;
                Item it;
                auto open = [&] {
                    it = load_unit(p, u);
                    if (!it.skip && it.ntiles == 0 && p.lse && head && g == 0)
                        p.lse[(int64_t)it.t * p.N1 + h] = it.rec[TR_VALID] ? sink : 0.f;
                    return !it.skip && it.ntiles > 0;
                };
                if (k > 0 && !open()) continue;
                bool ok;
                float rq = 0.f;
                // (without the wait an idle warp could give the next unit's arrival in place of another warp's)
                if (idle) ok = wait_on(sy, smem_u32(&hd->q_raw[kQStages - 1]), qc & 1);
                else rq = p.scale_log2 / split_q(sy, hd, trow, p.Dq / 64, qc & 1, ok);
                if (!ok) goto done;
                ++qc;
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&hd->q_full));
                if (k == 0) {
                    wait_resolved();
                    if (!open()) continue;
                }
                const int nt = it.j1 - it.j0;
                const uint64_t rq2 = pack2(rq, rq);
                float frame = -INFINITY, l = 0.f;  // of this thread's tiles: the sum of e 2^-frame
                for (int e = (sc0 & 1) == (uint32_t)g ? 0 : 1; e < nt; e += 2, ++mine) {
                    const uint32_t sc = sc0 + e;
                    if (idle) {
                        if (!wait_on(sy, smem_u32(&hd->s_full[g]), mine & 1)) goto done;
                        if (lane == 0) mbar_arrive(smem_u32(&hd->s_free[g]));
                        continue;
                    }
                    if (!wait_on(sy, smem_u32(&hd->c_full[sc % kConsts]), (sc / kConsts) & 1)) goto done;
                    // the maximum so far comes from the other warp's tile and goes on to its next
                    if (sc > 0 && !wait_on(sy, smem_u32(&hd->m_bar[warp & 3][g ^ 1]), ((sc - 1) >> 1) & 1)) goto done;
                    const float before = e > 0 ? hd->m[g ^ 1][h] : -INFINITY;
                    if (!wait_on(sy, smem_u32(&hd->s_full[g]), mine & 1)) goto done;
                    tc_fence_after();
                    const KeyConst &c = consts[sc % kConsts];
                    float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll 1
                    for (int i0 = 0; i0 < kBK; i0 += 16) {
                        uint32_t sr[16];
                        tmem_ld16(s_at + i0, sr);
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            const ulonglong2 s4 = *reinterpret_cast<const ulonglong2 *>(&c.s[i0 + i]);
                            const ulonglong2 l4 = *reinterpret_cast<const ulonglong2 *>(&c.ls[i0 + i]);
                            const float2 a = unpack2(fma2(mul2(pack2(__uint_as_float(sr[i]), __uint_as_float(sr[i + 1])), rq2), s4.x, l4.x));
                            const float2 b = unpack2(fma2(mul2(pack2(__uint_as_float(sr[i + 2]), __uint_as_float(sr[i + 3])), rq2), s4.y, l4.y));
                            mx0 = max3(mx0, a.x, a.y);
                            mx1 = max3(mx1, b.x, b.y);
                        }
                    }
                    const float mx = fmaxf(mx0, mx1);
                    const float mn = e == 0 || mx > before + kRise ? mx : before;
                    hd->m[g][h] = mn;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&hd->m_bar[warp & 3][g]));
                    const float mb = mn - (kTop - kRise);  // the tile's frame (rounded: scores may be as large as 2^60)
                    const uint64_t mb2 = pack2(-mb, -mb);
                    // the last message has arrived, so its copies have left the staging buffer
                    if (!wait_on(sy, smem_u32(&hd->p_sent[g]), (mine & 1) ^ 1, true)) goto done;
                    uint64_t sum0 = 0, sum1 = 0;
#pragma unroll 1
                    for (int i0 = 0; i0 < kBK; i0 += 16) {
                        uint32_t sr[16], hp[8];
                        tmem_ld16(s_at + i0, sr);
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            const ulonglong2 s4 = *reinterpret_cast<const ulonglong2 *>(&c.s[i0 + i]);
                            const ulonglong2 l4 = *reinterpret_cast<const ulonglong2 *>(&c.ls[i0 + i]);
                            const ulonglong2 v4 = *reinterpret_cast<const ulonglong2 *>(&c.inv[i0 + i]);
                            const float2 a = unpack2(add2(fma2(mul2(pack2(__uint_as_float(sr[i]), __uint_as_float(sr[i + 1])), rq2), s4.x, l4.x), mb2));
                            const float2 b = unpack2(add2(fma2(mul2(pack2(__uint_as_float(sr[i + 2]), __uint_as_float(sr[i + 3])), rq2), s4.y, l4.y), mb2));
                            const float2 p0 = make_float2(ex2_approx(a.x), ex2_approx(a.y)), p1 = make_float2(ex2_approx(b.x), ex2_approx(b.y));
                            sum0 = fma2(pack2(p0.x, p0.y), v4.x, sum0);
                            sum1 = fma2(pack2(p1.x, p1.y), v4.y, sum1);
                            hp[i >> 1] = pack_half(p0.x, p0.y);
                            hp[(i >> 1) + 1] = pack_half(p1.x, p1.y);
                        }
                        // 8 keys a granule; keys 0 .. 63 in the 128-byte row, 64 .. 95 in the 64-byte row
                        const uint32_t row = i0 < 64 ? row1 + ((2 * i0) ^ (sw1 & 0x60)) : row2 + ((2 * i0 - 128) ^ (sw2 & 0x20));
                        const uint32_t sw = (i0 < 64 ? sw1 : sw2) & 0x10;
#pragma unroll
                        for (int v = 0; v < 2; ++v)
                            st_shared_v4(row + ((v << 4) ^ sw), hp[4 * v], hp[4 * v + 1], hp[4 * v + 2], hp[4 * v + 3]);
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&hd->s_free[g]));
                    float alpha = e > 0 && mn != before ? exp2f(before - (kTop - kRise) - mb) : 1.f;
                    if (mb != frame) {
                        l *= exp2f(frame - mb);  // 0 before the first tile
                        frame = mb;
                    }
                    const float2 s0 = unpack2(sum0), s1 = unpack2(sum1);
                    l += (s0.x + s0.y) + (s1.x + s1.y);
                    float fin = 0.f;
                    if (e == nt - 2) {  // the other warp ends the unit: it needs this one's sum, in the frame it ends with
                        hd->l[lc & 1][0][h] = l;
                        hd->l[lc & 1][1][h] = frame;
                        __syncwarp();
                        if (lane == 0) mbar_arrive(smem_u32(&hd->l_bar[warp & 3]));
                    } else if (e == nt - 1) {
                        float total = l;
                        if (nt > 1) {
                            if (!wait_on(sy, smem_u32(&hd->l_bar[warp & 3]), lc & 1)) goto done;
                            const float other = hd->l[lc & 1][0][h], theirs = hd->l[lc & 1][1][h];
                            total += theirs == mb ? other : other * exp2f(theirs - mb);
                        }
                        const float own = mb + log2f(total);
                        fin = 1.f / total;
                        if (it.np == 1) {
                            const float lse2 = log2_add(own, sink * 1.4426950408889634f);
                            fin *= exp2f(own - lse2);
                            if (p.lse && head) p.lse[(int64_t)it.t * p.N1 + h] = lse2 * 0.6931471805599453f;
                        } else if (head) {
                            p.part_s[((int64_t)it.t * p.P + it.piece) * p.N1 + h] = own;
                        }
                    }
                    // the sign bit of the warp's first alpha: some row of the warp has one
                    if (!head) alpha = 1.f;
                    const bool some = __any_sync(0xffffffffu, alpha != 1.f);
                    *reinterpret_cast<float2 *>(stage + kMsgStats + h * 8) =
                        make_float2(__uint_as_float(__float_as_uint(alpha) | (lane == 0 && some ? 0x80000000u : 0u)), fin);
                    fence_proxy_async_smem();
                    // only now must the peer be done with the slot: S has been free since the second pass
                    const uint32_t ps = sc % kSlots;
                    if (!wait_on(sy, smem_u32(&hd->p_empty[ps]), ((sc / kSlots) & 1) ^ 1, true)) goto done;
                    if (lane == 0) {
                        const uint32_t peer_msg = peer_msgs + ps * kMsgBytes, peer_full = peer_full0 + ps * 8;
                        const uint32_t w32 = (warp & 3) * 32, src = smem_u32(stage);
                        bulk_to_peer(peer_msg + w32 * 128, src + w32 * 128, 32 * 128, peer_full);
                        bulk_to_peer(peer_msg + kMsgLo + w32 * 64, src + kMsgLo + w32 * 64, 32 * 64, peer_full);
                        bulk_to_peer(peer_msg + kMsgStats + w32 * 8, src + kMsgStats + w32 * 8, 32 * 8, peer_full);
                    }
                }
                sc0 += nt;
                if (nt > 1) ++lc;
            }
            // the last message must have been read before this CTA may exit
            if (sc0 > 0 && !wait_on(sy, smem_u32(&hd->p_empty[(sc0 - 1) % kSlots]), ((sc0 - 1) / kSlots) & 1, true)) goto done;
        }
    } else {
        // ======================= output CTA =======================
        uint8_t *ring = smem + kOutRing, *msgs = smem + kOutMsgs;
        if (warp == kAckWarp) {  // messages that have arrived: their slots expect the next one, their staging is free
            uint32_t pc = 0;
            for (uint32_t k = 0;; ++k) {
                int u;
                if (!tq_read(p, sy, rank, k, u)) goto done;
                if (u < 0) break;
                const Item it = load_unit(p, u);
                if (it.skip) continue;
                for (int j = it.j0; j < it.j1; ++j, ++pc) {
                    const uint32_t bar = smem_u32(&hd->p_full[pc % kSlots]);
                    if (!wait_on(sy, bar, (pc / kSlots) & 1, true)) goto done;
                    if (lane == 0) {
                        mbar_arrive_expect_tx(bar, msg_bytes);
                        mbar_arrive_remote(map_to_cta(smem_u32(&hd->p_sent[pc & 1]), 0));
                    }
                    __syncwarp();
                }
            }
        } else if (warp >= kProdWarp0) {
            producer<false>(p, sy, nullptr, ring, hd, nullptr);
        } else if (warp == kMmaWarp) {
            constexpr uint32_t idesc = idesc_f8(128, 256, 1, 0), idesc5 = idesc_f8(128, 256, 1, 1);
            uint32_t st = 0, phase = 0, pc = 0, oc = 0, rsc = 0;
            for (uint32_t k = 0;; ++k) {
                int u;
                if (!tq_read(p, sy, rank, k, u)) goto done;
                if (u < 0) break;
                const Item it = load_unit(p, u);
                if (it.skip || it.j1 <= it.j0) continue;
                if (!wait_on(sy, smem_u32(&hd->o_empty), (oc & 1) ^ 1)) goto done;
                ++oc;
                for (int j = it.j0; j < it.j1; ++j, ++pc) {
                    const int ps = pc % kSlots;
                    if (!wait_on(sy, smem_u32(&hd->p_ready[ps]), (pc / kSlots) & 1)) goto done;
                    const uint8_t *msg = msgs + ps * kMsgBytes;
                    const bool last = j == it.j1 - 1, rescale = j > it.j0 && some_alpha(msg);
                    if (!wait_on(sy, smem_u32(&hd->full[st]), phase)) goto done;
                    fence_proxy_async_smem();  // the rows were written by cp.async
                    const uint64_t a1 = sdesc_sw128(smem_u32(msg), 16, 1024), a2 = sdesc_sw64(smem_u32(msg) + kMsgLo, 512);
                    const uint64_t a3 = sdesc_sw32(smem_u32(smem + kOutThirds) + ps * kThirdBytes, 768);
                    const uint32_t base = smem_u32(ring) + st * kVStage;
#pragma unroll 1
                    for (int c = 0; c < 2; ++c) {  // 256 value dims each
                        if (rescale && !wait_on(sy, smem_u32(&hd->rs_done[c]), rsc & 1)) goto done;
                        tc_fence_after();
                        if (elect_one()) {
                            const uint64_t b = sdesc_sw128(base + c * 2 * kSlab, kSlab, 1024);
                            const uint32_t d = tmem + c * 256;
#pragma unroll
                            for (int i = 0; i < kBK / 32; ++i) {
                                const uint64_t a = i < 2 ? a1 + 4 * i : a2;
                                mma8_ss(d, a, b + 256 * i, idesc, (j > it.j0 || i > 0) ? 1u : 0u);
                                mma8_ss(d, a + 2, b + 256 * i, idesc5, 1u);
                                mma8_ss(d, a3 + 16 * i, b + 256 * i, idesc5, 1u);
                            }
                            tc_commit(smem_u32(&hd->pv_done[c][ps]));
                        }
                        __syncwarp();
                    }
                    if (rescale) ++rsc;
                    if (elect_one()) {
                        tc_commit(smem_u32(&hd->empty[st]));
                        tc_commit_mc(smem_u32(&hd->p_empty[ps]), (uint16_t)1);
                        if (last) tc_commit(smem_u32(&hd->o_full));
                    }
                    __syncwarp();
                    if (++st == kVStages) {
                        st = 0;
                        phase ^= 1;
                    }
                }
            }
        } else {
            const int g = warp >> 2, h = threadIdx.x & 127;  // which half of the columns, head row
            const bool head = h < p.N1;
            const uint32_t trow = tmem + ((uint32_t)((warp & 3) * 32) << 16);
            const uint32_t sw1 = (h & 7) << 4, sw2 = ((h >> 1) & 3) << 4, sw3 = ((h >> 2) & 1) << 4;
            uint8_t *const thirds = smem + kOutThirds + (h >> 3) * 768 + (h & 7) * 32;
            uint32_t ofc = 0, pc = 0;
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
                float fin = 1.f;
                for (int j = it.j0; j < it.j1; ++j, ++pc) {
                    const int ps = pc % kSlots;
                    uint8_t *msg = msgs + ps * kMsgBytes;
                    if (!wait_on(sy, smem_u32(&hd->p_full[ps]), (pc / kSlots) & 1, true)) goto done;
                    const float2 stat = reinterpret_cast<const float2 *>(msg + kMsgStats)[h];
                    const bool rescale = j > it.j0 && some_alpha(msg);
                    fin = stat.y;
                    if (g == (int)(pc & 1)) {  // this warp's tile: its 32 heads' weights into codes
                        if ((warp & 3) < quads) {
                            // 32 keys at a time, hi and mid in the place of their weights (short code: one stretch for all 96
                            // keys takes 0.8 % more of a prefill's time)
#pragma unroll 1
                            for (int i = 0; i < kBK / 32; ++i) {
                                uint8_t *const row = i < 2 ? msg + h * 128 : msg + kMsgLo + h * 64;
                                const uint32_t g0 = i == 1 ? 64 : 0, sw = i < 2 ? sw1 : sw2;
                                uint4 x[4], y[4];
#pragma unroll
                                for (int c = 0; c < 4; ++c) x[c] = *reinterpret_cast<const uint4 *>(row + ((g0 + c * 16) ^ sw));
#pragma unroll
                                for (int c = 0; c < 2; ++c) {
                                    uint4 z;
                                    split4w(x[2 * c].x, x[2 * c].y, y[c].x, y[2 + c].x, z.x);
                                    split4w(x[2 * c].z, x[2 * c].w, y[c].y, y[2 + c].y, z.y);
                                    split4w(x[2 * c + 1].x, x[2 * c + 1].y, y[c].z, y[2 + c].z, z.z);
                                    split4w(x[2 * c + 1].z, x[2 * c + 1].w, y[c].w, y[2 + c].w, z.w);
                                    *reinterpret_cast<uint4 *>(thirds + ps * kThirdBytes + i * 256 + ((c << 4) ^ sw3)) = z;
                                }
#pragma unroll
                                for (int c = 0; c < 4; ++c) *reinterpret_cast<uint4 *>(row + ((g0 + c * 16) ^ sw)) = y[c];
                            }
                            fence_proxy_async_smem();
                        }
                    }
                    // every warp, so that none reads the factors of a message that has been overwritten
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&hd->p_ready[ps]));
                    if (!rescale) continue;
                    const float a = fabsf(stat.x);
                    const bool any = __any_sync(0xffffffffu, a != 1.f);
#pragma unroll 1
                    for (int c = 0; c < 2; ++c) {
                        // the product of the tile before, of these columns (a barrier per slot: several products
                        // may be outstanding, which one barrier's two phases cannot tell apart)
                        if (!wait_on(sy, smem_u32(&hd->pv_done[c][(pc - 1) % kSlots]), ((pc - 1) / kSlots) & 1)) goto done;
                        if (any) {
                            tc_fence_after();
#pragma unroll 1
                            for (int e = 0; e < 128; e += 64) {
                                const uint32_t at = trow + c * 256 + g * 128 + e;
                                uint32_t r0[32], r1[32];
                                tmem_ld32(at, r0);
                                tmem_ld32(at + 32, r1);
                                tc_wait_ld();
#pragma unroll
                                for (int i = 0; i < 32; ++i) {
                                    r0[i] = __float_as_uint(__uint_as_float(r0[i]) * a);
                                    r1[i] = __float_as_uint(__uint_as_float(r1[i]) * a);
                                }
                                tmem_st32(at, r0);
                                tmem_st32(at + 32, r1);
                            }
                            tc_wait_st();
                            tc_fence_before();
                        }
                        __syncwarp();
                        if (lane == 0) mbar_arrive(smem_u32(&hd->rs_done[c]));
                    }
                }
                if (!wait_on(sy, smem_u32(&hd->o_full), ofc & 1)) goto done;
                ++ofc;
                tc_fence_after();
                const uint32_t tcol = trow + g * (kDv / 2);
                // Each warp stages 64 bytes of its 32 head rows (64-byte swizzle) and writes them out: one TMA
                // store, or 64-byte pieces of rows where a box would reach into the next token's heads.  Whole
                // tokens in bf16, pieces in fp32, normalised within the piece.  (Direct stores, 16 bytes a lane
                // to 32 rows, took 9.5 us for a piece.)
                if ((warp & 3) * 32 < p.N1) {
                    uint8_t *const at = smem + kOutStage + warp * kWarpSlab;
                    const uint32_t buf = smem_u32(at);
                    const bool piece = it.np > 1;
                    const int row = piece ? ((it.t * p.P + it.piece) * p.NP + (warp & 3) * 32) : it.t * p.N1 + (warp & 3) * 32;
                    const int step = piece ? 16 : 32;
#pragma unroll 1
                    for (int c = 0; c < kDv / 2; c += step) {
                        uint32_t r[32], w[16];
                        tmem_ld32(tcol + (c & ~31), r);
                        if (lane == 0) bulk_wait_read<0>();  // the last store has read buf
                        __syncwarp();
                        tc_wait_ld();
                        if (piece) {
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                w[i] = __float_as_uint(__uint_as_float(c & 16 ? r[16 + i] : r[i]) * fin);
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                w[i] = pack_bf16(__uint_as_float(r[2 * i]) * fin, __uint_as_float(r[2 * i + 1]) * fin);
                        }
#pragma unroll
                        for (int cc = 0; cc < 4; ++cc)
                            st_shared_v4(buf + lane * 64 + ((cc ^ ((lane >> 1) & 3)) << 4), w[4 * cc], w[4 * cc + 1], w[4 * cc + 2],
                                         w[4 * cc + 3]);
                        if (piece || p.N1 % 32 == 0) {
                            fence_proxy_async_smem();
                            __syncwarp();
                            if (lane == 0) {
                                tma_store_2d(piece ? &part_map : &out_map, buf, g * (kDv / 2) + c, row);
                                bulk_commit();
                            }
                        } else {
                            __syncwarp();
#pragma unroll
                            for (int i = 0; i < 32; i += 8) {
                                const int e = i + (lane >> 2), q = lane & 3;
                                const uint4 v = *reinterpret_cast<const uint4 *>(at + e * 64 + ((q ^ ((e >> 1) & 3)) << 4));
                                if ((warp & 3) * 32 + e < p.N1)
                                    *reinterpret_cast<uint4 *>(reinterpret_cast<__nv_bfloat16 *>(p.out) + (int64_t)(row + e) * kDv +
                                                               g * (kDv / 2) + c + q * 8) = v;
                            }
                            __syncwarp();  // buf is written again
                        }
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
// Block (t, h), thread = 4 columns.  Latency bound: the record, the sums and the first pieces' columns
// are loaded together, before the number of pieces is known (the slots of all P exist).  About 4 us for
// 23 pieces; two groups of threads with 12 pieces each ahead took 0.5 us off.
__global__ void __launch_bounds__(kDv / 4) fp8_combine_kernel(const TcArgs p) {
    constexpr int kAhead = 8;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int t = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
    const int64_t s0 = (int64_t)t * p.P;
    const float4 *po = reinterpret_cast<const float4 *>(p.part_o + (s0 * p.NP + h) * kDv) + tid;
    const int64_t stride = (int64_t)p.NP * kDv / 4;
    float4 o[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
        if (i < p.P) o[i] = __ldcg(po + i * stride);
    // every warp holds the sums of all pieces, two a lane
    const float r0 = lane < p.P ? __ldcg(p.part_s + (s0 + lane) * p.N1 + h) : -INFINITY;
    const float r1 = lane + 32 < p.P ? __ldcg(p.part_s + (s0 + lane + 32) * p.N1 + h) : -INFINITY;
    const float sink = p.sinks ? __ldg(p.sinks + h) * 1.4426950408889634f : -INFINITY;
    const int np = load_unit(p, t).np;
    if (np == 1) return;  // written by the attention kernel
    const float own0 = lane < np ? r0 : -INFINITY, own1 = lane + 32 < np ? r1 : -INFINITY;
    const bool bad = __any_sync(0xffffffffu, own0 != own0 || own1 != own1);
    float top = fmaxf(fmaxf(own0, own1), sink);
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    // pieces always hold a key, so that their sums are finite unless something is NaN
    float sum = exp2f(own0 - top) + exp2f(own1 - top);
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const float lse2 = bad ? NAN : top == INFINITY ? top : top + log2f(sum + exp2f(sink - top));
    const float w0 = exp2f(own0 - lse2), w1 = exp2f(own1 - lse2);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](int i, const float4 &v) {
        const float w = __shfl_sync(0xffffffffu, i < 32 ? w0 : w1, i & 31);
        acc.x = fmaf(w, v.x, acc.x);
        acc.y = fmaf(w, v.y, acc.y);
        acc.z = fmaf(w, v.z, acc.z);
        acc.w = fmaf(w, v.w, acc.w);
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
        if (i < np) add(i, o[i]);
#pragma unroll 4
    for (int i = kAhead; i < np; ++i) add(i, __ldcg(po + i * stride));
    uint2 *out = reinterpret_cast<uint2 *>(reinterpret_cast<__nv_bfloat16 *>(p.out) + ((int64_t)t * p.N1 + h) * kDv) + tid;
    *out = make_uint2(pack_bf16(acc.x, acc.y), pack_bf16(acc.z, acc.w));
    if (p.lse && tid == 0) p.lse[(int64_t)t * p.N1 + h] = lse2 * 0.6931471805599453f;
}

// Tensor map over [rows][D] bf16 or fp32, boxes of 32 rows x 128 bytes (128-byte swizzle) or 64 (64-byte).
int make_map(CUtensorMap *map, const void *base, int64_t rows, int D, bool fp32, uint32_t bytes) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return SAS_ERR_CUDA;
    if (rows >= INT32_MAX) return SAS_ERR_UNSUPPORTED;
    const uint32_t size = fp32 ? 4 : 2;
    cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)D * size};
    cuuint32_t box[2] = {bytes / size, 32};
    cuuint32_t estr[2] = {1, 1};
    const CUresult r = fn(map, fp32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                          const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? SAS_OK : SAS_ERR_CUDA;
}

constexpr int kClusters = 74;  // 148 SMs / 2
constexpr int kMinPieceTiles = 1;
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
    const int64_t est = (win + cmp + kBK - 1) / kBK;
    int64_t P = std::min<int64_t>(kClusters / a.num_tokens, (est + kMinPieceTiles - 1) / kMinPieceTiles);
    P = std::min<int64_t>(P, kMaxPieces);
    if (P <= 1) return pl;
    pl.M = (int)((est + P - 1) / P);
    pl.P = (int)((est + pl.M - 1) / pl.M);
    const int64_t bytes = (int64_t)a.num_tokens * pl.P * ((a.num_heads + 31) / 32 * 32) * kDv * 4;
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
    p.ori_div = make_div((uint32_t)p.ori_bs);
    p.cmp_div = make_div((uint32_t)p.cmp_bs);
    const Plan pl = plan(a);
    p.status = reinterpret_cast<uint32_t *>(p.rec + TR_STATUS);  // record 0 carries what no token is known for
    p.P = pl.P;
    p.M = pl.M;
    if ((int64_t)a.num_tokens * pl.P >= INT32_MAX) return SAS_ERR_UNSUPPORTED;
    p.U = a.num_tokens * pl.P;
    p.part_o = reinterpret_cast<float *>(ws + L.part_o);
    p.part_s = reinterpret_cast<float *>(ws + L.part_s);
    p.NP = (p.N1 + 31) / 32 * 32;
    CUtensorMap q_map, out_map, part_map;
    int rc = make_map(&q_map, p.q, (int64_t)p.T * p.N1, p.Dq, false, 128);
    if (!rc) rc = make_map(&out_map, p.out, (int64_t)p.T * p.N1, kDv, false, 64);
    part_map = out_map;
    if (!rc && p.P > 1) rc = make_map(&part_map, p.part_o, (int64_t)p.T * p.P * p.NP, kDv, true, 64);
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
    if (check_cuda(cudaLaunchKernelEx(&cfg, fp8_tc_kernel, p, q_map, out_map, part_map))) return SAS_ERR_CUDA;
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
