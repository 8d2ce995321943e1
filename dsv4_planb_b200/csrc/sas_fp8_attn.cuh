// What the kernels of the attention over an 8-bit cache share: arguments, token records, sink.
#pragma once

#include <algorithm>

#include "sas_common.cuh"
#include "sas_fp8.cuh"

namespace sas_fp8 {

// Per-token record of the resolve kernel, int32 each.
enum TokenRec : int {
    TR_B = 0,       // request
    TR_LEFT = 1,    // first window position
    TR_FIRST = 2,   // first positions in front of the window
    TR_NORI = 3,    // first + window keys
    TR_NCMP = 4,    // compressed keys
    TR_VALID = 5,   // the row belongs to a request
    TR_STATUS = 6,  // SAS_STATUS_* bits found for this token (resolve stores, attention ORs)
    TR_PAD = 7,
    TR_INTS = 8
};

struct Layout {
    size_t head;   // status word (for sas_kvq_read_status) and the unit counter
    size_t rec;    // int32 [T][TR_INTS]
    size_t rows;   // int32 [T][topk]: physical compressed rows (scenario 3), -1: a zero row
    size_t part_o; // split tokens: fp32 [T][P][N1 rounded up to 32][Dv]
    size_t part_s; // split tokens: fp32 [T][P][N1]: log2 of the piece's weight sum
    size_t total;
};
constexpr size_t kCounterOff = 64;

struct Args {
    const void *q;
    const uint8_t *ori, *cmp;
    const float *ori_scale, *cmp_scale, *sinks;
    const int32_t *ori_bt, *cmp_bt, *idx, *cu, *act_q, *act_kv;
    void *out;
    float *lse;
    int32_t *rec, *rows;
    int *counter;
    int B, T, q_rows, N1, Dq, Dv, K, ratio, scenario, win_left, first;
    int ori_block_num, ori_bs, ori_table_len, cmp_block_num, cmp_bs, cmp_table_len;
    float scale_log2;
};

// Physical row of position pos of request b, or -1 (a zero row): an unmapped block, a bad table entry
// or a position past the table (these two are reported).
__device__ __forceinline__ int32_t paged_row(const int32_t *__restrict__ table, int b, int len, int bs, int block_num,
                                             int pos, uint32_t &bits) {
    const int blk = pos / bs;
    int32_t phys = -1;
    if (blk < len) phys = __ldg(table + (int64_t)b * len + blk);
    else bits |= SAS_STATUS_BAD_BLOCK;
    if (phys >= block_num || phys < -1) bits |= SAS_STATUS_BAD_BLOCK;
    return phys < 0 || phys >= block_num ? -1 : phys * bs + (pos - blk * bs);
}

// The scale of a physical row, or 0 where its block has none: the row then reads as zeros.
__device__ __forceinline__ float row_scale(const float *__restrict__ scale, int bs, int32_t row, uint32_t &bits) {
    if (row < 0) return 0.f;
    const float s = __ldg(scale + row / bs);
    if (!scale_ok(s)) {
        bits |= SAS_STATUS_BAD_SCALE;
        return 0.f;
    }
    return s;
}

__device__ __forceinline__ int ori_position(const int32_t *rec, int slot) {
    return slot < rec[TR_FIRST] ? slot : rec[TR_LEFT] + slot - rec[TR_FIRST];
}

// log2(2^a + 2^b)
__device__ __forceinline__ float log2_add(float a, float b) {
    if (a != a || b != b) return NAN;  // fmaxf would drop it
    const float hi = fmaxf(a, b), lo = fminf(a, b);
    if (hi == INFINITY || lo == -INFINITY) return hi;
    return hi + log2f(1.f + exp2f(lo - hi));
}

} // namespace sas_fp8

namespace sas_host {
bool fp8_tc_supported(const SasFp8Args &a);
size_t fp8_tc_pieces(const SasFp8Args &a);  // pieces per token of the split plan (1: whole tokens)
int launch_fp8_tc(const SasFp8Args &a, const sas_fp8::Args &p, const sas_fp8::Layout &L, char *ws, cudaStream_t s);
int launch_fp8_simt(const SasFp8Args &a, const sas_fp8::Args &p, cudaStream_t s);
} // namespace sas_host
