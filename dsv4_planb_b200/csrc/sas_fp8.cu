// C entry points of the attention over an 8-bit cache (argument checks, workspace, launches) and the
// kernel that resolves every token's keys.
//
// resolve_kernel writes one record per flat row, whatever it belongs to, so that nothing has to be
// cleared before it: status bits live in the records and sas_kvq_read_status gathers them.  For
// scenario 3 it also maps the token's compressed indices to physical rows: the scan of a row of
// indices stops at the first -1 or after min(K, limit) slots, skips what is out of range, keeps
// duplicates and slot order.  Latency bound: its loads of the indices start before the request of
// the row is known.  About 3 us of a decode step's 29, most of them beside the launch of the attention.

#include "sas_fp8_attn.cuh"

using namespace sas_fp8;

namespace {

constexpr int kThreads = 256;
constexpr int kPer = 8;

__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Record of flat row t (warp-uniform; every lane calls).  `limit`: compressed rows below it are visible.
// `found(b)` runs as soon as the row's request is known (-1: none).
template <class F>
__device__ __forceinline__ void make_record(const Args &p, int t, int32_t (&r)[TR_INTS], int &limit, F found) {
    int b, s = 0, n = 0;
    if (p.cu) {
        b = find_request(p.cu, p.B, t);
        if (b >= 0) {
            const int c0 = __ldg(p.cu + b);
            s = t - c0;
            n = __ldg(p.cu + b + 1) - c0;
        }
    } else {
        b = t / p.q_rows;
        s = t - b * p.q_rows;
        if (b >= p.B) b = -1;
        else n = p.act_q ? min(__ldg(p.act_q + b), p.q_rows) : p.q_rows;
    }
    found(b);
    const bool valid = b >= 0 && s < n;
    const int64_t pos = valid ? (int64_t)__ldg(p.act_kv + b) - n + s : -1;
    const int g = (int)max(pos, (int64_t)-1);
    const int left = max(g - p.win_left, 0);
    const int first = g >= 0 ? min(p.first, left) : 0;
    limit = p.scenario >= 2 && g >= 0 ? (g + 1) / p.ratio : 0;
    r[TR_B] = b;
    r[TR_LEFT] = left;
    r[TR_FIRST] = first;
    r[TR_NORI] = g >= 0 ? first + g - left + 1 : 0;
    r[TR_NCMP] = p.scenario == 2 ? limit : 0;
    r[TR_VALID] = valid ? 1 : 0;
    r[TR_STATUS] = 0;
    r[TR_PAD] = 0;
}

__device__ __forceinline__ void store_record(const Args &p, int t, const int32_t (&r)[TR_INTS]) {
    int4 *d = reinterpret_cast<int4 *>(p.rec + (int64_t)t * TR_INTS);
    d[0] = make_int4(r[0], r[1], r[2], r[3]);
    d[1] = make_int4(r[4], r[5], r[6], r[7]);
}

// Scenarios 1 and 2: a warp per token.
__global__ void __launch_bounds__(kThreads) resolve_kernel(Args p) {
    launch_dependents();
    const int t = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    if (t == 0 && (threadIdx.x & 31) == 0) *p.counter = 0;
    if (t >= p.T) return;
    int32_t r[TR_INTS];
    int limit;
    make_record(p, t, r, limit, [](int) {});
    if ((threadIdx.x & 31) == 0) store_record(p, t, r);
}

// Scenario 3: a CTA per token.
__global__ void __launch_bounds__(kThreads) resolve_rows_kernel(Args p) {
    __shared__ int warp_sum[kThreads / 32];
    __shared__ int stop_s;
    __shared__ unsigned int bits_s;
    launch_dependents();
    const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (t == 0 && tid == 0) *p.counter = 0;
    const int32_t *idx = p.idx + (int64_t)t * p.K;
    int v[kPer];
    auto load = [&](int base) {
        const int i0 = base + tid * kPer;
        if (i0 + kPer <= p.K && (reinterpret_cast<uintptr_t>(idx + i0) & 15) == 0) {
            const int4 a = __ldg(reinterpret_cast<const int4 *>(idx + i0)), b = __ldg(reinterpret_cast<const int4 *>(idx + i0) + 1);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
#pragma unroll
            for (int k = 0; k < kPer; ++k) v[k] = i0 + k < p.K ? __ldg(idx + i0 + k) : -1;
        }
    };
    load(0);
    int32_t r[TR_INTS];
    int limit;
    // the table's entries need the request only: their loads run beside that of its length
    int32_t phys[kPer];
    auto look_up = [&](int b) {
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const int blk = max(v[k], 0) / p.cmp_bs;
            phys[k] = b >= 0 && blk < p.cmp_table_len ? __ldg(p.cmp_bt + (int64_t)b * p.cmp_table_len + blk) : -2;
        }
    };
    make_record(p, t, r, limit, look_up);
    if (tid == 0) {
        stop_s = 0x7fffffff;
        bits_s = 0;
    }
    __syncthreads();
    int32_t *rows = p.rows + (int64_t)t * p.K;
    int kept = 0;
    uint32_t bits = 0;
    // Every thread leaves by its own copy of `end`, which is the same in all of them: stop_s changes only between
    // a chunk's start and its first barrier, and is read only between the first and the second.
    int end = min(p.K, limit);
    for (int base = 0; base < end; base += kThreads * kPer) {
        if (base > 0) {
            load(base);
            look_up(r[TR_B]);
        }
        const int i0 = base + tid * kPer;
        int stop = 0x7fffffff;
#pragma unroll
        for (int k = kPer - 1; k >= 0; --k)
            if (v[k] == -1) stop = i0 + k;
        if (stop != 0x7fffffff) atomicMin(&stop_s, stop);
        __syncthreads();
        end = min(end, stop_s);
        int32_t row[kPer];
        int cnt = 0;
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            row[k] = -2;
            if (i0 + k < end) {
                if (v[k] < -1) bits |= SAS_STATUS_BAD_INDEX;
                if (v[k] >= 0 && v[k] < limit) {
                    const bool bad = phys[k] < -1 || phys[k] >= p.cmp_block_num;
                    if (bad) bits |= SAS_STATUS_BAD_BLOCK;
                    row[k] = bad || phys[k] < 0 ? -1 : phys[k] * p.cmp_bs + v[k] % p.cmp_bs;
                    ++cnt;
                }
            }
        }
        int incl = cnt;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        if (lane == 31) warp_sum[warp] = incl;
        __syncthreads();
        int at = kept + incl - cnt;
        for (int w = 0; w < kThreads / 32; ++w) {
            if (w < warp) at += warp_sum[w];
            kept += warp_sum[w];
        }
#pragma unroll
        for (int k = 0; k < kPer; ++k)
            if (row[k] != -2) rows[at++] = row[k];
    }
    if (bits) atomicOr(&bits_s, bits);
    __syncthreads();
    if (tid == 0) {
        r[TR_NCMP] = kept;
        r[TR_STATUS] = (int32_t)bits_s;
        store_record(p, t, r);
    }
}

__global__ void __launch_bounds__(kThreads) gather_status_kernel(const int32_t *rec, int T, uint32_t *word) {
    uint32_t bits = 0;
    for (int t = threadIdx.x; t < T; t += kThreads) bits |= (uint32_t)rec[(int64_t)t * TR_INTS + TR_STATUS];
    if (threadIdx.x == 0) *word = 0;
    __syncthreads();
    if (bits) atomicOr(word, bits);
}

int validate(const SasFp8Args &a) {
    if (a.batch < 0 || a.num_tokens < 0 || a.max_q_len < 0 || a.num_heads <= 0 || a.head_dim <= 0 || a.v_head_dim <= 0)
        return SAS_ERR_INVALID_ARG;
    if (a.scenario < 1 || a.scenario > 3 || a.ori_win_left < 0 || a.ori_first < 0 || a.topk < 0)
        return SAS_ERR_INVALID_ARG;
    if (a.dtype != SAS_DTYPE_BF16 && a.dtype != SAS_DTYPE_FP16) return SAS_ERR_INVALID_ARG;
    if (a.ori_block_num <= 0 || a.ori_block_size <= 0 || a.ori_table_len <= 0) return SAS_ERR_INVALID_ARG;
    if (a.scenario >= 2 &&
        (a.cmp_block_num <= 0 || a.cmp_block_size <= 0 || a.cmp_table_len <= 0 || a.cmp_ratio <= 0))
        return SAS_ERR_INVALID_ARG;
    if (a.kernel != SAS_KERNEL_AUTO && a.kernel != SAS_KERNEL_SIMT && a.kernel != SAS_KERNEL_TC) return SAS_ERR_INVALID_ARG;
    for (int i = 0; i < 4; ++i)
        if (a.reserved[i] != 0) return SAS_ERR_INVALID_ARG;
    if (a.head_dim % 16 != 0 || a.head_dim > 1024) return SAS_ERR_UNSUPPORTED;
    if (a.v_head_dim > a.head_dim || a.v_head_dim % 32 != 0 || a.v_head_dim > 512) return SAS_ERR_UNSUPPORTED;
    if (a.num_heads > 16 * 65535) return SAS_ERR_UNSUPPORTED;
    if ((int64_t)a.ori_block_num * a.ori_block_size >= ((int64_t)1 << 31)) return SAS_ERR_UNSUPPORTED;
    if (a.scenario >= 2 && (int64_t)a.cmp_block_num * a.cmp_block_size >= ((int64_t)1 << 31)) return SAS_ERR_UNSUPPORTED;
    if (a.kernel == SAS_KERNEL_TC && !sas_host::fp8_tc_supported(a)) return SAS_ERR_UNSUPPORTED;
    return SAS_OK;
}

bool use_tc(const SasFp8Args &a) { return a.kernel != SAS_KERNEL_SIMT && sas_host::fp8_tc_supported(a); }

Layout layout_of(const SasFp8Args &a) {
    Layout L{};
    size_t off = 0;
    auto take = [&](size_t bytes) { size_t o = off; off = sas::align_up(off + bytes); return o; };
    const size_t T = (size_t)a.num_tokens;
    L.head = take(sas::kAlign);
    L.rec = take(sizeof(int32_t) * TR_INTS * T);
    L.rows = take(a.scenario == 3 ? sizeof(int32_t) * (size_t)a.topk * T : 0);
    const size_t P = use_tc(a) ? sas_host::fp8_tc_pieces(a) : 1;
    const size_t slots = P > 1 ? T * P : 0, N1 = (size_t)a.num_heads;
    L.part_o = take(slots * ((N1 + 31) / 32 * 32) * (size_t)a.v_head_dim * sizeof(float));
    L.part_s = take(slots * N1 * sizeof(float));
    L.total = off;
    return L;
}

bool aligned(const void *p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

} // namespace

extern "C" {

int sas_kvq_workspace_size(const SasFp8Args *args, size_t *bytes) {
    if (!args || !bytes) return SAS_ERR_INVALID_ARG;
    const int rc = validate(*args);
    if (rc) return rc;
    *bytes = layout_of(*args).total;
    return SAS_OK;
}

int sas_kvq_forward(const SasFp8Args *args, const void *q, const void *ori_kv, const float *ori_scale,
                    const int32_t *ori_block_table, const void *cmp_kv, const float *cmp_scale,
                    const int32_t *cmp_block_table, const int32_t *cmp_indices, const int32_t *cu_seqlens_q,
                    const int32_t *act_q_len, const int32_t *act_kv_len, const float *sinks, void *out, float *lse,
                    void *workspace, size_t workspace_bytes, void *stream) {
    if (!args) return SAS_ERR_INVALID_ARG;
    const SasFp8Args &a = *args;
    const int rc = validate(a);
    if (rc) return rc;
    if (!cu_seqlens_q && a.num_tokens > 0 && (a.max_q_len <= 0 || (int64_t)a.batch * a.max_q_len != a.num_tokens))
        return SAS_ERR_INVALID_ARG;
    const Layout L = layout_of(a);
    if (!workspace || workspace_bytes < L.total) return SAS_ERR_WORKSPACE;
    const bool rows = a.num_tokens > 0, owned = rows && a.batch > 0;  // with no request the tables may be empty
    if (rows && (!q || !out || !ori_kv || !ori_scale)) return SAS_ERR_INVALID_ARG;
    if (owned && (!ori_block_table || !act_kv_len)) return SAS_ERR_INVALID_ARG;
    if (rows && a.scenario >= 2 && (!cmp_kv || !cmp_scale || (owned && !cmp_block_table))) return SAS_ERR_INVALID_ARG;
    if (a.num_tokens > 0 && a.scenario == 3 && a.topk > 0 && !cmp_indices) return SAS_ERR_INVALID_ARG;
    for (const void *x : {q, ori_kv, cmp_kv, (const void *)out, (const void *)workspace})
        if (!aligned(x, 16)) return SAS_ERR_INVALID_ARG;
    for (const void *x : {(const void *)ori_scale, (const void *)ori_block_table, (const void *)cmp_scale,
                          (const void *)cmp_block_table, (const void *)cmp_indices, (const void *)cu_seqlens_q,
                          (const void *)act_q_len, (const void *)act_kv_len, (const void *)sinks, (const void *)lse})
        if (!aligned(x, 4)) return SAS_ERR_INVALID_ARG;
    char *ws = static_cast<char *>(workspace);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a.num_tokens == 0) return SAS_OK;
    Args p;
    p.q = q;
    p.ori = static_cast<const uint8_t *>(ori_kv);
    p.cmp = static_cast<const uint8_t *>(cmp_kv);
    p.ori_scale = ori_scale;
    p.cmp_scale = cmp_scale;
    p.sinks = sinks;
    p.ori_bt = ori_block_table;
    p.cmp_bt = cmp_block_table;
    p.idx = cmp_indices;
    p.cu = cu_seqlens_q;
    p.act_q = act_q_len;
    p.act_kv = act_kv_len;
    p.out = out;
    p.lse = lse;
    p.rec = reinterpret_cast<int32_t *>(ws + L.rec);
    p.rows = reinterpret_cast<int32_t *>(ws + L.rows);
    p.counter = reinterpret_cast<int *>(ws + L.head + kCounterOff);
    p.B = a.batch;
    p.T = a.num_tokens;
    p.q_rows = std::max(a.max_q_len, 1);
    p.N1 = a.num_heads;
    p.Dq = a.head_dim;
    p.Dv = a.v_head_dim;
    p.K = a.scenario == 3 ? a.topk : 0;
    p.ratio = std::max(a.cmp_ratio, 1);
    p.scenario = a.scenario;
    p.win_left = a.ori_win_left;
    p.first = a.ori_first;
    p.ori_block_num = a.ori_block_num;
    p.ori_bs = a.ori_block_size;
    p.ori_table_len = a.ori_table_len;
    p.cmp_block_num = a.cmp_block_num;
    p.cmp_bs = std::max(a.cmp_block_size, 1);
    p.cmp_table_len = a.cmp_table_len;
    p.scale_log2 = a.softmax_scale * 1.4426950408889634f;
    if (a.scenario == 3) resolve_rows_kernel<<<a.num_tokens, kThreads, 0, s>>>(p);
    else resolve_kernel<<<(a.num_tokens + kThreads / 32 - 1) / (kThreads / 32), kThreads, 0, s>>>(p);
    if (sas_host::check_cuda(cudaGetLastError())) return SAS_ERR_CUDA;
    return use_tc(a) ? sas_host::launch_fp8_tc(a, p, L, ws, s) : sas_host::launch_fp8_simt(a, p, s);
}

int sas_kvq_read_status(const SasFp8Args *args, void *workspace, uint32_t *status, void *stream) {
    if (!args || !workspace || !status) return SAS_ERR_INVALID_ARG;
    const int rc = validate(*args);
    if (rc) return rc;
    *status = 0;
    if (args->num_tokens == 0) return SAS_OK;
    const Layout L = layout_of(*args);
    char *ws = static_cast<char *>(workspace);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    gather_status_kernel<<<1, kThreads, 0, s>>>(reinterpret_cast<const int32_t *>(ws + L.rec), args->num_tokens,
                                                reinterpret_cast<uint32_t *>(ws + L.head));
    if (sas_host::check_cuda(cudaGetLastError())) return SAS_ERR_CUDA;
    return sas_read_status(ws + L.head, status, stream);
}

} // extern "C"
