// Writing the paged K = V cache: new rows appended at their positions, with the rotation of the
// positional tail (of the rows and, where given, of the query heads) applied on the way.
//
// Token t of request b sits at position pos = act_kv[b] - n + s (s its index among the request's n
// new tokens) and goes to cache row (block_table[b][pos / bs], pos % bs).  Its last R dims turn by
// the angles of row rope_step * pos of a (cos | sin) table: (a, b) -> (a c - b s, a s + b c), pairs
// adjacent (interleaved) or R / 2 apart, in fp32, rounded once to the cache's type.  The other dims
// of a 16-bit cache are copied bit by bit.
//
// An 8-bit cache holds e4m3 codes and one power-of-two scale per block of tokens.  With A the
// largest finite |x| of the call's rows of a block, need = min 2^k >= A / 448 (k in [-60, 60]); a
// block whose row 0 is among the new rows takes need, any other max(old, need).  A scale that rises
// is shared by the rows already there: their codes are rounded again, code * old / new, which for
// powers of two moves the exponent and loses nothing above e4m3's subnormals.  Powers of two are
// taken for that reason: with scales A / 448 every growth would round every old row anew.
//
// Bound: bytes (each row read once and written once).  A decode call is one launch latency.

#include <algorithm>

#include "sas_common.cuh"
#include "sas_fp8.cuh"
#include "sas_tc_ptx.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kQHeads = 16;  // query heads per CTA of the q part
constexpr int kMaxChunks = 4;  // 16-byte chunks of a row per lane: D <= 1024

struct AppendArgs {
    const char *kv, *q;
    char *q_out, *cache;
    float *scale;
    const float *rope;
    const int32_t *table, *cu, *act_q, *act_kv;
    uint32_t *status;
    int64_t kv_stride;  // elements between kv rows
    int B, T, N1, D, R, interleaved, step, rope_rows;
    int block_num, bs, table_len, q_rows;  // q_rows: rows a request spans without cu (BSND)
    int nq;  // CTAs of the q part (a multiple of the cluster size)
};

template <typename T> __device__ __forceinline__ void unpack8(const uint4 v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = sas::DT<T>::to_f2(w[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}

template <typename T> __device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
    union { T h[8]; uint4 v; } u;
#pragma unroll
    for (int i = 0; i < 8; ++i) u.h[i] = sas::DT<T>::from_f(x[i]);
    return u.v;
}

// Chunk c (8 dims) of `row` in fp32, turned by the angles `cs` (R floats, cos then sin) where it
// lies in the last R dims.
template <typename T>
__device__ __forceinline__ void load_rotated(const AppendArgs &p, const uint4 *row, const float *cs, int c,
                                             float (&x)[8]) {
    unpack8<T>(row[c], x);  // a plain load: q may be turned in place
    const int d = c * 8 - (p.D - p.R);
    if (d < 0) return;
    const int half = p.R >> 1;
    if (p.interleaved) {
        const float4 co = __ldg(reinterpret_cast<const float4 *>(cs + (d >> 1)));
        const float4 si = __ldg(reinterpret_cast<const float4 *>(cs + half + (d >> 1)));
        const float cc[4] = {co.x, co.y, co.z, co.w}, ss[4] = {si.x, si.y, si.z, si.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = x[2 * i], b = x[2 * i + 1];
            x[2 * i] = a * cc[i] - b * ss[i];
            x[2 * i + 1] = a * ss[i] + b * cc[i];
        }
    } else {
        const bool low = d < half;
        const int e = low ? d : d - half;  // index of the pair
        float y[8];
        unpack8<T>(row[low ? c + half / 8 : c - half / 8], y);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float co = __ldg(cs + e + i), si = __ldg(cs + half + e + i);
            x[i] = low ? x[i] * co - y[i] * si : y[i] * si + x[i] * co;
        }
    }
}

// The new tokens of request b: the position of its first one, its first row among the T flat rows,
// and how many rows there are (clipped to T and to positions >= 0).
struct Span {
    int64_t pos;
    int row, n;
};
__device__ __forceinline__ Span span_of(const AppendArgs &p, int b) {
    int64_t row;
    int n;
    if (p.cu) {
        row = __ldg(p.cu + b);
        n = __ldg(p.cu + b + 1) - (int)row;
    } else {
        row = (int64_t)b * p.q_rows;
        n = p.act_q ? min(__ldg(p.act_q + b), p.q_rows) : p.q_rows;
    }
    Span sp;
    sp.pos = (int64_t)__ldg(p.act_kv + b) - n;
    if (sp.pos < 0) {  // tokens before the sequence's start have no place
        row -= sp.pos;
        n += (int)sp.pos;
        sp.pos = 0;
    }
    if (row < 0 || row >= p.T) n = 0;
    sp.row = (int)row;
    sp.n = (int)min((int64_t)n, (int64_t)p.T - row);
    return sp;
}

// Position of flat row t, or -1 where it belongs to no request (warp-uniform; every lane calls).
__device__ __forceinline__ int64_t position_of(const AppendArgs &p, int t, int &b) {
    b = p.cu ? sas_fp8::find_request(p.cu, p.B, t) : t / p.q_rows;
    if (b < 0 || b >= p.B) return -1;
    const Span sp = span_of(p, b);
    const int i = t - sp.row;
    return i >= 0 && i < sp.n ? sp.pos + i : -1;
}

// Angles of a position, or nullptr past the table's end.
__device__ __forceinline__ const float *angles(const AppendArgs &p, int64_t pos) {
    const int64_t r = pos * p.step;
    if (p.R > 0 && r >= p.rope_rows) {
        sas::set_status(p.status, SAS_STATUS_BAD_POSITION);
        return nullptr;
    }
    return p.rope + r * p.R;
}

__device__ __forceinline__ int64_t block_of(const AppendArgs &p, int b, int64_t blk) {
    int32_t phys = -1;
    if (blk < p.table_len) phys = __ldg(p.table + (int64_t)b * p.table_len + blk);
    if (phys < 0 || phys >= p.block_num) {
        sas::set_status(p.status, SAS_STATUS_BAD_BLOCK);
        return -1;
    }
    return phys;
}

// Query heads [16 y, 16 y + 16) of a token, turned by the token's angles; rows of no request (and of
// positions past the table) are copied as they are.  In place only the turned dims move.
template <typename T> __device__ void rotate_q(const AppendArgs &p, int cta) {
    const int groups = (p.N1 + kQHeads - 1) / kQHeads;
    const int t = cta / groups, h0 = (cta - t * groups) * kQHeads;
    if (t >= p.T) return;
    int b;
    const int64_t pos = position_of(p, t, b);
    const float *cs = pos >= 0 ? angles(p, pos) : nullptr;
    const bool in_place = p.q == p.q_out;
    if (in_place && cs == nullptr) return;
    const int c0 = in_place ? (p.D - p.R) / 8 : 0, nc = p.D / 8 - c0;
    const int heads = min(kQHeads, p.N1 - h0);
    const int64_t base = ((int64_t)t * p.N1 + h0) * (p.D / 8);
    const int total = heads * nc;
    // pairs that lie R / 2 apart are read by two threads: in place, all loads of a round come before
    // its stores, and a round holds whole heads
    const int round = in_place && !p.interleaved ? max(1, kThreads / nc) * nc : kThreads;
    for (int i0 = 0; i0 < total; i0 += round) {
        const int i = i0 + threadIdx.x;
        const bool live = (int)threadIdx.x < round && i < total;
        float x[8];
        uint4 raw = make_uint4(0, 0, 0, 0);
        int64_t at = 0;
        bool turned = false;
        if (live) {
            const int h = i / nc, c = c0 + i - h * nc;
            at = base + (int64_t)h * (p.D / 8);
            const uint4 *row = reinterpret_cast<const uint4 *>(p.q) + at;
            turned = cs != nullptr && c * 8 >= p.D - p.R;
            if (turned) load_rotated<T>(p, row, cs, c, x);
            else raw = row[c];
            at += c;
        }
        if (in_place) __syncthreads();
        if (live) reinterpret_cast<uint4 *>(p.q_out)[at] = turned ? pack8<T>(x) : raw;
    }
}

// 16-bit cache: a warp per new row.
template <typename T> __global__ void __launch_bounds__(kThreads) append16_kernel(AppendArgs p) {
    if ((int)blockIdx.x < p.nq) {
        rotate_q<T>(p, blockIdx.x);
        return;
    }
    const int t = ((int)blockIdx.x - p.nq) * kWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (t >= p.T) return;
    const uint4 *row = reinterpret_cast<const uint4 *>(p.kv + (int64_t)t * p.kv_stride * 2);
    const int nc = p.D / 8;
    int b;
    const int64_t pos = position_of(p, t, b);
    if (pos < 0) return;
    const int64_t blk = pos / p.bs, phys = block_of(p, b, blk);
    const float *cs = angles(p, pos);
    if (phys < 0 || cs == nullptr) return;
    uint4 *dst = reinterpret_cast<uint4 *>(p.cache) + (phys * p.bs + (pos - blk * p.bs)) * nc;
    for (int c = lane; c < nc; c += 32) {
        if (c * 8 < p.D - p.R) {
            dst[c] = __ldg(row + c);
        } else {
            float x[8];
            load_rotated<T>(p, row, cs, c, x);
            dst[c] = pack8<T>(x);
        }
    }
}

// 8-bit cache: a cluster per (request, block with new rows); its warps share the rows.
template <typename T> __global__ void __launch_bounds__(kThreads) append8_kernel(AppendArgs p) {
    __shared__ int warp_sum[kWarps];
    __shared__ int found[2];
    __shared__ float warp_max[kWarps];
    __shared__ float block_max;
    if ((int)blockIdx.x < p.nq) {
        rotate_q<T>(p, blockIdx.x);
        return;
    }
    const uint32_t rank = sas_ptx::cluster_rank();
    uint32_t ranks;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    const int unit = ((int)blockIdx.x - p.nq) / (int)ranks;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    // which request and block: the unit-th of all (request, touched block) pairs
    const int per = (p.B + kThreads - 1) / kThreads;
    int mine = 0;
    auto runs_of = [&](const Span &sp) {
        return sp.n > 0 ? (int)((sp.pos + sp.n - 1) / p.bs - sp.pos / p.bs) + 1 : 0;
    };
    for (int b = tid * per; b < min(p.B, (tid + 1) * per); ++b) mine += runs_of(span_of(p, b));
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    if (lane == 31) warp_sum[warp] = incl;
    if (tid == 0) found[0] = -1;
    __syncthreads();
    int before = incl - mine;
    for (int w = 0; w < warp; ++w) before += warp_sum[w];
    if (unit >= before && unit < before + mine) {
        for (int b = tid * per;; ++b) {
            const int n = runs_of(span_of(p, b));
            if (unit < before + n) {
                found[0] = b;
                found[1] = unit - before;
                break;
            }
            before += n;
        }
    }
    __syncthreads();
    const int b = found[0];
    if (b < 0) return;  // the whole cluster leaves: it has one unit
    const Span sp = span_of(p, b);
    const int64_t blk = sp.pos / p.bs + found[1];
    const int o0 = (int)max(sp.pos - blk * p.bs, (int64_t)0);                    // first new row in the block
    const int o1 = (int)min(sp.pos + sp.n - blk * p.bs, (int64_t)p.bs);          // one past the last
    const int64_t t0 = sp.row + (blk * p.bs + o0 - sp.pos);                      // flat row of o0
    const int64_t phys = block_of(p, b, blk);
    const bool any = phys >= 0;
    float old = any && o0 > 0 ? __ldg(p.scale + phys) : 0.f;
    const int nc = p.D / 8, w0 = (int)rank * kWarps + warp, nw = (int)ranks * kWarps;

    float amax = 0.f;
    if (any) {
        for (int o = o0 + w0; o < o1; o += nw) {
            const float *cs = angles(p, blk * p.bs + o);
            if (cs == nullptr) continue;
            const uint4 *row = reinterpret_cast<const uint4 *>(p.kv + (t0 + o - o0) * p.kv_stride * 2);
            for (int c = lane; c < nc; c += 32) {
                float x[8];
                load_rotated<T>(p, row, cs, c, x);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float a = fabsf(x[i]);
                    if (a <= 3.402823466e38f) amax = fmaxf(amax, a);  // neither infinity nor NaN
                }
            }
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (lane == 0) warp_max[warp] = amax;
    __syncthreads();
    amax = warp_max[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) amax = fmaxf(amax, warp_max[w]);
    if (ranks > 1) {
        if (tid == 0) block_max = amax;
        sas_ptx::cluster_sync();  // every rank has read the old scale and published its maximum
        for (uint32_t r = 0; r < ranks; ++r) {
            float v;
            asm volatile("ld.shared::cluster.f32 %0, [%1];"
                         : "=f"(v)
                         : "r"(sas_ptx::map_to_cta(sas_ptx::smem_u32(&block_max), r))
                         : "memory");
            amax = fmaxf(amax, v);
        }
        sas_ptx::cluster_sync();  // no rank leaves while its maximum may still be read
    } else {
        __syncthreads();  // every warp has read the old scale
    }
    if (!any) return;
    const float need = sas_fp8::scale_for(amax);
    float now = need;
    if (o0 > 0) {
        if (!sas_fp8::scale_ok(old)) {  // no scale: the rows before these were never written
            if (tid == 0) sas::set_status(p.status, SAS_STATUS_BAD_SCALE);
            old = need;
        }
        now = fmaxf(old, need);
    }
    if (rank == 0 && tid == 0) p.scale[phys] = now;
    uint8_t *block = reinterpret_cast<uint8_t *>(p.cache) + phys * p.bs * (int64_t)p.D;
    if (o0 > 0 && now > old) {  // the rows already there, rounded to the new scale
        const float f = old / now;
        const int n16 = o0 * (p.D / 16);
        uint4 *v = reinterpret_cast<uint4 *>(block);
        for (int i = (int)rank * kThreads + tid; i < n16; i += (int)ranks * kThreads) {
            uint4 x = v[i];
            x.x = sas_fp8::rescale4(x.x, f);
            x.y = sas_fp8::rescale4(x.y, f);
            x.z = sas_fp8::rescale4(x.z, f);
            x.w = sas_fp8::rescale4(x.w, f);
            v[i] = x;
        }
    }
    const float inv = 1.f / now;
    for (int o = o0 + w0; o < o1; o += nw) {  // the second read of a row finds it in L1
        const float *cs = angles(p, blk * p.bs + o);
        if (cs == nullptr) continue;
        const uint4 *row = reinterpret_cast<const uint4 *>(p.kv + (t0 + o - o0) * p.kv_stride * 2);
        uint2 *dst = reinterpret_cast<uint2 *>(block + (int64_t)o * p.D);
        for (int c = lane; c < nc; c += 32) {
            float x[8];
            load_rotated<T>(p, row, cs, c, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] *= inv;
            dst[c] = make_uint2(sas_fp8::to_e4m3x4(x[0], x[1], x[2], x[3]), sas_fp8::to_e4m3x4(x[4], x[5], x[6], x[7]));
        }
    }
}

bool aligned(const void *p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

} // namespace

using sas_host::check_cuda;

extern "C" int sas_cache_append(const SasAppendArgs *args, const void *kv, const void *q, void *q_out,
                                const float *rope_table, const int32_t *block_table, const int32_t *cu_seqlens_q,
                                const int32_t *act_q_len, const int32_t *act_kv_len, void *cache, float *cache_scale,
                                uint32_t *status, void *stream) {
    if (!args) return SAS_ERR_INVALID_ARG;
    const SasAppendArgs &a = *args;
    if (a.batch < 0 || a.num_tokens < 0 || a.num_heads < 0 || a.head_dim <= 0 || a.rope_dim < 0 || a.rope_step <= 0 ||
        a.rope_rows < 0 || a.block_num <= 0 || a.block_size <= 0 || a.table_len <= 0 || a.kv_row_stride < a.head_dim)
        return SAS_ERR_INVALID_ARG;
    for (int i = 0; i < 4; ++i)
        if (a.reserved[i] != 0) return SAS_ERR_INVALID_ARG;
    if (a.dtype != SAS_DTYPE_BF16 && a.dtype != SAS_DTYPE_FP16) return SAS_ERR_INVALID_ARG;
    const bool e4m3 = a.cache_dtype == SAS_DTYPE_E4M3;
    if (!e4m3 && a.cache_dtype != a.dtype) return SAS_ERR_UNSUPPORTED;
    if (a.head_dim % 16 != 0 || a.head_dim > 8 * 32 * kMaxChunks) return SAS_ERR_UNSUPPORTED;
    if (a.rope_dim > a.head_dim || a.rope_dim % 16 != 0 || a.kv_row_stride % 8 != 0) return SAS_ERR_UNSUPPORTED;
    if ((int64_t)a.block_num * a.block_size >= ((int64_t)1 << 31)) return SAS_ERR_UNSUPPORTED;
    if (!cu_seqlens_q && (a.max_q_len <= 0 || (int64_t)a.batch * a.max_q_len != a.num_tokens)) {
        if (a.num_tokens != 0) return SAS_ERR_INVALID_ARG;
    }
    if (a.num_tokens == 0 || a.batch == 0) return SAS_OK;
    if (!kv || !cache || !block_table || !act_kv_len || (a.rope_dim > 0 && !rope_table) || (e4m3 && !cache_scale) ||
        (a.num_heads > 0 && (!q || !q_out)))
        return SAS_ERR_INVALID_ARG;
    if (!aligned(kv, 16) || !aligned(q, 16) || !aligned(q_out, 16) || !aligned(cache, 16) || !aligned(rope_table, 16) ||
        !aligned(block_table, 4) || !aligned(cu_seqlens_q, 4) || !aligned(act_q_len, 4) || !aligned(act_kv_len, 4) ||
        !aligned(cache_scale, 4) || !aligned(status, 4))
        return SAS_ERR_INVALID_ARG;
    AppendArgs p;
    p.kv = static_cast<const char *>(kv);
    p.q = static_cast<const char *>(q);
    p.q_out = static_cast<char *>(q_out);
    p.cache = static_cast<char *>(cache);
    p.scale = cache_scale;
    // without a rotation the angles are never read, but a null address would mean "past the table"
    p.rope = a.rope_dim > 0 ? rope_table : reinterpret_cast<const float *>(act_kv_len);
    p.table = block_table;
    p.cu = cu_seqlens_q;
    p.act_q = act_q_len;
    p.act_kv = act_kv_len;
    p.status = status;
    p.kv_stride = a.kv_row_stride;
    p.B = a.batch;
    p.T = a.num_tokens;
    p.N1 = a.num_heads;
    p.D = a.head_dim;
    p.R = a.rope_dim;
    p.interleaved = a.rope_interleaved;
    p.step = a.rope_step;
    p.rope_rows = a.rope_rows;
    p.block_num = a.block_num;
    p.bs = a.block_size;
    p.table_len = a.table_len;
    p.q_rows = std::max(a.max_q_len, 1);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    int64_t nq = a.num_heads > 0 ? (int64_t)a.num_tokens * ((a.num_heads + kQHeads - 1) / kQHeads) : 0;
    const bool bf16 = a.dtype == SAS_DTYPE_BF16;
    if (!e4m3) {
        const int64_t grid = nq + (a.num_tokens + kWarps - 1) / kWarps;
        if (grid >= INT32_MAX) return SAS_ERR_UNSUPPORTED;
        p.nq = (int)nq;
        if (bf16) append16_kernel<__nv_bfloat16><<<(unsigned)grid, kThreads, 0, s>>>(p);
        else append16_kernel<__half><<<(unsigned)grid, kThreads, 0, s>>>(p);
        return check_cuda(cudaGetLastError());
    }
    // at most one unit per token, and n / bs + 2 per request of n tokens
    const int64_t units = std::min<int64_t>(a.num_tokens, a.num_tokens / a.block_size + 2 * (int64_t)a.batch);
    const int cluster = a.num_tokens >= 16 * units ? 8 : 1;
    nq = (nq + cluster - 1) / cluster * cluster;
    const int64_t grid = nq + units * cluster;
    if (grid >= INT32_MAX) return SAS_ERR_UNSUPPORTED;
    p.nq = (int)nq;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid, 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return check_cuda(bf16 ? cudaLaunchKernelEx(&cfg, append8_kernel<__nv_bfloat16>, p)
                           : cudaLaunchKernelEx(&cfg, append8_kernel<__half>, p));
}
