// CUDA-core attention over the 8-bit cache: every head count, D_qk <= 1024, D_v <= 512, fp32
// arithmetic throughout.  Serves the shapes and types the tensor-core kernel does not take.
//
// One CTA per (token, 16 heads).  Chunks of 32 keys pass through shared memory as fp16, which holds
// every e4m3 value exactly; a key's scale multiplies its score and its weight, so that rows are
// never scaled.  One online softmax (log2 domain) over all keys; the sink joins at the end:
//   lse2 = log2(2^(m + log2 l) + 2^sink2),  out = o / l * 2^(m + log2 l - lse2).
// Bound by the FP32 pipe: 2 N1 (D_qk + D_v) flops per key: 2.5 ms for 64 tokens of 2176 keys and 128 heads
// of 576 dims (15 TFLOP/s), which the tensor-core kernel does in 71 us.

#include "sas_fp8_attn.cuh"

namespace {

constexpr int kHG = 16, kKC = 32, kThreads = 256, kMaxPairs = 16;  // D_v / 32 <= 16

template <typename T> __global__ void __launch_bounds__(kThreads) fp8_simt_kernel(sas_fp8::Args p) {
    using namespace sas_fp8;
    extern __shared__ __align__(16) unsigned char smem[];
    const int KS = p.Dq + 8;
    float *qs = reinterpret_cast<float *>(smem);             // [kHG][Dq]
    __half *ks = reinterpret_cast<__half *>(qs + kHG * p.Dq);  // [kKC][KS]
    float *ps = reinterpret_cast<float *>(ks + kKC * KS);    // [kHG][kKC]
    float *ms = ps + kHG * kKC, *ls = ms + kHG, *al = ls + kHG;
    float *sc = al + kHG;                                    // [kKC]
    int32_t *rid = reinterpret_cast<int32_t *>(sc + kKC);    // [kKC]
    uint8_t *live = reinterpret_cast<uint8_t *>(rid + kKC);  // [kKC]: the slot holds a key
    __shared__ int32_t rec[TR_INTS];

    const int t = blockIdx.x, h0 = blockIdx.y * kHG;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid < TR_INTS) rec[tid] = p.rec[(int64_t)t * TR_INTS + tid];
    __syncthreads();
    const int npair = p.Dv >> 5, hq = tid >> 4, sub = tid & 15;
    T *out = reinterpret_cast<T *>(p.out);
    const int n_ori = rec[TR_NORI], n = rec[TR_VALID] ? n_ori + rec[TR_NCMP] : 0;
    const T *q = reinterpret_cast<const T *>(p.q) + (int64_t)t * p.N1 * p.Dq;
    for (int e = tid; e < kHG * p.Dq; e += kThreads) {
        const int h = e / p.Dq;
        qs[e] = h0 + h < p.N1 ? sas::DT<T>::to_f(q[(int64_t)h0 * p.Dq + e]) * p.scale_log2 : 0.f;
    }
    if (tid < kHG) {
        ms[tid] = -INFINITY;
        ls[tid] = 0.f;
    }
    float o[2 * kMaxPairs];
#pragma unroll
    for (int k = 0; k < 2 * kMaxPairs; ++k) o[k] = 0.f;
    uint32_t bits = 0;
    const int c16n = p.Dq >> 4;
    for (int c0 = 0; c0 < n; c0 += kKC) {
        __syncthreads();
        if (tid < kKC) {
            const int slot = c0 + tid;
            int32_t r = -1;
            float s = 0.f;
            if (slot < n_ori) {
                r = paged_row(p.ori_bt, rec[TR_B], p.ori_table_len, p.ori_bs, p.ori_block_num, ori_position(rec, slot),
                              bits);
                s = row_scale(p.ori_scale, p.ori_bs, r, bits);
            } else if (slot < n) {
                r = p.scenario == 3 ? p.rows[(int64_t)t * p.K + slot - n_ori]
                                    : paged_row(p.cmp_bt, rec[TR_B], p.cmp_table_len, p.cmp_bs, p.cmp_block_num,
                                                slot - n_ori, bits);
                s = row_scale(p.cmp_scale, p.cmp_bs, r, bits);
            }
            rid[tid] = s > 0.f ? r : -1;
            sc[tid] = s;
            live[tid] = slot < n;
        }
        __syncthreads();
        for (int e = tid; e < kKC * c16n; e += kThreads) {
            const int j = e / c16n, c = e - j * c16n;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (rid[j] >= 0)
                v = __ldg(reinterpret_cast<const uint4 *>((c0 + j < n_ori ? p.ori : p.cmp) + (int64_t)rid[j] * p.Dq) + c);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
            uint4 lo, hi;
            lo.x = e4m3x2_to_half2(w[0] & 0xffffu);
            lo.y = e4m3x2_to_half2(w[0] >> 16);
            lo.z = e4m3x2_to_half2(w[1] & 0xffffu);
            lo.w = e4m3x2_to_half2(w[1] >> 16);
            hi.x = e4m3x2_to_half2(w[2] & 0xffffu);
            hi.y = e4m3x2_to_half2(w[2] >> 16);
            hi.z = e4m3x2_to_half2(w[3] & 0xffffu);
            hi.w = e4m3x2_to_half2(w[3] >> 16);
            uint4 *d = reinterpret_cast<uint4 *>(ks + j * KS + c * 16);
            d[0] = lo;
            d[1] = hi;
        }
        __syncthreads();
        {  // scores and softmax: warp w owns heads 2 w, 2 w + 1; lane = key
            float a0 = 0.f, a1 = 0.f;
            const __half *kr = ks + lane * KS;
            const float *q0 = qs + 2 * warp * p.Dq, *q1 = q0 + p.Dq;
            for (int c = 0; c < p.Dq; c += 8) {
                const uint4 v = *reinterpret_cast<const uint4 *>(kr + c);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = sas::DT<__half>::to_f2(w[i]);
                    const float2 x = *reinterpret_cast<const float2 *>(q0 + c + 2 * i);
                    const float2 y = *reinterpret_cast<const float2 *>(q1 + c + 2 * i);
                    a0 = fmaf(x.x, f.x, fmaf(x.y, f.y, a0));
                    a1 = fmaf(y.x, f.x, fmaf(y.y, f.y, a1));
                }
            }
            const float s = sc[lane];
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                const int h = 2 * warp + hh;
                const float x = live[lane] ? (hh ? a1 : a0) * s : -INFINITY;
                float mx = x;
#pragma unroll
                for (int off = 16; off; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
                const float mo = ms[h], mn = fmaxf(mo, mx);
                const float e = live[lane] ? exp2f(x - mn) : 0.f;
                float sum = e;
#pragma unroll
                for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
                ps[h * kKC + lane] = e * s;
                __syncwarp();
                if (lane == 0) {
                    const float alpha = exp2f(mo - mn);
                    al[h] = alpha;
                    ls[h] = ls[h] * alpha + sum;
                    ms[h] = mn;
                }
            }
        }
        __syncthreads();
        const float alpha = al[hq];
#pragma unroll
        for (int k = 0; k < 2 * kMaxPairs; ++k) o[k] *= alpha;
        const int nk = min(kKC, n - c0);
        for (int j = 0; j < nk; ++j) {
            const float w = ps[hq * kKC + j];
            const uint32_t *row = reinterpret_cast<const uint32_t *>(ks + j * KS);
#pragma unroll
            for (int k = 0; k < kMaxPairs; ++k) {
                if (k < npair) {
                    const float2 f = sas::DT<__half>::to_f2(row[sub + 16 * k]);
                    o[2 * k] = fmaf(w, f.x, o[2 * k]);
                    o[2 * k + 1] = fmaf(w, f.y, o[2 * k + 1]);
                }
            }
        }
    }
    if (bits) atomicOr(reinterpret_cast<unsigned int *>(p.rec + (int64_t)t * TR_INTS + TR_STATUS), bits);
    __syncthreads();
    const int h = h0 + hq;
    if (h >= p.N1) return;
    const float l = ls[hq], own = n > 0 ? ms[hq] + log2f(l) : -INFINITY;
    const float sink = p.sinks ? p.sinks[h] : -INFINITY;
    const float lse2 = log2_add(own, sink * 1.4426950408889634f);
    const float f = n > 0 ? exp2f(own - lse2) / l : 0.f;
    if (p.lse && sub == 0)
        p.lse[(int64_t)t * p.N1 + h] = n > 0 ? lse2 * 0.6931471805599453f : rec[TR_VALID] ? sink : 0.f;
    T *orow = out + ((int64_t)t * p.N1 + h) * p.Dv;
#pragma unroll
    for (int k = 0; k < kMaxPairs; ++k) {
        if (k < npair) {
            orow[2 * (sub + 16 * k)] = sas::DT<T>::from_f(n > 0 ? o[2 * k] * f : 0.f);
            orow[2 * (sub + 16 * k) + 1] = sas::DT<T>::from_f(n > 0 ? o[2 * k + 1] * f : 0.f);
        }
    }
}

size_t simt_smem(int Dq) {
    return sizeof(float) * kHG * (size_t)Dq + 2 * (size_t)kKC * (Dq + 8) + sizeof(float) * (kHG * kKC + 3 * kHG + kKC) +
           4 * kKC + kKC + 64;
}

} // namespace

namespace sas_host {

int launch_fp8_simt(const SasFp8Args &a, const sas_fp8::Args &p, cudaStream_t s) {
    int dev = 0;
    if (check_cuda(cudaGetDevice(&dev))) return SAS_ERR_CUDA;
    if (dev < 0 || dev >= sas::kMaxDevices) return SAS_ERR_UNSUPPORTED;
    static sas::DeviceOnce attr_done[sas::kMaxDevices];
    const bool bf16 = a.dtype == SAS_DTYPE_BF16;
    const int rc = attr_done[dev].run(bf16 ? 1u : 2u, [&] {  // raised once to the largest layout
        return check_cuda(bf16 ? cudaFuncSetAttribute(fp8_simt_kernel<__nv_bfloat16>,
                                                      cudaFuncAttributeMaxDynamicSharedMemorySize, (int)simt_smem(1024))
                               : cudaFuncSetAttribute(fp8_simt_kernel<__half>,
                                                      cudaFuncAttributeMaxDynamicSharedMemorySize, (int)simt_smem(1024)));
    });
    if (rc) return rc;
    const dim3 grid(a.num_tokens, (a.num_heads + kHG - 1) / kHG);
    const size_t smem = simt_smem(a.head_dim);
    if (bf16) fp8_simt_kernel<__nv_bfloat16><<<grid, kThreads, smem, s>>>(p);
    else fp8_simt_kernel<__half><<<grid, kThreads, smem, s>>>(p);
    return check_cuda(cudaGetLastError());
}

} // namespace sas_host
