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
// Bound: bytes (each row read once and written once); a decode call is one launch latency, 6.4 us on the
// device.  4 x 8192 rows of 576 to 8 bits take 16.5 us, 57 MB at 3.4 TB/s: the rows are read twice, the
// second time from L1 or L2, and the two passes and the lookups before them follow one another in a CTA.
// Clusters of 4 x 128 threads with 4 loads under way per thread take 16.7 us, 2 x 128 18.7, 2 x 256 18.3,
// 8 x 256 43; one row per CTA (512 requests) takes 8.4 us with 128 threads and 12.4 with 256, which need
// two waves.  The largest value of the copied dims is found on the bits, two at a time: unpacked to
// floats, and with 64-bit positions, the kernel was bound by its instructions at 43 us.  Rows kept in
// registers between the passes cost occupancy, 63 us; two kernels with a warp per two rows, 47 us.  Calls one
// after the other, with the last one's codes still to be written back, take 20.6 us each; turning the tail in
// both passes, without the copy in shared memory, 22.5.

#include <algorithm>

#include "sas_common.cuh"
#include "sas_fp8.cuh"
#include "sas_tc_ptx.cuh"

namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kCluster = 4;  // CTAs per block that takes many rows
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
    int pos, row, n;
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
    int64_t pos = (int64_t)__ldg(p.act_kv + b) - n;
    if (pos < 0) {  // tokens before the sequence's start have no place
        if (n > 0) sas::set_status(p.status, SAS_STATUS_BAD_POSITION);
        row -= pos;
        n += (int)pos;
        pos = 0;
    }
    if (row < 0 || row >= p.T) n = 0;
    Span sp;
    sp.pos = (int)pos;
    sp.row = (int)row;
    sp.n = (int)min((int64_t)n, (int64_t)p.T - row);
    return sp;
}

// Position of flat row t, or -1 where it belongs to no request (warp-uniform; every lane calls).
__device__ __forceinline__ int position_of(const AppendArgs &p, int t, int &b) {
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

__device__ __forceinline__ int64_t block_of(const AppendArgs &p, int b, int blk) {
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
    const int pos = position_of(p, t, b);
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

// 16-bit cache: a warp per new row.  10,776 rows of 512 (25 MB) take 8.4 us, one row 6.4.
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
    const int pos = position_of(p, t, b);
    if (pos < 0) return;
    const int blk = pos / p.bs;
    const int64_t phys = block_of(p, b, blk);
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

// Bits of the 16-bit types' infinity.
template <typename T> __device__ constexpr uint32_t infinity_bits();
template <> __device__ constexpr uint32_t infinity_bits<__nv_bfloat16>() { return 0x7f80u; }
template <> __device__ constexpr uint32_t infinity_bits<__half>() { return 0x7c00u; }

__device__ __forceinline__ void note_finite(float x, float &amax) {
    x = fabsf(x);
    if (x <= 3.402823466e38f) amax = fmaxf(amax, x);  // neither infinity nor NaN
}

// Steps through the pieces of rows of `width` pieces: `from`, from + by, ...
struct Walk {
    int row, at, drow, dat, width;
    __device__ __forceinline__ Walk(int from, int by, int w)
        : row(from / w), at(from - from / w * w), drow(by / w), dat(by - by / w * w), width(w) {}
    __device__ __forceinline__ void next() {
        row += drow;
        at += dat;
        if (at >= width) {
            at -= width;
            ++row;
        }
    }
};

// 16 values of a 16-bit type times a power of two, to 16 codes.
template <typename T> __device__ __forceinline__ uint4 to_codes16(const uint4 (&v)[2], float inv) {
    float x[16];
    unpack8<T>(v[0], reinterpret_cast<float (&)[8]>(x[0]));
    unpack8<T>(v[1], reinterpret_cast<float (&)[8]>(x[8]));
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = sas_fp8::to_e4m3x4(x[4 * i] * inv, x[4 * i + 1] * inv, x[4 * i + 2] * inv, x[4 * i + 3] * inv);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Units of work: request b has those from c_b / bs + 2 b on (c_b its first flat row).  Its n rows touch at most
// n / bs + 2 blocks, so that each has a unit; there are T / bs + 2 B.  (A scan over all requests in each CTA
// took 770 us for 8192 of them.)
__device__ __forceinline__ int first_unit_of(const AppendArgs &p, int b) {
    const int row = p.cu ? min(max(__ldg(p.cu + b), 0), p.T) : b * p.q_rows;
    return row / p.bs + 2 * b;
}
__device__ __forceinline__ int request_of_unit(const AppendArgs &p, int unit) {  // warp-uniform; every lane calls
    const int lane = threadIdx.x & 31;
    int lo = 0, n = p.B;  // the request is in [lo, lo + n)
    while (n > 1) {
        const int step = (n + 31) / 32;
        const bool past = (lane + 1) * step < n && first_unit_of(p, lo + (lane + 1) * step) <= unit;
        const int k = __popc(__ballot_sync(0xffffffffu, past));
        lo += k * step;
        n = min(step, n - k * step);
    }
    return lo;
}

// 8-bit cache: a cluster per (request, block with new rows); its threads share the rows, 16 dims of the
// copied part or 8 of the turned part at a time.
template <typename T> __global__ void __launch_bounds__(kThreads) append8_kernel(AppendArgs p) {
    constexpr int kAhead = 4;  // loads of 16 dims under way per thread
    constexpr int kHeld = 2;   // turned pieces of 8 dims kept per thread: 32 rows of 64 dims in all
    __shared__ float warp_max[kWarps];
    __shared__ float block_max;
    __shared__ float4 held[kHeld][2][kThreads];  // turned values, from the first pass to the second
    if ((int)blockIdx.x < p.nq) {
        rotate_q<T>(p, blockIdx.x);
        return;
    }
    const uint32_t rank = sas_ptx::cluster_rank();
    uint32_t ranks;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    const int unit = ((int)blockIdx.x - p.nq) / (int)ranks;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    const int b = request_of_unit(p, unit);
    const Span sp = span_of(p, b);
    const int run = unit - first_unit_of(p, b), blk = sp.pos / p.bs + run;
    // no such run (the whole cluster leaves: it has one unit)
    if (sp.n <= 0 || run < 0 || blk > (sp.pos + sp.n - 1) / p.bs) return;
    const int first = blk * p.bs;           // the block's first position
    const int o0 = max(sp.pos - first, 0);  // first new row in the block
    int rows = min(sp.pos + sp.n - first, p.bs) - o0;
    const char *src = p.kv + ((int64_t)sp.row + (first + o0 - sp.pos)) * p.kv_stride * 2;
    const int64_t phys = block_of(p, b, blk);
    const float *cs0 = p.rope + (int64_t)(first + o0) * p.step * p.R;
    if (p.R > 0) {  // rows past the table's end have no place
        const int last = (int)min(((int64_t)p.rope_rows + p.step - 1) / p.step - (first + o0), (int64_t)rows);
        if (last < rows) sas::set_status(p.status, SAS_STATUS_BAD_POSITION);
        rows = max(last, 0);
    }
    if (phys < 0 || rows == 0) return;  // no row has a place: the block and its scale stay (in the whole cluster)
    float old = o0 > 0 ? __ldg(p.scale + phys) : 0.f;
    const int me = (int)rank * kThreads + tid, all = (int)ranks * kThreads;
    const int plain = (p.D - p.R) / 16, turned = p.R / 8;
    const int64_t src_bytes = p.kv_stride * 2;

    float amax = 0.f;
    auto turn = [&](const Walk &w, float (&x)[8]) {
        load_rotated<T>(p, reinterpret_cast<const uint4 *>(src + w.row * src_bytes), cs0 + (int64_t)w.row * p.step * p.R,
                        2 * plain + w.at, x);
    };
    if (turned) {
        Walk w(me, all, turned);
#pragma unroll
        for (int k = 0; k < kHeld; ++k, w.next()) {
            if (w.row >= rows) continue;
            float x[8];
            turn(w, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) note_finite(x[i], amax);
            held[k][0][tid] = make_float4(x[0], x[1], x[2], x[3]);
            held[k][1][tid] = make_float4(x[4], x[5], x[6], x[7]);
        }
        for (; w.row < rows; w.next()) {
            float x[8];
            turn(w, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) note_finite(x[i], amax);
        }
    }
    if (plain) {
        uint32_t m = 0;  // magnitudes order as their bits do, two at a time
        Walk w(me, all, plain);
        while (w.row < rows) {
            uint4 v[kAhead][2];
#pragma unroll
            for (int k = 0; k < kAhead; ++k, w.next()) {
                const uint4 *x = reinterpret_cast<const uint4 *>(src + w.row * src_bytes) + 2 * w.at;
                v[k][0] = w.row < rows ? __ldg(x) : make_uint4(0, 0, 0, 0);
                v[k][1] = w.row < rows ? __ldg(x + 1) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    m = __vmaxu2(m, v[k][i].x & 0x7fff7fffu);
                    m = __vmaxu2(m, v[k][i].y & 0x7fff7fffu);
                    m = __vmaxu2(m, v[k][i].z & 0x7fff7fffu);
                    m = __vmaxu2(m, v[k][i].w & 0x7fff7fffu);
                }
        }
        m = max(m >> 16, m & 0xffffu);
        if (m < infinity_bits<T>()) {
            amax = fmaxf(amax, sas::DT<T>::to_f2(m).x);
        } else {  // an infinity or a NaN: look again, past those
            for (Walk r(me, all, plain); r.row < rows; r.next()) {
                const uint4 *x = reinterpret_cast<const uint4 *>(src + r.row * src_bytes) + 2 * r.at;
                for (int h = 0; h < 2; ++h) {
                    float y[8];
                    unpack8<T>(__ldg(x + h), y);
                    for (int i = 0; i < 8; ++i) note_finite(y[i], amax);
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
    uint8_t *dst = block + (int64_t)o0 * p.D;  // the second read of a row finds it in L1 or L2
    if (plain) {
        Walk w(me, all, plain);
        while (w.row < rows) {
            uint4 v[kAhead][2];
            Walk r = w;
#pragma unroll
            for (int k = 0; k < kAhead; ++k, r.next()) {
                if (r.row >= rows) continue;
                const uint4 *x = reinterpret_cast<const uint4 *>(src + r.row * src_bytes) + 2 * r.at;
                v[k][0] = __ldg(x);
                v[k][1] = __ldg(x + 1);
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k, w.next())
                if (w.row < rows) reinterpret_cast<uint4 *>(dst + (int64_t)w.row * p.D)[w.at] = to_codes16<T>(v[k], inv);
        }
    }
    if (turned) {
        auto put = [&](const Walk &w, const float4 &a, const float4 &b) {
            reinterpret_cast<uint2 *>(dst + (int64_t)w.row * p.D)[2 * plain + w.at] =
                make_uint2(sas_fp8::to_e4m3x4(a.x * inv, a.y * inv, a.z * inv, a.w * inv),
                           sas_fp8::to_e4m3x4(b.x * inv, b.y * inv, b.z * inv, b.w * inv));
        };
        Walk w(me, all, turned);
#pragma unroll
        for (int k = 0; k < kHeld; ++k, w.next())
            if (w.row < rows) put(w, held[k][0][tid], held[k][1][tid]);
        for (; w.row < rows; w.next()) {
            float x[8];
            turn(w, x);
            put(w, make_float4(x[0], x[1], x[2], x[3]), make_float4(x[4], x[5], x[6], x[7]));
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
    // in place and without a rotation nothing of q moves
    const bool turn_q = a.num_heads > 0 && !(q && q == q_out && a.rope_dim == 0);
    if (a.num_tokens == 0 || (a.batch == 0 && (!turn_q || (q && q == q_out)))) return SAS_OK;
    if (!kv || !cache || (a.batch > 0 && (!block_table || !act_kv_len)) || (a.rope_dim > 0 && !rope_table) || (e4m3 && !cache_scale) ||
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
    int64_t nq = turn_q ? (int64_t)a.num_tokens * ((a.num_heads + kQHeads - 1) / kQHeads) : 0;
    const bool bf16 = a.dtype == SAS_DTYPE_BF16;
    if (!e4m3 || a.batch == 0) {  // rows of no request: their query heads are copied, and that is all
        const int64_t grid = nq + (a.batch > 0 ? (a.num_tokens + kWarps - 1) / kWarps : 0);
        if (grid >= INT32_MAX) return SAS_ERR_UNSUPPORTED;
        p.nq = (int)nq;
        if (bf16) append16_kernel<__nv_bfloat16><<<(unsigned)grid, kThreads, 0, s>>>(p);
        else append16_kernel<__half><<<(unsigned)grid, kThreads, 0, s>>>(p);
        return check_cuda(cudaGetLastError());
    }
    const int64_t units = a.num_tokens / a.block_size + 2 * (int64_t)a.batch;
    // a cluster where blocks take 16 rows and more: 128 rows per block as above; with one row its other CTAs are idle
    const int cluster = a.num_tokens >= 16 * units ? kCluster : 1;
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
