// Bounded waits, the abort flag and the unit queue of the cluster-pair tensor-core kernels, and the
// tensor-map encoder's address.  `P` below: a kernel's argument struct, with the unit count U and the
// global unit counter `counter`.
#pragma once

#include <cuda.h>

#include "sas_common.cuh"
#include "sas_tc_ptx.cuh"

namespace sas_tc {

using namespace sas_ptx;

constexpr uint64_t kTimeoutNs = 4000000000ull;

// Unit queue: one warp of the score CTA, the writer, takes unit ids from a global counter (the next one
// fetched while the current one runs) and publishes them to every role of both CTAs through a
// kTq-entry ring; an entry is reused once all reader warps have read it, whose number each kernel gives
// its tq_empty barriers.
constexpr int kTq = 8;
// Readers in the 16-bit kernel: every warp of its cluster but the writer, 8 in the score CTA, 9 in the output CTA.
constexpr uint32_t kTqReaders = 17;

// What the helpers below need of a kernel's shared header: its abort flag and its unit queue
// (each kernel lays these out in a header struct of its own).
struct Sync {
    volatile int *abort;
    uint32_t *status;
    uint32_t peer_abort;  // shared::cluster address of the peer CTA's abort flag
    uint64_t *tq_full, *tq_empty;
    volatile int *tq;
};

static __device__ __noinline__ void raise_abort(const Sync &s, uint32_t bits) {
    sas::set_status(s.status, bits);
    *s.abort = 1;
    st_cluster_u32(s.peer_abort, 1u);
}

// Wait for the phase of parity `parity` of mbarrier `bar`; false on abort / timeout.
__device__ __forceinline__ bool wait_bar(const Sync &s, uint32_t bar, uint32_t parity, bool cluster_scope = false) {
    uint64_t t0 = 0;
    for (uint32_t it = 0;; ++it) {
        if (cluster_scope ? mbar_try_cluster(bar, parity) : mbar_try(bar, parity)) return true;
        if ((it & 15u) == 15u) {
            if (*s.abort) return false;
            const uint64_t now = globaltimer();
            if (t0 == 0) t0 = now;
            else if (now - t0 > kTimeoutNs) {
                raise_abort(s, SAS_STATUS_WAIT_TIMEOUT);
                return false;
            }
        }
    }
}

// Warp-uniform wait: every lane polls; if any lane gives up, all do.
__device__ __forceinline__ bool wait_warp(const Sync &s, uint32_t bar, uint32_t parity, bool cluster_scope = false) {
    return __all_sync(0xffffffffu, wait_bar(s, bar, parity, cluster_scope));
}

// Warp-uniform poll: true (for every lane, each having acquired the phase) once
// any lane sees the phase complete.  Used on rs_req and o_full, whose next phase
// needs an arrival this warp makes later (rs_done / o_empty), so a phase one
// lane saw complete stays complete and the lanes that lagged acquire it on their
// first test.  The bound only guards that argument; it never binds.
__device__ __forceinline__ bool poll_warp(uint32_t bar, uint32_t parity) {
    // test_wait never suspends: a try_wait on one barrier could sleep through the other's phase
    const bool mine = mbar_test(bar, parity);
    if (!__any_sync(0xffffffffu, mine)) return false;
    if (!mine)
        for (uint32_t i = 0; i < (1u << 16) && !mbar_test(bar, parity); ++i) {
        }
    return true;
}

// Unit queue.  Cluster c's first unit is c (every role takes it without the queue); later ones
// come from the counter, offset by the cluster count, and pass through the queue: entry k >= 1
// lives in slot (k - 1) % kTq.
template <class P> __device__ __forceinline__ int first_unit(const P &p) {
    return (int)cluster_id_x() < p.U ? (int)cluster_id_x() : -1;
}

// Reader side (every warp of the cluster but the writer; warp-uniform): the k-th unit id of this
// cluster, or -1 once the counter has passed the last unit.  False on abort / timeout.
template <class P>
__device__ __forceinline__ bool tq_read(const P &p, const Sync &sy, uint32_t rank, uint32_t k, int &t) {
    if (k == 0) {
        t = first_unit(p);
        return true;
    }
    const int s = (k - 1) % kTq;
    if (!wait_warp(sy, smem_u32(&sy.tq_full[s]), ((k - 1) / kTq) & 1, true)) return false;
    t = sy.tq[s];
    __syncwarp();
    if ((threadIdx.x & 31) == 0) {
        const uint32_t e = smem_u32(&sy.tq_empty[s]);
        if (rank == 0)
            mbar_arrive(e);
        else
            mbar_arrive_remote(map_to_cta(e, 0));
    }
    return true;
}

// Writer side (one warp of the score CTA; warp-uniform).  `pend` (lane 0) holds the id taken while the
// previous unit's last tiles were being gathered (-1: none yet, take one now); taking it only
// then keeps a cluster from holding a unit it cannot start soon.
template <class P>
__device__ __forceinline__ bool tq_publish(const P &p, const Sync &sy, uint32_t k, int &pend, int &t) {
    if (k == 0) {
        t = first_unit(p);
        return true;
    }
    const int s = (k - 1) % kTq;
    const int lane = threadIdx.x & 31;
    if (k - 1 >= (uint32_t)kTq && !wait_warp(sy, smem_u32(&sy.tq_empty[s]), (((k - 1) / kTq) - 1) & 1))
        return false;
    int v = 0;
    if (lane == 0) {
        if (pend < 0) pend = (int)ncluster_x() + atomicAdd(p.counter, 1);
        v = pend < p.U ? pend : -1;
        pend = -1;
        sy.tq[s] = v;
        st_cluster_u32(map_to_cta(smem_u32((const void *)&sy.tq[s]), 1), (uint32_t)v);
        mbar_arrive(smem_u32(&sy.tq_full[s]));
        mbar_arrive_remote(map_to_cta(smem_u32(&sy.tq_full[s]), 1));
    }
    t = __shfl_sync(0xffffffffu, v, 0);
    return true;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = [] {
        void *ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            return reinterpret_cast<EncodeTiledFn>(ptr);
        return static_cast<EncodeTiledFn>(nullptr);
    }();
    return fn;
}

} // namespace sas_tc
