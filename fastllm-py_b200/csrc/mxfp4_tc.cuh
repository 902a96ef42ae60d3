// Shared by the products with matrices in 4 bits on the tensor cores (mxfp4_tc.cu, mxfp4_pair.cuh): how their warps wait, issue and
// give up, and how sums of tokens leave shared memory.
#pragma once

#include "mxfp4.cuh"
#include "tcgen05.cuh"

enum { MXT_ERR_WAIT = 121 };

__device__ __forceinline__ void mxt_tmem_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void mxt_umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
        "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// One lane of a warp that is together.  The issuing warps stay together and elect for each batch of instructions: what the matrix
// instructions take then is the same in the whole warp and lives in uniform registers.  Issued by a branch of lane 0 each of them
// cost 140 to 190 clocks, whatever its size (2048 tokens, K 4096, 22016 features: 472 us, and 331 with the election).
__device__ __forceinline__ bool mxt_elect() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ int mxt_warp() { return __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0); }
__device__ __forceinline__ void mxt_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Whether a barrier's phase is complete, without waiting.  The warps that issue matrix instructions ask for the next ones' barriers
// before they issue: the answer is there when they have.
__device__ __forceinline__ bool mxt_test(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
// (A wait names a phase by its parity, so whoever waits has to know that the phase before the one it means is over: because it waited
// for that itself, or because something that it waited for came after it.)
// A whole warp waits for a barrier's phase (limits as mbar_wait's; without a flag to the end).  All lanes ask, first without being put
// to sleep: a wait by one lane and a shuffle of the outcome took 190 clocks even where the phase was complete, and these kernels
// hand over from warp to warp several times a chunk (4096 x 8192 x 22016 in 4 bits: 384 us so, 313 this way; 64 tokens 22016 -> 8192:
// 40.8 and 36.8).  Where it is not they may be: asking over and over takes issue slots from the others (40 x 4096 x 12288 in 4 bits
// 9.6 us, and 9.0 so).
__device__ __forceinline__ bool mxt_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
    if (__all_sync(0xffffffffu, mxt_test(bar, parity))) return true;
    const uint64_t t0 = global_ns();
    for (uint32_t spins = 1;; ++spins) {
        if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity) != 0)) return true;
        if ((spins & 15u) == 0 && __any_sync(0xffffffffu, (abort_flag && *abort_flag) || global_ns() - t0 > TC_WAIT_LIMIT_NS)) return false;
    }
}
// Where the sums of a CTA's tokens are: [token][PITCH] floats of its own, and behind `parts` the other CTAs' of its cluster, in rank
// order, `stride` floats between them, from token `first` on.
struct MxtSums {
    const float* own;
    const float* parts;
    int ranks, rank, first, stride;
};
// Tokens t, t + STEP, .. (FEAT features, of a gated unit then their up values), added up in rank order, through the activation and out;
// `n`: how many features there are from the tile's first on.
template <int V> __device__ __forceinline__ void mxt_add(const float* from, float* to) {
    if (V == 4) {
        const float4 x = *reinterpret_cast<const float4*>(from);
        to[0] += x.x, to[V > 1 ? 1 : 0] += x.y, to[V > 2 ? 2 : 0] += x.z, to[V > 3 ? 3 : 0] += x.w;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) to[i] += from[i];
    }
}
template <typename TO, bool GATED, int FEAT, int PITCH, int V, int STEP>
__device__ __forceinline__ void mxt_rows(const MxtSums sums, int t, int last, TO* out, long ldo, int n, const FlGate act) {
    constexpr int PARTS = FEAT / (32 * V);                            // steps of 32 V features
    const int f0 = (threadIdx.x & 31) * V;
#pragma unroll 2
    for (; t < last; t += STEP) {
        float g[PARTS * V], u[PARTS * V];
#pragma unroll
        for (int i = 0; i < PARTS * V; ++i) g[i] = 0.0f, u[i] = GATED ? 0.0f : 1.0f;
        const float* own = sums.own + t * PITCH + f0;
        const float* part = sums.parts + (t - sums.first) * PITCH + f0;
#pragma unroll 4
        for (int q = 0; q < sums.ranks; ++q) {
            const float* row = q == sums.rank ? own : part;
            part += q == sums.rank ? 0 : sums.stride;
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
                mxt_add<V>(row + p * 32 * V, g + p * V);
                if (GATED) mxt_add<V>(row + FEAT + p * 32 * V, u + p * V);
            }
        }
        if (act.act != FL_ACT_NONE) gated_act(g, u, act);
        TO* dst = out + (long)t * ldo + f0;
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            if (f0 + p * 32 * V >= n) continue;                       // (n is a multiple of V)
            __align__(16) TO o[V];
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = from_f32<TO>(g[p * V + i]);
            TO* d = dst + p * 32 * V;
            if (V == 1) *d = o[0];
            else if (V * sizeof(TO) == 4) *reinterpret_cast<uint32_t*>(d) = *reinterpret_cast<const uint32_t*>(o);
            else if (V * sizeof(TO) == 8) *reinterpret_cast<uint2*>(d) = *reinterpret_cast<const uint2*>(o);
            else *reinterpret_cast<uint4*>(d) = *reinterpret_cast<const uint4*>(o);
        }
    }
}

__device__ __forceinline__ void mxt_give_up(volatile int* abort_flag, int* status) {
    if (!*abort_flag) {
        *abort_flag = 1;
        atomicCAS(status, 0, MXT_ERR_WAIT);
    }
}

__device__ __forceinline__ void mxt_copy(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src),
                 "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}

// Shared memory to the same place of CTA `rank` of the cluster, and to its barrier.
__device__ __forceinline__ void mxt_push(void* dst, const void* src, uint32_t bytes, uint64_t* bar, int rank) {
    uint32_t to, signal;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(dst)), "r"(rank));
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(signal) : "r"(smem_u32(bar)), "r"(rank));
    asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "r"(smem_u32(src)),
                 "r"(bytes), "r"(signal)
                 : "memory");
}
__device__ __forceinline__ void mxt_cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void mxt_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// ------------------------------------------------------------------ both operands in 4 bits
// A tile's codes as an operand of the block-scaled matrix instruction, no swizzle: `lead` bytes between core matrices along K, 128
// between those of neighbouring groups of 8 rows
__device__ __forceinline__ uint64_t mxq_desc(uint32_t saddr, uint32_t lead) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}
// float accumulator; A and B e2m1 with a scale 2^(s - 127) for 32 elements, which of the four bytes of a scale column `id` (0 or 2) and
// the next one are
__device__ __forceinline__ uint32_t mxq_idesc(int m, int n, int id) {
    return (uint32_t)id << 4 | 1u << 7 | 1u << 10 | (uint32_t)(n >> 3) << 17 | 1u << 23 | (uint32_t)(m >> 4) << 24 | (uint32_t)id << 29;
}
