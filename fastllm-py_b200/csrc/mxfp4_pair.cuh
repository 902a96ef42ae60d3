// Products of many rows with a matrix in microscaled 4-bit floating point on pairs of CTAs (cta_group::2): prompts.  First bfloat16 rows;
// rows in 4 bits themselves at the end.
//
// A pair's tile is 256 rows of W x up to 192 tokens.  Each CTA turns its 128 rows of W into bfloat16 in its own tensor memory (as
// mxfp4_tc.cu does) and loads half of the tokens; the MMA reads both halves, so a CTA moves and converts half of what two CTAs with
// tiles of 256 x 128 would.  Tensor memory holds two accumulators of 192 columns and two places of 64 columns for a chunk of W: the
// next tile's MMAs run while the epilogue's warps empty the last one's accumulator, 32 tokens a round through shared memory.  (With 256
// tokens there is room for one accumulator.)  Persistent: a pair walks over its tiles.
//
// Warps 0-15 convert, four of them half of a chunk of 128 along K, a thread one row; warps 16-23 are the epilogue, in two
// groups; warps 24 and 26 send for the tokens and the codes, warp 25 of the pair's even CTA (the leader) issues the MMAs.
//
// What bounds it: a chunk's way through wait, conversion, store to tensor memory and arrival, 1850 clocks of a warp for every other one;
// MMAs alone take 660 a chunk with 128 tokens, 770 with 192.  The issuing warp has few instructions to spare: with a barrier for each
// half of a chunk and one for its tokens a chunk took 1070 clocks, however small; it now waits for one, at which a converting
// warp arrives when it has seen the tokens too.  256 tokens 22016 -> 8192: 100 us, 86 so (81 now); 2048 tokens 11008 ->
// 4096 141 (1.31 PFLOP/s), 4096 -> the gated 2 x 11008 249 (1.48 PFLOP/s; launched on end 300, what the power limit leaves).  With one
// group of epilogue warps that 271, 517 tokens 2048 -> 5503 21.2 in place of 18.7: a tile's sums take about 5 us to leave.
#pragma once

#include "mxfp4_tc.cuh"

#define MXP_BN 192                                       // most tokens of a tile
// The tokens and the codes have rings of their own: a chunk's codes are needed a conversion earlier than its tokens, which would
// otherwise wait in shared memory for as long (2048 tokens, K 4096, 22016 features: 295 us with one ring of five stages).
#define MXP_X_RING (144 * 1024)
#define MXP_X_STAGES 8                                   // most of them: of bn / 2 x 128 elements, two boxes
#define MXP_W_STAGES 4
#define MXP_W_STAGE (MX_CODES + 1536)                    // 128 rows' codes, scales of up to 3 packed tiles
#define MXP_ROUND (32 * 128 * 4)                         // 32 tokens' sums
#define MXP_SMEM (MXP_X_RING + MXP_W_STAGES * MXP_W_STAGE + 2 * MXP_ROUND + 1024 + 512)
#define MXP_THREADS (27 * 32)

// ------------------------------------------------------------------ what a pair needs
// (What the leader's MMA reads of the other CTA is in tensor memory, which tcgen05's own fences order.  An arrival with a release at
// the cluster's scope waits for the thread's writes everywhere: it took this file's kernel from 297 to 466 us at 2048 tokens, K
// 4096, 22016 features.)
__device__ __forceinline__ void mxp_umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
        "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// The packed form as a tensor of 8-byte elements [chunks][4 pieces][256], for copies of 64 rows' codes of a chunk: a gated unit's rows.
// (As single copies of 1024 bytes they are eight a chunk: 2048 tokens, 4096 -> the gated 2 x 11008 306 us, and 292 with tensors.)
static int mxp_map_codes(CUtensorMap* map, const void* w, long rows, int chunks) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return (int)cudaErrorNotSupported;
    cuuint64_t dims[3] = {256, 4, (cuuint64_t)((rows + MX_ROWS - 1) / MX_ROWS * chunks)};
    cuuint64_t strides[2] = {2048, MX_CHUNK};
    cuuint32_t box[3] = {128, 4, 1}, elem[3] = {1, 1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_INT64, 3, const_cast<void*>(w), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : (int)cudaErrorInvalidValue;
}
// 64 rows' codes of a chunk, from the tile's row 0 or 64 on
__device__ __forceinline__ void mxp_copy_codes(void* dst, const CUtensorMap* map, uint64_t* bar, int row, int chunk) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
        "l"((uint64_t)map), "r"(smem_u32(bar)), "r"(row * 2), "r"(0), "r"(chunk)
        : "memory");
}
// A barrier of the epilogue's group `group`, and whether any of its threads came with `flag`: they leave together or not at all.
__device__ __forceinline__ bool mxp_vote(bool flag, int group) {
    uint32_t any;
    __syncwarp();
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "bar.red.or.pred q, %2, 128, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(any)
        : "r"((uint32_t)flag), "r"(2 + group)
        : "memory");
    return any != 0;
}

// The accumulator of a tile, emptied by a group of the epilogue's warps, which takes every other 32 tokens: this CTA's 128 rows, FEAT
// features of them on their way out.  `staged`: the group's.  False: given up.
template <typename TO, bool GATED>
__device__ __forceinline__ bool mxp_epilogue(uint32_t tmem_acc, float* staged, int group, int tokens, TO* __restrict__ out, long ldo, int n,
                                             const FlGate act, volatile int* abort_flag, uint64_t* acc_empty) {
    constexpr int FEAT = GATED ? 64 : 128, V = GATED ? 2 : 4;
    const int quarter = mxt_warp() & 3, r = quarter * 32 + (threadIdx.x & 31);
    const bool vec = (((uintptr_t)out | (uintptr_t)(ldo * (long)sizeof(TO))) & (V * sizeof(TO) - 1)) == 0 && (n & (V - 1)) == 0;
    bool read = false;                                    // the group's part of the accumulator has been
    for (int t = 32 * group; t < tokens; t += 64) {
        uint32_t v[32];
        tmem_ld16(tmem_acc + ((uint32_t)(quarter * 32) << 16) + (uint32_t)t, v);
        tmem_ld16(tmem_acc + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(t + 16), v + 16);
        tmem_ld_wait();
        if (t + 64 >= tokens) {
            tc_fence_before();
            __syncwarp();
            if ((threadIdx.x & 31) == 0) mbar_arrive_leader(acc_empty);
            read = true;
        }
        if (mxp_vote(false, group)) return false;         // the last round's rows have left
#pragma unroll
        for (int j = 0; j < 32; ++j) staged[j * 128 + r] = __uint_as_float(v[j]);
        if (mxp_vote(*abort_flag != 0, group)) return false;
        if (n <= 0) continue;
        const int last = min(32, tokens - t);
        if (vec) mxt_rows<TO, GATED, FEAT, 128, V, 4>(MxtSums{staged, staged, 1, 0, 0, 0}, quarter, last, out + (long)t * ldo, ldo, n, act);
        else mxt_rows<TO, GATED, FEAT, 128, 1, 4>(MxtSums{staged, staged, 1, 0, 0, 0}, quarter, last, out + (long)t * ldo, ldo, n, act);
    }
    __syncwarp();
    if (!read && (threadIdx.x & 31) == 0) mbar_arrive_leader(acc_empty);
    return true;
}

// row_tiles x token_tiles tiles; bn: tokens of a tile, a multiple of 32.
template <typename TO, bool GATED>
__global__ void __launch_bounds__(MXP_THREADS, 1)
mxp_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const uint8_t* __restrict__ w,
           TO* __restrict__ out, long ldo, int m, int n, int k, int bn, int x_stages, int token_tiles, int tiles, FlGate act,
           int* __restrict__ status) {
    constexpr int FEAT = GATED ? 64 : 128;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* ring = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    unsigned char* w_ring = ring + MXP_X_RING;
    float* staged = reinterpret_cast<float*>(w_ring + MXP_W_STAGES * MXP_W_STAGE);
    uint64_t* x_full = (uint64_t*)(staged + 2 * (MXP_ROUND / 4));                   // (the leader's: both CTAs' tokens)
    uint64_t* x_empty = x_full + MXP_X_STAGES;
    uint64_t* w_full = x_empty + MXP_X_STAGES;
    uint64_t* w_empty = w_full + MXP_W_STAGES;
    uint64_t* a_full = w_empty + MXP_W_STAGES;                                      // (the leader's)
    uint64_t* a_empty = a_full + 2;
    uint64_t* acc_full = a_empty + 2;
    uint64_t* acc_empty = acc_full + 2;                                             // (the leader's)
    uint32_t* tmem_slot = (uint32_t*)(acc_empty + 2);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    const int warp = mxt_warp(), lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank(), pair = (int)blockIdx.x >> 1, pairs = (int)gridDim.x >> 1;
    const int chunks = (k + 127) / 128;
    const int x_bytes = bn * 128;                                                   // of this CTA's half

    if (threadIdx.x == 0) {
        for (int s = 0; s < x_stages; ++s) {
            mbar_init(&x_full[s], 1);
            mbar_init(&x_empty[s], 1);
        }
        for (int s = 0; s < MXP_W_STAGES; ++s) {
            mbar_init(&w_full[s], 1);
            mbar_init(&w_empty[s], 8);
        }
        for (int p = 0; p < 2; ++p) {
            mbar_init(&a_full[p], 16);                       // eight warps in each CTA
            mbar_init(&a_empty[p], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], 16);                    // eight warps in each CTA
        }
        *abort_flag = (*(volatile int*)status != 0) ? 1 : 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 25) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();                                      // both CTAs' barriers exist before anyone signals them
    tc_fence_after();
    // accumulator b at 192 b, place p of W at 384 + 64 p.  (Launched in plain stream order, as every kernel with cta_group::2.)
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    bool ok = !*abort_flag;
    int issued = 0;
    if (warp < 16) {
        // ---- codes to bfloat16
        const int turn = warp >> 3, h = warp >> 2 & 1, r = threadIdx.x & 127;       // every other chunk, one half
        const uint32_t dst = tmem + 384u + (uint32_t)(turn * 64 + h * 32) + ((uint32_t)((warp & 3) * 32) << 16);
        // (a gated unit's 64 gate rows lie before its up rows)
        const int codes_at = GATED ? (r >> 6) * 4096 + h * 2048 + (r & 63) * 16 : h * 4096 + r * 16;
        int s = 0, x = 0, it = 0;                            // stages of the chunk's codes and tokens, chunks so far
        uint32_t ph = 0, xph = 0, pa = 0;
        const bool looks = rank == 0 && (warp & 7) == 0;     // for the tokens: the MMAs then need one barrier
        // (a stage of the tokens may have been the other group's before: a turn ago this one waited for the MMAs of four chunks back, and
        // there are more stages than that)
        for (int tile = pair; tile < tiles && ok; tile += pairs) {
            const int f0 = tile / token_tiles * (2 * FEAT) + rank * FEAT;
            // where the row's scales are: the gate rows lie in one packed tile, the up rows in one or two
            const int rr = !GATED ? r : r < 64 ? (f0 & (MX_ROWS - 1)) + r : (int)(((long)n + f0) & (MX_ROWS - 1)) + r - 64;
            const int scale_at = (!GATED || r < 64 ? 0 : 1 + (rr >> 7)) * 512 + (int)mx_scale_at(rr & 127) + 2 * h;
            for (int c = 0; c < chunks; ++c, ++it) {
                if ((it & 1) == turn) {
                    if (!mxt_wait(&w_full[s], ph, abort_flag)) {
                        if (lane == 0) mxt_give_up(abort_flag, status);
                        ok = false;
                        break;
                    }
                    const unsigned char* stage = w_ring + s * MXP_W_STAGE;
                    const uint4 qa = *reinterpret_cast<const uint4*>(stage + codes_at);
                    const uint4 qb = *reinterpret_cast<const uint4*>(stage + codes_at + (GATED ? 1024 : 2048));
                    const uint32_t sa = stage[scale_at], sb = stage[scale_at + 1];
                    const bool large = __any_sync(0xffffffffu, max(sa, sb) > 128u);
                    __syncwarp();
                    if (lane == 0) mxt_arrive(&w_empty[s]);
                    uint32_t v[32];
                    if (!large) {
                        mx_block(qa, mx_factor(sa), v);
                        mx_block(qb, mx_factor(sb), v + 16);
                    } else {
                        mx_block_large(qa, sa, v);
                        mx_block_large(qb, sb, v + 16);
                    }
                    if ((looks && !mxt_wait(&x_full[x], xph, abort_flag)) || !mxt_wait(&a_empty[turn], pa ^ 1u, abort_flag)) {
                        if (lane == 0) mxt_give_up(abort_flag, status);
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    mxt_tmem_st16(dst, v);
                    mxt_tmem_st16(dst + 16u, v + 16);
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if (rank == 0) mxt_arrive(&a_full[turn]);
                        else mbar_arrive_leader(&a_full[turn]);
                    }
                    pa ^= 1u;
                }
                if (++x == x_stages) { x = 0; xph ^= 1u; }
                if (++s == MXP_W_STAGES) { s = 0; ph ^= 1u; }
            }
        }
    } else if (warp < 24) {
        // ---- epilogue
        const int group = warp >> 2 & 1;
        int i = 0;
        for (int tile = pair; tile < tiles; tile += pairs, ++i) {
            const int b = i & 1;
            if (ok && !mxt_wait(&acc_full[b], (uint32_t)(i >> 1) & 1u, abort_flag)) {
                if (lane == 0) mxt_give_up(abort_flag, status);
                ok = false;
            }
            if (mxp_vote(!ok, group)) break;
            tc_fence_after();
            const int t0 = tile % token_tiles * bn, f0 = tile / token_tiles * (2 * FEAT) + rank * FEAT;
            if (!mxp_epilogue<TO, GATED>(tmem + (uint32_t)(b * 192), staged + group * (MXP_ROUND / 4), group, min(bn, m - t0),
                                         out + (long)t0 * ldo + f0, ldo, n - f0, act, abort_flag, &acc_empty[b]))
                break;
        }
    } else if (warp == 24) {
        // ---- this CTA's half of the tokens, signalled to the leader
        int s = 0;
        uint32_t ph = 0;
        for (int tile = pair; tile < tiles && ok; tile += pairs) {
            const int t0 = tile % token_tiles * bn + rank * (bn / 2);
            for (int c = 0; c < chunks; ++c) {
                if (!mxt_wait(&x_empty[s], ph ^ 1u, abort_flag)) {
                    if (lane == 0) mxt_give_up(abort_flag, status);
                    ok = false;
                    break;
                }
                if (mxt_elect()) {
                    unsigned char* dst = ring + s * x_bytes;
                    if (rank == 0) mbar_expect_tx(&x_full[s], 2 * (uint32_t)x_bytes);
                    tma_load_2d_pair(dst, &map_x, &x_full[s], c * 128, t0);
                    tma_load_2d_pair(dst + x_bytes / 2, &map_x, &x_full[s], c * 128 + 64, t0);
                }
                __syncwarp();
                ++issued;
                if (++s == x_stages) { s = 0; ph ^= 1u; }
            }
        }
    } else if (warp == 26) {
        // ---- this CTA's rows of W
        const long tile_bytes = (long)chunks * MX_CHUNK;
        int s = 0;
        uint32_t ph = 0;
        for (int tile = pair; tile < tiles && ok; tile += pairs) {
            const int f0 = tile / token_tiles * (2 * FEAT) + rank * FEAT;
            const long row1 = (long)n + f0;
            const int off0 = f0 & (MX_ROWS - 1), off1 = (int)(row1 & (MX_ROWS - 1)), first = min(64, MX_ROWS - off1);
            const int rest = (row1 / MX_ROWS + 1) * MX_ROWS < 2l * n ? 64 - first : 0;
            const uint8_t* src0 = w + (long)(f0 / MX_ROWS) * tile_bytes;
            const uint8_t* src1 = w + row1 / MX_ROWS * tile_bytes;
            // (a CTA whose rows lie behind the last has nothing to load and converts whatever is there: rows that go nowhere)
            const uint32_t w_bytes = f0 >= n ? 0 : !GATED ? MX_CHUNK : 4 * 1024 + 512 + 4 * first * 16 + 512 + (rest ? 4 * rest * 16 + 512 : 0);
            for (int c = 0; c < chunks; ++c) {
                if (!mxt_wait(&w_empty[s], ph ^ 1u, abort_flag)) {
                    if (lane == 0) mxt_give_up(abort_flag, status);
                    ok = false;
                    break;
                }
                if (mxt_elect()) {
                    unsigned char* dst = w_ring + s * MXP_W_STAGE;
                    mbar_expect_tx(&w_full[s], w_bytes);
                    const uint8_t* src = src0 + (long)c * MX_CHUNK;
                    if (w_bytes == 0) {
                    } else if (!GATED) {
                        mxt_copy(dst, src, MX_CHUNK, &w_full[s]);
                    } else {
                        mxp_copy_codes(dst, &map_w, &w_full[s], off0, (int)(f0 / MX_ROWS) * chunks + c);
                        mxt_copy(dst + MX_CODES, src + MX_CODES, 512, &w_full[s]);
                        src = src1 + (long)c * MX_CHUNK;
                        if ((off1 & 63) == 0) mxp_copy_codes(dst + 4096, &map_w, &w_full[s], off1, (int)(row1 / MX_ROWS) * chunks + c);
                        else
                            for (int b = 0; b < 4; ++b) mxt_copy(dst + 4096 + b * 1024, src + b * 2048 + off1 * 16, (uint32_t)first * 16, &w_full[s]);
                        mxt_copy(dst + MX_CODES + 512, src + MX_CODES, 512, &w_full[s]);
                        if (rest) {
                            src += tile_bytes;
                            for (int b = 0; b < 4; ++b)
                                mxt_copy(dst + 4096 + b * 1024 + first * 16, src + b * 2048, (uint32_t)rest * 16, &w_full[s]);
                            mxt_copy(dst + MX_CODES + 1024, src + MX_CODES, 512, &w_full[s]);
                        }
                    }
                }
                __syncwarp();
                ++issued;
                if (++s == MXP_W_STAGES) { s = 0; ph ^= 1u; }
            }
        }
    } else if (rank == 0) {
        // ---- MMA issuer, for both CTAs
        const uint32_t idesc = instr_desc_bf16(256, bn), ring_at = smem_u32(ring);
        const uint64_t half = (uint64_t)(x_bytes / 2) >> 4;
        int s = 0, i = 0;
        uint32_t turn = 0, pa = 0;
        bool there = false;                                  // the next chunk is known to be there, its tokens too
        for (int tile = pair; tile < tiles && ok; tile += pairs, ++i) {
            const int b = i & 1;
            ok = mxt_wait(&acc_empty[b], ((uint32_t)(i >> 1) & 1u) ^ 1u, abort_flag);
            const uint32_t acc = tmem + (uint32_t)(b * 192);
            for (int c = 0; c < chunks && ok; ++c) {
                if (!__all_sync(0xffffffffu, there) && !mxt_wait(&a_full[turn], pa, abort_flag)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                there = mxt_test(&a_full[turn ^ 1u], turn ? pa ^ 1u : pa);
                if (mxt_elect()) {
                    const uint64_t bdesc = smem_desc_sw128(ring_at + (uint32_t)(s * x_bytes));
#pragma unroll
                    for (int kk = 0; kk < 8; ++kk)
                        mxp_umma_ts(acc, tmem + 384u + turn * 64u + (uint32_t)(kk * 8), bdesc + (uint64_t)(2 * (kk & 3)) + (kk >= 4 ? half : 0),
                                    idesc, (c > 0 || kk > 0) ? 1u : 0u);
                    umma_commit_pair(&a_empty[turn]);
                    umma_commit_pair(&x_empty[s]);
                    if (c == chunks - 1) umma_commit_pair(&acc_full[b]);
                }
                __syncwarp();
                if (++s == x_stages) s = 0;
                pa ^= turn;
                turn ^= 1u;
            }
            if (!ok && lane == 0) mxt_give_up(abort_flag, status);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 24 && lane == 0 && *abort_flag) tma_drain(x_full, rank == 0 ? x_stages : 0, issued);
    if (warp == 26 && lane == 0 && *abort_flag) tma_drain(w_full, MXP_W_STAGES, issued);
    __syncthreads();
    cluster_sync_all();                                      // neither leaves while the other's MMAs or copies may reach it
    if (warp == 25) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// What a chunk takes, in ns: the conversion and its hand-overs up to 160 tokens, with 192 the MMAs (K 22016: 86 us with 64 and with 128
// tokens a tile, 104 with 192; 2048 tokens 4096 -> 12288 with 192 in eight rounds 162, with 160 in nine 168).
static int mxp_chunk(int bn) { return bn <= 160 ? 455 : 510; }
// Tokens of a tile: the multiple of 32 up to 192 with which the pairs take the least time for all their rounds; `rounds`: how many.
static int mxp_tokens(int m, int row_tiles, int pairs, long* rounds) {
    int best = 32;
    long least = 0;
    for (int bn = 32; bn <= MXP_BN; bn += 32) {
        const long r = ((long)row_tiles * ((m + bn - 1) / bn) + pairs - 1) / pairs;
        if (least == 0 || r * mxp_chunk(bn) < least) best = bn, least = r * mxp_chunk(bn), *rounds = r;
    }
    return best;
}

template <typename TO, bool GATED>
static int mxp_launch(const void* x, long ldx, const void* w, void* out, long ldo, int m, int n, int k, FlGate act, int num_sms, int* status,
                      cudaStream_t stream) {
    const int rows = GATED ? 128 : 256, chunks = (k + 127) / 128;
    long rounds;
    const int bn = mxp_tokens(m, (n + rows - 1) / rows, num_sms / 2, &rounds);
    const long tiles = (long)((n + rows - 1) / rows) * ((m + bn - 1) / bn);
    if (tiles > 0x3FFFFFFFl || rounds * chunks > 0x3FFFFFFFl) return (int)cudaErrorInvalidValue;
    CUtensorMap map;
    int rc = make_map(&map, x, m, k, ldx, bn / 2);
    if (rc) return rc;
    CUtensorMap map_w = map;                                 // (unused where W comes in whole chunks)
    if (GATED && (rc = mxp_map_codes(&map_w, w, 2l * n, chunks))) return rc;
    auto kernel = mxp_kernel<TO, GATED>;
    static bool configured[MX_DEVICES];
    const int device = mx_device();
    if (device < 0) return (int)cudaErrorInvalidDevice;
    if (!configured[device]) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MXP_SMEM);
        if (e != cudaSuccess) return (int)e;
        configured[device] = true;
    }
    const int stages = MXP_X_RING / (bn * 128);
    static_assert(MXP_X_RING / (MXP_BN * 128) >= 5 && MXP_X_STAGES >= 5 && MXP_W_STAGES % 2 == 0, "as the converting warps' waits need");
    const long pairs = tiles < num_sms / 2 ? tiles : num_sms / 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(2 * pairs));
    cfg.blockDim = dim3(MXP_THREADS);
    cfg.dynamicSmemBytes = MXP_SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, kernel, map, map_w, (const uint8_t*)w, (TO*)out, ldo, m, n, k, bn,
                                   stages < MXP_X_STAGES ? stages : MXP_X_STAGES, (m + bn - 1) / bn, (int)tiles, act, status);
}

// ---------------------------------------------------------------- both operands in 4 bits
// A pair's tile is 256 rows of W x 256 tokens, two packed tiles of each: a CTA copies one of W and one of A, in stages of two chunks
// (256 along K) that lie side by side in the packed form, one copy each, and the other CTA's tokens' scales.  A stage's MMAs take 512
// clocks and its 35 KB from L2 about as long, where single CTAs with tiles of 256 x 128 read 52 KB for half of the products.  Tensor
// memory holds one accumulator and the scales of every stage.
//
// What bounds it at 4096 x 8192 x 22016: the power limit, and then the operands from L2.  275 us after idle times, 327 launched on end (5.4
// and 4.5 PFLOP/s); a stage takes about 600 clocks.
//
// Warps 0-15, four of them a stage, move the scales (a lane 16 bytes of each block of them; every quarter of the lanes has all); warps
// 16-23 are the epilogue, in two groups; warp 24 sends for the copies, warp 25 of the leader issues the MMAs.
#define MXQP_STAGES 5
#define MXQP_STAGE (4 * MX_CHUNK + 1024)
#define MXQP_SF 24                                       // columns of a stage's scales: 4 of W and 8 of the tokens for each chunk
#define MXQP_SMEM (MXQP_STAGES * MXQP_STAGE + 2 * MXP_ROUND + 1024)
#define MXQP_THREADS (26 * 32)

__device__ __forceinline__ void mxqp_umma(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                          uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void mxqp_st4(uint32_t taddr, const uint4 v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// tiles: row pairs x token pairs (two packed tiles each).
template <typename TO>
__global__ void __launch_bounds__(MXQP_THREADS, 1)
mxqp_kernel(const uint8_t* __restrict__ a, const uint8_t* __restrict__ w, TO* __restrict__ out, long ldo, int m, int n, int chunks,
            int token_pairs, int tiles, int* __restrict__ status) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* ring = (unsigned char*)(((uintptr_t)smem_raw + 127) & ~(uintptr_t)127);
    float* staged = reinterpret_cast<float*>(ring + MXQP_STAGES * MXQP_STAGE);
    uint64_t* full_bar = (uint64_t*)(staged + 2 * (MXP_ROUND / 4));
    uint64_t* empty_bar = full_bar + MXQP_STAGES;
    uint64_t* scales_bar = empty_bar + MXQP_STAGES;              // (the leader's)
    uint64_t* acc_full = scales_bar + MXQP_STAGES;
    uint64_t* acc_empty = acc_full + 1;                          // (the leader's)
    uint32_t* tmem_slot = (uint32_t*)(acc_empty + 1);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    const int warp = mxt_warp(), lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank(), pair = (int)blockIdx.x >> 1, pairs = (int)gridDim.x >> 1;
    const int steps = (chunks + 1) / 2;                          // stages of a tile
    const int last_w = (n - 1) / MX_ROWS, last_a = (m - 1) / MX_ROWS;

    if (threadIdx.x == 0) {
        for (int s = 0; s < MXQP_STAGES; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
            mbar_init(&scales_bar[s], 8);                        // four warps in each CTA
        }
        mbar_init(acc_full, 1);
        mbar_init(acc_empty, 16);                                // eight warps in each CTA
        *abort_flag = (*(volatile int*)status != 0) ? 1 : 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 25) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();                                          // both CTAs' barriers exist before anyone signals them
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0), tmem_sf = tmem + 256u;
    bool ok = !*abort_flag;
    int issued = 0;
    if (warp < 16) {
        // ---- scales to tensor memory, every fourth stage
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        int it = 0;
        for (int tile = pair; tile < tiles && ok; tile += pairs)
            for (int step = 0; step < steps; ++step, ++it) {
                if ((it & 3) != warp >> 2) continue;
                const int s = it % MXQP_STAGES;
                const uint32_t ph = (uint32_t)(it / MXQP_STAGES) & 1u;
                // (The stage's use before was another group's, and copies land in any order: unless its MMAs are known to be done, this
                // use's parity may be that of a phase before it.  Those of this use need this group, so that barrier is not passed twice.)
                if (!mxt_wait(&empty_bar[s], ph ^ 1u, abort_flag) || !mxt_wait(&full_bar[s], ph, abort_flag)) {
                    if (lane == 0) mxt_give_up(abort_flag, status);
                    ok = false;
                    break;
                }
                tc_fence_after();                                // (the stage's columns: its last use's MMAs were done before it was filled again)
                const unsigned char* stage = ring + s * MXQP_STAGE;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    if (2 * step + c >= chunks) break;
                    const uint32_t at = tmem_sf + lanes + (uint32_t)(s * MXQP_SF + c * 12);
                    const uint4 own = *reinterpret_cast<const uint4*>(stage + 2 * MX_CHUNK + c * MX_CHUNK + MX_CODES + lane * 16);
                    const uint4 peer = *reinterpret_cast<const uint4*>(stage + 4 * MX_CHUNK + c * 512 + lane * 16);
                    mxqp_st4(at, *reinterpret_cast<const uint4*>(stage + c * MX_CHUNK + MX_CODES + lane * 16));
                    mxqp_st4(at + 4u, rank ? peer : own);
                    mxqp_st4(at + 8u, rank ? own : peer);
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_leader(&scales_bar[s]);
            }
    } else if (warp < 24) {
        // ---- epilogue: two groups of four warps, every other 32 tokens
        const int group = (warp >> 2) & 1, quarter = warp & 3, r = quarter * 32 + lane;
        float* mine = staged + group * (MXP_ROUND / 4);
        int i = 0;
        for (int tile = pair; tile < tiles; tile += pairs, ++i) {
            if (ok && !mxt_wait(acc_full, (uint32_t)i & 1u, abort_flag)) {
                if (lane == 0) mxt_give_up(abort_flag, status);
                ok = false;
            }
            if (mxp_vote(!ok, group)) break;
            tc_fence_after();
            const int t0 = tile % token_pairs * 256, f0 = tile / token_pairs * 256 + rank * 128, tokens = min(256, m - t0), left = n - f0;
            TO* dst = out + (long)t0 * ldo + f0;
            const bool vec = (((uintptr_t)dst | (uintptr_t)(ldo * (long)sizeof(TO))) & (4 * sizeof(TO) - 1)) == 0 && (n & 3) == 0;
            bool going = true;
            for (int t = 32 * group; t < 256 && going; t += 64) {
                uint32_t v[32];
                tmem_ld16(tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)t, v);
                tmem_ld16(tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(t + 16), v + 16);
                tmem_ld_wait();
                if (t + 64 >= 256) {                             // this group has read its part of the accumulator
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_leader(acc_empty);
                }
                if (t >= tokens || left <= 0) continue;          // (the same in the whole group)
                if (mxp_vote(false, group)) going = false;      // the last round's rows have left
#pragma unroll
                for (int j = 0; j < 32; ++j) mine[j * 128 + r] = __uint_as_float(v[j]);
                if (mxp_vote(*abort_flag != 0, group)) going = false;
                if (!going) break;
                const int last = min(32, tokens - t);
                const MxtSums from = {mine, mine, 1, 0, 0, 0};
                const FlGate none = {FL_ACT_NONE, 0.0f, 0.0f};
                if (vec) mxt_rows<TO, false, 128, 128, 4, 4>(from, quarter, last, dst + (long)t * ldo, ldo, left, none);
                else mxt_rows<TO, false, 128, 128, 1, 4>(from, quarter, last, dst + (long)t * ldo, ldo, left, none);
            }
            if (!going) break;
        }
    } else if (warp == 24) {
        // ---- producer: a tile of W, a tile of A, the other CTA's tokens' scales (tiles that do not exist: the last one again, whose
        // sums go nowhere)
        int s = 0;
        uint32_t ph = 0;
        for (int tile = pair; tile < tiles && ok; tile += pairs) {
            const long tile_bytes = (long)chunks * MX_CHUNK;
            const int wt = tile / token_pairs * 2 + rank, at = tile % token_pairs * 2;
            const uint8_t* src_w = w + min(wt, last_w) * tile_bytes;
            const uint8_t* src_a = a + min(at + rank, last_a) * tile_bytes;
            const uint8_t* src_p = a + min(at + 1 - rank, last_a) * tile_bytes + MX_CODES;
            for (int step = 0; step < steps; ++step) {
                if (!mxt_wait(&empty_bar[s], ph ^ 1u, abort_flag)) {
                    if (lane == 0) mxt_give_up(abort_flag, status);
                    ok = false;
                    break;
                }
                if (mxt_elect()) {
                    unsigned char* dst = ring + s * MXQP_STAGE;
                    const int two = 2 * step + 1 < chunks ? 2 : 1;
                    const long at_k = 2l * step * MX_CHUNK;
                    mbar_expect_tx(&full_bar[s], (uint32_t)(two * (2 * MX_CHUNK + 512)));
                    mxt_copy(dst, src_w + at_k, (uint32_t)(two * MX_CHUNK), &full_bar[s]);
                    mxt_copy(dst + 2 * MX_CHUNK, src_a + at_k, (uint32_t)(two * MX_CHUNK), &full_bar[s]);
                    mxt_copy(dst + 4 * MX_CHUNK, src_p + at_k, 512, &full_bar[s]);
                    if (two == 2) mxt_copy(dst + 4 * MX_CHUNK + 512, src_p + at_k + MX_CHUNK, 512, &full_bar[s]);
                }
                __syncwarp();
                ++issued;
                if (++s == MXQP_STAGES) { s = 0; ph ^= 1u; }
            }
        }
    } else if (rank == 0) {
        // ---- MMA issuer, for both CTAs.  (A stage's scales are in tensor memory once its copies have come, in either CTA.)
        const uint32_t idesc[2] = {mxq_idesc(256, 256, 0), mxq_idesc(256, 256, 2)}, ring_at = smem_u32(ring);
        int s = 0, i = 0;
        uint32_t ph = 0;
        bool there = false;                                      // the next stage is known to be there
        for (int tile = pair; tile < tiles && ok; tile += pairs, ++i) {
            ok = mxt_wait(acc_empty, ((uint32_t)i & 1u) ^ 1u, abort_flag);
            for (int step = 0; step < steps && ok; ++step) {
                if (!__all_sync(0xffffffffu, there)) ok = mxt_wait(&scales_bar[s], ph, abort_flag);
                if (!ok) break;
                tc_fence_after();
                const int next = s + 1 == MXQP_STAGES ? 0 : s + 1;
                there = mxt_test(&scales_bar[next], next ? ph : ph ^ 1u);
                const uint32_t at = ring_at + (uint32_t)(s * MXQP_STAGE), sf = tmem_sf + (uint32_t)(s * MXQP_SF);
                if (mxt_elect()) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        if (2 * step + c >= chunks) break;
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            mxqp_umma(tmem, mxq_desc(at + (uint32_t)(c * MX_CHUNK + h * 4096), 2048),
                                      mxq_desc(at + (uint32_t)((2 + c) * MX_CHUNK + h * 4096), 2048), idesc[h], sf + (uint32_t)(c * 12),
                                      sf + (uint32_t)(c * 12 + 4), (step > 0 || c > 0 || h > 0) ? 1u : 0u);
                    }
                    umma_commit_pair(&empty_bar[s]);
                    if (step == steps - 1) umma_commit_pair(acc_full);
                }
                __syncwarp();
                if (++s == MXQP_STAGES) { s = 0; ph ^= 1u; }
            }
            if (!ok && lane == 0) mxt_give_up(abort_flag, status);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 24 && lane == 0 && *abort_flag) tma_drain(full_bar, MXQP_STAGES, issued);
    __syncthreads();
    cluster_sync_all();                                          // neither leaves while the other's MMAs or copies may reach it
    if (warp == 25) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

template <typename TO>
static int mxqp_launch(const void* a, const void* w, void* out, long ldo, int m, int n, int k, int num_sms, int* status, cudaStream_t stream) {
    const int chunks = (k + 127) / 128, token_pairs = (m + 255) / 256;
    const long tiles = (long)((n + 255) / 256) * token_pairs, pairs = tiles < num_sms / 2 ? tiles : num_sms / 2;
    if (tiles > 0x3FFFFFFFl || (tiles / pairs + 1) * ((chunks + 1) / 2) > 0x3FFFFFFFl) return (int)cudaErrorInvalidValue;
    auto kernel = mxqp_kernel<TO>;
    static bool configured[MX_DEVICES];
    const int device = mx_device();
    if (device < 0) return (int)cudaErrorInvalidDevice;
    if (!configured[device]) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MXQP_SMEM);
        if (e != cudaSuccess) return (int)e;
        configured[device] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(2 * pairs));
    cfg.blockDim = dim3(MXQP_THREADS);
    cfg.dynamicSmemBytes = MXQP_SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, kernel, (const uint8_t*)a, (const uint8_t*)w, (TO*)out, ldo, m, n, chunks, token_pairs, (int)tiles, status);
}
