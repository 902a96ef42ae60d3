// Products of bfloat16 rows with a matrix in microscaled 4-bit floating point on the tensor cores (mxfp4.cuh says what the
// packed form is): out[t, f] = sum_k x[t, k] W[f, k], and the gated unit act(gate) * up of two such products.
//
// The weights are turned into bfloat16 on their way (exactly: a magnitude of two bits of significand times a power of two) and
// go to tensor memory as the MMA's A operand; the tokens come to shared memory by TMA as its B operand.  So the 16-bit form of
// the weights touches neither global nor shared memory, whose bandwidth the MMA needs for the tokens.
//
// A CTA takes two tiles of 128 rows of W (of a gated unit: a gate tile and the up tile of the same features) and up to 128
// tokens, K in stages of a chunk (128): one copy a row tile, two boxes of the tokens.  Warps 0-15 turn the codes into bfloat16, a
// thread one row of a chunk (warps 0-7 of every other one, 8-15 of those between), and write them to one of the two or
// three places in tensor memory; then they are the epilogue.  Warp 16 sends for the copies, warp 17 issues the MMAs.  Where there are
// fewer tiles than SMs a cluster of up to 8 CTAs shares K; each CTA is sent the others' sums of its share of the tokens, and adds them
// up in rank order.
//
// What bounds it: the conversion.  A word of 8 codes takes 9 instructions of the integer units, which take two clocks of a quarter of
// the SM each, and 8 multiplications: a chunk of 256 rows 600 clocks at the least, and 1050 with what the warps wait for one
// another; 16 MMAs take 620 clocks with 16 tokens, 820 with 64 and 1140 with 128.  64 tokens 22016 -> 8192: 35.1 us, 2.7 TB/s
// of codes, 0.66 PFLOP/s; 16 tokens 30.9; 128 tokens 44, 1.05 PFLOP/s.
#include "mxfp4_pair.cuh"
#include "mxfp4_tc.cuh"

#define MXT_BN 128                          // most tokens of a tile
#define MXT_A 3                             // most places of 2 x 64 columns in tensor memory
#define MXT_W_BYTES (2 * (MX_CODES + 1024)) // two row tiles of a chunk: codes, the scales of the one or two packed tiles they lie in
#define MXT_RING (224 * 1024)               // the epilogue's sums take its place: a CTA's own and what the others of its cluster send it
#define MXT_MAX_STAGES 10
#define MXT_FEW_ROWS 8                      // what fl_mx_few takes
#define MXT_FEW (-1)
#define MXT_PITCH 256                       // floats between the tokens of the sums
// (No other kernel that takes tensor memory fits an SM beside this much shared memory: an allocation never waits for a CTA that
// waits for its predecessor in the stream.)
#define MXT_SMEM (MXT_RING + 1024 + 1024)
#define MXT_WARPS 16                        // that convert, and of the epilogue
#define MXT_THREADS ((MXT_WARPS + 2) * 32)

// What the kernels with accumulators in tensor memory end with, by the whole CTA: the accumulators (valid where `any`, else zero)
// as float sums [token][2 x 128 rows] in shared memory, where the ring was (every copy has been read by an MMA that is done).  `ok`:
// of the first MXT_WARPS warps, whether the accumulators may be waited for.
//
// Of a cluster each CTA takes a share of the tokens; the others send it their sums of them, one copy each, to behind its own, where its
// ring is free too once its MMAs are done: the first meeting of the cluster, arrived at before the accumulators are read.  The second is
// arrived at when a CTA has all that it was sent, so the senders' sums have been read, and is waited for behind the output.  (With the
// sums fetched from the other CTAs by loads, 64 tokens 4096 -> 4096 took 11.6 us, 5.5 of them here.)  A CTA that gave up sends
// what it has: the status word tells that the results are not valid.
template <typename TO, bool GATED>
__device__ __forceinline__ void mxt_finish(float* sums, uint32_t tmem_d, int acc_cols, uint64_t* acc_bar, uint64_t* sent_bar,
                                           volatile int* abort_flag, int* status, bool ok, bool any, int rows, int ranks, int rank,
                                           TO* __restrict__ out, long ldo, int f0, int n, const FlGate act) {
    constexpr int FEAT = GATED ? 128 : 256, V = 4;
    const int warp = mxt_warp(), lane = threadIdx.x & 31;
    const int share = (rows + ranks - 1) / ranks, first = min(rows, rank * share), last = min(rows, first + share);
    float* parts = sums + rows * MXT_PITCH;
    if (warp < MXT_WARPS && ok && !mxt_wait(acc_bar, 0, abort_flag)) {
        if (lane == 0) mxt_give_up(abort_flag, status);
        ok = false;
    }
    __syncwarp();
    // 16 bytes or 8 of a lane's features at a time, where rows are aligned
    const bool vec = (((uintptr_t)(out + f0) | (uintptr_t)(ldo * (long)sizeof(TO))) & (V * sizeof(TO) - 1)) == 0 && (n & (V - 1)) == 0;
    if (ranks == 1 && (GATED || !vec)) {
        // Nothing to add up: a warp's 32 features side by side, a token a store.  Through shared memory as below 128 tokens, 4096 -> the
        // gated 2 x 11008, took 30.7 us, and 28.8 so; 517 tokens 2048 -> 5503 19.6 and 18.4; but with features by fours 256 x 1536 x
        // 1024 in 4 bits takes 7.2 that way, and 7.7 so.
        if (warp < MXT_WARPS && ok && !*abort_flag) {
            tc_fence_after();
            constexpr int TILES = GATED ? 1 : 2;                      // that warps share
            const int tile = GATED ? 0 : warp >> 2 & 1, f = f0 + tile * 128 + (threadIdx.x & 127);
            const uint32_t src = tmem_d + (uint32_t)(tile * acc_cols) + ((uint32_t)((warp & 3) * 32) << 16);
            for (int c = warp / (4 * TILES) * 16; c < rows; c += MXT_WARPS / (4 * TILES) * 16) {
                uint32_t v[16], w[16];
                tmem_ld16(src + (uint32_t)c, v);
                if (GATED) tmem_ld16(src + (uint32_t)(acc_cols + c), w);
                tmem_ld_wait();
                float g[16], u[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) g[j] = __uint_as_float(v[j]), u[j] = GATED ? __uint_as_float(w[j]) : 1.0f;
                if (act.act != FL_ACT_NONE) gated_act(g, u, act);
                TO* dst = out + (long)c * ldo + f;
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (c + j < rows && f < n) dst[(long)j * ldo] = from_f32<TO>(g[j]);
            }
        }
        __syncwarp();
        tc_fence_before();
        __syncthreads();
        return;
    }
    if (ranks > 1) mxt_cluster_arrive();
    if (warp < MXT_WARPS && ok) {
        tc_fence_after();
        const int tile = warp >> 2 & 1, f = tile * 128 + (threadIdx.x & 127);
        const uint32_t src = tmem_d + (uint32_t)(tile * acc_cols) + ((uint32_t)((warp & 3) * 32) << 16);
        for (int c = (warp >> 3) * 16; c < rows; c += 32) {
            uint32_t v[16];
            tmem_ld16(src + (uint32_t)c, v);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (c + j < rows) sums[(c + j) * MXT_PITCH + f] = any ? __uint_as_float(v[j]) : 0.0f;
        }
    }
    tc_fence_before();
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    tc_fence_after();
    if (ranks > 1) {
        mxt_cluster_wait();
        if (warp == MXT_WARPS && mxt_elect()) {
            if (last > first) mbar_expect_tx(sent_bar, (uint32_t)((ranks - 1) * (last - first) * MXT_PITCH * 4));
            for (int i = 1; i < ranks; ++i) {
                const int to = rank + i < ranks ? rank + i : rank + i - ranks, t0 = to * share, tokens = min(share, rows - t0);
                if (tokens > 0)
                    mxt_push(parts + (rank - (rank > to)) * tokens * MXT_PITCH, sums + t0 * MXT_PITCH,
                             (uint32_t)(tokens * MXT_PITCH * 4), sent_bar, to);
            }
        }
        // (a CTA that gave up waits for what is on its way to it all the same)
        if (warp < MXT_WARPS && last > first && !mxt_wait(sent_bar, 0, nullptr) && lane == 0) mxt_give_up(abort_flag, status);
        __syncwarp();
        mxt_cluster_arrive();
    }
    if (warp < MXT_WARPS && !*abort_flag) {
        const MxtSums from = {sums, parts, ranks, rank, first, (last - first) * MXT_PITCH};
        out += f0;
        // a warp takes a token: V features a lane and 32 V a step, or single ones side by side where rows are not aligned
        if (vec)
            mxt_rows<TO, GATED, FEAT, MXT_PITCH, V, MXT_WARPS>(from, first + warp, last, out, ldo, n - f0, act);
        else
            mxt_rows<TO, GATED, FEAT, MXT_PITCH, 1, MXT_WARPS>(from, first + warp, last, out, ldo, n - f0, act);
    }
    __syncwarp();
    if (ranks > 1) mxt_cluster_wait();
    else __syncthreads();
}

// The copies of a CTA's chunks c_begin .. c_end - 1, by one warp; returns how many stages were sent for.  A stage: bn x 128 elements
// of the tokens as two boxes, then the row tiles, each 8192 bytes of codes and the scales of the one or two packed tiles that its
// rows lie in.  Tile 0 begins with row f0 of W, tile 1 (if tiles is 2) with row row1.
__device__ __forceinline__ int mxt_produce(const CUtensorMap& map_x, const uint8_t* __restrict__ w, unsigned char* ring, uint64_t* full_bar,
                                           uint64_t* empty_bar, int stages, int stage_bytes, int bn, int t0, int n, int chunks, int f0, long row1,
                                           int tiles, int c_begin, int c_end, bool constant_w, bool ok, volatile int* abort_flag, int* status) {
    const int off = (int)(row1 & (MX_ROWS - 1)), x_bytes = bn * 256;
    const long tile_bytes = (long)chunks * MX_CHUNK;
    const uint8_t* src0 = w + (long)(f0 / MX_ROWS) * tile_bytes;
    const uint8_t* src1 = w + row1 / MX_ROWS * tile_bytes;
    const bool second = off != 0 && (row1 / MX_ROWS + 1) * MX_ROWS < 2l * n;             // (only up rows straddle)
    const uint32_t w_bytes = MX_CHUNK + (tiles < 2 ? 0 : off == 0 ? MX_CHUNK : 4 * (MX_ROWS - off) * 16 + 512 + (second ? 4 * off * 16 + 512 : 0));
    auto send_w = [&](int s, int c) {
        unsigned char* dst = ring + s * stage_bytes + x_bytes;
        mbar_expect_tx(&full_bar[s], (uint32_t)x_bytes + w_bytes);
        mxt_copy(dst, src0 + (long)c * MX_CHUNK, MX_CHUNK, &full_bar[s]);
        if (tiles < 2) return;
        dst += MX_CODES + 1024;
        const uint8_t* src = src1 + (long)c * MX_CHUNK;
        if (off == 0) {
            mxt_copy(dst, src, MX_CHUNK, &full_bar[s]);
            return;
        }
        for (int b = 0; b < 4; ++b) mxt_copy(dst + b * 2048, src + b * 2048 + off * 16, (uint32_t)(MX_ROWS - off) * 16, &full_bar[s]);
        mxt_copy(dst + MX_CODES, src + MX_CODES, 512, &full_bar[s]);
        if (!second) return;
        src += tile_bytes;
        for (int b = 0; b < 4; ++b) mxt_copy(dst + b * 2048 + (MX_ROWS - off) * 16, src + b * 2048, (uint32_t)off * 16, &full_bar[s]);
        mxt_copy(dst + MX_CODES + 512, src + MX_CODES, 512, &full_bar[s]);
    };
    auto send_x = [&](int s, int c) {
        tma_load_2d(ring + s * stage_bytes, &map_x, &full_bar[s], c * 128, t0);
        tma_load_2d(ring + s * stage_bytes + x_bytes / 2, &map_x, &full_bar[s], c * 128 + 64, t0);
    };
    // a constant W's first stages are sent for before the preceding kernel is waited for
    const int ahead = constant_w && ok ? max(0, min(stages, c_end - c_begin)) : 0;
    if (mxt_elect())
        for (int i = 0; i < ahead; ++i) send_w(i, c_begin + i);
    __syncwarp();
    pdl_wait();
    if (mxt_elect())
        for (int i = 0; i < ahead; ++i) send_x(i, c_begin + i);
    __syncwarp();
    int issued = ahead, s = issued % stages;
    uint32_t ph = (uint32_t)(issued / stages) & 1u;
    for (int c = c_begin + issued; c < c_end && ok; ++c) {
        if (!mxt_wait(&empty_bar[s], ph ^ 1u, abort_flag)) {
            if ((threadIdx.x & 31) == 0) mxt_give_up(abort_flag, status);
            break;
        }
        if (mxt_elect()) {
            send_w(s, c);
            send_x(s, c);
        }
        __syncwarp();
        ++issued;
        if (++s == stages) { s = 0; ph ^= 1u; }
    }
    return issued;
}

// grid: ranks of a cluster x token tiles x row tiles (pairs of them).  bn: tokens of a tile, a multiple of 16.  A stage is bn x 128
// tokens' elements as two boxes, then W.
template <typename TO, bool GATED>
__global__ void __launch_bounds__(MXT_THREADS, 1)
mxt_kernel(const __grid_constant__ CUtensorMap map_x, const uint8_t* __restrict__ w, TO* __restrict__ out, long ldo, int m, int n,
           int k, int bn, int stages, int ranks, int per_rank, bool constant_w, FlGate act, int* __restrict__ status) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* ring = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* full_bar = (uint64_t*)(ring + MXT_RING);
    uint64_t* empty_bar = full_bar + MXT_MAX_STAGES;
    uint64_t* a_full = empty_bar + MXT_MAX_STAGES;
    uint64_t* a_empty = a_full + MXT_A;
    uint64_t* acc_bar = a_empty + MXT_A;
    uint64_t* sent_bar = acc_bar + 1;
    uint32_t* tmem_slot = (uint32_t*)(sent_bar + 1);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    const int warp = mxt_warp(), lane = threadIdx.x & 31;
    const int rank = blockIdx.x;
    const int t0 = blockIdx.y * bn;
    const int f0 = blockIdx.z * (GATED ? 128 : 256);
    const int chunks = (k + 127) / 128;
    const int c_begin = rank * per_rank, c_end = min(chunks, c_begin + per_rank);
    const int x_bytes = bn * 256, stage_bytes = x_bytes + MXT_W_BYTES;
    // the second row tile: none, a packed tile, or (a gated unit's up rows) the end of one and the beginning of the next
    const int tiles = GATED || n - f0 > 128 ? 2 : 1;
    const long row1 = GATED ? (long)n + f0 : (long)f0 + 128;
    const int off = (int)(row1 & (MX_ROWS - 1));

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], MXT_WARPS / 2 + 1);
        }
        for (int s = 0; s < MXT_A; ++s) {
            mbar_init(&a_full[s], 8);
            mbar_init(&a_empty[s], 1);
        }
        mbar_init(acc_bar, 1);
        mbar_init(sent_bar, 1);
        *abort_flag = (*(volatile int*)status != 0) ? 1 : 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == MXT_WARPS + 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // two accumulators, then the places of A.  Up to 64 tokens leave room for three: a chunk's conversion then does not wait for the MMAs
    // of the last but one, which end about when it begins.
    const int acc_cols = bn <= 64 ? 64 : 128, places = bn <= 64 ? 3 : 2;
    const uint32_t tmem_d = __shfl_sync(0xffffffffu, *tmem_slot, 0), tmem_a = tmem_d + (uint32_t)(2 * acc_cols);
    pdl_trigger();
    int issued = 0;
    bool ok = !*abort_flag;
    if (warp < MXT_WARPS) {
        pdl_wait();                                              // (the output may still be read by the preceding kernel)
        // ---- codes to bfloat16: a thread's row of tile `tile`, every other chunk
        const int tile = warp >> 2 & 1, turn = warp >> 3, r = threadIdx.x & 127;
        const bool here = tile < tiles;
        const int rr = (tile ? off : 0) + r;                     // the row's place in the packed tiles
        const int codes_at = x_bytes + tile * (MX_CODES + 1024) + r * 16;
        const int scale_at = x_bytes + tile * (MX_CODES + 1024) + (rr >> 7) * 512 + mx_scale_at(rr & 127);
        const uint32_t lanes = tmem_a + (uint32_t)(tile * 64) + ((uint32_t)((warp & 3) * 32) << 16);
        // (a stage's or a place's use before may have been the other group's: this one has waited, a turn ago, for the MMAs of four or five
        // chunks back, and there are at least as many stages as that)
        int s = turn, place = turn;
        uint32_t ph = 0, pa = 0;
        if (s >= stages) s -= stages, ph ^= 1u;
        for (int c = c_begin + turn; c < c_end && ok; c += 2) {
            if (!mxt_wait(&full_bar[s], ph, abort_flag)) {
                if (lane == 0) mxt_give_up(abort_flag, status);
                ok = false;
                break;
            }
            const unsigned char* stage = ring + s * stage_bytes;
            uint4 q[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) q[b] = *reinterpret_cast<const uint4*>(stage + codes_at + b * 2048);
            const uint32_t sc = *reinterpret_cast<const uint32_t*>(stage + scale_at);
            __syncwarp();
            if (lane == 0) mxt_arrive(&empty_bar[s]);
            // (a byte above 128: its top bit is set, and it is not 128 itself)
            const bool large = __any_sync(0xffffffffu, (sc & 0x80808080u & ((sc & 0x7F7F7F7Fu) + 0x7F7F7F7Fu)) != 0);
            uint32_t v[32];
            auto two = [&](int b) {
                if (!large) {
                    mx_block(q[b], mx_factor(sc >> (8 * b) & 255u), v);
                    mx_block(q[b + 1], mx_factor(sc >> (8 * b + 8) & 255u), v + 16);
                } else {
                    mx_block_large(q[b], sc >> (8 * b) & 255u, v);
                    mx_block_large(q[b + 1], sc >> (8 * b + 8) & 255u, v + 16);
                }
            };
            if (here) two(0);
            if (!mxt_wait(&a_empty[place], pa ^ 1u, abort_flag)) {
                if (lane == 0) mxt_give_up(abort_flag, status);
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t dst = lanes + (uint32_t)(place * 128);
            if (here) {
                mxt_tmem_st16(dst, v);
                mxt_tmem_st16(dst + 16u, v + 16);
                two(2);
                mxt_tmem_st16(dst + 32u, v);
                mxt_tmem_st16(dst + 48u, v + 16);
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mxt_arrive(&a_full[place]);
            if ((place += 2) >= places) place -= places, pa ^= 1u;
            s += 2;
            if (s >= stages) s -= stages, ph ^= 1u;
        }
    } else if (warp == MXT_WARPS) {
        issued = mxt_produce(map_x, w, ring, full_bar, empty_bar, stages, stage_bytes, bn, t0, n, chunks, f0, row1, tiles, c_begin, c_end, constant_w,
                             ok, abort_flag, status);
    } else {
        // ---- MMA issuer.  (No chunk comes before the preceding kernel is over, and the limit of a wait is not for that kernel's time.)
        pdl_wait();
        const uint32_t idesc = instr_desc_bf16(128, bn), ring_at = smem_u32(ring);
        int s = 0;
        uint32_t place = 0, pa = 0;
        bool there = false;                                      // the next chunk is known to be there
        for (int c = c_begin; c < c_end && ok; ++c) {
            // (the tokens are there too: the converting warps had waited for the stage's barrier)
            if (!__all_sync(0xffffffffu, there) && !mxt_wait(&a_full[place], pa, abort_flag)) {
                if (lane == 0) mxt_give_up(abort_flag, status);
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t next = place + 1 == (uint32_t)places ? 0 : place + 1;
            there = mxt_test(&a_full[next], next ? pa : pa ^ 1u);
            const uint64_t bdesc = smem_desc_sw128(ring_at + (uint32_t)(s * stage_bytes));
            const uint64_t half = (uint64_t)(x_bytes / 2) >> 4;
            if (mxt_elect()) {
                for (int tile = 0; tile < tiles; ++tile)
#pragma unroll
                    for (int kk = 0; kk < 8; ++kk)
                        mxt_umma_ts(tmem_d + (uint32_t)(tile * acc_cols), tmem_a + place * 128u + (uint32_t)(tile * 64 + kk * 8),
                                    bdesc + (uint64_t)(2 * (kk & 3)) + (kk >= 4 ? half : 0), idesc, (c > c_begin || kk > 0) ? 1u : 0u);
                umma_commit(&a_empty[place]);
                umma_commit(&empty_bar[s]);
            }
            __syncwarp();
            if (++s == stages) s = 0;
            place = next;
            if (next == 0) pa ^= 1u;
        }
        if (ok && mxt_elect()) umma_commit(acc_bar);
    }
    mxt_finish<TO, GATED>(reinterpret_cast<float*>(ring), tmem_d, acc_cols, acc_bar, sent_bar, abort_flag, status, ok, c_end > c_begin,
                          min(bn, m - t0), ranks, rank, out + (long)t0 * ldo, ldo, f0, n, act);
    if (warp == MXT_WARPS && lane == 0 && *abort_flag) tma_drain(full_bar, stages, issued);
    __syncthreads();
    if (warp == MXT_WARPS + 1) tmem_dealloc(tmem_d, 512);
}

// A cluster of CTAs along the grid's x.
template <typename... KArgs, typename... Args>
static int mxt_launch_cluster(void (*kernel)(KArgs...), int threads, int smem, dim3 grid, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = grid.x;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = fl_pdl_enabled() ? 2 : 1;
    return (int)cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

// What a kernel takes, in ns: `launch`, and for each round of the device's clusters of `ranks` CTAs a chunk's time for each of a CTA's,
// and a tile's beginning and end: `tile`, more for each token, and for each whose sums it is sent.
struct MxtTimes {
    int launch, chunk, tile, token, sent;
};
// The clusters' size of least time for tiles of `bn` tokens, which it returns in `time`.  slots[r]: clusters of r CTAs that the device
// holds at once.
static int mxt_ranks(long tiles, int chunks, int bn, const int* slots, const MxtTimes& t, long* time) {
    int best = 1;
    *time = 0;
    for (int r = 1; r <= 8 && r <= chunks; ++r) {
        const int sent = (r - 1) * ((bn + r - 1) / r);
        if (slots[r] < 1 || (bn + sent) * MXT_PITCH * 4 > MXT_RING) continue;
        const long round = (long)((chunks + r - 1) / r) * t.chunk + t.tile + t.token * bn + t.sent * sent;
        const long all = (tiles + slots[r] - 1) / slots[r] * round + t.launch;
        if (*time == 0 || all < *time) best = r, *time = all;
    }
    return best;
}
static int mxt_failed() {
    const cudaError_t e = cudaGetLastError();
    return (int)(e == cudaSuccess ? cudaErrorInvalidDevice : e);
}
// Asked of the driver at a kernel's first launch on a device, which is also when the kernel gets its shared memory there.
struct MxtSlots {
    int of[MX_DEVICES][9];                  // [device][0]: asked
};
template <typename... KArgs>
static const int* mxt_slots(void (*kernel)(KArgs...), int threads, int smem, MxtSlots& found) {
    const int device = mx_device();
    if (device < 0) return nullptr;
    int* slots = found.of[device];
    if (slots[0]) return slots;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
        cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) != cudaSuccess)
        return nullptr;
    for (int r = 1; r <= 8; ++r) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(r);
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = r;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        if (cudaOccupancyMaxActiveClusters(&slots[r], kernel, &cfg) != cudaSuccess) return nullptr;
    }
    slots[0] = 1;
    return slots;
}

template <typename TO, bool GATED>
static int mxt_launch(const void* x, long ldx, const void* w, void* out, long ldo, int m, int n, int k, bool constant_w, FlGate act,
                      int which, int num_sms, int* status, cudaStream_t stream) {
    const int row_tiles = (n + (GATED ? 127 : 255)) / (GATED ? 128 : 256), chunks = (k + 127) / 128;
    static MxtSlots found;
    const int* slots = mxt_slots(mxt_kernel<TO, GATED>, MXT_THREADS, MXT_SMEM, found);
    if (!slots) return mxt_failed();
    // Tokens of a tile and CTAs of a cluster, by what the kernel takes (fitted to 190 measured products, 16 to 517 tokens, K 1024 to 22016,
    // 1536 to 12288 features, within 4% on average): a chunk a little more than half a us whatever the tokens, so as many of them
    // as there are, unless the tiles are too few for the SMs.  128 tokens 11008 -> 4096: 64 a tile with four CTAs 22.1 us, 128 with four
    // 28.1; 22016 -> 8192: 128 with four 44.7, 64 with two 63.1; 517 tokens 4096 -> 4096: 64 with one 26.9, 112 with one 34.1.
    int bn = 0, ranks = 1;
    long time = 0, rounds;
    for (int most = MXT_BN; most >= 64; most -= 32) {
        const int even = (m + most - 1) / most, tokens = (int)(((long)m + even - 1) / even + 15) / 16 * 16;
        if (tokens == bn) continue;
        long t;
        const MxtTimes times = {300, tokens <= 64 ? 560 + tokens * 3 / 2 : 790, 3800, 24, 22};
        const int r = mxt_ranks((long)((m + tokens - 1) / tokens) * row_tiles, chunks, tokens, slots, times, &t);
        if (bn == 0 || t < time) bn = tokens, ranks = r, time = t;
    }
    const int tokens_y = (m + bn - 1) / bn;
    // The kernel for few rows takes 0.19 ns for 1000 elements of W: one token 22016 -> 8192: 35.7 us, 29.7 here; 4096 -> the gated 2 x
    // 11008: 16.5, 22 here.
    if (which == 0 && m <= MXT_FEW_ROWS && 1500 + (long)n * (GATED ? 2 : 1) * k / 1000 * 19 / 100 < time) return MXT_FEW;
    // On pairs of CTAs: the way in and out, which no neighbour in the stream overlaps, the chunks, and the last tile's epilogue.  517 tokens
    // 4096 -> 4096: 24.4 us, 26.4 here; 192 tokens 4096 -> 12288: 25.4 and 26.9; 2048 tokens 4096 -> 12288: 141 and 224.
    const int pair_bn = mxp_tokens(m, row_tiles, num_sms / 2, &rounds);
    const bool fits = tokens_y <= 65535 && row_tiles <= 65535;       // a grid's y and z; pairs walk over any number of tiles
    if (which == 2 || (which == 0 && (!fits || 6000 + mxp_chunk(pair_bn) * rounds * chunks + 30 * pair_bn < time)))
        return mxp_launch<TO, GATED>(x, ldx, w, out, ldo, m, n, k, act, num_sms, status, stream);
    if (!fits) return (int)cudaErrorInvalidValue;
    const int per_rank = (chunks + ranks - 1) / ranks;
    int stages = MXT_RING / (bn * 256 + MXT_W_BYTES);               // (up to 64 tokens six at the least, else four)
    if (stages > MXT_MAX_STAGES) stages = MXT_MAX_STAGES;
    static_assert(MXT_RING / (64 * 256 + MXT_W_BYTES) >= 5 && MXT_RING / (MXT_BN * 256 + MXT_W_BYTES) >= 4, "as the converting warps' waits need");
    CUtensorMap map;
    int rc = make_map(&map, x, m, k, ldx, bn);
    if (rc) return rc;
    return mxt_launch_cluster(mxt_kernel<TO, GATED>, MXT_THREADS, MXT_SMEM, dim3(ranks, tokens_y, row_tiles), stream, map, (const uint8_t*)w,
                              (TO*)out, ldo, m, n, k, bn, stages, ranks, per_rank, constant_w, act, status);
}

// x: bfloat16 rows, 16-byte aligned, `ldx` elements apart (a multiple of 8).  n: output features (gated: half of w's rows).
// constant_w: nothing that may still run writes w, so its first bytes may be read while the kernels before this one run.
// which: 0 the kernel that takes less time, 1 the one above, 2 the one on pairs of CTAs (mxfp4_pair.cuh).  MXT_FEW: nothing has been
// launched, the kernel for few rows (fl_mx_few) takes less.
FL_API int fl_mxt_product(const void* x, long ldx, const void* w, void* out, int out_code, long ldo, int m, int n, int k, int gated,
                          int act, float p0, float p1, int constant_w, int which, int num_sms, int* status, cudaStream_t stream) {
    const FlGate gate = {act, p0, p1};
    FL_DISPATCH(out_code, TO, {
        return gated ? mxt_launch<TO, true>(x, ldx, w, out, ldo, m, n, k, constant_w != 0, gate, which, num_sms, status, stream)
                     : mxt_launch<TO, false>(x, ldx, w, out, ldo, m, n, k, constant_w != 0, gate, which, num_sms, status, stream);
    })
    return (int)cudaErrorInvalidValue;
}

// ---------------------------------------------------------------- both operands in 4 bits
// out[t, f] = sum_k A[t, k] W[f, k] on the block-scaled matrix instruction: codes in shared memory as they lie in the packed form (a
// row's 16 bytes of a block are a line of an 8 x 16-byte core matrix; core matrices 128 bytes apart along the rows, 2048 along
// K), the scales copied from there to tensor memory, 4 columns for 128 rows x 4 blocks.  A stage is two chunks of 128 along K, side by
// side in the packed form, of two tiles of W's rows and of one of A's: three copies.
//
// What bounds it: few rows the bytes (64 x 8192 x 22016 21.2 us, 4.5 TB/s), small products the way in and out (16 x 256 x 128 takes
// 2.8 us, 261 x 1537 x 1000 7.8, about 4 of them after its last stage).  A stage takes 0.56 us, its MMAs 0.27: the rest is the
// issuing warp's, which has three instructions for the scales of each chunk.  (Stages of one chunk: 0.33 us, and 128 x 4096 x 11008
// 15.5 us in place of 14.1.)
#define MXQ_STAGE (6 * MX_CHUNK)
#define MXQ_STAGES 4
#define MXQ_SF 24                                              // columns of a stage's scales: 12 for each chunk
#define MXQ_SMEM MXT_SMEM
static_assert(MXQ_STAGES * MXQ_STAGE <= MXT_RING, "the stages lie in the ring");

__device__ __forceinline__ void mxq_copy_scales(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
__device__ __forceinline__ void mxq_umma(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                         uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

template <typename TO>
__global__ void __launch_bounds__(MXT_THREADS, 1)
mxq_kernel(const uint8_t* __restrict__ a, const uint8_t* __restrict__ w, TO* __restrict__ out, long ldo, int m, int n, int chunks,
           int ranks, int per_rank, int* __restrict__ status) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* ring = (unsigned char*)(((uintptr_t)smem_raw + 127) & ~(uintptr_t)127);
    uint64_t* full_bar = (uint64_t*)(ring + MXT_RING);
    uint64_t* empty_bar = full_bar + MXQ_STAGES;
    uint64_t* acc_bar = empty_bar + MXQ_STAGES;
    uint64_t* sent_bar = acc_bar + 1;
    uint32_t* tmem_slot = (uint32_t*)(sent_bar + 1);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    const int warp = mxt_warp(), lane = threadIdx.x & 31;
    const int rank = blockIdx.x;
    const int t0 = blockIdx.y * 128, f0 = blockIdx.z * 256;
    const int rows = min(128, m - t0), tiles = n - f0 > 128 ? 2 : 1;
    const int c_begin = rank * per_rank, c_end = min((chunks + 1) / 2, c_begin + per_rank);       // stages along K

    if (threadIdx.x == 0) {
        for (int s = 0; s < MXQ_STAGES; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        mbar_init(acc_bar, 1);
        mbar_init(sent_bar, 1);
        *abort_flag = (*(volatile int*)status != 0) ? 1 : 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == MXT_WARPS + 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_d = __shfl_sync(0xffffffffu, *tmem_slot, 0), tmem_sf = tmem_d + 256;
    pdl_trigger();
    pdl_wait();
    int issued = 0;
    const bool ok = !*abort_flag;
    if (warp == MXT_WARPS) {
        // ---- producer
        const uint8_t* src_a = a + (long)blockIdx.y * chunks * MX_CHUNK;
        const uint8_t* src_w = w + (long)blockIdx.z * 2 * chunks * MX_CHUNK;
        int s = 0;
        uint32_t ph = 0;
        for (int c = c_begin; c < c_end && ok; ++c) {
            if (!mxt_wait(&empty_bar[s], ph ^ 1u, abort_flag)) {
                if (lane == 0) mxt_give_up(abort_flag, status);
                break;
            }
            if (mxt_elect()) {
                unsigned char* dst = ring + s * MXQ_STAGE;
                const uint32_t bytes = 2 * c + 1 < chunks ? 2 * MX_CHUNK : MX_CHUNK;
                mbar_expect_tx(&full_bar[s], (uint32_t)(tiles + 1) * bytes);
                mxt_copy(dst, src_a + 2l * c * MX_CHUNK, bytes, &full_bar[s]);
                for (int t = 0; t < tiles; ++t)
                    mxt_copy(dst + (1 + t) * 2 * MX_CHUNK, src_w + ((long)t * chunks + 2 * c) * MX_CHUNK, bytes, &full_bar[s]);
            }
            __syncwarp();
            ++issued;
            if (++s == MXQ_STAGES) { s = 0; ph ^= 1u; }
        }
    } else if (warp == MXT_WARPS + 1) {
        const int bn = (rows + 15) / 16 * 16;
        const uint32_t idesc[2] = {mxq_idesc(128, bn, 0), mxq_idesc(128, bn, 2)}, ring_at = smem_u32(ring);
        int s = 0;
        uint32_t ph = 0;
        bool going = ok;
        bool there = false;                                      // the next stage is known to be there
        for (int c = c_begin; c < c_end && going; ++c) {
            if (!__all_sync(0xffffffffu, there) && !mxt_wait(&full_bar[s], ph, abort_flag)) {
                if (lane == 0) mxt_give_up(abort_flag, status);
                going = false;
                break;
            }
            tc_fence_after();
            const int next = s + 1 == MXQ_STAGES ? 0 : s + 1;
            there = mxt_test(&full_bar[next], next ? ph : ph ^ 1u);
            const uint32_t at = ring_at + (uint32_t)(s * MXQ_STAGE), sf = tmem_sf + (uint32_t)(s * MXQ_SF);
            if (mxt_elect()) {
                // (the stage's columns: its last use's MMAs were done before its copies were sent for)
                const int two = 2 * c + 1 < chunks ? 2 : 1;
                for (int i = 0; i < two; ++i) {
                    const uint32_t from = at + (uint32_t)(i * MX_CHUNK), to = sf + (uint32_t)(12 * i);
                    for (int t = 0; t <= tiles; ++t)
                        mxq_copy_scales(to + (uint32_t)(4 * t), mxq_desc(from + (uint32_t)(t * 2 * MX_CHUNK + MX_CODES), 128));
                    for (int t = 0; t < tiles; ++t)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            mxq_umma(tmem_d + (uint32_t)(t * 128), mxq_desc(from + (uint32_t)((1 + t) * 2 * MX_CHUNK + h * 4096), 2048),
                                     mxq_desc(from + (uint32_t)(h * 4096), 2048), idesc[h], to + (uint32_t)(4 + 4 * t), to,
                                     (c > c_begin || i > 0 || h > 0) ? 1u : 0u);
                }
                umma_commit(&empty_bar[s]);
            }
            __syncwarp();
            if (++s == MXQ_STAGES) { s = 0; ph ^= 1u; }
        }
        if (going && mxt_elect()) umma_commit(acc_bar);
    }
    mxt_finish<TO, false>(reinterpret_cast<float*>(ring), tmem_d, 128, acc_bar, sent_bar, abort_flag, status, ok, c_end > c_begin, rows, ranks, rank,
                          out + (long)t0 * ldo, ldo, f0, n, FlGate{FL_ACT_NONE, 0.0f, 0.0f});
    if (warp == MXT_WARPS && lane == 0 && *abort_flag) tma_drain(full_bar, MXQ_STAGES, issued);
    __syncthreads();
    if (warp == MXT_WARPS + 1) tmem_dealloc(tmem_d, 512);
}

// a [m, k] and w [n, k] packed.  which: 0 the kernel that takes less time, 1 the one above, 2 the one on pairs of CTAs
// (mxfp4_pair.cuh).
FL_API int fl_mxq_product(const void* a, const void* w, void* out, int out_code, long ldo, int m, int n, int k, int which, int num_sms,
                          int* status, cudaStream_t stream) {
    const int chunks = (k + 127) / 128, stages = (chunks + 1) / 2, token_tiles = (m + 127) / 128, row_tiles = (n + 255) / 256;
    FL_DISPATCH(out_code, TO, {
        static MxtSlots found;
        const int* slots = mxt_slots(mxq_kernel<TO>, MXT_THREADS, MXQ_SMEM, found);
        if (!slots) return mxt_failed();
        // 14.1 us for 128 tokens 11008 -> 4096 with four CTAs, 16.2 with three, 19.0 with two, 28.0 with one; 8.5 for 16 tokens
        // 4096 -> 12288 with two, 12.4 with four.  On pairs 24.9 us for 517 tokens 4096 -> 12288, 28.8 here; 21.7 for 192 tokens 11008 ->
        // 4096, 14.8 here.
        long time;
        const int ranks = mxt_ranks((long)token_tiles * row_tiles, stages, m < 128 ? m : 128, slots, MxtTimes{340, 564, 2800, 16, 31}, &time);
        const long rounds = ((long)row_tiles * ((token_tiles + 1) / 2) + num_sms / 2 - 1) / (num_sms / 2);
        const bool fits = token_tiles <= 65535 && row_tiles <= 65535;
        if (which == 2 || (which == 0 && (!fits || (m > 128 && 6000 + rounds * (chunks * 170 + 2000) < time))))
            return mxqp_launch<TO>(a, w, out, ldo, m, n, k, num_sms, status, stream);
        if (!fits) return (int)cudaErrorInvalidValue;
        const int per_rank = (stages + ranks - 1) / ranks;
        return mxt_launch_cluster(mxq_kernel<TO>, MXT_THREADS, MXQ_SMEM, dim3(ranks, token_tiles, row_tiles), stream, (const uint8_t*)a,
                                  (const uint8_t*)w, (TO*)out, ldo, m, n, chunks, ranks, per_rank, status);
    })
    return (int)cudaErrorInvalidValue;
}
