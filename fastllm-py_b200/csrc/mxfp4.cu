// Microscaled 4-bit floating point (mxfp4.cuh says what the packed form is): rounding to it and back, and products of few rows with a
// matrix held in it.
#include "mxfp4.cuh"

// ---------------------------------------------------------------- rounding
// s = max(exponent byte of the block's largest magnitude - 2, 0): the largest then lies in [4, 8) units of S, or all are below
// that.  x / S is exact (a product with a power of two; what underflows rounds to 0 either way); the conversion rounds to
// nearest, ties to even codes, and saturates at 6.  A block with a NaN or an infinity has s = 255 and codes 0.
//
// Bound by memory: k (2 or 4) bytes of a row in, 17 k / 32 out.  A warp takes 8 rows of a chunk, 4 lanes a row: a lane's 8
// elements of each of the four blocks are loaded before the first is used.  The rows are two neighbours in each quarter of the
// tile: their scales are 32 bytes side by side, as two rows' codes of a block are, so that every 32-byte sector is written whole.
// Rows that do not begin on 16 bytes go through shared memory, an element a lane.  bfloat16 [2048, 11008] 10.4 us (5.5 TB/s), float
// [5503, 4096] 17.2 (5.9 TB/s).
__device__ __forceinline__ int mx_row_of(int unit, int i) { return 2 * unit + (i & 1) + 32 * (i >> 1); }      // unit 0 .. 15, i 0 .. 7

// 8 elements of a row from element c on, zeros behind k
__device__ __forceinline__ uint4 mx_tokens8(const bf16* row, int c, int k) {
    if (c + 8 <= k) return *reinterpret_cast<const uint4*>(row + c);
    uint32_t v[4] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (c + i < k) v[i >> 1] |= (uint32_t)__bfloat16_as_ushort(row[c + i]) << (16 * (i & 1));
    return make_uint4(v[0], v[1], v[2], v[3]);
}
struct MxFloat8 {
    float4 a, b;
};
__device__ __forceinline__ MxFloat8 mx_tokens8(const float* row, int c, int k) {
    if (c + 8 <= k) return {reinterpret_cast<const float4*>(row + c)[0], reinterpret_cast<const float4*>(row + c)[1]};
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < k ? row[c + i] : 0.0f;
    return {make_float4(v[0], v[1], v[2], v[3]), make_float4(v[4], v[5], v[6], v[7])};
}
// 8 rows of a chunk in a warp's shared memory, elements between rows so that 16 bytes of four lanes a row meet no bank twice
template <typename T> constexpr int MX_PITCH = sizeof(T) == 2 ? 160 : 132;
// a word of codes: a conversion makes a byte of two neighbouring nibbles
__device__ __forceinline__ uint32_t mx_word(const float (&v)[8]) {
    uint32_t word;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\tmov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(word)
        : "f"(v[0]), "f"(v[2]), "f"(v[4]), "f"(v[6]), "f"(v[1]), "f"(v[3]), "f"(v[5]), "f"(v[7]));
    return word;
}
// the scale byte of a block whose largest magnitude has these bits (magnitudes compare as integers do, a NaN above all)
__device__ __forceinline__ int mx_scale_byte(uint32_t top) {
    const int e = (int)(top >> 23);
    return e == 255 ? 255 : max(e - 2, 0);
}
__device__ __forceinline__ float mx_inverse(int s) { return __uint_as_float((uint32_t)(254 - min(s, 253)) << 23); }   // 2^(127 - s)
// A lane's 8 elements of a block that 4 lanes have: their largest magnitude's scale byte, and the word of codes.  bfloat16 pairs are
// compared as pairs of 16-bit integers, and multiplied as pairs: with a power of two that is exact but for what is far below a code.
__device__ __forceinline__ uint32_t mx_codes(const uint4& x, int& s) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    uint32_t top = __vmaxu2(__vmaxu2(w[0] & 0x7FFF7FFFu, w[1] & 0x7FFF7FFFu), __vmaxu2(w[2] & 0x7FFF7FFFu, w[3] & 0x7FFF7FFFu));
    top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 2));
    s = mx_scale_byte(max(top, top << 16));
    const uint32_t inv = (uint32_t)(254 - min(s, 253)) * 0x00800080u;
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t y = mx_mul(w[i], inv);
        v[2 * i] = __uint_as_float(y << 16);
        v[2 * i + 1] = __uint_as_float(y & 0xFFFF0000u);
    }
    return mx_word(v);
}
__device__ __forceinline__ uint32_t mx_codes(const MxFloat8& x, int& s) {
    float v[8] = {x.a.x, x.a.y, x.a.z, x.a.w, x.b.x, x.b.y, x.b.z, x.b.w};
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    s = mx_scale_byte(top);
    const float inv = mx_inverse(s);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= inv;
    return mx_word(v);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) mx_quantize_kernel(const T* __restrict__ x, long ld, uint8_t* __restrict__ data, int m,
                                                          int k, int chunks) {
    pdl_wait();
    pdl_trigger();
    const int chunk = blockIdx.y * 8 + (threadIdx.x >> 5);           // a unit of 8 rows x one chunk; 16 units fill a tile's chunk
    if (chunk >= chunks) return;                                     // (whole warps)
    const int lane = threadIdx.x & 31, t = lane & 3;
    const long tile = blockIdx.x >> 4;
    const int u = blockIdx.x & 15;
    uint8_t* dst = data + (tile * chunks + chunk) * MX_CHUNK;
    const int r = mx_row_of(u, lane >> 2);
    const long row = tile * MX_ROWS + r;
    decltype(mx_tokens8(x, 0, 0)) v[4];
    if constexpr (VEC) {
#pragma unroll
        for (int b = 0; b < 4; ++b) v[b] = mx_tokens8(x + row * ld, row < m ? chunk * 128 + b * 32 + t * 8 : k, k);
    } else {
        __shared__ __align__(16) T staged[8][8 * MX_PITCH<T>];
        T* mine = staged[threadIdx.x >> 5];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const long from = tile * MX_ROWS + mx_row_of(u, i);
                const int c = chunk * 128 + b * 32 + lane;
                mine[i * MX_PITCH<T> + b * 32 + lane] = from < m && c < k ? x[from * ld + c] : from_f32<T>(0.0f);
            }
        __syncwarp();
#pragma unroll
        for (int b = 0; b < 4; ++b) v[b] = mx_tokens8(mine + (lane >> 2) * MX_PITCH<T>, b * 32 + t * 8, 128);
    }
    uint32_t scales = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        int s;
        const uint32_t word = mx_codes(v[b], s);
        scales |= (uint32_t)s << (8 * b);
        *reinterpret_cast<uint32_t*>(dst + b * 2048 + r * 16 + t * 4) = s == 255 ? 0 : word;
    }
    if (t == 0) *reinterpret_cast<uint32_t*>(dst + mx_scale_at(r)) = scales;
}

FL_API int fl_mx_quantize(const void* x, int code, long ld, void* data, int m, int k, cudaStream_t stream) {
    const int chunks = (k + 127) / 128;
    const dim3 grid((unsigned)((m + MX_ROWS - 1) / MX_ROWS) * 16, (chunks + 7) / 8);
    if (grid.y > 65535) return (int)cudaErrorInvalidValue;
    FL_DISPATCH(code, T, {
        const bool vec = (((uintptr_t)x | (uintptr_t)(ld * (long)sizeof(T))) & 15) == 0;
        return fl_launch(vec ? mx_quantize_kernel<T, true> : mx_quantize_kernel<T, false>, grid, dim3(256), 0, stream,
                         (const T*)x, ld, (uint8_t*)data, m, k, chunks);
    })
    return (int)cudaErrorInvalidValue;
}

// Back: the same division of the work, bound by memory; rows that do not begin on 16 bytes are written an element a lane, the words of
// a row handed round by shuffles, and are bound by issue: 19.9 million instructions where the same rows aligned take 7.1, 85% of the
// issue slots, and as many sectors written.  (Through shared memory they took as long, and twice that after a kernel without any:
// the SMs' memory is then divided anew.)  [2048, 11008] to bfloat16 11.4 us (5.0 TB/s), [5503, 4096] to float 18.0 (5.7 TB/s),
// [5503, 4097] 23.3.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(const uint8_t* __restrict__ data, T* __restrict__ out, long ld, int m,
                                                            int k, int chunks) {
    pdl_wait();
    pdl_trigger();
    const int chunk = blockIdx.y * 8 + (threadIdx.x >> 5);
    if (chunk >= chunks) return;
    const int lane = threadIdx.x & 31, t = lane & 3;
    const long tile = blockIdx.x >> 4;
    const int u = blockIdx.x & 15, r = mx_row_of(u, lane >> 2);
    const uint8_t* src = data + (tile * chunks + chunk) * MX_CHUNK;
    const uint32_t scales = *reinterpret_cast<const uint32_t*>(src + mx_scale_at(r));
    // 16 bytes of output a lane and store, side by side: 8 bfloat16 of a word, or 4 floats of each of two words
    constexpr int WORDS = VEC ? sizeof(T) / 2 : 1, N = 16 / sizeof(T);
    uint32_t word[4][WORDS];
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int j = 0; j < WORDS; ++j)
            word[b][j] = *reinterpret_cast<const uint32_t*>(src + b * 2048 + r * 16 + (WORDS == 1 ? t : 2 * j + (t >> 1)) * 4);
    if constexpr (VEC) {
        const long row = tile * MX_ROWS + r;
        const bool large = __any_sync(0xffffffffu, (scales & 0x80808080u & ((scales & 0x7F7F7F7Fu) + 0x7F7F7F7Fu)) != 0);
        if (row >= m) return;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const uint32_t s = scales >> (8 * b) & 255u;
#pragma unroll
            for (int j = 0; j < WORDS; ++j) {
                uint32_t w[4];                                        // in bfloat16, which has all that float has of these values
                mx_pairs(WORDS == 1 ? word[b][j] : word[b][j] >> (8 * (t & 1)), large ? mx_factor_large(s) : mx_factor(s), w);
                if (large)
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = mx_mul(w[i], mx_factor_rest(s));
                __align__(16) T v[N];
#pragma unroll
                for (int i = 0; i < N / 2; ++i) {
                    if (sizeof(T) == 2) {
                        reinterpret_cast<uint32_t*>(v)[i] = w[i];
                    } else {
                        reinterpret_cast<uint32_t*>(v)[2 * i] = w[i] << 16;
                        reinterpret_cast<uint32_t*>(v)[2 * i + 1] = w[i] & 0xFFFF0000u;
                    }
                }
                const int c = chunk * 128 + b * 32 + (j * 4 + t) * N;
                T* dst = out + row * ld + c;
                if (c + N <= k) {
                    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(v);
                } else {
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (c + i < k) dst[i] = v[i];
                }
            }
        }
    } else {
        const int place = 4 * ((lane & 1) * 4 + (lane >> 1 & 3));         // of element lane % 8 in its word
#pragma unroll 2
        for (int i = 0; i < 8; ++i) {
            const long row = tile * MX_ROWS + mx_row_of(u, i);
            const uint32_t sc = __shfl_sync(0xffffffffu, scales, 4 * i);
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const uint32_t code = __shfl_sync(0xffffffffu, word[b][0], 4 * i + (lane >> 3)) >> place;
                const int c = chunk * 128 + b * 32 + lane;
                if (row < m && c < k) out[row * ld + c] = from_f32<T>(mx_value(code) * mx_scale((int)(sc >> (8 * b)) & 255));
            }
        }
    }
}

FL_API int fl_mx_dequantize(const void* data, void* out, int code, long ld, int m, int k, cudaStream_t stream) {
    const int chunks = (k + 127) / 128;
    const dim3 grid((unsigned)((m + MX_ROWS - 1) / MX_ROWS) * 16, (chunks + 7) / 8);
    if (grid.y > 65535) return (int)cudaErrorInvalidValue;
    FL_DISPATCH(code, T, {
        const bool vec = (((uintptr_t)out | (uintptr_t)(ld * (long)sizeof(T))) & 15) == 0;
        return fl_launch(vec ? mx_dequantize_kernel<T, true> : mx_dequantize_kernel<T, false>, grid, dim3(256), 0,
                         stream, (const uint8_t*)data, (T*)out, ld, m, k, chunks);
    })
    return (int)cudaErrorInvalidValue;
}

// ---------------------------------------------------------------- products of few rows
// out[t, f] = sum_k x[t, k] W[f, k] for up to 8 tokens, or of a gated unit act(gate, up) of features f and n + f.  A CTA takes 2 x 16
// rows of W (of a gated unit 16 gate rows and the 16 up rows of the same features), a warp of it every WARPS-th chunk of K.  The rows
// are the 16 of m16n8k16 and the tokens its 8 columns.
// Lane 4 g + q reads the 16 bytes of rows g and g + 8 of block q, so a lane has one scale for 32 codes; which elements of K meet in
// one instruction does not matter as long as both operands agree, and a lane's 8 consecutive elements of a token are the partners of
// one word of codes.  The warps' sums meet in shared memory and are added in order.
//
// LB warps fit an SM.  With 20 and more a warp has registers for one chunk: its rows are loaded anew for the next one as soon as
// their codes have been read, and its tokens at the end.  With 16 the next codes are on their way during the whole chunk.
//
// What bounds it: the wait for the codes, and then issue.  One token 4096 -> 12288 takes 10.1 us (2.6 TB/s), 4096 -> the gated 2 x 11008
// 16.6 (2.9 TB/s).  With 20 and 17 warps an SM a warp issues every 9.5 and 7.5 clocks, of which it waits 4.0 and 3.3 for memory; the
// issue slots are 53% and 59% taken while an SM has work, and SMs have it for 86% and 90% of the busiest one's time.  The conversion of 256 values takes 18 clocks of a quarter's integer units: 3 us and 5.5 at the least.  The matrix instructions
// bound nothing: 8 clocks of a quarter each, 21 for a link of a chain on one accumulator, which three warps a quarter hide; their pipe
// is 0.16 and 0.19 busy.  2 to 8 tokens take 1 to 5% more.
__device__ __forceinline__ void mx_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <typename TO, int WARPS, bool GATED, int LB>
__global__ void __launch_bounds__(WARPS * 32, LB / WARPS)
mx_few_kernel(const bf16* __restrict__ x, long ldx, const uint8_t* __restrict__ w, TO* __restrict__ out, long ldo, int m, int n, int k,
              bool constant_w, FlGate act) {
    constexpr int MT = 2, ROWS = GATED ? 16 : 32;                    // tiles of 16 rows, output features of a CTA
    constexpr bool EARLY = LB <= 16;
    __shared__ float red[WARPS][8][MT * 16 + 1];
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const int chunks = (k + 127) / 128;
    const int f0 = blockIdx.x * ROWS;
    // codes of block q of a row, of the warp's next chunk (a row that does not exist: of the last one; not stored)
    const uint8_t* src[MT][2];
    int sc_at[MT][2];                                                // from there to the block's scale
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int f = min(f0 + (GATED ? 0 : 16 * t) + 8 * h + g, n - 1);
            const long row = (GATED ? (long)t * n : 0) + f;
            const int r = (int)(row & (MX_ROWS - 1));
            src[t][h] = w + (row / MX_ROWS * chunks + warp) * (long)MX_CHUNK + q * 2048 + r * 16;
            sc_at[t][h] = (int)mx_scale_at(r) + q - (q * 2048 + r * 16);
        }
    uint4 z[MT][2];
    uint32_t s[MT][2];
    auto fetch = [&](int t) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            z[t][h] = *reinterpret_cast<const uint4*>(src[t][h]);
            s[t][h] = src[t][h][sc_at[t][h]];
            src[t][h] += WARPS * MX_CHUNK;
        }
    };
    const bf16* token = x + (long)min(g, m - 1) * ldx;               // (likewise)
    uint4 xs[4];
    auto fetch_x = [&](int c, int e) {                               // 8 elements; zeros behind k
        const bf16* at = token + c * 128 + q * 32 + e * 8;
        if (c * 128 + 128 <= k) xs[e] = *reinterpret_cast<const uint4*>(at);       // (the same in all lanes)
        else xs[e] = mx_tokens8(token, c * 128 + q * 32 + e * 8, k);
    };
    if (!constant_w) pdl_wait();
    if (warp < chunks)
#pragma unroll
        for (int t = 0; t < MT; ++t) fetch(t);
    if (constant_w) pdl_wait();
    if (!EARLY && warp < chunks)
#pragma unroll
        for (int e = 0; e < 4; ++e) fetch_x(warp, e);
    float acc[MT][4] = {};
#pragma unroll 1
    for (int c = warp; c < chunks; c += WARPS) {
        const bool more = c + WARPS < chunks;
        uint4 y[MT][2];
        uint32_t sy[MT][2], most = 0;
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                y[t][h] = z[t][h];
                sy[t][h] = s[t][h];
                most = max(most, sy[t][h]);
            }
        if (EARLY) {
#pragma unroll
            for (int e = 0; e < 4; ++e) fetch_x(c, e);
            if (more)
#pragma unroll
                for (int t = 0; t < MT; ++t) fetch(t);
        }
        if (!__any_sync(0xffffffffu, most > 128u)) {
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const uint32_t m1[2] = {mx_factor(sy[t][0]), mx_factor(sy[t][1])};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t v[2][4];
#pragma unroll
                    for (int h = 0; h < 2; ++h) mx_pairs(e == 0 ? y[t][h].x : e == 1 ? y[t][h].y : e == 2 ? y[t][h].z : y[t][h].w, m1[h], v[h]);
                    mx_mma(acc[t], v[0][0], v[1][0], v[0][1], v[1][1], xs[e].x, xs[e].y);
                    mx_mma(acc[t], v[0][2], v[1][2], v[0][3], v[1][3], xs[e].z, xs[e].w);
                }
                if (!EARLY && more) fetch(t);
            }
        } else {                                                     // some block's scale takes two factors
#pragma unroll
            for (int t = 0; t < MT; ++t) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t v[2][4];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        mx_pairs(e == 0 ? y[t][h].x : e == 1 ? y[t][h].y : e == 2 ? y[t][h].z : y[t][h].w, mx_factor_large(sy[t][h]), v[h]);
#pragma unroll
                        for (int j = 0; j < 4; ++j) v[h][j] = mx_mul(v[h][j], mx_factor_rest(sy[t][h]));
                    }
                    mx_mma(acc[t], v[0][0], v[1][0], v[0][1], v[1][1], xs[e].x, xs[e].y);
                    mx_mma(acc[t], v[0][2], v[1][2], v[0][3], v[1][3], xs[e].z, xs[e].w);
                }
                if (!EARLY && more) fetch(t);
            }
        }
        if (!EARLY && more)
#pragma unroll
            for (int e = 0; e < 4; ++e) fetch_x(c + WARPS, e);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[warp][2 * q + (e & 1)][t * 16 + g + 8 * (e >> 1)] = acc[t][e];
    __syncthreads();
    for (int i = threadIdx.x; i < ROWS * m; i += WARPS * 32) {
        const int t = i / ROWS, f = i % ROWS;
        if (f0 + f >= n) continue;
        float v = 0.0f, u = 1.0f;
#pragma unroll
        for (int j = 0; j < WARPS; ++j) v += red[j][t][f];
        if (GATED) {
            u = 0.0f;
#pragma unroll
            for (int j = 0; j < WARPS; ++j) u += red[j][t][(MT - 1) * 16 + f];
        }
        out[(long)t * ldo + f0 + f] = from_f32<TO>(act.act == FL_ACT_NONE ? v : fl_gated(v, u, act));
    }
}

template <typename TO, int WARPS, bool GATED, int LB>
static int mx_launch_few(const bf16* x, long ldx, const uint8_t* w, TO* out, long ldo, int m, int n, int k, bool constant_w,
                         FlGate act, cudaStream_t stream) {
    constexpr int ROWS = GATED ? 16 : 32;
    return fl_launch(mx_few_kernel<TO, WARPS, GATED, LB>, dim3((n + ROWS - 1) / ROWS), dim3(WARPS * 32), 0, stream, x, ldx, w, out, ldo, m, n, k,
                     constant_w, act);
}

// x: up to 8 bfloat16 rows with `ldx` elements between them (a multiple of 8, from 16 bytes on).  n: output features (gated: half
// of w's rows).  act: an FlAct or FL_ACT_NONE; a product that is not gated has f(v, 1).  constant_w: nothing that may still
// run writes w, so its first bytes may be read while the kernels before this one in the stream run.
FL_API int fl_mx_few(const void* x, long ldx, const void* w, void* out, int out_code, long ldo, int m, int n, int k, int gated,
                     int act, float p0, float p1, int constant_w, int num_sms, cudaStream_t stream) {
    const FlGate gate = {act, p0, p1};
    if (m > 8) return (int)cudaErrorInvalidValue;
    // Warps of a CTA, and CTAs an SM, by how many CTAs there are: all of them at once, as far as that goes, and then as many registers a
    // thread as that leaves.  One token, in us, with 16 warps an SM in CTAs of 16 and 8, with 24 in CTAs of 8, with 20 in CTAs of 4:
    // 128 CTAs (11008 -> 4096) 9.5, 18, 21, 24; 256 (22016 -> 8192) 38, 36, 45, 72; 384 (4096 -> 12288) 13.3, 12.7, 10.6, 15.5; 688
    // (4096 -> the gated 2 x 11008) 24.9, 22.8, 19.2, 17.1.
    const int ctas = gated ? (n + 15) / 16 : (n + 31) / 32;
    FL_DISPATCH(out_code, TO, {
#define MX_FEW(WARPS, LB)                                                                                                              \
    return gated ? mx_launch_few<TO, WARPS, true, LB>((const bf16*)x, ldx, (const uint8_t*)w, (TO*)out, ldo, m, n, k, constant_w != 0, gate, stream) \
                 : mx_launch_few<TO, WARPS, false, LB>((const bf16*)x, ldx, (const uint8_t*)w, (TO*)out, ldo, m, n, k, constant_w != 0, gate, stream)
        if (ctas <= num_sms) MX_FEW(16, 16);
        if (ctas <= 2 * num_sms) MX_FEW(8, 16);
        if (ctas <= 3 * num_sms) MX_FEW(8, 24);
        MX_FEW(4, 20);
    })
    return (int)cudaErrorInvalidValue;
}
