// Microscaled 4-bit floating point (MXFP4, the OCP microscaling format): rounding to it and back, and products of a matrix
// held in it.
//
// Along K a matrix is cut into blocks of 32.  A block has one scale S = 2^(s - 127) with a byte s (255: the block is NaN) and
// 32 elements of 4 bits, a sign and the magnitude 0, 0.5, 1, 1.5, 2, 3, 4 or 6 (e2m1).
//
// The packed form, as every kernel here reads it: [row tiles of 128][K chunks of 128][MX_CHUNK bytes].  A chunk holds four
// pieces, one for each block, of 128 rows x 16 bytes of codes, then 512 bytes of scales: row r's four in one word at
// (r % 32) * 16 + (r / 32) * 4.  Nibble j of a 4-byte word of codes is element 2 j for j < 4 and 2 (j - 4) + 1 after that, so
// that one shift and one mask give two neighbours in the two halves of a word.  A row's codes of a block are 16 bytes in one
// piece and a tile's rows lie side by side: what an 8 x 16-byte core matrix of a tcgen05 operand is, and a chunk is one
// copy.  The scales lie as tcgen05.cp takes them to tensor memory.
#include "common.cuh"

#define MX_ROWS 128
#define MX_CODES 8192
#define MX_CHUNK 8704

__device__ __forceinline__ long mx_scale_at(int r) { return MX_CODES + (r & 31) * 16 + (r >> 5) * 4; }
__device__ __forceinline__ float mx_scale(int s) {          // 2^(s - 127)
    return s == 255 ? CUDART_NAN_F : (s == 0 ? __uint_as_float(0x00400000u) : __uint_as_float((uint32_t)s << 23));
}
// Element j of a word (the order above) in float, without its block's scale: sign and magnitude put where a float of exponent
// 2^-126 has them, a subnormal for the magnitudes 0 and 0.5, and multiplied by 2^126, exactly.
__device__ __forceinline__ float mx_value(uint32_t word, int j) {
    const uint32_t code = word >> (((j & 1) * 4 + (j >> 1)) * 4);
    return __uint_as_float(((code & 8u) << 28) | ((code & 7u) << 22)) * 8.507059173023462e37f;
}

// ---------------------------------------------------------------- rounding
// s = max(exponent byte of the block's largest magnitude - 2, 0): the largest then lies in [4, 8) units of S, or all are below
// that.  x / S is exact (a product with a power of two; what underflows rounds to 0 either way); the conversion rounds to
// nearest, ties to even codes, and saturates at 6.  A block with a NaN or an infinity has s = 255 and codes 0.
//
// Bound by memory: k (2 or 4) bytes of a row in, 17 k / 32 out.  A warp takes 8 rows of a chunk, 4 lanes a row: a lane's 8
// elements of each of the four blocks are loaded before the first is used, and a warp's codes of a block are 128 bytes side
// by side.
template <typename T> __device__ __forceinline__ void mx_load8(const T* src, int n, bool vec, float (&v)[8]) {
    if (vec && n >= 8) {
        if (sizeof(T) == 2) {
            const uint4 r = *reinterpret_cast<const uint4*>(src);
            const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
            }
        } else {
            const float4 a = reinterpret_cast<const float4*>(src)[0], b = reinterpret_cast<const float4*>(src)[1];
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? to_f32<T>(src[i]) : 0.0f;
}

template <typename T>
__global__ void __launch_bounds__(256) mx_quantize_kernel(const T* __restrict__ x, long ld, uint8_t* __restrict__ data, int m,
                                                          int k, int chunks, long units, bool vec) {
    pdl_wait();
    pdl_trigger();
    const long unit = (long)blockIdx.x * 8 + (threadIdx.x >> 5);     // 8 rows x one chunk; 16 units fill a tile's chunk
    if (unit >= units) return;                                       // (whole warps)
    const int lane = threadIdx.x & 31, t = lane & 3;
    const int chunk = (int)(unit % chunks);
    const long row0 = unit / chunks * 8;
    const long row = row0 + (lane >> 2);
    const int r = (int)(row & (MX_ROWS - 1));
    uint8_t* dst = data + (row / MX_ROWS * chunks + chunk) * MX_CHUNK;
    float v[4][8];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const int c = chunk * 128 + b * 32 + t * 8;
        mx_load8(x + row * ld + c, row < m ? k - c : 0, vec, v[b]);
    }
    uint32_t scales = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        // magnitudes compare as integers do, a NaN above all
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[b][i]) & 0x7FFFFFFFu);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = (int)(top >> 23);
        const int s = e == 255 ? 255 : max(e - 2, 0);
        scales |= (uint32_t)s << (8 * b);
        const float inv = __uint_as_float((uint32_t)(254 - min(s, 253)) << 23);     // 2^(127 - s)
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t two;                                             // element 2 i in the low nibble, 2 i + 1 in the high one
            asm("{\n\t.reg .b8 q;\n\tcvt.rn.satfinite.e2m1x2.f32 q, %2, %1;\n\tcvt.u32.u8 %0, q;\n\t}"
                : "=r"(two)
                : "f"(v[b][2 * i] * inv), "f"(v[b][2 * i + 1] * inv));
            word |= (two & 0xFu) << (4 * i) | (two >> 4) << (16 + 4 * i);
        }
        if (s == 255) word = 0;
        *reinterpret_cast<uint32_t*>(dst + b * 2048 + r * 16 + t * 4) = word;
    }
    if (t == 0) *reinterpret_cast<uint32_t*>(dst + mx_scale_at(r)) = scales;
}

FL_API int fl_mx_quantize(const void* x, int code, long ld, void* data, int m, int k, cudaStream_t stream) {
    const int chunks = (k + 127) / 128;
    const long units = (long)((m + MX_ROWS - 1) / MX_ROWS) * 16 * chunks;
    if ((units + 7) / 8 > 0x7FFFFFFFl) return (int)cudaErrorInvalidValue;
    FL_DISPATCH(code, T, {
        const bool vec = (((uintptr_t)x | (uintptr_t)(ld * (long)sizeof(T))) & 15) == 0;
        return fl_launch(mx_quantize_kernel<T>, dim3((unsigned)((units + 7) / 8)), dim3(256), 0, stream, (const T*)x, ld,
                         (uint8_t*)data, m, k, chunks, units, vec);
    })
    return (int)cudaErrorInvalidValue;
}

template <typename T>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(const uint8_t* __restrict__ data, T* __restrict__ out, long ld, int m,
                                                            int k, int chunks, long units, bool vec) {
    pdl_wait();
    pdl_trigger();
    const long unit = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (unit >= units) return;
    const int lane = threadIdx.x & 31, t = lane & 3;
    const int chunk = (int)(unit % chunks);
    const long row = unit / chunks * 8 + (lane >> 2);
    if (row >= m) return;
    const int r = (int)(row & (MX_ROWS - 1));
    const uint8_t* src = data + (row / MX_ROWS * chunks + chunk) * MX_CHUNK;
    const uint32_t scales = *reinterpret_cast<const uint32_t*>(src + mx_scale_at(r));
    uint32_t word[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) word[b] = *reinterpret_cast<const uint32_t*>(src + b * 2048 + r * 16 + t * 4);
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const int c = chunk * 128 + b * 32 + t * 8;
        const float scale = mx_scale((int)(scales >> (8 * b)) & 255);
        T v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = from_f32<T>(mx_value(word[b], i) * scale);
        T* dst = out + row * ld + c;
        if (vec && c + 8 <= k) {
#pragma unroll
            for (int i = 0; i < (int)(8 * sizeof(T) / 16); ++i) reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(v)[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < k) dst[i] = v[i];
        }
    }
}

FL_API int fl_mx_dequantize(const void* data, void* out, int code, long ld, int m, int k, cudaStream_t stream) {
    const int chunks = (k + 127) / 128;
    const long units = (long)((m + 7) / 8) * chunks;
    if ((units + 7) / 8 > 0x7FFFFFFFl) return (int)cudaErrorInvalidValue;
    FL_DISPATCH(code, T, {
        const bool vec = (((uintptr_t)out | (uintptr_t)(ld * (long)sizeof(T))) & 15) == 0;
        return fl_launch(mx_dequantize_kernel<T>, dim3((unsigned)((units + 7) / 8)), dim3(256), 0, stream, (const uint8_t*)data,
                         (T*)out, ld, m, k, chunks, units, vec);
    })
    return (int)cudaErrorInvalidValue;
}

// ---------------------------------------------------------------- products
// out[t, f] = sum_k x[t, k] W[f, k], or of a gated unit act(gate, up) of features f and n + f.  A warp sums one feature for 8
// tokens: 16 lanes share a chunk, 8 elements each.  x comes in bfloat16 or packed as W is.
template <typename TO, bool PACKED, bool GATED>
__global__ void __launch_bounds__(256) mx_product_kernel(const void* __restrict__ x, long ldx, const uint8_t* __restrict__ w,
                                                         TO* __restrict__ out, long ldo, int m, int n, int k, FlGate act) {
    pdl_wait();
    pdl_trigger();
    const int chunks = (k + 127) / 128;
    const int lane = threadIdx.x & 31;
    const int groups = (n + 7) / 8;
    const int f = blockIdx.x % groups * 8 + (threadIdx.x >> 5);
    const int t0 = blockIdx.x / groups * 8;
    if (f >= n) return;                                               // (whole warps)
    float acc[GATED ? 2 : 1][8] = {};
    for (int chunk = lane >> 4; chunk < chunks; chunk += 2) {
        const int b = (lane >> 2) & 3, word = lane & 3;
        float v[GATED ? 2 : 1][8];
#pragma unroll
        for (int g = 0; g < (GATED ? 2 : 1); ++g) {
            const long row = (long)g * n + f;
            const int r = (int)(row & (MX_ROWS - 1));
            const uint8_t* src = w + (row / MX_ROWS * chunks + chunk) * MX_CHUNK;
            const uint32_t codes = *reinterpret_cast<const uint32_t*>(src + b * 2048 + r * 16 + word * 4);
            const float scale = mx_scale(src[mx_scale_at(r) + b]);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[g][i] = mx_value(codes, i) * scale;
        }
        const int c = chunk * 128 + b * 32 + word * 8;
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            if (t0 + t >= m) break;
            float a[8];
            if (PACKED) {
                const int r = (t0 + t) & (MX_ROWS - 1);
                const uint8_t* src = (const uint8_t*)x + ((long)((t0 + t) / MX_ROWS) * chunks + chunk) * MX_CHUNK;
                const uint32_t codes = *reinterpret_cast<const uint32_t*>(src + b * 2048 + r * 16 + word * 4);
                const float scale = mx_scale(src[mx_scale_at(r) + b]);
#pragma unroll
                for (int i = 0; i < 8; ++i) a[i] = mx_value(codes, i) * scale;
            } else {
                mx_load8((const bf16*)x + (long)(t0 + t) * ldx + c, k - c, true, a);
            }
#pragma unroll
            for (int g = 0; g < (GATED ? 2 : 1); ++g)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (c + i < k) acc[g][t] = fmaf(a[i], v[g][i], acc[g][t]);
        }
    }
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        const float g = warp_sum(acc[0][t]);
        const float u = GATED ? warp_sum(acc[GATED ? 1 : 0][t]) : 1.0f;
        if (lane == 0 && t0 + t < m) out[(long)(t0 + t) * ldo + f] = from_f32<TO>(act.act == FL_ACT_NONE ? g : fl_gated(g, u, act));
    }
}

template <typename TO, bool PACKED, bool GATED>
static int mx_launch_product(const void* x, long ldx, const void* w, void* out, long ldo, int m, int n, int k, FlGate act,
                             cudaStream_t stream) {
    const long blocks = (long)((n + 7) / 8) * ((m + 7) / 8);
    if (blocks > 0x7FFFFFFFl) return (int)cudaErrorInvalidValue;
    return fl_launch(mx_product_kernel<TO, PACKED, GATED>, dim3((unsigned)blocks), dim3(256), 0, stream, x, ldx,
                     (const uint8_t*)w, (TO*)out, ldo, m, n, k, act);
}

// x: bfloat16 rows with `ldx` elements between them (a multiple of 8, from 16 bytes on), or, ldx 0, packed.  n: output features
// (gated: half of w's rows).  act: an FlAct or FL_ACT_NONE; a product that is not gated has f(v, 1).
FL_API int fl_mx_product(const void* x, long ldx, const void* w, void* out, int out_code, long ldo, int m, int n, int k, int gated,
                         int act, float p0, float p1, cudaStream_t stream) {
    const FlGate gate = {act, p0, p1};
    FL_DISPATCH(out_code, TO, {
        if (gated) return mx_launch_product<TO, false, true>(x, ldx, w, out, ldo, m, n, k, gate, stream);
        if (ldx == 0) return mx_launch_product<TO, true, false>(x, ldx, w, out, ldo, m, n, k, gate, stream);
        return mx_launch_product<TO, false, false>(x, ldx, w, out, ldo, m, n, k, gate, stream);
    })
    return (int)cudaErrorInvalidValue;
}
