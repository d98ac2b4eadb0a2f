// Quantisation to FP8 e4m3 with one power-of-two scale for each block of 128 elements, along the rows of a matrix, along
// its columns, or both from one read; the same from a matrix already held that way (the 8-bit activation checkpoint of a
// training step turned into the operand of its weight gradient); and the way back.
//
//   E(block) = the least integer e >= -127 with max |x| <= 448 * 2^e     (0 for a block of zeros)
//   code     = round_to_nearest_even_e4m3(x * 2^-E),  scale byte = E + 127 (ue8m0: the value 2^E)
//   a block that holds an infinity or a NaN is a NaN as a whole: scale byte 255, every code 0x7f.
// With the rounding of E upwards nothing saturates, and x * 2^-E is exact, so a code's one rounding is the conversion's.
//
// What bounds these passes is HBM: one read of the source, one byte per element and form written. A CTA owns a tile of 128 x
// 128 elements, the block of either direction, and holds it in registers (8 rows x 8 columns a thread), so the maxima, the
// scales and both forms' codes come from one read. The column form leaves through a 16 KB shared-memory tile as rows of 128
// contiguous bytes; its eight-byte pieces are exchanged by an XOR of the column group so that neither the writes (one column
// group a lane) nor the reads (one column a half-warp) meet in a bank.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "gemm_launch.cuh"
#include "qgemm_internal.h"

namespace qgemm {

namespace {

constexpr int kQbThreads = 256;
constexpr int kQb = 128;  // block length, and the side of a CTA's tile

struct QuantBlockParams {
    const void* in;
    long long ld_in;
    const uint8_t* in_scale;  // source held in 8 bits: its scales [ceil(cols / 128), rows]
    uint8_t *q, *qt;          // row form [rows, cols], column form [cols, rows]
    long long ld_q, ld_qt;
    uint8_t *scale, *scale_t;  // [ceil(cols/128), rows or ceil(rows/128)], [ceil(rows/128), cols or ceil(cols/128)]
    int rows, cols;
    int vec_in, vec_q, vec_qt;  // 8 elements can be loaded, 8 codes stored, in whole vectors
};

// Scale byte from the bit pattern of max |x| (infinities and NaN order above every number).
__device__ __forceinline__ uint32_t scale_byte(uint32_t b) {
    if (b >= 0x7f800000u) return 255u;
    if (b == 0u) return 127u;
    // 448 = 1.75 * 2^8: one more when the mantissa is above 1.75
    return static_cast<uint32_t>(max(0, static_cast<int>((b + 0x1fffffu) >> 23) - 8));
}
// 2^-E, or NaN for byte 255. E <= 120 for a block of finite floats, so the result is a normal number.
__device__ __forceinline__ float inverse_scale(uint32_t byte) {
    return byte == 255u ? __uint_as_float(0x7fffffffu) : __uint_as_float((254u - byte) << 23);
}

// Four codes from four scaled values (cvt: two values an instruction, nearest even; NaN gives 0x7f).
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

// Eight consecutive elements of a row. `maxima` folds their absolute values' bit patterns into m[] (kWords words, as
// they lie in the source's type), `widen` gives the eight floats, `as_float_bits` the float pattern of one maximum.
template <typename T>
struct Eight;

template <>
struct Eight<float> {
    uint32_t w[8];
    static constexpr int kWords = 8;  // one column a word
    __device__ __forceinline__ void load(const float* p) {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(p)), b = __ldg(reinterpret_cast<const uint4*>(p) + 1);
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
    }
    __device__ __forceinline__ void set(int j, const float* p) { w[j] = __ldg(reinterpret_cast<const uint32_t*>(p)); }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = 0u;
    }
    __device__ __forceinline__ uint32_t mag(int i) const { return w[i] & 0x7fffffffu; }
    static __device__ __forceinline__ uint32_t fold(uint32_t a, uint32_t b) { return max(a, b); }
    static __device__ __forceinline__ uint32_t float_bits(uint32_t word, int) { return word; }
    static __device__ __forceinline__ uint32_t both_halves(uint32_t word) { return word; }
    __device__ __forceinline__ float value(int j) const { return __uint_as_float(w[j]); }
};

template <bool BF>
struct Eight16 {
    uint32_t w[4];
    static constexpr int kWords = 4;  // two columns a word
    __device__ __forceinline__ void load(const uint16_t* p) {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    }
    __device__ __forceinline__ void set(int j, const uint16_t* p) {
        const uint32_t v = __ldg(p);
        w[j >> 1] |= v << (16 * (j & 1));
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = 0u;
    }
    __device__ __forceinline__ uint32_t mag(int i) const { return w[i] & 0x7fff7fffu; }
    static __device__ __forceinline__ uint32_t fold(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }
    // the float pattern of one half of a word of maxima
    static __device__ __forceinline__ uint32_t float_bits(uint32_t word, int half) {
        const uint32_t h = half ? word >> 16 : word & 0xffffu;
        if constexpr (BF) return h << 16;
        else return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(h))));
    }
    static __device__ __forceinline__ uint32_t both_halves(uint32_t word) {
        const uint32_t h = max(word >> 16, word & 0xffffu);
        return float_bits(h, 0);
    }
    __device__ __forceinline__ float value(int j) const {
        const uint32_t word = w[j >> 1];
        if constexpr (BF) return __uint_as_float((j & 1) ? (word & 0xffff0000u) : (word << 16));
        else {
            const __half2 h = *reinterpret_cast<const __half2*>(&word);
            return (j & 1) ? __high2float(h) : __low2float(h);
        }
    }
};
struct Bf16Tag {};
struct Fp16Tag {};
template <>
struct Eight<Bf16Tag> : Eight16<true> {};
template <>
struct Eight<Fp16Tag> : Eight16<false> {};
template <typename T>
struct Elem {
    using type = uint16_t;
};
template <>
struct Elem<float> {
    using type = float;
};

// Where the eight-byte piece `piece` (rows 8 * piece ..) of column `c` lies in the shared tile of the column form.
__device__ __forceinline__ uint32_t turned_offset(int c, int piece) {
    return static_cast<uint32_t>(c * kQb + ((piece ^ (c >> 3)) & 15) * 8);
}

// The finished column form of a tile, 128 columns x 128 bytes in shared memory, to qt. A half-warp takes one column.
__device__ __forceinline__ void store_turned(const uint8_t* turned, const QuantBlockParams& p, int row0, int col0) {
    const int piece = static_cast<int>(threadIdx.x) & 15;
    const int r = row0 + piece * 8;
    const int n = min(8, p.rows - r);
    if (n <= 0) return;
#pragma unroll
    for (int i = 0; i < kQb / (kQbThreads / 16); ++i) {
        const int c = i * (kQbThreads / 16) + (static_cast<int>(threadIdx.x) >> 4);
        if (col0 + c >= p.cols) break;
        const uint2 v = *reinterpret_cast<const uint2*>(turned + turned_offset(c, piece));
        uint8_t* dst = p.qt + static_cast<long long>(col0 + c) * p.ld_qt + r;
        if (n == 8 && p.vec_qt) {
            *reinterpret_cast<uint2*>(dst) = v;
        } else {
            for (int j = 0; j < n; ++j) dst[j] = static_cast<uint8_t>((j < 4 ? v.x >> (8 * j) : v.y >> (8 * (j - 4))) & 0xffu);
        }
    }
}

// One thread's 8 x 8 codes of the column form into the shared tile: code[i] holds the codes of columns 0..3 (lo) and 4..7
// (hi) of row i; eight rows of one column make the eight bytes that are stored together.
__device__ __forceinline__ void put_turned(uint8_t* turned, int cgroup, int piece, const uint32_t (&lo)[8], const uint32_t (&hi)[8]) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const uint32_t(&w)[8] = half ? hi : lo;
        uint32_t t[4][2];  // a 4 x 4 byte transposition, twice
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const uint32_t a = __byte_perm(w[4 * g], w[4 * g + 1], 0x5140), b = __byte_perm(w[4 * g + 2], w[4 * g + 3], 0x5140);
            const uint32_t c = __byte_perm(w[4 * g], w[4 * g + 1], 0x7362), d = __byte_perm(w[4 * g + 2], w[4 * g + 3], 0x7362);
            t[0][g] = __byte_perm(a, b, 0x5410);
            t[1][g] = __byte_perm(a, b, 0x7632);
            t[2][g] = __byte_perm(c, d, 0x5410);
            t[3][g] = __byte_perm(c, d, 0x7632);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            *reinterpret_cast<uint2*>(turned + turned_offset(cgroup * 8 + half * 4 + j, piece)) = make_uint2(t[j][0], t[j][1]);
    }
}

// A thread's place in the tile: rows 8 * piece .. + 8 with piece = 0..15, columns 8 * cgroup .. + 8 with cgroup = lane & 15;
// a load instruction of a warp covers two rows of 128 elements.
template <typename T, bool ROW, bool COL, bool SQUARE>
__global__ void __launch_bounds__(kQbThreads)
quantize_block_kernel(const QuantBlockParams p) {
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
    using E = typename Elem<T>::type;
    using V = Eight<T>;
    __shared__ __align__(16) uint8_t turned[COL ? kQb * kQb : 16];
    __shared__ uint32_t part[8][COL && !SQUARE ? kQb : 1];  // column (or whole-tile) maxima of each warp's sixteen rows
    __shared__ float col_inv[COL && !SQUARE ? kQb : 1];

    const int lane = static_cast<int>(threadIdx.x) & 31, warp = static_cast<int>(threadIdx.x) >> 5;
    const int cgroup = lane & 15, piece = warp * 2 + (lane >> 4);
    const int row0 = static_cast<int>(blockIdx.y) * kQb, col0 = static_cast<int>(blockIdx.x) * kQb;
    const int r0 = row0 + piece * 8, c0 = col0 + cgroup * 8;
    const E* src = static_cast<const E*>(p.in) + static_cast<long long>(r0) * p.ld_in + c0;
    const int n_cols = min(8, p.cols - c0);

    V v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (r0 + i < p.rows && n_cols == 8 && p.vec_in) {
            v[i].load(src + i * p.ld_in);
        } else {
            v[i].clear();
            if (r0 + i < p.rows) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j < n_cols) v[i].set(j, src + i * p.ld_in + j);
            }
        }
    }

    float row_inv[8];
    float tile_inv = 1.0f;
    if constexpr (SQUARE) {
        uint32_t m = 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int k = 0; k < V::kWords; ++k) m = V::fold(m, v[i].mag(k));
        m = V::both_halves(m);
        m = __reduce_max_sync(0xffffffffu, m);
        if (lane == 0) part[warp][0] = m;
        __syncthreads();
        m = part[lane & 7][0];
        m = __reduce_max_sync(0xffffffffu, m);
        const uint32_t byte = scale_byte(m);
        tile_inv = inverse_scale(byte);
        if (threadIdx.x == 0) {
            const long long nb_r = (p.rows + kQb - 1) / kQb, nb_c = (p.cols + kQb - 1) / kQb;
            if (ROW) p.scale[blockIdx.x * nb_r + blockIdx.y] = static_cast<uint8_t>(byte);
            if (COL) p.scale_t[blockIdx.y * nb_c + blockIdx.x] = static_cast<uint8_t>(byte);
        }
    } else {
        if constexpr (ROW) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint32_t m = v[i].mag(0);
#pragma unroll
                for (int k = 1; k < V::kWords; ++k) m = V::fold(m, v[i].mag(k));
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) m = V::fold(m, __shfl_xor_sync(0xffffffffu, m, o));
                const uint32_t byte = scale_byte(V::both_halves(m));
                row_inv[i] = inverse_scale(byte);
                if (cgroup == i && r0 + i < p.rows)
                    p.scale[static_cast<long long>(blockIdx.x) * p.rows + r0 + i] = static_cast<uint8_t>(byte);
            }
        }
        if constexpr (COL) {
#pragma unroll
            for (int k = 0; k < V::kWords; ++k) {
                uint32_t m = v[0].mag(k);
#pragma unroll
                for (int i = 1; i < 8; ++i) m = V::fold(m, v[i].mag(k));
                m = V::fold(m, __shfl_xor_sync(0xffffffffu, m, 16));
                if (lane < 16) {
                    if constexpr (V::kWords == 8) {
                        part[warp][cgroup * 8 + k] = m;
                    } else {
                        part[warp][cgroup * 8 + 2 * k] = V::float_bits(m, 0);
                        part[warp][cgroup * 8 + 2 * k + 1] = V::float_bits(m, 1);
                    }
                }
            }
            __syncthreads();
            if (threadIdx.x < kQb) {
                const int c = static_cast<int>(threadIdx.x);
                uint32_t m = part[0][c];
#pragma unroll
                for (int w = 1; w < 8; ++w) m = max(m, part[w][c]);
                const uint32_t byte = scale_byte(m);
                col_inv[c] = inverse_scale(byte);
                if (col0 + c < p.cols)
                    p.scale_t[static_cast<long long>(blockIdx.y) * p.cols + col0 + c] = static_cast<uint8_t>(byte);
            }
            __syncthreads();
        }
    }

    if constexpr (ROW) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (r0 + i < p.rows && n_cols > 0) {
                const float s = SQUARE ? tile_inv : row_inv[i];
                const uint2 codes = make_uint2(
                    pack4(v[i].value(0) * s, v[i].value(1) * s, v[i].value(2) * s, v[i].value(3) * s),
                    pack4(v[i].value(4) * s, v[i].value(5) * s, v[i].value(6) * s, v[i].value(7) * s));
                uint8_t* dst = p.q + static_cast<long long>(r0 + i) * p.ld_q + c0;
                if (n_cols == 8 && p.vec_q) {
                    *reinterpret_cast<uint2*>(dst) = codes;
                } else {
                    for (int j = 0; j < n_cols; ++j)
                        dst[j] = static_cast<uint8_t>((j < 4 ? codes.x >> (8 * j) : codes.y >> (8 * (j - 4))) & 0xffu);
                }
            }
        }
    }
    if constexpr (COL) {
        float s[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] = SQUARE ? tile_inv : col_inv[cgroup * 8 + j];
        uint32_t lo[8], hi[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            lo[i] = pack4(v[i].value(0) * s[0], v[i].value(1) * s[1], v[i].value(2) * s[2], v[i].value(3) * s[3]);
            hi[i] = pack4(v[i].value(4) * s[4], v[i].value(5) * s[5], v[i].value(6) * s[6], v[i].value(7) * s[7]);
        }
        put_turned(turned, cgroup, piece, lo, hi);
        __syncthreads();
        store_turned(turned, p, row0, col0);
    }
}

// ------------------------------------------------------------------------------------------------ from 8 bits
__device__ __forceinline__ void decode4(uint32_t codes, float (&x)[4]) {
    const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes & 0xffffu), __NV_E4M3);
    const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes >> 16), __NV_E4M3);
    const float2 fa = __half22float2(__half2(a)), fb = __half22float2(__half2(b));
    x[0] = fa.x; x[1] = fa.y; x[2] = fb.x; x[3] = fb.y;
}

// Values are carried as code * 2^(E - 8): the largest, 448 * 2^(127 - 8), and the smallest step, 2^(-9 - 127 - 8), are both
// exact in fp32 (the latter as a subnormal), so no value a scale byte can express overflows or loses a bit on the way.
__device__ __forceinline__ float shifted_scale(uint32_t byte) {
    if (byte == 255u) return __uint_as_float(0x7fffffffu);
    return byte > 8u ? __uint_as_float((byte - 8u) << 23) : __uint_as_float(1u << (14u + byte));
}
__device__ __forceinline__ uint32_t scale_byte_shifted(uint32_t b) {  // from the pattern of max |x| * 2^-8
    if (b >= 0x7f800000u) return 255u;
    if (b == 0u) return 127u;
    if (b < 0x800000u) return b > 0x700000u ? 1u : 0u;
    return (b + 0x1fffffu) >> 23;
}

// Row form -> column form: the 128 x 1 blocks of the values quantised anew. One byte read and one written an element.
__global__ void __launch_bounds__(kQbThreads)
requantize_block_kernel(const QuantBlockParams p) {
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
    __shared__ __align__(16) uint8_t turned[kQb * kQb];
    __shared__ uint32_t part[8][kQb];
    __shared__ float col_inv[kQb];

    const int lane = static_cast<int>(threadIdx.x) & 31, warp = static_cast<int>(threadIdx.x) >> 5;
    const int cgroup = lane & 15, piece = warp * 2 + (lane >> 4);
    const int row0 = static_cast<int>(blockIdx.y) * kQb, col0 = static_cast<int>(blockIdx.x) * kQb;
    const int r0 = row0 + piece * 8, c0 = col0 + cgroup * 8;
    const uint8_t* src = static_cast<const uint8_t*>(p.in) + static_cast<long long>(r0) * p.ld_in + c0;
    const int n_cols = min(8, p.cols - c0);

    uint2 v[8];
    uint32_t byte[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] = make_uint2(0u, 0u);
        byte[i] = 127u;
        if (r0 + i < p.rows && n_cols > 0) {
            byte[i] = __ldg(p.in_scale + static_cast<long long>(blockIdx.x) * p.rows + r0 + i);
            if (n_cols == 8 && p.vec_in) {
                v[i] = __ldg(reinterpret_cast<const uint2*>(src + i * p.ld_in));
            } else {
                for (int j = 0; j < n_cols; ++j) {
                    const uint32_t c = __ldg(src + i * p.ld_in + j);
                    if (j < 4) v[i].x |= c << (8 * j);
                    else v[i].y |= c << (8 * (j - 4));
                }
            }
        }
    }
    float s[8];
    uint32_t m[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        s[i] = shifted_scale(byte[i]);
        float x[4];
        decode4(v[i].x, x);
#pragma unroll
        for (int j = 0; j < 4; ++j) m[j] = max(m[j], __float_as_uint(x[j] * s[i]) & 0x7fffffffu);
        decode4(v[i].y, x);
#pragma unroll
        for (int j = 0; j < 4; ++j) m[4 + j] = max(m[4 + j], __float_as_uint(x[j] * s[i]) & 0x7fffffffu);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        m[j] = max(m[j], __shfl_xor_sync(0xffffffffu, m[j], 16));
        if (lane < 16) part[warp][cgroup * 8 + j] = m[j];
    }
    __syncthreads();
    if (threadIdx.x < kQb) {
        const int c = static_cast<int>(threadIdx.x);
        uint32_t b = part[0][c];
#pragma unroll
        for (int w = 1; w < 8; ++w) b = max(b, part[w][c]);
        const uint32_t e = scale_byte_shifted(b);
        // 2^(8 - E) as a float; below E = -119 it does not exist: those columns carry 2^127 and the missing factor is
        // applied to the values first, marked by the sign
        col_inv[c] = e == 255u ? __uint_as_float(0x7fffffffu)
                               : (e >= 8u ? __uint_as_float((262u - e) << 23) : -__uint_as_float((254u - e) << 23));
        if (col0 + c < p.cols) p.scale_t[static_cast<long long>(blockIdx.y) * p.cols + col0 + c] = static_cast<uint8_t>(e);
    }
    __syncthreads();
    float t[8];
    bool small = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        t[j] = col_inv[cgroup * 8 + j];
        small = small || t[j] < 0.0f;
    }
    uint32_t lo[8], hi[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float x[4], y[4];
        decode4(v[i].x, x);
        decode4(v[i].y, y);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[j] *= s[i];
            y[j] *= s[i];
        }
        if (small) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[j] = t[j] < 0.0f ? x[j] * 256.0f * -t[j] : x[j] * t[j];
                y[j] = t[4 + j] < 0.0f ? y[j] * 256.0f * -t[4 + j] : y[j] * t[4 + j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[j] *= t[j];
                y[j] *= t[4 + j];
            }
        }
        lo[i] = pack4(x[0], x[1], x[2], x[3]);
        hi[i] = pack4(y[0], y[1], y[2], y[3]);
    }
    put_turned(turned, cgroup, piece, lo, hi);
    __syncthreads();
    store_turned(turned, p, row0, col0);
}

// out = round(code * 2^E). The product is exact in fp32 (or overflows to an infinity, as the rounded value does), so the
// conversion to the output type is the one rounding. Eight elements a thread and step.
template <int OUT>
__global__ void __launch_bounds__(kQbThreads)
dequantize_block_kernel(const uint8_t* __restrict__ q, long long ld_q, const uint8_t* __restrict__ scale, int block_shift,
                        long long scale_rows, int rows, int cols, uint8_t* __restrict__ out, long long ld_out, int vec_in,
                        int vec_out) {
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
    constexpr int OB = OUT == OUT_F32 ? 4 : 2;
    const int groups = (cols + 7) / 8;
    const long long total = static_cast<long long>(groups) * rows;
    const long long step = static_cast<long long>(gridDim.x) * kQbThreads;
    for (long long g = static_cast<long long>(blockIdx.x) * kQbThreads + threadIdx.x; g < total; g += step) {
        const long long r = g / groups;
        const int c = static_cast<int>(g - r * groups) * 8;
        const int n = min(8, cols - c);
        const uint8_t* src = q + r * ld_q + c;
        uint2 v = make_uint2(0u, 0u);
        if (n == 8 && vec_in) {
            v = __ldg(reinterpret_cast<const uint2*>(src));
        } else {
            for (int j = 0; j < n; ++j) {
                const uint32_t b = __ldg(src + j);
                if (j < 4) v.x |= b << (8 * j);
                else v.y |= b << (8 * (j - 4));
            }
        }
        const uint32_t byte = __ldg(scale + static_cast<long long>(c >> 7) * scale_rows + (r >> block_shift));
        const float s = byte == 255u ? __uint_as_float(0x7fffffffu)
                                     : (byte == 0u ? __uint_as_float(0x400000u) : __uint_as_float(byte << 23));
        float x[8];
        decode4(v.x, *reinterpret_cast<float(*)[4]>(&x[0]));
        decode4(v.y, *reinterpret_cast<float(*)[4]>(&x[4]));
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= s;
        uint8_t* dst = out + (r * ld_out + c) * OB;
        if constexpr (OUT == OUT_F32) {
            if (n == 8 && vec_out) {
                reinterpret_cast<float4*>(dst)[0] = make_float4(x[0], x[1], x[2], x[3]);
                reinterpret_cast<float4*>(dst)[1] = make_float4(x[4], x[5], x[6], x[7]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j < n) reinterpret_cast<float*>(dst)[j] = x[j];
            }
        } else {
            uint32_t u[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (OUT == OUT_BF16) {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
                    u[j] = *reinterpret_cast<const uint32_t*>(&h);
                } else {
                    const __half2 h = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
                    u[j] = *reinterpret_cast<const uint32_t*>(&h);
                }
            }
            if (n == 8 && vec_out) {
                *reinterpret_cast<uint4*>(dst) = make_uint4(u[0], u[1], u[2], u[3]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j < n)
                        reinterpret_cast<uint16_t*>(dst)[j] =
                            static_cast<uint16_t>((j & 1) ? (u[j >> 1] >> 16) : (u[j >> 1] & 0xffffu));
            }
        }
    }
}

template <typename T>
cudaError_t launch_quantize(const QuantBlockParams& p, bool square, dim3 grid, cudaStream_t stream) {
    const bool row = p.q != nullptr, col = p.qt != nullptr;
    if (square) {
        if (row && col) return launch_pdl(quantize_block_kernel<T, true, true, true>, grid, dim3(kQbThreads), 0, stream, p);
        if (row) return launch_pdl(quantize_block_kernel<T, true, false, true>, grid, dim3(kQbThreads), 0, stream, p);
        return launch_pdl(quantize_block_kernel<T, false, true, true>, grid, dim3(kQbThreads), 0, stream, p);
    }
    if (row && col) return launch_pdl(quantize_block_kernel<T, true, true, false>, grid, dim3(kQbThreads), 0, stream, p);
    if (row) return launch_pdl(quantize_block_kernel<T, true, false, false>, grid, dim3(kQbThreads), 0, stream, p);
    return launch_pdl(quantize_block_kernel<T, false, true, false>, grid, dim3(kQbThreads), 0, stream, p);
}

bool aligned(const void* ptr, size_t ld_bytes, size_t to) {
    return reinterpret_cast<uintptr_t>(ptr) % to == 0 && ld_bytes % to == 0;
}

constexpr size_t kMaxSide = 65535ull * kQb;  // a grid's second dimension counts blocks of 128 rows

}  // namespace

int quantize_block_launch(int in_dtype, const void* in, size_t ld_in, size_t rows, size_t cols, int block_rows, void* q,
                          size_t ld_q, uint8_t* scale, void* qt, size_t ld_qt, uint8_t* scale_t, cudaStream_t stream) {
    if (in_dtype != QGEMM_DTYPE_FP32 && in_dtype != QGEMM_DTYPE_BF16 && in_dtype != QGEMM_DTYPE_FP16)
        return QGEMM_ERR_UNSUPPORTED;
    if (block_rows != 1 && block_rows != kQb) return QGEMM_ERR_INVALID_ARG;
    if ((q == nullptr) != (scale == nullptr) || (qt == nullptr) != (scale_t == nullptr)) return QGEMM_ERR_INVALID_ARG;
    if (rows == 0 || cols == 0) return QGEMM_OK;
    if (in == nullptr || (q == nullptr && qt == nullptr)) return QGEMM_ERR_INVALID_ARG;
    if (ld_in < cols || (q != nullptr && ld_q < cols) || (qt != nullptr && ld_qt < rows)) return QGEMM_ERR_INVALID_ARG;
    if (rows > kMaxSide || cols > kMaxSide) return QGEMM_ERR_INVALID_ARG;
    const size_t es = in_dtype == QGEMM_DTYPE_FP32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(in) % es != 0) return QGEMM_ERR_ALIGNMENT;
    QuantBlockParams p = {};
    p.in = in;
    p.ld_in = static_cast<long long>(ld_in);
    p.q = static_cast<uint8_t*>(q);
    p.qt = static_cast<uint8_t*>(qt);
    p.ld_q = static_cast<long long>(ld_q);
    p.ld_qt = static_cast<long long>(ld_qt);
    p.scale = scale;
    p.scale_t = scale_t;
    p.rows = static_cast<int>(rows);
    p.cols = static_cast<int>(cols);
    p.vec_in = aligned(in, ld_in * es, 16);
    p.vec_q = aligned(q, ld_q, 8);
    p.vec_qt = aligned(qt, ld_qt, 8);
    const dim3 grid(static_cast<unsigned>((cols + kQb - 1) / kQb), static_cast<unsigned>((rows + kQb - 1) / kQb));
    cudaError_t e;
    switch (in_dtype) {
        case QGEMM_DTYPE_FP32: e = launch_quantize<float>(p, block_rows == kQb, grid, stream); break;
        case QGEMM_DTYPE_BF16: e = launch_quantize<Bf16Tag>(p, block_rows == kQb, grid, stream); break;
        default: e = launch_quantize<Fp16Tag>(p, block_rows == kQb, grid, stream); break;
    }
    return e == cudaSuccess ? QGEMM_OK : QGEMM_ERR_CUDA;
}

int requantize_block_launch(const void* q, size_t ld_q, const uint8_t* scale, size_t rows, size_t cols, void* qt,
                            size_t ld_qt, uint8_t* scale_t, cudaStream_t stream) {
    if (rows == 0 || cols == 0) return QGEMM_OK;
    if (q == nullptr || scale == nullptr || qt == nullptr || scale_t == nullptr || ld_q < cols || ld_qt < rows)
        return QGEMM_ERR_INVALID_ARG;
    if (rows > kMaxSide || cols > kMaxSide) return QGEMM_ERR_INVALID_ARG;
    QuantBlockParams p = {};
    p.in = q;
    p.ld_in = static_cast<long long>(ld_q);
    p.in_scale = scale;
    p.qt = static_cast<uint8_t*>(qt);
    p.ld_qt = static_cast<long long>(ld_qt);
    p.scale_t = scale_t;
    p.rows = static_cast<int>(rows);
    p.cols = static_cast<int>(cols);
    p.vec_in = aligned(q, ld_q, 8);
    p.vec_qt = aligned(qt, ld_qt, 8);
    const dim3 grid(static_cast<unsigned>((cols + kQb - 1) / kQb), static_cast<unsigned>((rows + kQb - 1) / kQb));
    return launch_pdl(requantize_block_kernel, grid, dim3(kQbThreads), 0, stream, p) == cudaSuccess ? QGEMM_OK : QGEMM_ERR_CUDA;
}

int dequantize_block_launch(int out_dtype, const void* q, size_t ld_q, const uint8_t* scale, int block_rows, size_t rows,
                            size_t cols, void* out, size_t ld_out, cudaStream_t stream) {
    if (out_dtype != QGEMM_DTYPE_FP32 && out_dtype != QGEMM_DTYPE_BF16 && out_dtype != QGEMM_DTYPE_FP16)
        return QGEMM_ERR_UNSUPPORTED;
    if (block_rows != 1 && block_rows != kQb) return QGEMM_ERR_INVALID_ARG;
    if (rows == 0 || cols == 0) return QGEMM_OK;
    if (q == nullptr || scale == nullptr || out == nullptr || ld_q < cols || ld_out < cols) return QGEMM_ERR_INVALID_ARG;
    if (rows > kMaxSide || cols > kMaxSide) return QGEMM_ERR_INVALID_ARG;
    const size_t es = out_dtype == QGEMM_DTYPE_FP32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(out) % es != 0) return QGEMM_ERR_ALIGNMENT;
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) != cudaSuccess) return QGEMM_ERR_CUDA;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return QGEMM_ERR_CUDA;
    const size_t groups = ((cols + 7) / 8) * rows;
    const size_t want = (groups + kQbThreads - 1) / kQbThreads;
    const unsigned blocks = static_cast<unsigned>(want < static_cast<size_t>(sms) * 8 ? want : static_cast<size_t>(sms) * 8);
    const long long scale_rows = static_cast<long long>(block_rows == kQb ? (rows + kQb - 1) / kQb : rows);
    const int shift = block_rows == kQb ? 7 : 0;
    const int vec_in = aligned(q, ld_q, 8), vec_out = aligned(out, ld_out * es, 16);
    auto go = [&](auto kernel) {
        return launch_pdl(kernel, dim3(blocks), dim3(kQbThreads), 0, stream, static_cast<const uint8_t*>(q),
                          static_cast<long long>(ld_q), scale, shift, scale_rows, static_cast<int>(rows),
                          static_cast<int>(cols), static_cast<uint8_t*>(out), static_cast<long long>(ld_out), vec_in, vec_out);
    };
    const cudaError_t e = out_dtype == QGEMM_DTYPE_FP32   ? go(dequantize_block_kernel<OUT_F32>)
                          : out_dtype == QGEMM_DTYPE_BF16 ? go(dequantize_block_kernel<OUT_BF16>)
                                                          : go(dequantize_block_kernel<OUT_F16>);
    return e == cudaSuccess ? QGEMM_OK : QGEMM_ERR_CUDA;
}

}  // namespace qgemm
