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

enum : int { kAnywhere = 0, kEights = 1, kVectors = 2 };

struct QuantBlockParams {
    const void* in;
    long long ld_in;
    const uint8_t* in_scale;  // source held in 8 bits: its scales [ceil(cols / 128), rows]
    uint8_t *q, *qt;          // row form [rows, cols], column form [cols, rows]
    long long ld_q, ld_qt;
    uint8_t *scale, *scale_t;  // [ceil(cols/128), rows or ceil(rows/128)], [ceil(rows/128), cols or ceil(cols/128)]
    int rows, cols;
    int source;         // what the source's rows are aligned to
    int vec_q, vec_qt;  // 8 codes can be stored in whole vectors
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

// Two and four codes from scaled values (cvt: two values an instruction, nearest even; NaN gives 0x7f).
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) { return __byte_perm(pack2(a, b), pack2(c, d), 0x5410); }

// Eight consecutive elements of a row. `maxima` folds their absolute values' bit patterns into m[] (kWords words, as
// they lie in the source's type), `widen` gives the eight floats, `as_float_bits` the float pattern of one maximum.
template <typename T>
struct Eight;

template <>
struct Eight<float> {
    uint32_t w[8];
    static constexpr int kWords = 8;  // one column a word
    __device__ __forceinline__ void load(const float* p) {
        const uint4* at = reinterpret_cast<const uint4*>(p);
        const uint4 a = ptx::ld_global(at), b = ptx::ld_global(at + 1);
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
    }
    __device__ __forceinline__ void load_by_eights(const float* p) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint2 a = ptx::ld_global(reinterpret_cast<const uint2*>(p) + k);
            w[2 * k] = a.x;
            w[2 * k + 1] = a.y;
        }
    }
    __device__ __forceinline__ void load_any(const float* p) {
        if ((reinterpret_cast<uintptr_t>(p) & 7u) == 0) {
            load_by_eights(p);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) w[k] = ptx::ld_global(reinterpret_cast<const uint32_t*>(p) + k);
        }
    }
    __device__ __forceinline__ void set(int j, const float* p) { w[j] = ptx::ld_global(reinterpret_cast<const uint32_t*>(p)); }
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
        const uint4 a = ptx::ld_global(reinterpret_cast<const uint4*>(p));
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    }
    __device__ __forceinline__ void load_by_eights(const uint16_t* p) {
        const uint2* at = reinterpret_cast<const uint2*>(p);
        const uint2 a = ptx::ld_global(at), b = ptx::ld_global(at + 1);
        w[0] = a.x; w[1] = a.y; w[2] = b.x; w[3] = b.y;
    }
    // from any address: the words that hold the elements, shifted by half a word where they start inside one
    __device__ __forceinline__ void load_any(const uint16_t* p) {
        const uint32_t half = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) >> 1) & 1u;
        const uint32_t* words = reinterpret_cast<const uint32_t*>(p - half);
        uint32_t v[5];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = ptx::ld_global(words + k);
        v[4] = ptx::ld_global(words + 3 + half);
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(v[k], v[k + 1], 16u * half);
    }
    __device__ __forceinline__ void set(int j, const uint16_t* p) {
        const uint32_t v = ptx::ld_global(p);
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
template <bool WHOLE>
__device__ __forceinline__ void store_turned(const uint8_t* turned, const QuantBlockParams& p, int row0, int col0) {
    const int piece = static_cast<int>(threadIdx.x) & 15, first = static_cast<int>(threadIdx.x) >> 4;
    const int r = row0 + piece * 8;
    const int n = min(8, p.rows - r);
    if (!WHOLE && n <= 0) return;
    uint8_t* dst = p.qt + static_cast<long long>(col0 + first) * p.ld_qt + r;
    const long long step = (kQbThreads / 16) * p.ld_qt;
#pragma unroll
    for (int i = 0; i < kQb / (kQbThreads / 16); ++i, dst += step) {
        const int c = i * (kQbThreads / 16) + first;
        if (!WHOLE && col0 + c >= p.cols) break;
        const uint2 v = *reinterpret_cast<const uint2*>(turned + turned_offset(c, piece));
        if (WHOLE || (n == 8 && p.vec_qt)) {
            *reinterpret_cast<uint2*>(dst) = v;
        } else {
            for (int j = 0; j < n; ++j) dst[j] = static_cast<uint8_t>((j < 4 ? v.x >> (8 * j) : v.y >> (8 * (j - 4))) & 0xffu);
        }
    }
}

// One thread's 8 x 8 codes of the column form into the shared tile: pair[i][k] holds row i's codes of columns 2 k and 2 k + 1
// in its low half; eight rows of one column make the eight bytes that are stored together.
__device__ __forceinline__ void put_turned(uint8_t* turned, int cgroup, int piece, const uint32_t (&pair)[8][4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        uint32_t even[2], odd[2];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const uint32_t a = __byte_perm(pair[4 * g][k], pair[4 * g + 1][k], 0x5140);
            const uint32_t b = __byte_perm(pair[4 * g + 2][k], pair[4 * g + 3][k], 0x5140);
            even[g] = __byte_perm(a, b, 0x5410);
            odd[g] = __byte_perm(a, b, 0x7632);
        }
        *reinterpret_cast<uint2*>(turned + turned_offset(cgroup * 8 + 2 * k, piece)) = make_uint2(even[0], even[1]);
        *reinterpret_cast<uint2*>(turned + turned_offset(cgroup * 8 + 2 * k + 1, piece)) = make_uint2(odd[0], odd[1]);
    }
}

// The maxima of a warp's sixteen rows from each lane's of its eight (rows of its half-warp): a butterfly that halves the
// rows a lane is responsible for at every step, 8 exchanges instead of 32; lanes 2 j and 2 j + 1 of a half-warp end up with
// row j.
template <typename V>
__device__ __forceinline__ uint32_t row_maximum(const uint32_t (&m)[8], int lane) {
    uint32_t a[4], b[2];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const bool up = lane & 8;
        const uint32_t give = up ? m[k] : m[4 + k], keep = up ? m[4 + k] : m[k];
        a[k] = V::fold(keep, __shfl_xor_sync(0xffffffffu, give, 8));
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const bool up = lane & 4;
        const uint32_t give = up ? a[k] : a[2 + k], keep = up ? a[2 + k] : a[k];
        b[k] = V::fold(keep, __shfl_xor_sync(0xffffffffu, give, 4));
    }
    const bool up = lane & 2;
    uint32_t c = V::fold(up ? b[1] : b[0], __shfl_xor_sync(0xffffffffu, up ? b[0] : b[1], 2));
    return V::fold(c, __shfl_xor_sync(0xffffffffu, c, 1));
}

template <bool COL, bool SQUARE>
struct QuantShared {
    uint8_t turned[COL ? kQb * kQb : 16];
    uint32_t part[8][COL && !SQUARE ? kQb : 1];  // column (or whole-tile) maxima of each warp's sixteen rows
    float col_inv[COL && !SQUARE ? kQb : 1];
};

// A thread's place in the tile: rows 8 * piece .. + 8 with piece = 0..15, columns 8 * cgroup .. + 8 with cgroup = lane & 15;
// a load instruction of a warp covers two rows of 128 elements. WHOLE: the tile lies inside the matrix and the codes are
// aligned to whole vectors. SOURCE: what the source's rows are aligned to, vectors of 16 bytes, eight bytes or nothing.
template <typename T, bool ROW, bool COL, bool SQUARE, bool WHOLE, int SOURCE>
__device__ __forceinline__ void quantize_tile(const QuantBlockParams& p, QuantShared<COL, SQUARE>& sh) {
    using E = typename Elem<T>::type;
    using V = Eight<T>;
    const int lane = static_cast<int>(threadIdx.x) & 31, warp = static_cast<int>(threadIdx.x) >> 5;
    const int cgroup = lane & 15, piece = warp * 2 + (lane >> 4);
    const int row0 = static_cast<int>(blockIdx.y) * kQb, col0 = static_cast<int>(blockIdx.x) * kQb;
    const int r0 = row0 + piece * 8, c0 = col0 + cgroup * 8;
    const E* src = static_cast<const E*>(p.in) + static_cast<long long>(r0) * p.ld_in + c0;
    const int n_cols = WHOLE ? 8 : min(8, p.cols - c0);

    V v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i, src += p.ld_in) {
        if (WHOLE && SOURCE == kVectors) {
            v[i].load(src);
        } else if (WHOLE && SOURCE == kEights) {
            v[i].load_by_eights(src);
        } else if (WHOLE || (r0 + i < p.rows && n_cols == 8)) {
            v[i].load_any(src);
        } else {
            v[i].clear();
            if (r0 + i < p.rows) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j < n_cols) v[i].set(j, src + j);
            }
        }
    }

    float row_inv = 1.0f;  // of row (lane >> 1) & 7 of this half-warp
    float tile_inv = 1.0f;
    if constexpr (SQUARE) {
        uint32_t m = 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int k = 0; k < V::kWords; ++k) m = V::fold(m, v[i].mag(k));
        m = V::both_halves(m);
        m = __reduce_max_sync(0xffffffffu, m);
        if (lane == 0) sh.part[warp][0] = m;
        __syncthreads();
        m = sh.part[lane & 7][0];
        m = __reduce_max_sync(0xffffffffu, m);
        const uint32_t byte = scale_byte(m);
        tile_inv = inverse_scale(byte);
        if (threadIdx.x == 0) {
            const long long nb_r = (p.rows + kQb - 1) / kQb, nb_c = (p.cols + kQb - 1) / kQb;
            if (ROW) p.scale[blockIdx.x * nb_r + blockIdx.y] = static_cast<uint8_t>(byte);
            if (COL) p.scale_t[blockIdx.y * nb_c + blockIdx.x] = static_cast<uint8_t>(byte);
        }
    } else {
        if constexpr (COL) {
#pragma unroll
            for (int k = 0; k < V::kWords; ++k) {
                uint32_t m = v[0].mag(k);
#pragma unroll
                for (int i = 1; i < 8; ++i) m = V::fold(m, v[i].mag(k));
                m = V::fold(m, __shfl_xor_sync(0xffffffffu, m, 16));
                if (lane < 16) {
                    if constexpr (V::kWords == 8) {
                        sh.part[warp][cgroup * 8 + k] = m;
                    } else {
                        sh.part[warp][cgroup * 8 + 2 * k] = V::float_bits(m, 0);
                        sh.part[warp][cgroup * 8 + 2 * k + 1] = V::float_bits(m, 1);
                    }
                }
            }
        }
        if constexpr (ROW) {
            uint32_t m[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                m[i] = v[i].mag(0);
#pragma unroll
                for (int k = 1; k < V::kWords; ++k) m[i] = V::fold(m[i], v[i].mag(k));
            }
            const uint32_t byte = scale_byte(V::both_halves(row_maximum<V>(m, lane)));
            row_inv = inverse_scale(byte);
            const int r = r0 + ((lane >> 1) & 7);
            if ((lane & 1) == 0 && (WHOLE || r < p.rows))
                p.scale[static_cast<long long>(blockIdx.x) * p.rows + r] = static_cast<uint8_t>(byte);
        }
        if constexpr (COL) {
            __syncthreads();
            if (threadIdx.x < kQb) {
                const int c = static_cast<int>(threadIdx.x);
                uint32_t m = sh.part[0][c];
#pragma unroll
                for (int w = 1; w < 8; ++w) m = max(m, sh.part[w][c]);
                const uint32_t byte = scale_byte(m);
                sh.col_inv[c] = inverse_scale(byte);
                if (WHOLE || col0 + c < p.cols)
                    p.scale_t[static_cast<long long>(blockIdx.y) * p.cols + col0 + c] = static_cast<uint8_t>(byte);
            }
        }
    }

    if constexpr (ROW) {
        uint8_t* dst = p.q + static_cast<long long>(r0) * p.ld_q + c0;
#pragma unroll
        for (int i = 0; i < 8; ++i, dst += p.ld_q) {
            const float s = SQUARE ? tile_inv : __shfl_sync(0xffffffffu, row_inv, (lane & 16) + 2 * i);
            const uint2 codes = make_uint2(
                pack4(v[i].value(0) * s, v[i].value(1) * s, v[i].value(2) * s, v[i].value(3) * s),
                pack4(v[i].value(4) * s, v[i].value(5) * s, v[i].value(6) * s, v[i].value(7) * s));
            if (WHOLE || (r0 + i < p.rows && n_cols == 8 && p.vec_q)) {
                *reinterpret_cast<uint2*>(dst) = codes;
            } else if (r0 + i < p.rows) {
                for (int j = 0; j < n_cols; ++j)
                    dst[j] = static_cast<uint8_t>((j < 4 ? codes.x >> (8 * j) : codes.y >> (8 * (j - 4))) & 0xffu);
            }
        }
    }
    if constexpr (COL) {
        if (!SQUARE) __syncthreads();
        float s[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] = SQUARE ? tile_inv : sh.col_inv[cgroup * 8 + j];
        uint32_t pair[8][4];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) pair[i][k] = pack2(v[i].value(2 * k) * s[2 * k], v[i].value(2 * k + 1) * s[2 * k + 1]);
        put_turned(sh.turned, cgroup, piece, pair);
        __syncthreads();
        store_turned<WHOLE>(sh.turned, p, row0, col0);
    }
}

__device__ __forceinline__ bool whole_tile(const QuantBlockParams& p) {
    return p.vec_q && p.vec_qt && static_cast<int>(blockIdx.y + 1) * kQb <= p.rows &&
           static_cast<int>(blockIdx.x + 1) * kQb <= p.cols;
}

// Tiles that share an SM, by the registers a tile can be held in: what a CTA has in flight is its tile, so this sets the
// bandwidth. (16-bit, 4096 x 7168, column form: four 16.4 us, two 21.3, five, with spilled registers, 18.7; both forms:
// three 22.3, two 25.9, four 23.2.)
template <typename T, bool ROW, bool COL, bool SQUARE>
constexpr int tiles_per_sm() {
    if (sizeof(typename Elem<T>::type) == 2) return SQUARE ? (ROW ? 4 : 5) : (ROW && COL ? 3 : 4);
    return ROW ? 2 : 3;
}

template <typename T, bool ROW, bool COL, bool SQUARE>
__global__ void __launch_bounds__(kQbThreads, (tiles_per_sm<T, ROW, COL, SQUARE>()))
quantize_block_kernel(const QuantBlockParams p) {
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
    __shared__ __align__(16) QuantShared<COL, SQUARE> sh;
    if (!whole_tile(p)) quantize_tile<T, ROW, COL, SQUARE, false, kAnywhere>(p, sh);
    else if (p.source == kVectors) quantize_tile<T, ROW, COL, SQUARE, true, kVectors>(p, sh);
    else if (p.source == kEights) quantize_tile<T, ROW, COL, SQUARE, true, kEights>(p, sh);
    else quantize_tile<T, ROW, COL, SQUARE, true, kAnywhere>(p, sh);
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

// Row form -> column form: the 128 x 1 blocks of the values quantised anew. One byte read and one written an element, so
// what bounds it besides HBM is the arithmetic, and that is done two elements at a time in fp16 wherever fp16 is exact:
//   u = code * 2^(E_row - S), S the largest of the tile's 128 row scales, is a whole multiple of 2^-24 with 4 significant
//   bits when all rows are within 2^15 of S, so it is exact (as a subnormal, too), and so are the columns' maxima;
//   y = u * 2^(S - E_col) has a factor that fp16 holds when the column's maximum is at least 2^-6 (or 0); it is exact, or
//   below 2^-14 and a zero among the codes however it is rounded.
// A tile that is not like that (rows far apart, a column of nothing but tiny codes, a NaN) takes the fp32 form below: a
// tile's choice is the same for all its threads. (All in fp32: 77 us at 16384 x 7168, 15 instructions an element.)
struct RequantShared {
    uint8_t turned[kQb * kQb];
    uint32_t part[8][kQb];
    uint32_t factor[kQb];
};

// Maxima of eight warps' parts -> the columns' scale bytes, stored; `factor` keeps what multiplies a column's values.
template <bool WHOLE, typename Byte, typename Factor>
__device__ __forceinline__ void column_scales(RequantShared& sh, const QuantBlockParams& p, int col0, Byte byte_of, Factor factor_of) {
    if (threadIdx.x < kQb) {
        const int c = static_cast<int>(threadIdx.x);
        uint32_t b = sh.part[0][c];
#pragma unroll
        for (int w = 1; w < 8; ++w) b = max(b, sh.part[w][c]);
        const uint32_t e = byte_of(b);
        sh.factor[c] = factor_of(e);
        if (WHOLE || col0 + c < p.cols) p.scale_t[static_cast<long long>(blockIdx.y) * p.cols + col0 + c] = static_cast<uint8_t>(e);
    }
}

// A thread's codes of the tile; zeros where there is no row or column.
template <bool WHOLE>
__device__ __forceinline__ void load_codes(const QuantBlockParams& p, int r0, int c0, uint2 (&v)[8]) {
    const uint8_t* src = static_cast<const uint8_t*>(p.in) + static_cast<long long>(r0) * p.ld_in + c0;
    const int n_cols = WHOLE ? 8 : min(8, p.cols - c0);
#pragma unroll
    for (int i = 0; i < 8; ++i, src += p.ld_in) {
        if (WHOLE || (r0 + i < p.rows && n_cols == 8 && p.source == kEights)) {
            v[i] = ptx::ld_global(reinterpret_cast<const uint2*>(src));
        } else {
            v[i] = make_uint2(0u, 0u);
            if (r0 + i < p.rows) {
                for (int j = 0; j < n_cols; ++j) {
                    const uint32_t c = ptx::ld_global(src + j);
                    if (j < 4) v[i].x |= c << (8 * j);
                    else v[i].y |= c << (8 * (j - 4));
                }
            }
        }
    }
}

// The fp32 form, for any codes and scales.
template <bool WHOLE>
__device__ __noinline__ void requantize_tile_fp32(const QuantBlockParams& p, RequantShared& sh) {
    const int lane = static_cast<int>(threadIdx.x) & 31, warp = static_cast<int>(threadIdx.x) >> 5;
    const int cgroup = lane & 15, piece = warp * 2 + (lane >> 4);
    const int row0 = static_cast<int>(blockIdx.y) * kQb, col0 = static_cast<int>(blockIdx.x) * kQb;
    uint2 v[8];
    load_codes<WHOLE>(p, row0 + piece * 8, col0 + cgroup * 8, v);
    const uint8_t* scales = p.in_scale + static_cast<long long>(blockIdx.x) * p.rows + row0 + piece * 8;
    float s[8];
    uint32_t m[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        s[i] = shifted_scale(WHOLE || row0 + piece * 8 + i < p.rows ? ptx::ld_global(scales + i) : 127u);
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
        if (lane < 16) sh.part[warp][cgroup * 8 + j] = m[j];
    }
    __syncthreads();
    // 2^(8 - E) as a float; below E = -119 it does not exist: those columns carry 2^(-E - 1) with the sign set, and 2^9
    // is applied to the values first
    column_scales<WHOLE>(
        sh, p, col0, [](uint32_t b) { return scale_byte_shifted(b); },
        [](uint32_t e) { return e == 255u ? 0x7fffffffu : (e >= 8u ? (262u - e) << 23 : 0x80000000u | ((253u - e) << 23)); });
    __syncthreads();
    float t[8];
    bool small = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        t[j] = __uint_as_float(sh.factor[cgroup * 8 + j]);
        small = small || t[j] < 0.0f;
    }
    uint32_t pair[8][4];
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
                x[j] = t[j] < 0.0f ? x[j] * 512.0f * -t[j] : x[j] * t[j];
                y[j] = t[4 + j] < 0.0f ? y[j] * 512.0f * -t[4 + j] : y[j] * t[4 + j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[j] *= t[j];
                y[j] *= t[4 + j];
            }
        }
        pair[i][0] = pack2(x[0], x[1]);
        pair[i][1] = pack2(x[2], x[3]);
        pair[i][2] = pack2(y[0], y[1]);
        pair[i][3] = pack2(y[2], y[3]);
    }
    put_turned(sh.turned, cgroup, piece, pair);
    __syncthreads();
    store_turned<WHOLE>(sh.turned, p, row0, col0);
}

__device__ __forceinline__ __half2 half2_of(uint32_t w) { return *reinterpret_cast<const __half2*>(&w); }
__device__ __forceinline__ uint32_t bits_of(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ __half2 decode2(uint32_t codes) {
    return __half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes & 0xffffu), __NV_E4M3));
}
__device__ __forceinline__ uint32_t encode2(__half2 y) { return __nv_cvt_halfraw2_to_fp8x2(static_cast<__half2_raw>(y), __NV_SATFINITE, __NV_E4M3); }

template <bool WHOLE>
__device__ __forceinline__ void requantize_tile(const QuantBlockParams& p, RequantShared& sh) {
    const int lane = static_cast<int>(threadIdx.x) & 31, warp = static_cast<int>(threadIdx.x) >> 5;
    const int cgroup = lane & 15, piece = warp * 2 + (lane >> 4);
    const int row0 = static_cast<int>(blockIdx.y) * kQb, col0 = static_cast<int>(blockIdx.x) * kQb;
    uint2 v[8];
    load_codes<WHOLE>(p, row0 + piece * 8, col0 + cgroup * 8, v);
    // this lane's row's scale, and the largest and smallest of the tile's, in every warp
    const uint8_t* scales = p.in_scale + static_cast<long long>(blockIdx.x) * p.rows + row0;
    const int own = piece * 8 + (cgroup >> 1);
    const bool exists = WHOLE || row0 + own < p.rows;
    const uint32_t byte = exists ? ptx::ld_global(scales + own) : 0u;
    uint32_t top = 0u, low = 255u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int r = 32 * j + lane;
        if (WHOLE || row0 + r < p.rows) {
            const uint32_t b = ptx::ld_global(scales + r);
            top = max(top, b);
            low = min(low, b);
        }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    low = __reduce_min_sync(0xffffffffu, low);
    if (top == 255u || top - low > 15u) {
        requantize_tile_fp32<WHOLE>(p, sh);
        return;
    }
    // 2^(E_row - S) in both halves: normal down to 2^-14, 2^-15 a subnormal; the codes of rows that do not exist are zeros
    const uint32_t below = top - byte;
    const uint32_t factor_bits = (!exists || below == 15u ? 0x200u : (15u - below) << 10) * 0x10001u;
    // The codes stay as they are and are decoded twice: that takes half the registers, so five tiles fit on an SM.
    __half2 f[8], m[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) m[k] = half2_of(0u);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        f[i] = half2_of(__shfl_sync(0xffffffffu, factor_bits, (lane & 16) + 2 * i));
        m[0] = __hmax2_nan(m[0], __habs2(__hmul2(decode2(v[i].x), f[i])));
        m[1] = __hmax2_nan(m[1], __habs2(__hmul2(decode2(v[i].x >> 16), f[i])));
        m[2] = __hmax2_nan(m[2], __habs2(__hmul2(decode2(v[i].y), f[i])));
        m[3] = __hmax2_nan(m[3], __habs2(__hmul2(decode2(v[i].y >> 16), f[i])));
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        m[k] = __hmax2_nan(m[k], half2_of(__shfl_xor_sync(0xffffffffu, bits_of(m[k]), 16)));
        if (lane < 16) {
            sh.part[warp][cgroup * 8 + 2 * k] = bits_of(m[k]) & 0xffffu;
            sh.part[warp][cgroup * 8 + 2 * k + 1] = bits_of(m[k]) >> 16;
        }
    }
    __syncthreads();
    bool other = false;
    if (threadIdx.x < kQb) {
        const int c = static_cast<int>(threadIdx.x);
        uint32_t b = sh.part[0][c];
#pragma unroll
        for (int w = 1; w < 8; ++w) b = max(b, sh.part[w][c]);
        // a column's maximum lies in [2^-6, 448] or is 0, or the tile takes the other form (a NaN's pattern lies above)
        other = b != 0u && (b < 0x2400u || b > 0x5f00u);
        // E_col - S = exponent - 8, one more when the mantissa is above 1.75, -14 .. 0 here; E_col is at least -127
        uint32_t e = 127u, factor = 0u;
        if (b != 0u && !other) {
            const int d = static_cast<int>((b + 0xffu) >> 10) - 15 - 8;
            const int byte_of_column = max(0, static_cast<int>(top) + d);
            e = static_cast<uint32_t>(byte_of_column);
            factor = static_cast<uint32_t>(15 - (byte_of_column - static_cast<int>(top))) << 10;
        }
        sh.factor[c] = factor;
        if (!other && (WHOLE || col0 + c < p.cols))
            p.scale_t[static_cast<long long>(blockIdx.y) * p.cols + col0 + c] = static_cast<uint8_t>(e);
    }
    if (__syncthreads_or(other)) {
        requantize_tile_fp32<WHOLE>(p, sh);
        return;
    }
    __half2 t[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) t[k] = half2_of(sh.factor[cgroup * 8 + 2 * k] | (sh.factor[cgroup * 8 + 2 * k + 1] << 16));
    uint32_t pair[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        pair[i][0] = encode2(__hmul2(__hmul2(decode2(v[i].x), f[i]), t[0]));
        pair[i][1] = encode2(__hmul2(__hmul2(decode2(v[i].x >> 16), f[i]), t[1]));
        pair[i][2] = encode2(__hmul2(__hmul2(decode2(v[i].y), f[i]), t[2]));
        pair[i][3] = encode2(__hmul2(__hmul2(decode2(v[i].y >> 16), f[i]), t[3]));
    }
    put_turned(sh.turned, cgroup, piece, pair);
    __syncthreads();
    store_turned<WHOLE>(sh.turned, p, row0, col0);
}

__global__ void __launch_bounds__(kQbThreads, 5)
requantize_block_kernel(const QuantBlockParams p) {
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
    __shared__ __align__(16) RequantShared sh;
    if (p.source == kEights && whole_tile(p)) requantize_tile<true>(p, sh);
    else requantize_tile<false>(p, sh);
}

// out = round(code * 2^E). The product is exact in fp32 (or overflows to an infinity, as the rounded value does), so the
// conversion to the output type is the one rounding. A thread has W neighbouring columns (16 bytes of output) of four rows
// at a time (eight took more registers: 16384 x 7168 to bf16 75 us instead of 59): their loads are all in flight together, a
// warp's stores cover whole lines, and rows and columns come without a division. Where rows of `out` do not start on 16
// bytes (VEC false) an fp32 thread stores its columns one by one, and a 16-bit thread has two columns of eight rows, a word
// of output where a row starts on one (4001 x 7167 to bf16: by eight single columns 80 us, by one 52).
template <int OUT>
__device__ __forceinline__ void store_value(uint8_t* dst, float x) {
    if constexpr (OUT == OUT_F32) *reinterpret_cast<float*>(dst) = x;
    else if constexpr (OUT == OUT_BF16) *reinterpret_cast<__nv_bfloat16*>(dst) = __float2bfloat16_rn(x);
    else *reinterpret_cast<__half*>(dst) = __float2half_rn(x);
}
__device__ __forceinline__ float scale_value(uint32_t byte) {
    return byte == 255u ? __uint_as_float(0x7fffffffu) : (byte == 0u ? __uint_as_float(0x400000u) : __uint_as_float(byte << 23));
}
template <int OUT, bool VEC>
struct DequantShape {
    static constexpr int kCols = OUT == OUT_F32 ? 4 : (VEC ? 8 : 2);
    static constexpr int kRows = OUT == OUT_F32 || VEC ? 4 : 8;
};
template <int OUT, bool VEC>
__global__ void __launch_bounds__(kQbThreads, 4)
dequantize_block_kernel(const uint8_t* q, long long ld_q, const uint8_t* scale, int block_shift, long long scale_rows, int rows,
                        int cols, uint8_t* out, long long ld_out, int vec_in) {
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();
    constexpr int OB = OUT == OUT_F32 ? 4 : 2;
    constexpr int W = DequantShape<OUT, VEC>::kCols, U = DequantShape<OUT, VEC>::kRows;
    const int c = (static_cast<int>(blockIdx.x) * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)) * W;
    if (c >= cols) return;
    const int n = min(W, cols - c);
    const uint8_t* scales = scale + static_cast<long long>(c >> 7) * scale_rows;
    const long long step = static_cast<long long>(gridDim.y) * blockDim.y * U;
    for (long long r0 = (static_cast<long long>(blockIdx.y) * blockDim.y + threadIdx.y) * U; r0 < rows; r0 += step) {
        const int nr = static_cast<int>(min(static_cast<long long>(U), rows - r0));
        const uint8_t* src = q + r0 * ld_q + c;
        if constexpr (W == 2) {
            uint32_t code[U], byte[U];
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int k = min(i, nr - 1);
                const uint8_t* at = src + k * ld_q;
                if (vec_in && n == 2) code[i] = ptx::ld_global(reinterpret_cast<const uint16_t*>(at));
                else code[i] = ptx::ld_global(at) | (n == 2 ? ptx::ld_global(at + 1) << 8 : 0u);
                byte[i] = ptx::ld_global(scales + ((r0 + k) >> block_shift));
            }
            uint8_t* dst = out + (r0 * ld_out + c) * OB;
#pragma unroll
            for (int i = 0; i < U; ++i, dst += ld_out * OB) {
                if (i >= nr) continue;
                const float2 x = __half22float2(decode2(code[i]));
                const float s = scale_value(byte[i]);
                if (n == 2 && (reinterpret_cast<uintptr_t>(dst) & 3u) == 0) {
                    uint32_t u;
                    if constexpr (OUT == OUT_BF16) {
                        const __nv_bfloat162 h = __floats2bfloat162_rn(x.x * s, x.y * s);
                        u = *reinterpret_cast<const uint32_t*>(&h);
                    } else {
                        u = bits_of(__floats2half2_rn(x.x * s, x.y * s));
                    }
                    *reinterpret_cast<uint32_t*>(dst) = u;
                } else {
                    store_value<OUT>(dst, x.x * s);
                    if (n == 2) store_value<OUT>(dst + OB, x.y * s);
                }
            }
            continue;
        } else {
            uint32_t v[U][W / 4], byte[U];
#pragma unroll
            for (int i = 0; i < U; ++i) {
#pragma unroll
                for (int k = 0; k < W / 4; ++k) v[i][k] = 0u;
                byte[i] = 127u;
                if (i < nr) {
                    byte[i] = ptx::ld_global(scales + ((r0 + i) >> block_shift));
                    if (n == W && vec_in) {
                        if constexpr (W == 8) {
                            const uint2 w = ptx::ld_global(reinterpret_cast<const uint2*>(src + i * ld_q));
                            v[i][0] = w.x;
                            v[i][1] = w.y;
                        } else {
                            v[i][0] = ptx::ld_global(reinterpret_cast<const uint32_t*>(src + i * ld_q));
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < W; ++j)
                            if (j < n) v[i][j >> 2] |= ptx::ld_global(src + i * ld_q + j) << (8 * (j & 3));
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < U; ++i) {
                if (i >= nr) break;
                const float s = scale_value(byte[i]);
                float x[W];
#pragma unroll
                for (int k = 0; k < W / 4; ++k) decode4(v[i][k], *reinterpret_cast<float(*)[4]>(&x[4 * k]));
#pragma unroll
                for (int j = 0; j < W; ++j) x[j] *= s;
                uint8_t* dst = out + ((r0 + i) * ld_out + c) * OB;
                if (n < W || !VEC) {
#pragma unroll
                    for (int j = 0; j < W; ++j)
                        if (j < n) store_value<OUT>(dst + j * OB, x[j]);
                } else if constexpr (OUT == OUT_F32) {
                    *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
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
                    *reinterpret_cast<uint4*>(dst) = make_uint4(u[0], u[1], u[2], u[3]);
                }
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
    p.source = aligned(in, ld_in * es, 16) ? kVectors : (aligned(in, ld_in * es, 8) ? kEights : kAnywhere);
    p.vec_q = q == nullptr || aligned(q, ld_q, 8);
    p.vec_qt = qt == nullptr || aligned(qt, ld_qt, 8);
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
    p.source = aligned(q, ld_q, 8) ? kEights : kAnywhere;
    p.vec_q = 1;
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
    const long long scale_rows = static_cast<long long>(block_rows == kQb ? (rows + kQb - 1) / kQb : rows);
    const int shift = block_rows == kQb ? 7 : 0;
    const bool vec_out = aligned(out, ld_out * es, 16);
    const int vec_in = aligned(q, ld_q, es == 4 ? 4 : (vec_out ? 8 : 2));
    // a block: as many neighbouring pieces of a row as there are, up to 256, and rows for the rest of its threads
    const size_t piece = es == 4 ? 4 : (vec_out ? 8 : 2), rows_at_once = es == 4 || vec_out ? 4 : 8;
    const size_t pieces = (cols + piece - 1) / piece;
    unsigned bx = 1;
    while (bx < static_cast<unsigned>(kQbThreads) && bx < pieces) bx *= 2;
    const unsigned by = kQbThreads / bx;
    const size_t row_steps = (rows + by * rows_at_once - 1) / (by * rows_at_once);
    const dim3 grid(static_cast<unsigned>((pieces + bx - 1) / bx), static_cast<unsigned>(row_steps < 65535 ? row_steps : 65535));
    auto go = [&](auto vec_kernel, auto any_kernel) {
        return launch_pdl(vec_out ? vec_kernel : any_kernel, grid, dim3(bx, by), 0, stream, static_cast<const uint8_t*>(q),
                          static_cast<long long>(ld_q), scale, shift, scale_rows, static_cast<int>(rows),
                          static_cast<int>(cols), static_cast<uint8_t*>(out), static_cast<long long>(ld_out), vec_in);
    };
    cudaError_t e;
    switch (out_dtype) {
        case QGEMM_DTYPE_FP32: e = go(dequantize_block_kernel<OUT_F32, true>, dequantize_block_kernel<OUT_F32, false>); break;
        case QGEMM_DTYPE_BF16: e = go(dequantize_block_kernel<OUT_BF16, true>, dequantize_block_kernel<OUT_BF16, false>); break;
        default: e = go(dequantize_block_kernel<OUT_F16, true>, dequantize_block_kernel<OUT_F16, false>); break;
    }
    return e == cudaSuccess ? QGEMM_OK : QGEMM_ERR_CUDA;
}

}  // namespace qgemm
