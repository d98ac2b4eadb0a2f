// FP8 e4m3 GEMM with power-of-two (ue8m0) scales on blocks of 128 along K, applied by the tensor cores.
//
//   C[m,n] (+)= sum_kb 2^(ea[kb,m] + eb[kb,n]) * sum_{k in block kb} A[m,k] * B[n,k]        fp32 accumulation
//
// gemm_blockscale.cu serves the same product for fp32 scales, which the tensor cores cannot apply: it drains a partial sum
// from tensor memory and rescales it in CUDA cores for every 128 of K, and stops at 1.7 PFLOP/s. A scale that is a power of
// two is the operand form of tcgen05.mma.kind::mxf8f6f4: the scales are multiplied in on the way into the accumulator,
// which stays in tensor memory for the whole of K, and the product runs at the plain FP8 kernels' pace.
//
// The instruction takes one scale per row and 32 elements of K; a 128-wide block is four instructions with the same scale
// id. One tensor-memory word holds a row's scales of four K blocks (a "chunk"); the 128 rows of an operand take four columns
// of 32 lanes, repeated over the four lane quadrants. They come from global memory in the caller's plain layout ([K
// block][row], or [K block][row / 128]) through four warps, one a quadrant: a warp a 128 rows loads words and turns them into
// a row's four K blocks, and after an exchange through shared memory every warp stores all of them to its quadrant.
// (Through tcgen05.cp instead, from shared memory and in the issuing thread's own order, the issuer had two more waits, the
// copies and two more commits for every chunk: 256 x 128 tiles took 21.9 us for 1024 x 2048 x 8192, with stores 19.4.)
//
// Barriers besides the ring's full / empty and the accumulators': sfull[c] (a chunk's scales are in columns c), sdone[c]
// (the chunk's last MMA has completed: columns c are free). All waits are bounded as in gemm_sm100.cuh.
#pragma once
#include "gemm_sm100.cuh"

namespace qgemm {

struct E8m0Params {
    void* C;
    long long ldc;
    int M, N, K;
    int m_tiles, n_tiles;
    int kb_total;
    int group_m;
    uint32_t idesc;
    const uint8_t* a_scale;  // [kb_total][a_rows], entry of row m: m >> a_shift
    const uint8_t* b_scale;
    long long a_rows, b_rows;
    int a_shift, b_shift;  // 0: a scale per row, 7: per 128 rows
    int out;               // OUT_F32 / OUT_BF16 / OUT_F16
    int accumulate;        // fp32 C: add to what it holds
    int c_tma_ok, c_vec_ok;
    int n_tma;         // boxes of C that begin before this column are stored by TMA (tma_store_columns)
    int test_skip_kb;  // failure-detection test hook: the producers leave out this K block (-1 = none)
    int* status;
};

constexpr int kE8Cols = 4;       // chunks of scales in tensor memory
constexpr int kE8Threads = 320;  // producer, MMA issuer, four epilogue warps, four scale warps (6 .. 9)
enum : int { ROLE_SCALES = 4 };

// wait_bounded by a whole warp, with one answer: what follows is executed by all its lanes or by none.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int role,
                                          int where, uint32_t peer_abort = 0) {
    return __all_sync(0xffffffffu, wait_bounded(bar, parity, abort_flag, status, role, where, peer_abort));
}

// One operand's scales on their way from global to shared memory.
struct ScaleSource {
    const uint8_t* scale;
    long long ld;
    int shift, rows;
};

// A lane's part of a chunk (K blocks kb0 .. kb0 + n, n <= 4) of 128 rows from row0: for each K block the word that holds the
// scales of rows 4 lane .. + 4, or the two words they lie across when the block's row of scales does not start on a word
// boundary (any M, any base address). No word is touched that holds none of the operand's scales. A row or K block that
// does not exist gets some other one's scale: its products are zeros in rows of C that are not stored, or are not made.
//
// load_scales uses nothing that it loads, and a scale warp keeps kE8Ahead chunks loading: a chunk must not cost a memory
// latency each, which under the ring's own traffic is more than the tensor cores take for it (measured at 4096 x 7168 x
// 7168, row-scaled B: 404 us with one load waited for at a time, 194 with one chunk at a time, 157 with four in flight).
constexpr int kE8Ahead = 4;
struct ScaleWords {
    uint32_t lo[4], hi[4];
};
__device__ __forceinline__ const uint8_t* scale_row(const ScaleSource& s, int row0, int kb) {
    return s.scale + kb * s.ld + (min(row0, s.rows - 1) >> s.shift);
}
__device__ __forceinline__ void load_scales(ScaleWords& out, const ScaleSource& s, int row0, int kb0, int n, int lane) {
    if (s.shift != 0) {  // one scale for the 128 rows
#pragma unroll
        for (int i = 0; i < 4; ++i) out.lo[i] = ptx::ld_global(scale_row(s, row0, kb0 + min(i, n - 1)));
        return;
    }
    const int bytes = min(128, s.rows - min(row0, s.rows - 1));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint8_t* at = scale_row(s, row0, kb0 + min(i, n - 1));
        const int off = static_cast<int>(reinterpret_cast<uintptr_t>(at) & 3u);
        const int last = (off + bytes - 1) >> 2;
        const uint32_t* words = reinterpret_cast<const uint32_t*>(at - off);
        out.lo[i] = ptx::ld_global(words + min(lane, last));
        if (off != 0) out.hi[i] = ptx::ld_global(words + min(lane + 1, last));
    }
}
// Into 512 bytes of shared memory: row r's four K blocks as a word at (r % 32) * 16 + (r / 32) * 4, so that lane l finds the
// words of its four columns, rows l, 32 + l, 64 + l and 96 + l, side by side.
__device__ __forceinline__ void put_scales(uint32_t dst, const ScaleWords& c, const ScaleSource& s, int row0, int kb0, int n,
                                           int lane) {
    if (s.shift != 0) {
        const uint32_t w = c.lo[0] | (c.lo[1] << 8) | (c.lo[2] << 16) | (c.lo[3] << 24);
        ptx::st_shared_v4(dst + lane * 16, w, w, w, w);
        return;
    }
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(scale_row(s, row0, kb0 + min(i, n - 1))) & 3u);
        v[i] = off != 0 ? __funnelshift_r(c.lo[i], c.hi[i], 8 * off) : c.lo[i];
    }
    const uint32_t x = __byte_perm(v[0], v[1], 0x5140), y = __byte_perm(v[2], v[3], 0x5140);
    const uint32_t z = __byte_perm(v[0], v[1], 0x7362), t = __byte_perm(v[2], v[3], 0x7362);
    const uint32_t w[4] = {__byte_perm(x, y, 0x5410), __byte_perm(x, y, 0x7632), __byte_perm(z, t, 0x5410),
                           __byte_perm(z, t, 0x7632)};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t r = static_cast<uint32_t>(4 * lane + j);
        ptx::st_shared_u32(dst + (r & 31u) * 16u + (r >> 5) * 4u, w[j]);
    }
}

// The four scale warps, over the chunks of K blocks [kb0, kb1) of work items first, first + step, ... < last. Unit u = 0 ..
// UNITS - 1 is 128 rows of an operand, loaded by scale warp u from row rows(work item). `start` sends the first loads on their
// way, before the CTA-wide barrier in a kernel whose producer waits for memory there too. `run` needs tensor memory, and is
// executed by all four warps to the end whatever happens, because they meet at a barrier of their own for every chunk: after
// a wait that ran out they only meet.
template <int UNITS>
struct ScaleFeeder {
    ScaleSource src;
    int g, lane;  // scale warp 0 .. 3
    int first, last, step, kb0, kb1;
    ScaleWords buf[kE8Ahead];
    struct Place {
        int w, kb, row0;
    } ahead;
    template <typename Rows>
    __device__ __forceinline__ void advance(Place& c, Rows rows) {
        c.kb += 4;
        if (c.kb >= kb1) {
            c.kb = kb0;
            c.w += step;
            if (c.w < last) c.row0 = rows(c.w);
        }
    }
    template <typename Rows>
    __device__ __forceinline__ void fetch(ScaleWords& to, Rows rows) {
        if (g >= UNITS || ahead.w >= last) return;
        load_scales(to, src, ahead.row0, ahead.kb, min(4, kb1 - ahead.kb), lane);
        advance(ahead, rows);
    }
    template <typename Rows>
    __device__ __forceinline__ void start(Rows rows) {
        ahead = {first, kb0, rows(first)};
#pragma unroll
        for (int i = 0; i < kE8Ahead; ++i) fetch(buf[i], rows);
    }
    // exchange: 2 * UNITS * 512 bytes of shared memory; tmem: the scale columns (chunk c's at (c % kE8Cols) * 4 * UNITS);
    // free(column, parity) waits for a column's MMAs, ready(column) arrives on its sfull.
    template <typename Rows, typename Free, typename Ready>
    __device__ __forceinline__ void run(Rows rows, uint32_t exchange, uint32_t tmem, int quadrant, Free free, Ready ready) {
        static_assert(kE8Ahead == kE8Cols && kE8Ahead % 2 == 0, "one buffer a column set, two exchange areas");
        const uint32_t mine = tmem + (static_cast<uint32_t>(quadrant * 32) << 16);
        Place put = {first, kb0, rows(first)};
        uint32_t parity = 1;  // the first pass over the columns finds them free
        bool ok = true;
        while (put.w < last) {
#pragma unroll
            for (int i = 0; i < kE8Ahead; ++i) {
                if (put.w >= last) break;
                const uint32_t area = exchange + (i & 1) * (UNITS * 512);
                if (g < UNITS) put_scales(area + g * 512, buf[i], src, put.row0, put.kb, min(4, kb1 - put.kb), lane);
                fetch(buf[i], rows);
                asm volatile("bar.sync 1, 128;" ::: "memory");
                ok = ok && free(i, parity, put.kb);
                if (ok) {
                    ptx::tc_fence_after();
                    uint4 v[UNITS];
#pragma unroll
                    for (int u = 0; u < UNITS; ++u) v[u] = ptx::ld_shared_v4(area + u * 512 + lane * 16);
#pragma unroll
                    for (int u = 0; u < UNITS; ++u) ptx::tmem_st_32x32b_x4(mine + i * (4 * UNITS) + u * 4, v[u]);
                    ptx::tmem_st_wait();
                    ptx::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) ready(i);
                }
                advance(put, rows);
            }
            parity ^= 1u;
        }
    }
};

__device__ __forceinline__ void e8_decode(int w, const E8m0Params& p, int& m_blk, int& n_blk) {
    const int group_sz = p.group_m * p.n_tiles;
    const int g = w / group_sz;
    const int first_m = g * p.group_m;
    const int gm = min(p.m_tiles - first_m, p.group_m);
    const int r = w - g * group_sz;
    n_blk = r / gm;
    m_blk = first_m + (r - n_blk * gm);
}

constexpr int kE8RowWords = 128 + 4;  // a row of 128 partial sums in shared memory, padded

// Four sums to C[row][..]: columns n .. n + 3 as a vector, or (VEC false) those of n, n + 32, n + 64, n + 96 that exist. One
// thread of the whole launch adds to an element, so the order of the additions is fixed; it waits for no old value (read and
// written back, 1024 x 1024 x 4096 took 15.3 us instead of 11, and 24.5 instead of 11.5 without vectors).
template <bool VEC>
__device__ __forceinline__ void store_four(const E8m0Params& p, long long row, int n, const float (&acc)[4]) {
    const long long at = row * p.ldc + n;
    if (p.out == OUT_F32) {
        float* dst = static_cast<float*>(p.C) + at;
        if constexpr (VEC) {
            if (p.accumulate) ptx::red_add_v4_f32(dst, acc[0], acc[1], acc[2], acc[3]);
            else *reinterpret_cast<float4*>(dst) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (n + 32 * j >= p.N) continue;
                if (p.accumulate) ptx::red_add_f32(dst + 32 * j, acc[j]);
                else dst[32 * j] = acc[j];
            }
        }
        return;
    }
    uint32_t u[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        if (p.out == OUT_BF16) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(acc[2 * j], acc[2 * j + 1]);
            u[j] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
            const __half2 h = __floats2half2_rn(acc[2 * j], acc[2 * j + 1]);
            u[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    uint16_t* dst = static_cast<uint16_t*>(p.C) + at;
    if constexpr (VEC) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(u[0], u[1]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n + 32 * j < p.N) dst[32 * j] = static_cast<uint16_t>((j & 1) ? (u[j >> 1] >> 16) : (u[j >> 1] & 0xffffu));
    }
}

// Adds up the S partial tiles ([rows][kE8RowWords] fp32 at the start of the shared memory of cluster CTAs first, first + STEP,
// ...) in that order and stores the sums to C[m0 ..][n0 .. n0 + 128]. The `rows` valid rows are dealt out over the S CTAs, of
// which this is number `part`; a warp takes a row, a lane four columns: neighbouring ones where C takes vectors of four,
// 32 apart where it does not, so that a warp's store is contiguous either way.
template <int S, int STEP>
__device__ __forceinline__ void sum_and_store(const E8m0Params& p, uint32_t smem_base, uint32_t first, uint32_t part, int m0,
                                              int rows, int n0) {
    const int warp = static_cast<int>(threadIdx.x) >> 5, lane = static_cast<int>(threadIdx.x) & 31;
    const int per = (rows + S - 1) / S;
    const int r1 = min(rows, (static_cast<int>(part) + 1) * per);
    const bool vec = p.c_vec_ok != 0 && n0 + 128 <= p.N;
    for (int r = static_cast<int>(part) * per + warp; r < r1; r += kE8Threads / 32) {
        const uint32_t row = smem_base + static_cast<uint32_t>(r * kE8RowWords * 4);
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        uint32_t w[S][4];
#pragma unroll
        for (uint32_t k = 0; k < static_cast<uint32_t>(S); ++k) {
            const uint32_t at = S > 1 ? ptx::mapa_shared(row, first + k * STEP) : row;
            if (vec) {
                ptx::ld_shared_cluster_v4(at + lane * 16, w[k][0], w[k][1], w[k][2], w[k][3]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) w[k][j] = ptx::ld_shared_cluster_u32(at + (lane + 32 * j) * 4);
            }
        }
#pragma unroll
        for (int k = 0; k < S; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] += __uint_as_float(w[k][j]);
        if (vec) store_four<true>(p, m0 + r, n0 + lane * 4, acc);
        else store_four<false>(p, m0 + r, n0 + lane, acc);
    }
}

// ==================================================================================== small and middling M
// Roles of the operands exchanged: the 128 rows of the instruction are rows of B (output columns), its N = TM columns are
// rows of A (tokens), 16 to 64 of them, so a few tokens cost a few columns of work instead of 128 rows of padding,
// and a lane of the accumulator is an output column: C's rows leave as contiguous runs.
//
// With few tokens the product is one pass over B, bounded by HBM. Every SM has to pull, so K is cut over the S CTAs of a
// cluster, whose partial sums meet in distributed shared memory (fixed slice order: results are reproducible); and a ring of
// about 100 KB lets two CTAs share an SM, so that one's start and end hide behind the other's loads.
template <int TM>
struct E8SmallSmem {
    static constexpr int kBStage = 128 * 128;
    static constexpr int kAStage = TM * 128;
    static constexpr int kStages = TM <= 32 ? 5 : 4;
    static constexpr int kTiles = kStages * (kBStage + kAStage);
    static_assert(TM * kE8RowWords * 4 <= kTiles, "the partial tile lies over the ring");
    static constexpr int kScaleOffset = kTiles;  // exchange areas: 128 rows of B, 128 of A
    static constexpr int kBarOffset = kScaleOffset + 2 * 2 * 512;
    static constexpr int kBars = 2 * kStages + 2 * kE8Cols + 1;
    static constexpr int kMiscOffset = kBarOffset + kBars * 8;
    static constexpr int kTotal = kMiscOffset + 16;
    static constexpr int kDynamicBytes = kTotal + 1024;
    static constexpr uint32_t kScaleCol = TM < 32 ? 32 : TM;  // accumulator columns before the scales'
    static constexpr uint32_t kTmemCols = TM <= 32 ? 64 : 128;
    static_assert(kScaleCol + kE8Cols * 8 <= kTmemCols, "tensor-memory columns");
};

template <int TM, int S>
__global__ void __launch_bounds__(kE8Threads, 2)
gemm_e8m0_small_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                       const E8m0Params p) {
    using L = E8SmallSmem<TM>;
    constexpr int STAGES = L::kStages;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = ptx::smem_u32(smem_raw);
    const uint32_t pad = ((raw_addr + 1023u) & ~1023u) - raw_addr;
    uint8_t* smem = smem_raw + pad;
    const uint32_t smem_base = raw_addr + pad;
    const uint32_t smem_b = smem_base;
    const uint32_t smem_a = smem_base + STAGES * L::kBStage;
    const uint32_t smem_s = smem_base + L::kScaleOffset;
    const uint32_t bar_full = smem_base + L::kBarOffset;
    const uint32_t bar_empty = bar_full + STAGES * 8;
    const uint32_t bar_sfull = bar_empty + STAGES * 8;
    const uint32_t bar_sdone = bar_sfull + kE8Cols * 8;
    const uint32_t bar_tfull = bar_sdone + kE8Cols * 8;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + L::kMiscOffset);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMiscOffset + 4);

    const int warp = static_cast<int>(threadIdx.x) >> 5;
    const int lane = static_cast<int>(threadIdx.x) & 31;
    const uint32_t rank = S > 1 ? ptx::cluster_ctarank() : 0u;
    const int tile = static_cast<int>(blockIdx.x) / S;
    const int n_blk = tile / p.m_tiles, m_blk = tile - n_blk * p.m_tiles;  // the token tiles of a piece of B side by side
    const int n0 = n_blk * 128, m0 = m_blk * TM;
    const int kb0 = static_cast<int>(static_cast<long long>(rank) * p.kb_total / S);
    const int kb1 = static_cast<int>(static_cast<long long>(rank + 1) * p.kb_total / S);

    auto load_block = [&](int kb, uint32_t stage) {
        if (kb == p.test_skip_kb) return;
        const uint32_t full = bar_full + stage * 8;
        ptx::mbar_arrive_expect_tx(full, L::kBStage + L::kAStage);
        ptx::tma_load_2d(smem_b + stage * L::kBStage, &tmap_b, full, kb * 128, n0);
        ptx::tma_load_2d(smem_a + stage * L::kAStage, &tmap_a, full, kb * 128, m0);
    };
    int prod_kb = kb0;
    if (warp == 0) {
        if (lane < STAGES) {
            ptx::mbar_init(bar_full + lane * 8, 1);
            ptx::mbar_init(bar_empty + lane * 8, 1);
        }
        if (lane < kE8Cols) {
            ptx::mbar_init(bar_sfull + lane * 8, 4);  // the scale warps
            ptx::mbar_init(bar_sdone + lane * 8, 1);
        }
        if (lane == 0) {
            ptx::mbar_init(bar_tfull, 1);
            *abort_flag = 0;
            ptx::prefetch_tensormap(&tmap_a);
            ptx::prefetch_tensormap(&tmap_b);
        }
        ptx::fence_barrier_init();
        __syncwarp();
        // the ring's first fill is on its way before the CTA-wide barrier
        if (ptx::elect_one()) {
            ptx::pdl_wait();
            for (int s = 0; s < STAGES && prod_kb < kb1; ++s, ++prod_kb) load_block(prod_kb, s);
        }
        __syncwarp();
    }
    if (warp == 1) {
        ptx::tmem_alloc(ptx::smem_u32(const_cast<uint32_t*>(tmem_slot)), L::kTmemCols);
        ptx::tmem_relinquish();
    }
    // the first loads of the scales, B's (unit 0) and A's (unit 1), are on their way too
    const bool of_a = warp == 7;
    ScaleFeeder<2> feeder;
    auto scale_rows = [&](int) { return of_a ? m0 : n0; };
    if (warp >= 6) {
        feeder.src = of_a ? ScaleSource{p.a_scale, p.a_rows, p.a_shift, p.M} : ScaleSource{p.b_scale, p.b_rows, p.b_shift, p.N};
        feeder.g = warp - 6;
        feeder.lane = lane;
        feeder.first = 0;
        feeder.last = feeder.step = 1;
        feeder.kb0 = kb0;
        feeder.kb1 = kb1;
        ptx::pdl_wait();
        feeder.start(scale_rows);
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    // only now, with this CTA's tensor memory in hand: a successor's CTA may share the SM and take what is left of it
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();

    auto raise_peers = [&]() {
        if constexpr (S > 1) {
            const uint32_t own = ptx::smem_u32(const_cast<int*>(abort_flag));
            for (uint32_t r = 0; r < static_cast<uint32_t>(S); ++r)
                if (r != rank) ptx::st_shared_cluster_u32(ptx::mapa_shared(own, r), 1u);
        }
    };

    if (warp == 0) {
        // ------------------------------------------------------------ TMA producer (after the first fill)
        if (ptx::elect_one()) {
            uint32_t stage = 0, phase = 0;  // parity of the `empty` completion that frees the slot again
            for (int kb = kb0 + STAGES; kb < kb1; ++kb) {
                if (!wait_bounded(bar_empty + stage * 8, phase, abort_flag, p.status, ROLE_PRODUCER, kb)) {
                    raise_peers();
                    break;
                }
                load_block(kb, stage);
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer
        if (ptx::elect_one()) {
            uint32_t stage = 0, phase = 0, col = 0, cphase = 0;
            bool ok = true;
            for (int kc = kb0; ok && kc < kb1; kc += 4) {
                if (!wait_bounded(bar_sfull + col * 8, cphase, abort_flag, p.status, ROLE_MMA, -1 - kc)) {
                    ok = false;
                    break;
                }
                const uint32_t sb_tmem = tmem_base + L::kScaleCol + col * 8, sa_tmem = sb_tmem + 4;
                const int n = min(4, kb1 - kc);
                for (int i = 0; i < n; ++i) {
                    if (!wait_bounded(bar_full + stage * 8, phase, abort_flag, p.status, ROLE_MMA, kc + i)) {
                        ok = false;
                        break;
                    }
                    ptx::tc_fence_after();
                    const uint64_t b_desc = ptx::make_kmajor_sw128_desc(smem_b + stage * L::kBStage);
                    const uint64_t a_desc = ptx::make_kmajor_sw128_desc(smem_a + stage * L::kAStage);
                    const uint32_t idesc = p.idesc | ptx::idesc_scale_id(static_cast<uint32_t>(i));
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        ptx::umma_e8m0(tmem_base, b_desc + 2u * k, a_desc + 2u * k, idesc, sb_tmem, sa_tmem,
                                       (kc + i > kb0 || k > 0) ? 1u : 0u);
                    ptx::tc_commit(bar_empty + stage * 8);
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                ptx::tc_commit(bar_sdone + col * 8);
                if (++col == kE8Cols) {
                    col = 0;
                    cphase ^= 1u;
                }
            }
            if (ok) ptx::tc_commit(bar_tfull);
            else raise_peers();
        }
    } else if (warp >= 6) {
        // ------------------------------------------------------------ scales
        auto free = [&](int col, uint32_t parity, int kb) {
            const bool ok = warp_wait(bar_sdone + col * 8, parity, abort_flag, p.status, ROLE_SCALES, kb);
            if (!ok) raise_peers();
            return ok;
        };
        auto ready = [&](int col) { ptx::mbar_arrive(bar_sfull + col * 8); };
        feeder.run(scale_rows, smem_s, tmem_base + L::kScaleCol, warp & 3, free, ready);
    } else {
        // ------------------------------------------------------------ accumulator -> own shared memory, a token a row
        const int quad = warp & 3;
        if (warp_wait(bar_tfull, 0u, abort_flag, p.status, ROLE_EPILOGUE, tile)) {
            ptx::tc_fence_after();
            // the ring is idle: every load has landed and every MMA that read it has completed
            float* col = reinterpret_cast<float*>(smem) + quad * 32 + lane;
            const int tokens = min(TM, p.M - m0);
#pragma unroll 1
            for (int c = 0; c < TM && c < tokens; c += 32) {
                uint32_t v[32];
                ptx::tmem_ld_32x32b_x32(tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + c, v);
                ptx::tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    if (c + j < tokens) col[(c + j) * kE8RowWords] = __uint_as_float(v[j]);
            }
            ptx::tc_fence_before();
        } else {
            raise_peers();
        }
    }

    // ---------------------------------------------------------------- every CTA's partial tile is in place
    __syncthreads();
    if constexpr (S > 1) {
        ptx::cluster_arrive();
        ptx::cluster_wait();
    }
    if (*abort_flag == 0)  // the cluster's CTAs share the tokens out
        sum_and_store<S, 1>(p, smem_base, 0u, rank, m0, min(TM, p.M - m0), n0);

    // ---------------------------------------------------------------- teardown
    ptx::tc_fence_before();
    __syncthreads();
    if constexpr (S > 1) {  // no CTA's shared memory goes away while a peer may still read it
        ptx::cluster_arrive();
        ptx::cluster_wait();
    }
    if (*abort_flag != 0) {
        // let copies and MMAs that were already issued finish before the memory they touch is released
        for (int i = 0; i < 64; ++i) __nanosleep(20000);
        __syncthreads();
    }
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem_base, L::kTmemCols);
    }
}

// ==================================================================================== large products
// CTA pairs on 256 x 256 tiles (tcgen05.mma.cta_group::2; the ring, the pair's barriers and the persistent tile loop as in
// gemm_sm100_2cta.cuh). Each CTA's tensor memory has 512 columns: two 256-column accumulators would leave none for scales,
// so the second accumulator starts at column 192 and the last 64 columns hold four chunks of scales. The accumulators
// share columns 192..255: the epilogue drains those first and hands them over (`tfree`), and the next tile's MMAs run under
// the rest of the drain. The first instruction of a tile waits only for a quarter of its predecessor's epilogue; the arrival
// that tells the issuer is in its way, so it orders no more than it must (mbar_arrive_remote; as a cluster-scope release it
// made 6144 x 7168 x 2048 take 91 us instead of 85).
//
// Scales: the leader's instruction multiplies each CTA's 128 rows by that CTA's A scales, and all 256 columns by the B
// scales, which both CTAs hold in full; the scale warps of either CTA arrive on the leader's `sfull`.
//
// With 256 x 128 tiles (twice as many, for problems that have too few of the larger) both accumulators fit side by side.
template <int BN>
struct E8PairSmem {
    static constexpr int kUnits = 1 + BN / 128;  // 128 rows of scales each: this CTA's of A, all of B
    static constexpr int kStages = BN == 256 ? 6 : 8;
    static constexpr int kAStage = 128 * 128;
    static constexpr int kBStage = (BN / 2) * 128;
    static constexpr int kTiles = kStages * (kAStage + kBStage);
    static constexpr int kOutOffset = kTiles;  // one 4 KB staging box per epilogue warp
    static constexpr int kScaleOffset = kOutOffset + 4 * 4096;
    static constexpr int kBarOffset = kScaleOffset + 2 * kUnits * 512;
    static constexpr int kBars = 2 * kStages + 2 * kE8Cols + 4;  // full, empty, sfull, sdone, tfull[2], tfree[2]
    static constexpr int kMiscOffset = kBarOffset + kBars * 8;
    static constexpr int kTotal = kMiscOffset + 16;
    static constexpr int kDynamicBytes = kTotal + 1024;
    static constexpr uint32_t kAccStep = BN == 256 ? 192 : 128;  // first column of the second accumulator
    static constexpr uint32_t kScaleCol = BN == 256 ? 448 : 256;  // first column of the scales
    static constexpr uint32_t kScaleCols = 4 * kUnits;  // columns of a chunk: A's, then B's
    static_assert(kAccStep + BN <= kScaleCol && kScaleCol + kE8Cols * kScaleCols <= 512, "tensor-memory columns");
};

// A staged box to a C that TMA cannot address (any ldc, any base aligned to its element), or to the last columns of one that
// do not end on 16 bytes: a warp writes a row's 128 bytes at a time; 16-bit rows as words where the row starts on one. fp32
// rows are read from the box eight at a time before the first of them is written, and an accumulating product adds without
// reading C: row after row 8192 x 4096 x 4096 took 126 us instead of 106, and 890 instead of 110 accumulating. (16-bit rows
// gain nothing by eights; rows that start inside a word, shifted between the lanes and stored as words, took 164 us there
// instead of 95. From registers, a row a lane, 2500 x 2500 x 8192 took 115 us.)
template <int OUT>
__device__ __forceinline__ void store_box_rows(const E8m0Params& p, uint32_t box, int row0, int n0, int lane) {
    constexpr int OB = OutBytes<OUT>::value;
    constexpr int U = OUT == OUT_F32 ? 8 : 1;
    const int rows = min(32, p.M - row0);
    const long long step = p.ldc * OB;
    uint8_t* dst = static_cast<uint8_t*>(p.C) + (static_cast<long long>(row0) * p.ldc + n0) * OB;
#pragma unroll(OUT == OUT_F32 ? 1 : 4)
    for (int r0 = 0; r0 < rows; r0 += U, dst += U * step) {
        uint32_t w[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {  // 16-byte units of row r lie exchanged by r % 8
            const int r = r0 + i;
            w[i] = ptx::ld_shared_u32(box + static_cast<uint32_t>(r * 128 + (((lane >> 2) ^ (r & 7)) * 16) + (lane & 3) * 4));
        }
        if constexpr (OUT == OUT_F32) {
            if (n0 + lane >= p.N) continue;
            uint8_t* at = dst + 4 * lane;
            if (p.accumulate) {
#pragma unroll
                for (int i = 0; i < U; ++i)
                    if (r0 + i < rows) ptx::red_add_f32(reinterpret_cast<float*>(at + i * step), __uint_as_float(w[i]));
            } else {
#pragma unroll
                for (int i = 0; i < U; ++i)
                    if (r0 + i < rows) *reinterpret_cast<uint32_t*>(at + i * step) = w[i];
            }
        } else {
            uint16_t* h = reinterpret_cast<uint16_t*>(dst) + 2 * lane;
            if ((reinterpret_cast<uintptr_t>(dst) & 3u) == 0 && n0 + 64 <= p.N) {
                *reinterpret_cast<uint32_t*>(h) = w[0];
            } else {
                if (n0 + 2 * lane < p.N) h[0] = static_cast<uint16_t>(w[0] & 0xffffu);
                if (n0 + 2 * lane + 1 < p.N) h[1] = static_cast<uint16_t>(w[0] >> 16);
            }
        }
    }
}

template <int OUT, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kE8Threads, 1)
gemm_e8m0_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                      const __grid_constant__ CUtensorMap tmap_c, const E8m0Params p) {
    using L = E8PairSmem<BN>;
    static_assert(BN == 256 || BN == 128, "pair tile width");
    constexpr int STAGES = L::kStages;
    constexpr bool kOverlap = BN == 256;  // the accumulators share columns
    constexpr int OB = OutBytes<OUT>::value;
    constexpr int CW = 128 / OB;  // columns of a staged box: 64 (16-bit out) or 32

    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = ptx::smem_u32(smem_raw);
    const uint32_t pad = ((raw_addr + 1023u) & ~1023u) - raw_addr;
    uint8_t* smem = smem_raw + pad;
    const uint32_t smem_base = raw_addr + pad;
    const uint32_t smem_a = smem_base;
    const uint32_t smem_b = smem_base + STAGES * L::kAStage;
    const uint32_t smem_s = smem_base + L::kScaleOffset;
    const uint32_t bar_full = smem_base + L::kBarOffset;
    const uint32_t bar_empty = bar_full + STAGES * 8;
    const uint32_t bar_sfull = bar_empty + STAGES * 8;
    const uint32_t bar_sdone = bar_sfull + kE8Cols * 8;
    const uint32_t bar_tfull = bar_sdone + kE8Cols * 8;
    // tfree[0] with overlapping accumulators: a tile's share of the common columns is out; else tfree[a]: accumulator a is
    const uint32_t bar_tfree = bar_tfull + 2 * 8;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + L::kMiscOffset);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMiscOffset + 4);

    const int warp = static_cast<int>(threadIdx.x) >> 5;
    const int lane = static_cast<int>(threadIdx.x) & 31;
    const uint32_t rank = ptx::cluster_ctarank();  // 0 = leader
    const int cluster_id = static_cast<int>(blockIdx.x) >> 1;
    const int n_clusters = static_cast<int>(gridDim.x) >> 1;
    const int total_work = p.m_tiles * p.n_tiles;
    const uint32_t peer_abort = ptx::mapa_shared(ptx::smem_u32(const_cast<int*>(abort_flag)), rank ^ 1u);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            ptx::mbar_init(bar_full + s * 8, 1);
            ptx::mbar_init(bar_empty + s * 8, 1);
        }
        for (int c = 0; c < kE8Cols; ++c) {
            ptx::mbar_init(bar_sfull + c * 8, 8);  // four scale warps of each CTA
            ptx::mbar_init(bar_sdone + c * 8, 1);
        }
        ptx::mbar_init(bar_tfull, 1);
        ptx::mbar_init(bar_tfull + 8, 1);
        ptx::mbar_init(bar_tfree, 8);  // four epilogue warps of each CTA
        ptx::mbar_init(bar_tfree + 8, 8);
        *abort_flag = 0;
        ptx::fence_barrier_init();
    }
    if (warp == 0 && lane == 0) {
        ptx::prefetch_tensormap(&tmap_a);
        ptx::prefetch_tensormap(&tmap_b);
        if (p.c_tma_ok) ptx::prefetch_tensormap(&tmap_c);
    }
    if (warp == 1) {
        ptx::tmem_alloc_pair(ptx::smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
        ptx::tmem_relinquish_pair();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::cluster_arrive();
    ptx::cluster_wait();
    ptx::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();

    if (warp == 0) {
        // ------------------------------------------------------------ TMA producer (both CTAs)
        if (ptx::elect_one()) {
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            for (int w = cluster_id; ok && w < total_work; w += n_clusters) {
                int m_blk, n_blk;
                e8_decode(w, p, m_blk, n_blk);
                const int row_a = (m_blk * 2 + static_cast<int>(rank)) * 128;
                const int row_b = n_blk * BN + static_cast<int>(rank) * (BN / 2);
                for (int kb = 0; kb < p.kb_total; ++kb) {
                    if (!wait_bounded(bar_empty + stage * 8, phase ^ 1u, abort_flag, p.status, ROLE_PRODUCER, kb, peer_abort)) {
                        ok = false;
                        break;
                    }
                    if (kb != p.test_skip_kb) {
                        if (rank == 0) ptx::mbar_arrive_expect_tx(bar_full + stage * 8, 2 * (L::kAStage + L::kBStage));
                        const uint32_t leader_full = ptx::mapa_shared(bar_full + stage * 8, 0);
                        ptx::tma_load_2d_pair(smem_a + stage * L::kAStage, &tmap_a, leader_full, kb * 128, row_a);
                        ptx::tma_load_2d_pair(smem_b + stage * L::kBStage, &tmap_b, leader_full, kb * 128, row_b);
                    }
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer (leader CTA only)
        if (rank == 0 && ptx::elect_one()) {
            uint32_t stage = 0, phase = 0, col = 0, cphase = 0;
            uint32_t it = 0;
            bool ok = true;
            for (int w = cluster_id; ok && w < total_work; w += n_clusters, ++it) {
                const uint32_t acc = it & 1u;
                const uint32_t d_tmem = tmem_base + acc * L::kAccStep;
                if constexpr (kOverlap) {
                    // the previous tile's share of the common columns is out (and with it everything of the tile before)
                    if (it > 0 && !wait_bounded(bar_tfree, (it - 1) & 1u, abort_flag, p.status, ROLE_MMA, -1, peer_abort)) break;
                } else {
                    if (!wait_bounded(bar_tfree + acc * 8, ((it >> 1) & 1u) ^ 1u, abort_flag, p.status, ROLE_MMA, -1, peer_abort)) break;
                }
                for (int kc = 0; ok && kc < p.kb_total; kc += 4) {
                    if (!wait_bounded(bar_sfull + col * 8, cphase, abort_flag, p.status, ROLE_MMA, -2 - kc, peer_abort)) {
                        ok = false;
                        break;
                    }
                    const uint32_t sa_tmem = tmem_base + L::kScaleCol + col * L::kScaleCols, sb_tmem = sa_tmem + 4;
                    const int n = min(4, p.kb_total - kc);
                    for (int i = 0; i < n; ++i) {
                        if (!wait_bounded(bar_full + stage * 8, phase, abort_flag, p.status, ROLE_MMA, kc + i, peer_abort)) {
                            ok = false;
                            break;
                        }
                        ptx::tc_fence_after();
                        const uint64_t a_desc = ptx::make_kmajor_sw128_desc(smem_a + stage * L::kAStage);
                        const uint64_t b_desc = ptx::make_kmajor_sw128_desc(smem_b + stage * L::kBStage);
                        const uint32_t idesc = p.idesc | ptx::idesc_scale_id(static_cast<uint32_t>(i));
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            ptx::umma_e8m0_pair(d_tmem, a_desc + 2u * k, b_desc + 2u * k, idesc, sa_tmem, sb_tmem,
                                                (kc + i > 0 || k > 0) ? 1u : 0u);
                        ptx::tc_commit_pair(bar_empty + stage * 8, 3);
                        if (++stage == STAGES) {
                            stage = 0;
                            phase ^= 1u;
                        }
                    }
                    if (!ok) break;
                    ptx::tc_commit_pair(bar_sdone + col * 8, 3);
                    if (++col == kE8Cols) {
                        col = 0;
                        cphase ^= 1u;
                    }
                }
                if (ok) ptx::tc_commit_pair(bar_tfull + acc * 8, 3);
            }
        }
    } else if (warp >= 6) {
        // ------------------------------------------------------------ scales (both CTAs)
        const bool of_a = warp == 6;
        ScaleFeeder<L::kUnits> feeder;
        auto scale_rows = [&](int w) {
            int m_blk, n_blk;
            e8_decode(w, p, m_blk, n_blk);
            return of_a ? (m_blk * 2 + static_cast<int>(rank)) * 128 : n_blk * BN + (warp - 7) * 128;
        };
        feeder.src = of_a ? ScaleSource{p.a_scale, p.a_rows, p.a_shift, p.M} : ScaleSource{p.b_scale, p.b_rows, p.b_shift, p.N};
        feeder.g = warp - 6;
        feeder.lane = lane;
        feeder.first = cluster_id;
        feeder.last = total_work;
        feeder.step = n_clusters;
        feeder.kb0 = 0;
        feeder.kb1 = p.kb_total;
        feeder.start(scale_rows);
        auto free = [&](int col, uint32_t parity, int kb) {
            return warp_wait(bar_sdone + col * 8, parity, abort_flag, p.status, ROLE_SCALES, kb, peer_abort);
        };
        auto ready = [&](int col) { ptx::mbar_arrive_remote(ptx::mapa_shared(bar_sfull + col * 8, 0)); };
        feeder.run(scale_rows, smem_s, tmem_base + L::kScaleCol, warp & 3, free, ready);
    } else {
        // ------------------------------------------------------------ epilogue (both CTAs)
        const int quad = warp & 3;
        const uint32_t stage_base = smem_base + L::kOutOffset + quad * 4096u;
        uint32_t it = 0;
        for (int w = cluster_id; w < total_work; w += n_clusters, ++it) {
            int m_blk, n_blk;
            e8_decode(w, p, m_blk, n_blk);
            const uint32_t acc = it & 1u;
            if (!warp_wait(bar_tfull + acc * 8, (it >> 1) & 1u, abort_flag, p.status, ROLE_EPILOGUE, w, peer_abort)) break;
            ptx::tc_fence_after();
            const uint32_t t_addr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + acc * L::kAccStep;
            const int row0 = (m_blk * 2 + static_cast<int>(rank)) * 128 + quad * 32;
            // the columns that both accumulators use come first: the last 64 of the first, the first 64 of the second
            const int first = kOverlap && acc == 0 ? static_cast<int>(L::kAccStep) / CW : 0;
            // boxes after which the issuer may go on: those, or all of them
            constexpr int kShared = kOverlap ? (BN - static_cast<int>(L::kAccStep)) / CW : BN / CW;
#pragma unroll 1
            for (int b = 0; b < BN / CW; ++b) {
                const int c = (first + b) & (BN / CW - 1);
                const int n0 = n_blk * BN + c * CW;
                const bool live = row0 < p.M && n0 < p.N;  // warp-uniform
                uint32_t v[CW];
                if (live) {
                    ptx::tmem_ld_32x32b_x32(t_addr + c * CW, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
                    if constexpr (CW == 64)
                        ptx::tmem_ld_32x32b_x32(t_addr + c * CW + 32, *reinterpret_cast<uint32_t(*)[32]>(&v[32]));
                    ptx::tmem_ld_wait();
                }
                if (b == kShared - 1) {
                    ptx::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive_remote(ptx::mapa_shared(bar_tfree + (kOverlap ? 0 : acc * 8), 0));
                }
                if (!live) continue;
                uint32_t u[32];
                if constexpr (OUT == OUT_F32) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) u[j] = v[j];
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        if constexpr (OUT == OUT_BF16) {
                            const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
                            u[j] = *reinterpret_cast<const uint32_t*>(&h);
                        } else {
                            const __half2 h = __floats2half2_rn(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
                            u[j] = *reinterpret_cast<const uint32_t*>(&h);
                        }
                    }
                }
                // a staged box of 32 rows x 128 bytes; it is free once the store before has read it
                const bool by_tma = p.c_tma_ok && n0 < p.n_tma;
                if (p.c_tma_ok && ptx::elect_one()) ptx::tma_store_wait_read<0>();
                __syncwarp();
                const uint32_t row_addr = stage_base + static_cast<uint32_t>(lane) * 128u;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    ptx::st_shared_v4(row_addr + static_cast<uint32_t>((j ^ (lane & 7)) * 16), u[4 * j], u[4 * j + 1],
                                      u[4 * j + 2], u[4 * j + 3]);
                if (by_tma) {
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    if (ptx::elect_one()) {
                        if (OUT == OUT_F32 && p.accumulate) ptx::tma_add_3d(&tmap_c, stage_base, n0, row0, 0);
                        else ptx::tma_store_3d(&tmap_c, stage_base, n0, row0, 0);
                        ptx::tma_store_commit();
                    }
                } else {
                    __syncwarp();
                    store_box_rows<OUT>(p, stage_base, row0, n0, lane);
                    __syncwarp();
                }
            }
        }
        if (lane == 0) ptx::tma_store_wait_read<0>();
    }

    // ---------------------------------------------------------------- teardown
    ptx::tc_fence_before();
    __syncthreads();
    // neither CTA may release its shared or tensor memory while the other can still touch it
    ptx::cluster_arrive();
    ptx::cluster_wait();
    if (*abort_flag != 0) {
        for (int i = 0; i < 64; ++i) __nanosleep(20000);
        __syncthreads();
    }
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc_pair(tmem_base, 512);
    }
}

// ==================================================================================== few tiles, long K
// 256 x 128 tiles on CTA pairs with K cut over the S pairs of a cluster, one tile per cluster; the partial sums meet in
// distributed shared memory as in the small kernel (each CTA's 128 rows with the same rows of the other pairs).
struct E8PairKSmem {
    static constexpr int kStages = 8;
    static constexpr int kAStage = 128 * 128;
    static constexpr int kBStage = 64 * 128;
    static constexpr int kTiles = kStages * (kAStage + kBStage);
    static_assert(128 * kE8RowWords * 4 <= kTiles, "the partial tile lies over the ring");
    static constexpr int kScaleOffset = kTiles;
    static constexpr int kBarOffset = kScaleOffset + 2 * 2 * 512;
    static constexpr int kBars = 2 * kStages + 2 * kE8Cols + 1;
    static constexpr int kMiscOffset = kBarOffset + kBars * 8;
    static constexpr int kTotal = kMiscOffset + 16;
    static constexpr int kDynamicBytes = kTotal + 1024;
    static constexpr uint32_t kScaleCol = 128;
    static constexpr uint32_t kTmemCols = 256;
};

template <int S>
__global__ void __launch_bounds__(kE8Threads, 1)
gemm_e8m0_pair_split_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                            const E8m0Params p) {
    using L = E8PairKSmem;
    constexpr int STAGES = L::kStages;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = ptx::smem_u32(smem_raw);
    const uint32_t pad = ((raw_addr + 1023u) & ~1023u) - raw_addr;
    uint8_t* smem = smem_raw + pad;
    const uint32_t smem_base = raw_addr + pad;
    const uint32_t smem_a = smem_base;
    const uint32_t smem_b = smem_base + STAGES * L::kAStage;
    const uint32_t smem_s = smem_base + L::kScaleOffset;
    const uint32_t bar_full = smem_base + L::kBarOffset;
    const uint32_t bar_empty = bar_full + STAGES * 8;
    const uint32_t bar_sfull = bar_empty + STAGES * 8;
    const uint32_t bar_sdone = bar_sfull + kE8Cols * 8;
    const uint32_t bar_tfull = bar_sdone + kE8Cols * 8;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + L::kMiscOffset);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kMiscOffset + 4);

    const int warp = static_cast<int>(threadIdx.x) >> 5;
    const int lane = static_cast<int>(threadIdx.x) & 31;
    const uint32_t crank = ptx::cluster_ctarank();
    const uint32_t rank = crank & 1u;        // in the pair; 0 = leader
    const uint32_t leader = crank & ~1u;
    const uint32_t slice = crank >> 1;
    int m_blk, n_blk;
    e8_decode(static_cast<int>(blockIdx.x) / (2 * S), p, m_blk, n_blk);
    const int m0 = (m_blk * 2 + static_cast<int>(rank)) * 128, n0 = n_blk * 128;
    const int kb0 = static_cast<int>(static_cast<long long>(slice) * p.kb_total / S);
    const int kb1 = static_cast<int>(static_cast<long long>(slice + 1) * p.kb_total / S);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            ptx::mbar_init(bar_full + s * 8, 1);
            ptx::mbar_init(bar_empty + s * 8, 1);
        }
        for (int c = 0; c < kE8Cols; ++c) {
            ptx::mbar_init(bar_sfull + c * 8, 8);  // four scale warps of each CTA of the pair
            ptx::mbar_init(bar_sdone + c * 8, 1);
        }
        ptx::mbar_init(bar_tfull, 1);
        *abort_flag = 0;
        ptx::fence_barrier_init();
        ptx::prefetch_tensormap(&tmap_a);
        ptx::prefetch_tensormap(&tmap_b);
    }
    if (warp == 1) {
        ptx::tmem_alloc_pair(ptx::smem_u32(const_cast<uint32_t*>(tmem_slot)), L::kTmemCols);
        ptx::tmem_relinquish_pair();
    }
    const bool of_a = warp == 6;
    ScaleFeeder<2> feeder;
    auto scale_rows = [&](int) { return of_a ? m0 : n0; };
    if (warp >= 6) {
        feeder.src = of_a ? ScaleSource{p.a_scale, p.a_rows, p.a_shift, p.M} : ScaleSource{p.b_scale, p.b_rows, p.b_shift, p.N};
        feeder.g = warp - 6;
        feeder.lane = lane;
        feeder.first = 0;
        feeder.last = feeder.step = 1;
        feeder.kb0 = kb0;
        feeder.kb1 = kb1;
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::cluster_arrive();
    ptx::cluster_wait();
    ptx::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    ptx::pdl_launch_dependents();
    ptx::pdl_wait();

    auto raise_peers = [&]() {
        const uint32_t own = ptx::smem_u32(const_cast<int*>(abort_flag));
        for (uint32_t r = 0; r < 2u * S; ++r)
            if (r != crank) ptx::st_shared_cluster_u32(ptx::mapa_shared(own, r), 1u);
    };

    if (warp == 0) {
        // ------------------------------------------------------------ TMA producer (every CTA)
        if (ptx::elect_one()) {
            uint32_t stage = 0, phase = 0;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!wait_bounded(bar_empty + stage * 8, phase ^ 1u, abort_flag, p.status, ROLE_PRODUCER, kb)) {
                    raise_peers();
                    break;
                }
                if (kb != p.test_skip_kb) {
                    if (rank == 0) ptx::mbar_arrive_expect_tx(bar_full + stage * 8, 2 * (L::kAStage + L::kBStage));
                    const uint32_t leader_full = ptx::mapa_shared(bar_full + stage * 8, leader);
                    ptx::tma_load_2d_pair(smem_a + stage * L::kAStage, &tmap_a, leader_full, kb * 128, m0);
                    ptx::tma_load_2d_pair(smem_b + stage * L::kBStage, &tmap_b, leader_full, kb * 128,
                                          n0 + static_cast<int>(rank) * 64);
                }
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer (the pair's leader)
        if (rank == 0 && ptx::elect_one()) {
            const uint16_t both = static_cast<uint16_t>(3u << leader);
            uint32_t stage = 0, phase = 0, col = 0, cphase = 0;
            bool ok = true;
            for (int kc = kb0; ok && kc < kb1; kc += 4) {
                if (!wait_bounded(bar_sfull + col * 8, cphase, abort_flag, p.status, ROLE_MMA, -1 - kc)) {
                    ok = false;
                    break;
                }
                const uint32_t sa_tmem = tmem_base + L::kScaleCol + col * 8, sb_tmem = sa_tmem + 4;
                const int n = min(4, kb1 - kc);
                for (int i = 0; i < n; ++i) {
                    if (!wait_bounded(bar_full + stage * 8, phase, abort_flag, p.status, ROLE_MMA, kc + i)) {
                        ok = false;
                        break;
                    }
                    ptx::tc_fence_after();
                    const uint64_t a_desc = ptx::make_kmajor_sw128_desc(smem_a + stage * L::kAStage);
                    const uint64_t b_desc = ptx::make_kmajor_sw128_desc(smem_b + stage * L::kBStage);
                    const uint32_t idesc = p.idesc | ptx::idesc_scale_id(static_cast<uint32_t>(i));
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        ptx::umma_e8m0_pair(tmem_base, a_desc + 2u * k, b_desc + 2u * k, idesc, sa_tmem, sb_tmem,
                                            (kc + i > kb0 || k > 0) ? 1u : 0u);
                    ptx::tc_commit_pair(bar_empty + stage * 8, both);
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                ptx::tc_commit_pair(bar_sdone + col * 8, both);
                if (++col == kE8Cols) {
                    col = 0;
                    cphase ^= 1u;
                }
            }
            if (ok) ptx::tc_commit_pair(bar_tfull, both);
            else raise_peers();
        }
    } else if (warp >= 6) {
        // ------------------------------------------------------------ scales (every CTA)
        auto free = [&](int col, uint32_t parity, int kb) {
            const bool ok = warp_wait(bar_sdone + col * 8, parity, abort_flag, p.status, ROLE_SCALES, kb);
            if (!ok) raise_peers();
            return ok;
        };
        auto ready = [&](int col) { ptx::mbar_arrive_remote(ptx::mapa_shared(bar_sfull + col * 8, leader)); };
        feeder.start(scale_rows);
        feeder.run(scale_rows, smem_s, tmem_base + L::kScaleCol, warp & 3, free, ready);
    } else {
        // ------------------------------------------------------------ accumulator -> own shared memory
        const int quad = warp & 3;
        if (warp_wait(bar_tfull, 0u, abort_flag, p.status, ROLE_EPILOGUE, m_blk)) {
            ptx::tc_fence_after();
            // the ring is idle: every load has landed and every MMA that read it, in either CTA, has completed
            if (m0 + quad * 32 < p.M) {  // rows that exist
                const uint32_t row_addr = smem_base + static_cast<uint32_t>((quad * 32 + lane) * kE8RowWords * 4);
#pragma unroll 1
                for (int c = 0; c < 128; c += 32) {
                    uint32_t v[32];
                    ptx::tmem_ld_32x32b_x32(tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + c, v);
                    ptx::tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        ptx::st_shared_v4(row_addr + static_cast<uint32_t>((c + 4 * j) * 4), v[4 * j], v[4 * j + 1], v[4 * j + 2],
                                          v[4 * j + 3]);
                }
            }
            ptx::tc_fence_before();
        } else {
            raise_peers();
        }
    }

    // ---------------------------------------------------------------- every CTA's partial tile is in place
    __syncthreads();
    ptx::cluster_arrive();
    ptx::cluster_wait();
    if (*abort_flag == 0 && m0 < p.M) sum_and_store<S, 2>(p, smem_base, rank, slice, m0, min(128, p.M - m0), n0);

    // ---------------------------------------------------------------- teardown
    ptx::tc_fence_before();
    __syncthreads();
    ptx::cluster_arrive();
    ptx::cluster_wait();
    if (*abort_flag != 0) {
        for (int i = 0; i < 64; ++i) __nanosleep(20000);
        __syncthreads();
    }
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc_pair(tmem_base, L::kTmemCols);
    }
}

// tokens_per_tile: 16, 32 or 64; slices: 1, 2, 4 or 8, at most kb_total (gemm_e8m0.cu).
cudaError_t launch_e8m0_small(int tokens_per_tile, int slices, const CUtensorMap& ta, const CUtensorMap& tb,
                              const E8m0Params& p, cudaStream_t stream);
// tile_n: 256 or 128 (slices == 1: persistent), 128 with slices == 2.
cudaError_t launch_e8m0_pair(int tile_n, int slices, const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc,
                             const E8m0Params& p, int clusters, cudaStream_t stream);

}  // namespace qgemm
