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
// id. One tensor-memory word holds a row's scales of four K blocks (a "chunk"), so a chunk's scales are 512 bytes per 128
// rows. They come from global memory in the caller's plain layout ([K block][row], or [K block][row / 128]) through a warp
// that transposes them into words, 16 bytes a lane, and from there with tcgen05.cp.
//
// Barriers besides the ring's full / empty and the accumulators': sfull[slot] (a chunk's scales are in shared memory),
// sempty[slot] (the chunk's last MMA has completed: its shared-memory slot and its tensor-memory columns, same index, are
// free). All waits are bounded as in gemm_sm100.cuh.
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
    int* status;
};

constexpr int kE8Slots = 4;  // chunks of scales in flight
constexpr int kE8Threads = 256;  // producer, MMA issuer, four epilogue warps, two scale warps
enum : int { ROLE_SCALES = 4 };

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
// load_scales uses nothing that it loads, and the warps that fill the slots keep kE8Ahead chunks loading: a chunk must not
// cost a memory latency each, which under the ring's own traffic is more than the tensor cores take for it (measured at
// 4096 x 7168 x 7168, row-scaled B: 404 us with one load waited for at a time, 194 with one chunk at a time, 157 with
// four in flight).
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
        for (int i = 0; i < 4; ++i) out.lo[i] = __ldg(scale_row(s, row0, kb0 + min(i, n - 1)));
        return;
    }
    const int bytes = min(128, s.rows - min(row0, s.rows - 1));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint8_t* at = scale_row(s, row0, kb0 + min(i, n - 1));
        const int off = static_cast<int>(reinterpret_cast<uintptr_t>(at) & 3u);
        const int last = (off + bytes - 1) >> 2;
        const uint32_t* words = reinterpret_cast<const uint32_t*>(at - off);
        out.lo[i] = __ldg(words + min(lane, last));
        if (off != 0) out.hi[i] = __ldg(words + min(lane + 1, last));
    }
}
// Into the 512 bytes that tc_copy_scales reads: row r's four K blocks as a word at (r % 32) * 16 + (r / 32) * 4.
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

// The scale warp of a kernel whose CTA has one K range [kb0, kb1) of one tile: `start` loads the first chunks (before the
// CTA-wide barrier), `run` fills the slots and arrives on sfull (at cluster address full_at(slot)).
struct ScaleFeeder {
    ScaleSource src;
    int row0, kb0, kb1, lane;
    ScaleWords buf[kE8Ahead];
    __device__ __forceinline__ void start() {
#pragma unroll
        for (int i = 0; i < kE8Ahead; ++i)
            if (kb0 + 4 * i < kb1) load_scales(buf[i], src, row0, kb0 + 4 * i, min(4, kb1 - kb0 - 4 * i), lane);
    }
    // Chunk c goes to slot c % kE8Slots; free(slot, parity) waits for it and says whether to go on.
    template <typename Free, typename Put>
    __device__ __forceinline__ bool run(Free free, Put filled, uint32_t slots, uint32_t slot_bytes) {
        static_assert(kE8Ahead == kE8Slots, "one buffer a slot");
        uint32_t parity = 1;  // the first pass over the slots finds them free
        for (int kc = kb0; kc < kb1; kc += 4 * kE8Ahead, parity ^= 1u) {
#pragma unroll
            for (int i = 0; i < kE8Ahead; ++i) {
                const int k = kc + 4 * i;
                if (k >= kb1) break;
                if (!free(i, parity, k)) return false;
                put_scales(slots + i * slot_bytes, buf[i], src, row0, k, min(4, kb1 - k), lane);
                const int ahead = k + 4 * kE8Ahead;
                __syncwarp();
                filled(i);
                if (ahead < kb1) load_scales(buf[i], src, row0, ahead, min(4, kb1 - ahead), lane);
            }
        }
        return true;
    }
};

// wait_bounded for a barrier that another CTA of the cluster arrives on after writing its own shared memory.
__device__ __forceinline__ bool wait_bounded_cluster(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status,
                                                     int role, int where, uint32_t peer_abort) {
    if (!wait_bounded(bar, parity, abort_flag, status, role, where, peer_abort)) return false;
    return ptx::mbar_try_wait_cluster(bar, parity);  // complete already: this orders the peer's writes
}

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

// Adds up the S partial tiles ([rows][kE8RowWords] fp32 at the start of the shared memory of cluster CTAs first, first + STEP,
// ...) in that order and stores the sums to C[m0 ..][n0 .. n0 + 128]. The `rows` valid rows are dealt out over the S CTAs, of
// which this is number `part`; a warp takes a row, a lane four columns.
template <int S, int STEP, int WARPS = kE8Threads / 32>
__device__ __forceinline__ void sum_and_store(const E8m0Params& p, uint32_t smem_base, uint32_t first, uint32_t part, int m0,
                                              int rows, int n0) {
    const int warp = static_cast<int>(threadIdx.x) >> 5, lane = static_cast<int>(threadIdx.x) & 31;
    const int per = (rows + S - 1) / S;
    const int r1 = min(rows, (static_cast<int>(part) + 1) * per);
    const int n = n0 + lane * 4;
    const int n_valid = min(4, p.N - n);
    if (n_valid <= 0) return;
    const bool vec = p.c_vec_ok != 0 && n_valid == 4;
    for (int r = static_cast<int>(part) * per + warp; r < r1; r += WARPS) {
        const uint32_t own = smem_base + static_cast<uint32_t>((r * kE8RowWords + lane * 4) * 4);
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        uint32_t w[S][4];
#pragma unroll
        for (uint32_t k = 0; k < static_cast<uint32_t>(S); ++k) {
            if constexpr (S > 1) ptx::ld_shared_cluster_v4(ptx::mapa_shared(own, first + k * STEP), w[k][0], w[k][1], w[k][2], w[k][3]);
            else ptx::ld_shared_cluster_v4(own, w[k][0], w[k][1], w[k][2], w[k][3]);
        }
#pragma unroll
        for (int k = 0; k < S; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] += __uint_as_float(w[k][j]);
        const long long at = static_cast<long long>(m0 + r) * p.ldc + n;
        if (p.out == OUT_F32) {
            float* dst = static_cast<float*>(p.C) + at;
            if (vec) {
                float4 o = make_float4(acc[0], acc[1], acc[2], acc[3]);
                if (p.accumulate) {
                    const float4 old = *reinterpret_cast<const float4*>(dst);
                    o = make_float4(old.x + o.x, old.y + o.y, old.z + o.z, old.w + o.w);
                }
                *reinterpret_cast<float4*>(dst) = o;
            } else {
                for (int j = 0; j < n_valid; ++j) dst[j] = p.accumulate ? dst[j] + acc[j] : acc[j];
            }
        } else {
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
            if (vec) {
                *reinterpret_cast<uint2*>(dst) = make_uint2(u[0], u[1]);
            } else {
                for (int j = 0; j < n_valid; ++j)
                    dst[j] = static_cast<uint16_t>((j & 1) ? (u[j >> 1] >> 16) : (u[j >> 1] & 0xffffu));
            }
        }
    }
}

// ==================================================================================== small and middling M
// Roles of the operands exchanged: the 128 rows of the instruction are rows of B (output columns), its N = TM columns are
// rows of A (tokens), 16 to 128 of them, so a few tokens cost a few columns of work instead of a 128-row tile of padding,
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
    static constexpr int kScaleOffset = kTiles;
    static constexpr int kScaleSlot = 1024;  // 128 rows of B, then up to 128 of A
    static constexpr int kBarOffset = kScaleOffset + kE8Slots * kScaleSlot;
    static constexpr int kBars = 2 * kStages + 2 * kE8Slots + 1;
    static constexpr int kMiscOffset = kBarOffset + kBars * 8;
    static constexpr int kTotal = kMiscOffset + 16;
    static constexpr int kDynamicBytes = kTotal + 1024;
    static constexpr uint32_t kScaleCol = TM < 32 ? 32 : TM;  // accumulator columns before the scales'
    static constexpr uint32_t kTmemCols = TM <= 32 ? 64 : (TM == 64 ? 128 : 256);
    static_assert(kScaleCol + kE8Slots * 8 <= kTmemCols, "tensor-memory columns");
};

template <int TM, int S>
__global__ void __launch_bounds__(kE8Threads)
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
    const uint32_t bar_sempty = bar_sfull + kE8Slots * 8;
    const uint32_t bar_tfull = bar_sempty + kE8Slots * 8;
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
        if (lane < kE8Slots) {
            ptx::mbar_init(bar_sfull + lane * 8, 2);
            ptx::mbar_init(bar_sempty + lane * 8, 1);
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
    // the scale warps (6: B's, 7: A's) send their first loads on their way
    const bool of_a = warp == 7;
    ScaleFeeder feeder;
    if (warp >= 6) {
        feeder.src = of_a ? ScaleSource{p.a_scale, p.a_rows, p.a_shift, p.M} : ScaleSource{p.b_scale, p.b_rows, p.b_shift, p.N};
        feeder.row0 = of_a ? m0 : n0;
        feeder.kb0 = kb0;
        feeder.kb1 = kb1;
        feeder.lane = lane;
        ptx::pdl_wait();
        feeder.start();
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
            uint32_t stage = 0, phase = 0, slot = 0, sphase = 0;
            bool ok = true;
            for (int kc = kb0; ok && kc < kb1; kc += 4) {
                if (!wait_bounded(bar_sfull + slot * 8, sphase, abort_flag, p.status, ROLE_MMA, -1 - kc)) {
                    ok = false;
                    break;
                }
                ptx::fence_proxy_async_smem();  // what the scale warps wrote, for the copy
                ptx::tc_fence_after();
                const uint32_t sb_tmem = tmem_base + L::kScaleCol + slot * 8, sa_tmem = sb_tmem + 4;
                ptx::tc_copy_scales(sb_tmem, ptx::make_scale_desc(smem_s + slot * L::kScaleSlot));
                ptx::tc_copy_scales(sa_tmem, ptx::make_scale_desc(smem_s + slot * L::kScaleSlot + 512));
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
                ptx::tc_commit(bar_sempty + slot * 8);
                if (++slot == kE8Slots) {
                    slot = 0;
                    sphase ^= 1u;
                }
            }
            if (ok) ptx::tc_commit(bar_tfull);
            else raise_peers();
        }
    } else if (warp >= 6) {
        // ------------------------------------------------------------ scales
        auto free = [&](int slot, uint32_t parity, int kc) {
            return wait_bounded(bar_sempty + slot * 8, parity, abort_flag, p.status, ROLE_SCALES, kc);
        };
        auto filled = [&](int slot) {
            if (lane == 0) ptx::mbar_arrive(bar_sfull + slot * 8);
        };
        if (!feeder.run(free, filled, smem_s + (of_a ? 512 : 0), L::kScaleSlot)) raise_peers();
    } else {
        // ------------------------------------------------------------ accumulator -> own shared memory, a token a row
        const int quad = warp & 3;
        if (wait_bounded(bar_tfull, 0u, abort_flag, p.status, ROLE_EPILOGUE, tile)) {
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
// share columns 192..255: the epilogue drains those first and hands them over (`ovl`), and the next tile's MMAs run under
// the rest of the drain. The first instruction of a tile waits only for a quarter of its predecessor's epilogue.
//
// Scales: the leader's instruction multiplies each CTA's 128 rows by that CTA's A scales, and all 256 columns by the B
// scales, which both CTAs hold in full; the scale warps of either CTA write their own shared memory and arrive on the
// leader's `sfull`; one tcgen05.cp of the leader copies in both CTAs.
//
// With 256 x 128 tiles (twice as many, for problems that have too few of the larger) both accumulators fit side by side.
template <int BN>
struct E8PairSmem {
    static constexpr int kScaleWarps = 1 + BN / 128;  // a warp for each 128 rows of scales
    static constexpr int kThreads = 32 * (7 + kScaleWarps);  // and one that hands their slots over
    static constexpr int kStages = BN == 256 ? 6 : 8;
    static constexpr int kAStage = 128 * 128;
    static constexpr int kBStage = (BN / 2) * 128;
    static constexpr int kTiles = kStages * (kAStage + kBStage);
    static constexpr int kOutOffset = kTiles;  // one 4 KB staging box per epilogue warp
    static constexpr int kScaleOffset = kOutOffset + 4 * 4096;
    static constexpr int kScaleSlot = 512 + (BN / 128) * 512;  // this CTA's 128 rows of A, all rows of B
    static constexpr int kBarOffset = kScaleOffset + kE8Slots * kScaleSlot;
    static constexpr int kBars = 2 * kStages + 3 * kE8Slots + 4;  // full, empty, sfull, sempty, sput, tfull[2], tfree[2]
    static constexpr int kMiscOffset = kBarOffset + kBars * 8;
    static constexpr int kTotal = kMiscOffset + 16;
    static constexpr int kDynamicBytes = kTotal + 1024;
    static constexpr uint32_t kAccStep = BN == 256 ? 192 : 128;  // first column of the second accumulator
    static constexpr uint32_t kScaleCol = BN == 256 ? 448 : 256;  // first column of the scales
    static constexpr uint32_t kScaleCols = 4 + BN / 32;  // columns of a chunk: A's, then B's
    static_assert(kAccStep + BN <= kScaleCol && kScaleCol + kE8Slots * kScaleCols <= 512, "tensor-memory columns");
};

template <int OUT, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(E8PairSmem<BN>::kThreads, 1)
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
    const uint32_t bar_sempty = bar_sfull + kE8Slots * 8;
    const uint32_t bar_sput = bar_sempty + kE8Slots * 8;  // this CTA's scale warps have written their part of a slot
    const uint32_t bar_tfull = bar_sput + kE8Slots * 8;
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
        for (int s = 0; s < kE8Slots; ++s) {
            ptx::mbar_init(bar_sfull + s * 8, 2);  // both CTAs
            ptx::mbar_init(bar_sput + s * 8, L::kScaleWarps);
            ptx::mbar_init(bar_sempty + s * 8, 1);
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
                    if (rank == 0) ptx::mbar_arrive_expect_tx(bar_full + stage * 8, 2 * (L::kAStage + L::kBStage));
                    const uint32_t leader_full = ptx::mapa_shared(bar_full + stage * 8, 0);
                    ptx::tma_load_2d_pair(smem_a + stage * L::kAStage, &tmap_a, leader_full, kb * 128, row_a);
                    ptx::tma_load_2d_pair(smem_b + stage * L::kBStage, &tmap_b, leader_full, kb * 128, row_b);
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
            uint32_t stage = 0, phase = 0, slot = 0, sphase = 0;
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
                    if (!wait_bounded_cluster(bar_sfull + slot * 8, sphase, abort_flag, p.status, ROLE_MMA, -2 - kc, peer_abort)) {
                        ok = false;
                        break;
                    }
                    ptx::tc_fence_after();
                    const uint32_t sa_tmem = tmem_base + L::kScaleCol + slot * L::kScaleCols, sb_tmem = sa_tmem + 4;
                    const uint32_t src = smem_s + slot * L::kScaleSlot;
                    ptx::tc_copy_scales_pair(sa_tmem, ptx::make_scale_desc(src));
#pragma unroll
                    for (int h = 0; h < BN / 128; ++h)
                        ptx::tc_copy_scales_pair(sb_tmem + 4 * h, ptx::make_scale_desc(src + 512 + 512 * h));
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
                    ptx::tc_commit_pair(bar_sempty + slot * 8, 3);
                    if (++slot == kE8Slots) {
                        slot = 0;
                        sphase ^= 1u;
                    }
                }
                if (ok) ptx::tc_commit_pair(bar_tfull + acc * 8, 3);
            }
        }
    } else if (warp == 6 + L::kScaleWarps) {
        // ------------------------------------------------------------ scale slots handed to the issuer (both CTAs). The
        // proxy fence waits for the memory operations of the warp that executes it, so it has a warp without loads
        if (ptx::elect_one()) {
            uint32_t slot = 0, phase = 0;
            const int chunks = (p.kb_total + 3) / 4;
            bool ok = true;
            for (int w = cluster_id; ok && w < total_work; w += n_clusters) {
                for (int c = 0; c < chunks; ++c) {
                    if (!wait_bounded(bar_sput + slot * 8, phase, abort_flag, p.status, ROLE_SCALES, -1 - c, peer_abort)) {
                        ok = false;
                        break;
                    }
                    ptx::fence_proxy_async_smem();
                    ptx::mbar_arrive_cluster(ptx::mapa_shared(bar_sfull + slot * 8, 0));
                    if (++slot == kE8Slots) {
                        slot = 0;
                        phase ^= 1u;
                    }
                }
            }
        }
    } else if (warp >= 6) {
        // ------------------------------------------------------------ scales (both CTAs): warp 6 A's, warp 7 B's first 128
        // rows, warp 8 (BN = 256) B's others; chunk c, counted through all tiles, goes to slot c % 4
        const bool of_a = warp == 6;
        const ScaleSource src = of_a ? ScaleSource{p.a_scale, p.a_rows, p.a_shift, p.M}
                                     : ScaleSource{p.b_scale, p.b_rows, p.b_shift, p.N};
        const uint32_t slots = smem_s + static_cast<uint32_t>(warp - 6) * 512u;
        struct Place {
            int w, kc, row0;
        };
        auto tile_row = [&](Place& c) {
            if (c.w >= total_work) return;
            int m_blk, n_blk;
            e8_decode(c.w, p, m_blk, n_blk);
            c.row0 = of_a ? (m_blk * 2 + static_cast<int>(rank)) * 128 : n_blk * BN + (warp - 7) * 128;
        };
        auto advance = [&](Place& c) {
            c.kc += 4;
            if (c.kc >= p.kb_total) {
                c.kc = 0;
                c.w += n_clusters;
                tile_row(c);
            }
        };
        Place put = {cluster_id, 0, 0};
        tile_row(put);
        Place ahead = put;
        ScaleWords buf[kE8Ahead];
        static_assert(kE8Ahead == kE8Slots, "one buffer a slot");
#pragma unroll
        for (int i = 0; i < kE8Ahead; ++i) {
            if (ahead.w < total_work) {
                load_scales(buf[i], src, ahead.row0, ahead.kc, min(4, p.kb_total - ahead.kc), lane);
                advance(ahead);
            }
        }
        uint32_t parity = 1;  // the first pass over the slots finds them free
        bool ok = true;
        while (ok && put.w < total_work) {
#pragma unroll
            for (int i = 0; i < kE8Ahead; ++i) {
                if (put.w >= total_work) break;
                if (!wait_bounded(bar_sempty + i * 8, parity, abort_flag, p.status, ROLE_SCALES, put.kc, peer_abort)) {
                    ok = false;
                    break;
                }
                put_scales(slots + i * L::kScaleSlot, buf[i], src, put.row0, put.kc, min(4, p.kb_total - put.kc), lane);
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(bar_sput + i * 8);
                advance(put);
                if (ahead.w < total_work) {
                    load_scales(buf[i], src, ahead.row0, ahead.kc, min(4, p.kb_total - ahead.kc), lane);
                    advance(ahead);
                }
            }
            parity ^= 1u;
        }
    } else {
        // ------------------------------------------------------------ epilogue (both CTAs)
        const int quad = warp & 3;
        const uint32_t stage_base = smem_base + L::kOutOffset + quad * 4096u;
        uint32_t it = 0;
        for (int w = cluster_id; w < total_work; w += n_clusters, ++it) {
            int m_blk, n_blk;
            e8_decode(w, p, m_blk, n_blk);
            const uint32_t acc = it & 1u;
            if (!wait_bounded(bar_tfull + acc * 8, (it >> 1) & 1u, abort_flag, p.status, ROLE_EPILOGUE, w, peer_abort)) break;
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
                    if (lane == 0) ptx::mbar_arrive_cluster(ptx::mapa_shared(bar_tfree + (kOverlap ? 0 : acc * 8), 0));
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
                if (p.c_tma_ok) {
                    // the box is free once the store before has read it
                    if (ptx::elect_one()) ptx::tma_store_wait_read<0>();
                    __syncwarp();
                    const uint32_t row_addr = stage_base + static_cast<uint32_t>(lane) * 128u;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        ptx::st_shared_v4(row_addr + static_cast<uint32_t>((j ^ (lane & 7)) * 16), u[4 * j], u[4 * j + 1],
                                          u[4 * j + 2], u[4 * j + 3]);
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    if (ptx::elect_one()) {
                        if (OUT == OUT_F32 && p.accumulate) ptx::tma_add_3d(&tmap_c, stage_base, n0, row0, 0);
                        else ptx::tma_store_3d(&tmap_c, stage_base, n0, row0, 0);
                        ptx::tma_store_commit();
                    }
                } else if (row0 + lane < p.M) {
                    uint8_t* dst = static_cast<uint8_t*>(p.C) + (static_cast<long long>(row0 + lane) * p.ldc + n0) * OB;
#pragma unroll
                    for (int j = 0; j < CW; ++j) {
                        if (n0 + j < p.N) {
                            if constexpr (OUT == OUT_F32) {
                                float* f = reinterpret_cast<float*>(dst) + j;
                                *f = p.accumulate ? *f + __uint_as_float(u[j]) : __uint_as_float(u[j]);
                            } else {
                                reinterpret_cast<uint16_t*>(dst)[j] =
                                    static_cast<uint16_t>((j & 1) ? (u[j >> 1] >> 16) : (u[j >> 1] & 0xffffu));
                            }
                        }
                    }
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
    static constexpr int kScaleSlot = 1024;  // this CTA's 128 rows of A, 128 rows of B
    static constexpr int kBarOffset = kScaleOffset + kE8Slots * kScaleSlot;
    static constexpr int kBars = 2 * kStages + 3 * kE8Slots + 1;
    static constexpr int kMiscOffset = kBarOffset + kBars * 8;
    static constexpr int kTotal = kMiscOffset + 16;
    static constexpr int kDynamicBytes = kTotal + 1024;
    static constexpr int kThreads = kE8Threads + 32;  // and a warp that hands the scale slots over
    static constexpr uint32_t kScaleCol = 128;
    static constexpr uint32_t kTmemCols = 256;
};

template <int S>
__global__ void __launch_bounds__(E8PairKSmem::kThreads, 1)
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
    const uint32_t bar_sempty = bar_sfull + kE8Slots * 8;
    const uint32_t bar_sput = bar_sempty + kE8Slots * 8;
    const uint32_t bar_tfull = bar_sput + kE8Slots * 8;
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
        for (int s = 0; s < kE8Slots; ++s) {
            ptx::mbar_init(bar_sfull + s * 8, 2);  // both CTAs of the pair
            ptx::mbar_init(bar_sput + s * 8, 2);   // A's and B's scale warp
            ptx::mbar_init(bar_sempty + s * 8, 1);
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
    ScaleFeeder feeder;
    if (warp == 6 || warp == 7) {
        feeder.src = of_a ? ScaleSource{p.a_scale, p.a_rows, p.a_shift, p.M} : ScaleSource{p.b_scale, p.b_rows, p.b_shift, p.N};
        feeder.row0 = of_a ? m0 : n0;
        feeder.kb0 = kb0;
        feeder.kb1 = kb1;
        feeder.lane = lane;
        ptx::pdl_wait();
        feeder.start();
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
                if (rank == 0) ptx::mbar_arrive_expect_tx(bar_full + stage * 8, 2 * (L::kAStage + L::kBStage));
                const uint32_t leader_full = ptx::mapa_shared(bar_full + stage * 8, leader);
                ptx::tma_load_2d_pair(smem_a + stage * L::kAStage, &tmap_a, leader_full, kb * 128, m0);
                ptx::tma_load_2d_pair(smem_b + stage * L::kBStage, &tmap_b, leader_full, kb * 128,
                                      n0 + static_cast<int>(rank) * 64);
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
            uint32_t stage = 0, phase = 0, slot = 0, sphase = 0;
            bool ok = true;
            for (int kc = kb0; ok && kc < kb1; kc += 4) {
                if (!wait_bounded_cluster(bar_sfull + slot * 8, sphase, abort_flag, p.status, ROLE_MMA, -1 - kc, 0)) {
                    ok = false;
                    break;
                }
                ptx::tc_fence_after();
                const uint32_t sa_tmem = tmem_base + L::kScaleCol + slot * 8, sb_tmem = sa_tmem + 4;
                ptx::tc_copy_scales_pair(sa_tmem, ptx::make_scale_desc(smem_s + slot * L::kScaleSlot));
                ptx::tc_copy_scales_pair(sb_tmem, ptx::make_scale_desc(smem_s + slot * L::kScaleSlot + 512));
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
                ptx::tc_commit_pair(bar_sempty + slot * 8, both);
                if (++slot == kE8Slots) {
                    slot = 0;
                    sphase ^= 1u;
                }
            }
            if (ok) ptx::tc_commit_pair(bar_tfull, both);
            else raise_peers();
        }
    } else if (warp == 8) {
        // ------------------------------------------------------------ scale slots handed to the issuer (every CTA)
        if (ptx::elect_one()) {
            uint32_t slot = 0, phase = 0;
            for (int kc = kb0; kc < kb1; kc += 4) {
                if (!wait_bounded(bar_sput + slot * 8, phase, abort_flag, p.status, ROLE_SCALES, -1 - kc)) {
                    raise_peers();
                    break;
                }
                ptx::fence_proxy_async_smem();
                ptx::mbar_arrive_cluster(ptx::mapa_shared(bar_sfull + slot * 8, leader));
                if (++slot == kE8Slots) {
                    slot = 0;
                    phase ^= 1u;
                }
            }
        }
    } else if (warp >= 6) {
        // ------------------------------------------------------------ scales (every CTA)
        auto free = [&](int slot, uint32_t parity, int kc) {
            return wait_bounded(bar_sempty + slot * 8, parity, abort_flag, p.status, ROLE_SCALES, kc);
        };
        auto filled = [&](int slot) {
            if (lane == 0) ptx::mbar_arrive(bar_sput + slot * 8);
        };
        if (!feeder.run(free, filled, smem_s + (of_a ? 0 : 512), L::kScaleSlot)) raise_peers();
    } else {
        // ------------------------------------------------------------ accumulator -> own shared memory
        const int quad = warp & 3;
        if (wait_bounded(bar_tfull, 0u, abort_flag, p.status, ROLE_EPILOGUE, m_blk)) {
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
    if (*abort_flag == 0 && m0 < p.M) sum_and_store<S, 2, L::kThreads / 32>(p, smem_base, rank, slice, m0, min(128, p.M - m0), n0);

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

// tokens_per_tile: 16, 32, 64 or 128; slices: 1, 2, 4 or 8, at most kb_total (gemm_e8m0.cu).
cudaError_t launch_e8m0_small(int tokens_per_tile, int slices, const CUtensorMap& ta, const CUtensorMap& tb,
                              const E8m0Params& p, cudaStream_t stream);
// tile_n: 256 or 128 (slices == 1: persistent), 128 with slices 2 or 4.
cudaError_t launch_e8m0_pair(int tile_n, int slices, const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc,
                             const E8m0Params& p, int clusters, cudaStream_t stream);

}  // namespace qgemm
