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
    int a_words, b_words;  // four rows' scales can be loaded as a word
    int out;               // OUT_F32 / OUT_BF16 / OUT_F16
    int accumulate;        // fp32 C: add to what it holds
    int c_tma_ok, c_vec_ok;
    int* status;
};

constexpr int kE8Slots = 4;  // chunks of scales in flight
constexpr int kE8Threads = 256;  // producer, MMA issuer, four epilogue warps, two scale warps
constexpr int kE8PairThreads = 320;  // four scale warps
enum : int { ROLE_SCALES = 4 };

// One operand's scales on their way from global to shared memory.
struct ScaleSource {
    const uint8_t* scale;
    long long ld;
    int shift, rows;
    int words;  // the scales of four neighbouring rows can be loaded as a word
};

// A lane's part of a chunk (K blocks kb0 .. kb0 + n, n <= 4) of 128 rows, as it was loaded: of rows 4 lane .. + 4, a word a
// K block (`by_fours`), or of rows 32 j + lane, a byte a row and block. load_scales uses nothing that it loads, so a caller
// that loads a chunk ahead waits for memory only where it packs. (With conditional loads, each waited for in turn, a chunk
// of a row-scaled 256-row B took 4 us, and the product 404 us instead of 194 at 4096 x 7168 x 7168.)
struct ScaleWords {
    uint32_t v[16];
    int row0, n;
    bool by_fours;
};
__device__ __forceinline__ void load_scales(ScaleWords& out, const ScaleSource& s, int row0, int kb0, int n, int lane) {
    out.row0 = row0;
    out.n = n;
    out.by_fours = s.words != 0 && s.shift == 0 && row0 + 128 <= s.rows;
    const uint8_t* at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) at[i] = s.scale + (kb0 + min(i, n - 1)) * s.ld;
    if (out.by_fours) {
#pragma unroll
        for (int i = 0; i < 4; ++i) out.v[i] = __ldg(reinterpret_cast<const uint32_t*>(at[i] + row0) + lane);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int row = min(row0 + 32 * j + lane, s.rows - 1) >> s.shift;
#pragma unroll
            for (int i = 0; i < 4; ++i) out.v[4 * j + i] = __ldg(at[i] + row);
        }
    }
}
// Into the 512 bytes that tc_copy_scales reads: row r's four K blocks as a word at (r % 32) * 16 + (r / 32) * 4. Rows and
// blocks that do not exist get the scale 1.
__device__ __forceinline__ void put_scales(uint32_t dst, const ScaleWords& c, int rows, int lane) {
    if (c.by_fours) {
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = i < c.n ? c.v[i] : 0x7f7f7f7fu;
        const uint32_t x = __byte_perm(v[0], v[1], 0x5140), y = __byte_perm(v[2], v[3], 0x5140);
        const uint32_t z = __byte_perm(v[0], v[1], 0x7362), t = __byte_perm(v[2], v[3], 0x7362);
        const uint32_t w[4] = {__byte_perm(x, y, 0x5410), __byte_perm(x, y, 0x7632), __byte_perm(z, t, 0x5410),
                               __byte_perm(z, t, 0x7632)};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t r = static_cast<uint32_t>(4 * lane + j);
            ptx::st_shared_u32(dst + (r & 31u) * 16u + (r >> 5) * 4u, w[j]);
        }
    } else {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) b[i] = i < c.n ? c.v[4 * j + i] : 127u;
            w[j] = c.row0 + 32 * j + lane < rows ? b[0] | (b[1] << 8) | (b[2] << 16) | (b[3] << 24) : 0x7f7f7f7fu;
        }
        ptx::st_shared_v4(dst + lane * 16, w[0], w[1], w[2], w[3]);
    }
}

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
    static constexpr int kRowWords = 128 + 4;  // a token's 128 partial sums, padded
    static_assert(TM * kRowWords * 4 <= kTiles, "the partial tile lies over the ring");
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
    const ScaleSource src = of_a ? ScaleSource{p.a_scale, p.a_rows, p.a_shift, p.M, p.a_words}
                                 : ScaleSource{p.b_scale, p.b_rows, p.b_shift, p.N, p.b_words};
    ScaleWords next;
    if (warp >= 6) {
        ptx::pdl_wait();
        load_scales(next, src, of_a ? m0 : n0, kb0, min(4, kb1 - kb0), lane);
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
        // ------------------------------------------------------------ scales, loaded a chunk ahead
        uint32_t slot = 0, sphase = 1;  // the first pass over the slots finds them free
        for (int kc = kb0; kc < kb1; kc += 4) {
            const ScaleWords now = next;
            if (kc + 4 < kb1) load_scales(next, src, of_a ? m0 : n0, kc + 4, min(4, kb1 - kc - 4), lane);
            if (!wait_bounded(bar_sempty + slot * 8, sphase, abort_flag, p.status, ROLE_SCALES, kc)) {
                raise_peers();
                break;
            }
            put_scales(smem_s + slot * L::kScaleSlot + (of_a ? 512 : 0), now, src.rows, lane);
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(bar_sfull + slot * 8);
            if (++slot == kE8Slots) {
                slot = 0;
                sphase ^= 1u;
            }
        }
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
                    if (c + j < tokens) col[(c + j) * L::kRowWords] = __uint_as_float(v[j]);
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
    if (*abort_flag == 0) {
        // a warp takes a token, a lane four output columns; the cluster's CTAs share the tokens out
        const int tokens = min(TM, p.M - m0);
        const int per = (tokens + S - 1) / S;
        const int t1 = min(tokens, (static_cast<int>(rank) + 1) * per);
        const int n = n0 + lane * 4;
        const int n_valid = min(4, p.N - n);
        if (n_valid > 0) {
            for (int t = static_cast<int>(rank) * per + warp; t < t1; t += kE8Threads / 32) {
                const uint32_t own = smem_base + static_cast<uint32_t>((t * L::kRowWords + lane * 4) * 4);
                float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                if constexpr (S > 1) {
                    uint32_t w[S][4];
#pragma unroll
                    for (uint32_t k = 0; k < static_cast<uint32_t>(S); ++k)
                        ptx::ld_shared_cluster_v4(ptx::mapa_shared(own, k), w[k][0], w[k][1], w[k][2], w[k][3]);
#pragma unroll
                    for (int k = 0; k < S; ++k)
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[j] += __uint_as_float(w[k][j]);
                } else {
                    const float4 v = *reinterpret_cast<const float4*>(smem + (own - smem_base));
                    acc[0] = v.x; acc[1] = v.y; acc[2] = v.z; acc[3] = v.w;
                }
                const long long at = static_cast<long long>(m0 + t) * p.ldc + n;
                const bool vec = p.c_vec_ok != 0 && n_valid == 4;
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
    }

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
struct E8PairSmem {
    static constexpr int kBN = 256;
    static constexpr int kStages = 6;
    static constexpr int kAStage = 128 * 128;
    static constexpr int kBStage = (kBN / 2) * 128;
    static constexpr int kTiles = kStages * (kAStage + kBStage);
    static constexpr int kOutOffset = kTiles;  // one 4 KB staging box per epilogue warp
    static constexpr int kScaleOffset = kOutOffset + 4 * 4096;
    static constexpr int kScaleSlot = 512 + (kBN / 128) * 512;  // this CTA's 128 rows of A, all rows of B
    static constexpr int kBarOffset = kScaleOffset + kE8Slots * kScaleSlot;
    static constexpr int kBars = 2 * kStages + 2 * kE8Slots + 3;  // full, empty, sfull, sempty, tfull[2], ovl
    static constexpr int kMiscOffset = kBarOffset + kBars * 8;
    static constexpr int kTotal = kMiscOffset + 16;
    static constexpr int kDynamicBytes = kTotal + 1024;
    static constexpr uint32_t kAccStep = 192;   // first column of the second accumulator
    static constexpr uint32_t kScaleCol = 448;  // first column of the scales
    static constexpr uint32_t kScaleCols = 4 + kBN / 32;  // columns of a chunk: A's, then B's
    static_assert(kAccStep + kBN <= kScaleCol && kScaleCol + kE8Slots * kScaleCols <= 512, "tensor-memory columns");
};

template <int OUT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kE8PairThreads, 1)
gemm_e8m0_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                      const __grid_constant__ CUtensorMap tmap_c, const E8m0Params p) {
    using L = E8PairSmem;
    constexpr int STAGES = L::kStages, BN = L::kBN;
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
    const uint32_t bar_tfull = bar_sempty + kE8Slots * 8;
    const uint32_t bar_ovl = bar_tfull + 2 * 8;
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
            ptx::mbar_init(bar_sfull + s * 8, 4);  // A's and B's scale warp of each CTA
            ptx::mbar_init(bar_sempty + s * 8, 1);
        }
        ptx::mbar_init(bar_tfull, 1);
        ptx::mbar_init(bar_tfull + 8, 1);
        ptx::mbar_init(bar_ovl, 8);  // four epilogue warps of each CTA
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
                // the previous tile's share of the common columns is out (and with it everything of the tile before)
                if (it > 0 && !wait_bounded(bar_ovl, (it - 1) & 1u, abort_flag, p.status, ROLE_MMA, -1, peer_abort)) break;
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
    } else if (warp >= 6) {
        // ------------------------------------------------------------ scales (both CTAs): warps 6 and 7 A's, 8 and 9 B's, the
        // even and the odd chunks (counted through all tiles) of each, loaded one ahead: four chunks of an operand are in
        // flight or in their slots, which covers the latency of a loaded L2
        const bool of_a = warp < 8;
        const ScaleSource src = of_a ? ScaleSource{p.a_scale, p.a_rows, p.a_shift, p.M, p.a_words}
                                     : ScaleSource{p.b_scale, p.b_rows, p.b_shift, p.N, p.b_words};
        int w = cluster_id, kc = 0, row0 = 0;  // the chunk to load next
        auto place = [&]() {
            if (w >= total_work) return;
            int m_blk, n_blk;
            e8_decode(w, p, m_blk, n_blk);
            row0 = of_a ? (m_blk * 2 + static_cast<int>(rank)) * 128 : n_blk * BN;
        };
        auto advance = [&]() {
            kc += 4;
            if (kc >= p.kb_total) {
                kc = 0;
                w += n_clusters;
                place();
            }
        };
        ScaleWords lo, hi;
        auto load = [&]() {
            const int n = min(4, p.kb_total - kc);
            load_scales(lo, src, row0, kc, n, lane);
            if (!of_a) load_scales(hi, src, row0 + 128, kc, n, lane);
        };
        place();
        uint32_t slot = static_cast<uint32_t>(warp) & 1u, sphase = 1;  // the first pass over the slots finds them free
        if (slot != 0) advance();
        if (w < total_work) load();
        while (w < total_work) {
            const ScaleWords lo_now = lo, hi_now = hi;
            const int kc_now = kc;
            advance();
            if (w < total_work) advance();
            if (w < total_work) load();
            if (!wait_bounded(bar_sempty + slot * 8, sphase, abort_flag, p.status, ROLE_SCALES, kc_now, peer_abort)) break;
            const uint32_t dst = smem_s + slot * L::kScaleSlot;
            put_scales(of_a ? dst : dst + 512, lo_now, src.rows, lane);
            if (!of_a) put_scales(dst + 1024, hi_now, src.rows, lane);
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive_cluster(ptx::mapa_shared(bar_sfull + slot * 8, 0));
            slot += 2;
            if (slot >= kE8Slots) {
                slot -= kE8Slots;
                sphase ^= 1u;
            }
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
            const int first = acc == 0 ? static_cast<int>(L::kAccStep) / CW : 0;
            constexpr int kShared = (BN - static_cast<int>(L::kAccStep)) / CW;  // boxes they make up
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
                    if (lane == 0) ptx::mbar_arrive_cluster(ptx::mapa_shared(bar_ovl, 0));
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

// tokens_per_tile: 16, 32, 64 or 128; slices: 1, 2, 4 or 8, at most kb_total (gemm_e8m0.cu).
cudaError_t launch_e8m0_small(int tokens_per_tile, int slices, const CUtensorMap& ta, const CUtensorMap& tb,
                              const E8m0Params& p, cudaStream_t stream);
cudaError_t launch_e8m0_pair(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, const E8m0Params& p,
                             int clusters, cudaStream_t stream);

}  // namespace qgemm
