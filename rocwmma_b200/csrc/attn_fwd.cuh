// Forward attention on tcgen05.
//
// A CTA owns 256 queries of one head as two tiles of 128 and walks the key tiles that either of them sees.  (Where the grid is
// small it owns one tile of queries, whose even and odd key tiles take the places of the two: PER = 1.)  Per tile
//   S = Q K^T (tensor cores, fp32 in tensor memory) -> softmax warps: running maximum and sum, P = 2^(x - m) in 16 bits over S
//   -> O += P V (tensor cores, P from tensor memory).
// The two tiles take turns: while the tensor cores work on one, 128 threads (one to a query) do the softmax of the other.
// The running maximum of a row is only moved when a score passes it by more than 2^14 (RESCALE_STEP), so O is rescaled rarely and
// a tile's weights mostly take one pass over its scores.  Key tiles come from the last to the first: under a causal mask the
// nearest ones, which a distance bias makes the largest, are first (2 x 16 heads of 4096 x 128 with slopes: 173 us; 270 the other
// way round, where the maximum moves in every tile, at that step).
// Bound: a pair of tiles takes 1.9 us at a head of 128, 1.55 us of which remain without any softmax: M = 128, N = 128 products
// read shared memory at its full 128 bytes a cycle next to the copies' writes, and 2 x 2 of them are 1.1 us by the tensor cores'
// rate.  Measured, bf16: 1 x 16 heads of 16384 x 128 1.1-1.2 PFLOP/s, 2 x 16 heads of 4096 x 128 0.28 ms (990 TFLOP/s), causal
// 0.15 ms (930), causal with cap 0.19-0.21 ms, with slopes 0.15 ms, 5 packed documents of 8192 tokens 0.11 ms.  What was tried and not kept: announcing
// P in halves (931 instead of 1064 TFLOP/s then), part of the exponentials as polynomials (892-938).
#pragma once
#include "attn_tc05.cuh"

namespace b200wmma
{
    namespace attn
    {
        constexpr uint32_t FWD_THREADS  = 320; // warps 0-3: softmax of tile 0, 4-7: of tile 1, 8: TMA, 9: MMA

        template <uint32_t HD>
        struct FwdSmem
        {
            static constexpr uint32_t TILE_BYTES = HD / 64 * BOX_BYTES;
            static constexpr uint32_t STAGES     = HD == 128 ? 4 : 8; // key and value tiles in turn
            static constexpr uint32_t Q          = 0;
            static constexpr uint32_t KV         = Q + 2 * TILE_BYTES;
            static constexpr uint32_t LIST       = KV + STAGES * TILE_BYTES; // SEG words
            static constexpr uint32_t RAW        = LIST + SEG * 4; // SEG bytes of flags before they are listed
            static constexpr uint32_t STATS      = RAW + SEG; // 2 x 128 maxima, 2 x 128 sums
            static constexpr uint32_t BARS       = STATS + 4 * TILE * 4;
            static constexpr uint32_t Q_FULL = BARS, KV_FULL = Q_FULL + 8, KV_EMPTY = KV_FULL + 8 * STAGES, S_FULL = KV_EMPTY + 8 * STAGES,
                                      P_FULL = S_FULL + 16, O_DONE = P_FULL + 16;
            static constexpr uint32_t MISC  = O_DONE + 16; // tensor memory address, abort flag, list length
            static constexpr uint32_t TOTAL = MISC + 16;
            static constexpr uint32_t BYTES = TOTAL + 1024;
        };

        enum FwdRole : uint32_t
        {
            FWD_PRODUCER = 0x31,
            FWD_MMA      = 0x32,
            FWD_SOFTMAX  = 0x33
        };

        template <typename T, uint32_t HD, bool CAP, bool BIAS, bool PLAIN, uint32_t PER>
        __global__ void __launch_bounds__(FWD_THREADS, 1)
            fwd_tc05_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                            const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_o,
                            const __grid_constant__ Params p,
                            float* __restrict__ lse, const DocTile* __restrict__ doc_tiles_q, const DocTile* __restrict__ doc_tiles_kv,
                            uint32_t q_blocks, unsigned* status)
        {
            using L = FwdSmem<HD>;
            extern __shared__ uint8_t smem_raw[];
            const uint32_t            base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
            uint8_t*                  smem = smem_raw + (base - ptx::smem_u32(smem_raw));
            uint32_t*                 list = reinterpret_cast<uint32_t*>(smem + L::LIST);
            uint8_t*                  raw  = smem + L::RAW;
            uint32_t*                 misc = reinterpret_cast<uint32_t*>(smem + L::MISC);
            volatile uint32_t*        cta_abort = misc + 1;

            const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
            // the last queries first: under a causal mask they take longest
            const uint32_t bh = blockIdx.x % (p.batch * p.heads_q), q_block = q_blocks - 1 - blockIdx.x / (p.batch * p.heads_q);
            const uint32_t h = bh % p.heads_q, b = bh / p.heads_q, g = h / (p.heads_q / p.heads_kv);
            const uint32_t row0 = q_block * PER * TILE, q_tiles = (p.len_q + TILE - 1) / TILE, kv_tiles = (p.len_kv + TILE - 1) / TILE;
            const int32_t  prefix = p.prefix ? p.prefix[b] : 0;
            const bool     docs   = p.doc_q != nullptr;
            constexpr uint32_t ahead = PER == 2 ? 1 : 2; // key tiles whose scores are asked for before the weights of one are there

            if(threadIdx.x == 0)
            {
                ptx::prefetch_tensormap(&map_q);
                ptx::prefetch_tensormap(&map_k);
                ptx::prefetch_tensormap(&map_v);
                ptx::mbar_init(base + L::Q_FULL, 1);
                for(uint32_t s = 0; s < L::STAGES; ++s)
                {
                    ptx::mbar_init(base + L::KV_FULL + 8 * s, 1);
                    ptx::mbar_init(base + L::KV_EMPTY + 8 * s, 1);
                }
                for(uint32_t t = 0; t < 2; ++t)
                {
                    ptx::mbar_init(base + L::S_FULL + 8 * t, 1);
                    ptx::mbar_init(base + L::P_FULL + 8 * t, 4); // warps
                    ptx::mbar_init(base + L::O_DONE + 8 * t, 1);
                }
                *cta_abort = 0u;
                ptx::fence_barrier_init();
                ptx::fence_proxy_async_smem();
            }
            if(warp == 9)
            {
                ptx::tmem_alloc(base + L::MISC, 512);
                ptx::tmem_relinquish();
            }
            ptx::tc_fence_before_sync();
            __syncthreads();
            ptx::tc_fence_after_sync();
            const uint32_t tmem = misc[0];
            const uint32_t s_tmem[2] = {tmem, tmem + TILE}, o_tmem[2] = {tmem + 2 * TILE, tmem + 2 * TILE + HD};

            // roles keep their place in the rings from one segment of the key tiles to the next
            uint32_t   c = 0; // producer, MMA: place in the ring
            uint32_t   done[2] = {0, 0}; // MMA: S tiles so far of each query tile
            const uint32_t t   = warp >> 2; // softmax: this thread's query tile
            const uint32_t row = row0 + (PER == 2 ? t * TILE : 0) + (threadIdx.x & 127u), quad = warp & 3u;
            const int32_t  at  = int32_t(row) + p.off;
            uint32_t       n_s = 0; // softmax: S tiles so far
            float          m = -INFINITY, l = 0.0f;
            bool           ok = true, q_here = false, steep = false, wild = false;
            const ScoreConst sc = score_const(p, h);
            const int32_t    doc = (docs && row < p.len_q) ? p.doc_q[size_t(b) * p.len_q + row] : 0;
            // keys [0, lim) of this row are visible as far as causality and lengths go
            const int32_t lim = (row >= p.len_q || doc < 0) ? 0 : (p.causal ? min(max(at + 1, prefix), int32_t(p.len_kv)) : int32_t(p.len_kv));

            // TILE_NEED, TILE_MASK of the e-th key tile (of `entries`, from the last) for place u
            const auto flags = [&](uint32_t entries, uint32_t e, uint32_t u) {
                const uint32_t f = list[entries - 1 - e] >> 24;
                return PER == 2 ? f >> (2 * u) : ((e ^ u) & 1u) ? 0u : f;
            };
            for(uint32_t seg = (kv_tiles - 1) / SEG * SEG;; seg -= SEG)
            {
                // the key tiles of this segment that a query of the CTA sees, with the flags of both query tiles
                const uint32_t entries = list_tiles<FWD_THREADS>(seg, min(SEG, kv_tiles - seg), list, raw, misc + 2, [&](uint32_t tile) {
                    uint32_t       f  = 0;
                    const DocTile* dk = docs ? doc_tiles_kv + size_t(b) * kv_tiles + tile : nullptr;
                    for(uint32_t u = 0; u < PER; ++u)
                    {
                        const uint32_t r0 = row0 + u * TILE;
                        if(r0 < p.len_q)
                            f |= tile_flags(p, r0, tile * TILE, prefix, docs ? doc_tiles_q + size_t(b) * q_tiles + r0 / TILE : nullptr, dk)
                                 << (2 * u);
                    }
                    return f && docs && dk->neg ? f | TILE_DIRTY : f;
                });

                if(warp < 8)
                    q_here |= entries != 0;
                if(warp == 8)
                {
                    // ------------------------------ TMA producer ------------------------------
                    if(lane == 0 && ok && entries)
                    {
                        if(!q_here)
                        {
                            const uint32_t n = PER == 2 && row0 + TILE < p.len_q ? 2u : 1u;
                            ptx::mbar_arrive_expect_tx(base + L::Q_FULL, n * L::TILE_BYTES);
                            for(uint32_t u = 0; u < n; ++u)
                                load_tile<HD>(base + L::Q + u * L::TILE_BYTES, &map_q, row0 + u * TILE, h, b, base + L::Q_FULL);
                            q_here = true;
                        }
                        const auto load = [&](const CUtensorMap* map, uint32_t e) {
                            const uint32_t st = c % L::STAGES, ph = (c / L::STAGES) & 1u;
                            ok = ok
                                 && ptx::mbar_wait_bounded(base + L::KV_EMPTY + 8 * st, ph ^ 1u, cta_abort, status,
                                                           FWD_PRODUCER << 24 | (blockIdx.x & 0xFFFFFFu), tc05::WAIT_TIMEOUT_NS);
                            if(!ok)
                                return;
                            ++c;
                            ptx::mbar_arrive_expect_tx(base + L::KV_FULL + 8 * st, L::TILE_BYTES);
                            load_tile<HD>(base + L::KV + st * L::TILE_BYTES, map, (list[entries - 1 - e] & 0xFFFFFFu) * TILE, g, b,
                                          base + L::KV_FULL + 8 * st);
                        };
                        // in the order of their use: the keys of the first tiles, then values and the keys `ahead` tiles on
                        for(uint32_t e = 0; e < min(ahead, entries); ++e)
                            load(&map_k, e);
                        for(uint32_t e = 0; ok && e < entries; ++e)
                        {
                            load(&map_v, e);
                            if(e + ahead < entries)
                                load(&map_k, e + ahead);
                        }
                    }
                    __syncwarp();
                }
                else if(warp == 9)
                {
                    // ------------------------------- MMA issuer -------------------------------
                    // The whole warp waits (rows of padding are cleared by all lanes); lane 0 issues.
                    const auto wait = [&](uint32_t bar, uint32_t parity, uint32_t what) {
                        ok = ok
                             && wait_bounded_warp(bar, parity, cta_abort, status,
                                                            FWD_MMA << 24 | what << 20 | (blockIdx.x & 0xFFFFFu));
                        ptx::tc_fence_after_sync();
                        return ok;
                    };
                    const auto arrive_kv = [&](uint32_t n, uint32_t e) { // waits for stage n, makes it fit for a product
                        const uint32_t st = n % L::STAGES;
                        if(!wait(base + L::KV_FULL + 8 * st, (n / L::STAGES) & 1u, 1))
                            return false;
                        if(list[entries - 1 - e] >> 24 & TILE_DIRTY)
                        {
                            const uint32_t c0 = (list[entries - 1 - e] & 0xFFFFFFu) * TILE;
                            clear_padding<HD>(smem + L::KV + st * L::TILE_BYTES, p.doc_kv + size_t(b) * p.len_kv + c0, min(TILE, p.len_kv - c0),
                                              lane);
                        }
                        return true;
                    };
                    const auto scores = [&](uint32_t u, uint32_t e, uint32_t n) { // S of query tile u
                        if((flags(entries, e, u) & TILE_NEED) && elect_one())
                        {
                            mma_over_head<T, HD>(s_tmem[u], base + L::Q + (PER == 2 ? u : 0) * L::TILE_BYTES,
                                                 base + L::KV + (n % L::STAGES) * L::TILE_BYTES);
                            ptx::tc_commit(base + L::S_FULL + 8 * u);
                        }
                    };
                    const auto free_stage = [&](uint32_t n) {
                        if(elect_one())
                            ptx::tc_commit(base + L::KV_EMPTY + 8 * (n % L::STAGES));
                    };
                    if(entries && ok)
                    {
                        if(!q_here)
                            wait(base + L::Q_FULL, 0, 0);
                        q_here = true;
                        for(uint32_t e = 0; ok && e < min(ahead, entries); ++e)
                            if(arrive_kv(c, e))
                            {
                                scores(0, e, c);
                                scores(1, e, c);
                                free_stage(c++);
                            }
                        for(uint32_t e = 0; ok && e < entries; ++e)
                        {
                            if(!arrive_kv(c, e))
                                break;
                            const bool more = e + ahead < entries;
                            if(more && !arrive_kv(c + 1, e + ahead))
                                break;
                            for(uint32_t u = 0; ok && u < 2; ++u)
                            {
                                if(flags(entries, e, u) & TILE_NEED)
                                {
                                    if(!wait(base + L::P_FULL + 8 * u, done[u] & 1u, 2 + u))
                                        break;
                                    if(elect_one())
                                    {
                                        mma_over_tokens<T, HD>(o_tmem[u], s_tmem[u], base + L::KV + (c % L::STAGES) * L::TILE_BYTES,
                                                               done[u] != 0);
                                        ptx::tc_commit(base + L::O_DONE + 8 * u);
                                    }
                                    ++done[u];
                                }
                                if(more)
                                    scores(u, e + ahead, c + 1);
                            }
                            if(!ok)
                                break;
                            free_stage(c++);
                            if(more)
                                free_stage(c++);
                        }
                    }
                    __syncwarp();
                }
                else
                {
                    // --------------------------------- softmax --------------------------------
                    const uint32_t lane_tmem = (quad * 32u) << 16;
                    for(uint32_t e = 0; ok && e < entries; ++e)
                    {
                        const uint32_t f = flags(entries, e, t);
                        if(!(f & TILE_NEED))
                            continue;
                        const uint32_t c0 = (list[entries - 1 - e] & 0xFFFFFFu) * TILE;
                        int32_t        key_docs[4]; // on their way while the product is
                        if(docs && (f & TILE_MASK))
#pragma unroll
                            for(uint32_t i = 0; i < 4; ++i)
                                key_docs[i] = c0 + 32 * i + lane < p.len_kv ? __ldg(p.doc_kv + size_t(b) * p.len_kv + c0 + 32 * i + lane) : -1;
                        ok = wait_bounded_warp(base + L::S_FULL + 8 * t, n_s & 1u, cta_abort, status, FWD_SOFTMAX << 24 | (blockIdx.x & 0xFFFFFFu));
                        if(!ok)
                            break;
                        ptx::tc_fence_after_sync();
                        const uint32_t s_row = s_tmem[t] + lane_tmem;
                        const float    from  = static_cast<float>(at - int32_t(c0));
                        const auto     transform_as = [&](auto how, int at_col, auto& x) {
#pragma unroll
                            for(int k = 0; k < int(sizeof(x) / 4); k += 2)
                            {
                                uint64_t unused;
                                float    lo, hi;
                                unpair(score2<CAP, BIAS, decltype(how)::value>(sc, pair(__uint_as_float(x[k]), __uint_as_float(x[k + 1])),
                                                                               from - static_cast<float>(at_col + k), -1.0f, unused),
                                       lo, hi);
                                x[k] = __float_as_uint(lo), x[k + 1] = __float_as_uint(hi);
                            }
                        };
                        const auto transform = [&](int at_col, auto& x) {
                            if constexpr(!PLAIN)
                            {
                                const bool small = tame<CAP>(sc, x);
                                wild |= !small;
                                bend<CAP>(sc, small, [&](auto how) { transform_as(how, at_col, x); });
                            }
                        };
                        uint32_t see[4] = {~0u, ~0u, ~0u, ~0u};
                        if(f & TILE_MASK)
                        {
#pragma unroll
                            for(int i = 0; i < 4; ++i)
                                see[i] = below(lim - int32_t(c0), i);
                            if(docs)
                            {
                                uint32_t same[4] = {0, 0, 0, 0};
                                same_docs(key_docs, doc, same);
#pragma unroll
                                for(int i = 0; i < 4; ++i)
                                    see[i] &= same[i];
                            }
                        }
                        const auto masked = [&](int at_col, auto& x) {
#pragma unroll
                            for(int k = 0; k < int(sizeof(x) / 4); ++k)
                                if(!(see[at_col / 32] >> (at_col % 32 + k) & 1u))
                                    x[k] = 0xFF800000u; // -infinity
                        };
                        // One pass with the maximum as it stands and, under a cap, small scores taken for granted.  Where that turns
                        // out wrong, two passes; and two at once in the tile after that.
                        float top;
                        bool  moved = n_s == 0 || steep || wild;
                        if(!moved)
                        {
                            uint32_t    w[4][16];
                            const float sub = m == -INFINITY ? 0.0f : -m, c = PLAIN ? sc.c : 1.0f;
                            float       most = 0.0f;
                            const auto  guess = [&](int at_col, auto& x) {
                                if constexpr(CAP)
                                    most = magnitude(x, most);
                                if constexpr(!PLAIN)
                                    transform_as(Bent<TAME>{}, at_col, x);
                            };
                            const float more = f & TILE_MASK ? weights_at<T>(s_row, c, sub, w, top,
                                                                             [&](int at_col, auto& x) {
                                                                                 guess(at_col, x);
                                                                                 masked(at_col, x);
                                                                             })
                                                             : weights_at<T>(s_row, c, sub, w, top, guess);
                            moved = __any_sync(0xFFFFFFFFu, top * c > m + RESCALE_STEP || (CAP && !(most * fabsf(sc.k2) <= TAME_LIMIT)));
                            if(!moved)
                            {
                                l += more;
#pragma unroll
                                for(int i = 0; i < 4; ++i)
                                    tmem_st_32x32b_x16(s_row + 16 * i, w[i]);
                            }
                        }
                        if(moved)
                        {
                            wild = false;
                            top = row_max<true>(s_row, [&](int at_col, auto& x) {
                                transform(at_col, x);
                                masked(at_col, x);
                            });
                            if constexpr(PLAIN)
                                top *= sc.c; // scale > 0
                            // move the maximum where some row of this warp has outgrown it
                            const bool outgrown = __any_sync(0xFFFFFFFFu, top > m + RESCALE_STEP);
                            steep = outgrown && n_s != 0;
                            if(outgrown)
                            {
                                const float m2 = fmaxf(m, top);
                                const float by = m2 == -INFINITY ? 1.0f : ex2(m - m2);
                                l *= by;
                                m = m2;
                                if(n_s != 0)
                                {
                                    ok = wait_bounded_warp(base + L::O_DONE + 8 * t, (n_s - 1) & 1u, cta_abort, status,
                                                                     FWD_SOFTMAX << 24 | 1u << 20 | (blockIdx.x & 0xFFFFFu));
                                    if(!ok)
                                        break;
                                    ptx::tc_fence_after_sync();
#pragma unroll 1
                                    for(uint32_t c = 0; c < HD; c += 32)
                                    {
                                        uint32_t w[32];
                                        ptx::tmem_ld_32x32b_x32(o_tmem[t] + lane_tmem + c, w);
                                        ptx::tmem_ld_wait();
#pragma unroll
                                        for(int i = 0; i < 32; ++i)
                                            w[i] = __float_as_uint(__uint_as_float(w[i]) * by);
                                        tmem_st_32x32b_x32(o_tmem[t] + lane_tmem + c, w);
                                    }
                                }
                            }
                            const float sub = m == -INFINITY ? 0.0f : -m;
                            l += weights<T>(s_row, PLAIN ? sc.c : 1.0f, sub);
                        }
                        tmem_st_wait();
                        ptx::tc_fence_before_sync();
                        __syncwarp();
                        if(lane == 0)
                            ptx::mbar_arrive(base + L::P_FULL + 8 * t);
                        ++n_s;
                    }
                }
                if(seg == 0)
                    break;
                __syncthreads(); // the list is written anew
            }

            // ---- results ----
            if(warp < 8)
            {
                const bool have = n_s != 0;
                if(q_here && ok) // the copies of Q, whose place is used below, are over also where this tile sees nothing
                    ok = wait_bounded_warp(base + L::Q_FULL, 0, cta_abort, status, FWD_SOFTMAX << 24 | 3u << 20 | (blockIdx.x & 0xFFFFFu));
                if(have && ok)
                {
                    ok = wait_bounded_warp(base + L::O_DONE + 8 * t, (n_s - 1) & 1u, cta_abort, status,
                                                     FWD_SOFTMAX << 24 | 2u << 20 | (blockIdx.x & 0xFFFFFu));
                    ptx::tc_fence_after_sync();
                }
                // every product of this tile is done: its Q makes room for the results
                const uint32_t tile_smem = L::Q + (PER == 2 ? t * L::TILE_BYTES : 0), tile_row = threadIdx.x & 127u, lane_tmem = (quad * 32u) << 16;
                if(PER == 2)
                {
                    if(ok)
                        stage_row<T>(smem + tile_smem, tile_row, o_tmem[t] + lane_tmem, 0, HD, have && l != 0.0f ? inverse(l) : 0.0f);
                }
                else
                {
                    // the even and the odd key tiles meet; each group of threads takes half of the columns
                    float* stats = reinterpret_cast<float*>(smem + L::STATS);
                    stats[threadIdx.x] = m, stats[2 * TILE + threadIdx.x] = l;
                    ptx::tc_fence_before_sync();
                    ptx::named_bar_sync(1, 2 * TILE); // warps that gave up come here too
                    ptx::tc_fence_after_sync();
                    const float m0 = stats[tile_row], m1 = stats[TILE + tile_row];
                    const float l0 = stats[2 * TILE + tile_row], l1 = stats[3 * TILE + tile_row];
                    m = fmaxf(m0, m1);
                    // a sum without a maximum is NaN and stays it
                    const float by0 = l0 == 0.0f ? 0.0f : m0 == -INFINITY ? l0 : ex2(m0 - m);
                    const float by1 = l1 == 0.0f ? 0.0f : m1 == -INFINITY ? l1 : ex2(m1 - m);
                    l = by0 * l0 + by1 * l1;
                    if(ok)
                        stage_row<T>(smem + tile_smem, tile_row, o_tmem[0] + lane_tmem, t * (HD / 2), (t + 1) * (HD / 2),
                                     by0 != 0.0f ? by0 * inverse(l) : 0.0f, o_tmem[1] + lane_tmem, by1 != 0.0f ? by1 * inverse(l) : 0.0f);
                }
                if(ok)
                    ptx::fence_proxy_async_smem();
                if(ok && lse && row < p.len_q && (PER == 2 || t == 0))
                    lse[(size_t(b) * p.heads_q + h) * p.len_q + row] = l == 0.0f ? -INFINITY : (m + log2f(l)) * LN2;
                if(PER == 2)
                    ptx::named_bar_sync(1 + t, TILE);
                else
                    ptx::named_bar_sync(1, 2 * TILE);
                if(tile_row == 0 && (PER == 2 || t == 0) && row < p.len_q && !*cta_abort)
                    store_tile<HD>(&map_o, base + tile_smem, row, h, b);
            }
            ptx::tc_fence_before_sync();
            __syncthreads();
            if(*cta_abort)
            {
                // A wait was abandoned: copies or products of this CTA may still be in flight.  Give them a bounded grace
                // period before shared and tensor memory are released.
                const uint64_t t0 = ptx::globaltimer_ns();
                while(ptx::globaltimer_ns() - t0 < 2000000ull)
                    __nanosleep(1000);
                __syncthreads();
            }
            if(warp == 9)
            {
                ptx::tc_fence_after_sync();
                ptx::tmem_dealloc(tmem, 512);
            }
        }
    } // namespace attn
} // namespace b200wmma
