// Backward attention on tcgen05: delta = rowsum(dout * o) in one pass over the rows, then two kernels that both recompute
// P = 2^(x - lse), so that no sum is shared between blocks and no atomics are needed (eight products where one kernel
// with shared sums would do five).
//   dkv: a block owns 128 keys of one key head and walks the queries of all its heads, with keys as tensor memory lanes:
//        S^T = K Q^T, dP^T = V dO^T, dV += P^T dO, dK += dS^T Q
//   dq:  a block owns 128 queries and walks the keys:  S = Q K^T, dP = dO V^T, dQ += dS K
// The dq kernel runs first and sets delta right (see there).
// with dS = P (dP - delta) (1 - tanh^2).  P^T and dS overwrite the products that they come from in tensor memory.
// 256 or 512 threads compute; one warp issues the products, one the copies.
// Bound: the products.  Each kernel has four to a pair of tiles (2048 cycles at a head of 128); S of the next step runs while dS
// of this one is computed, dP of the next one while its P is.  Measured, bf16, gradients of 2 x 16 heads of 4096 x 128: 0.92 ms
// (735-750 TFLOP/s counting five products), causal 0.51 ms, causal with cap and 4 key heads 0.65 ms; both kernels take about the
// same.
#pragma once
#include "attn_tc05.cuh"

namespace b200wmma
{
    namespace attn
    {
        // Four warps compute a part of a tile's columns, COLS to a lane; then come the warps for TMA and MMA.  Two parts, or four under
        // a cap, whose longer chain of instructions more warps hide: forward and backward of 2 x 8 heads of 1027 x 80 with cap and
        // slopes 97 us (at that step 99, 109 with two parts); without a cap four parts lose (2 x 16 heads of 4096 x 128, causal: 0.57 ms,
        // 0.52).
        template <bool CAP>
        struct BwdWarps
        {
            static constexpr uint32_t PARTS = CAP ? 4 : 2, COLS = TILE / PARTS, CHUNKS = COLS / 32;
            static constexpr uint32_t COMPUTE = 4 * PARTS, TMA = COMPUTE, MMA = COMPUTE + 1, THREADS = 32 * (COMPUTE + 2);
        };

        template <uint32_t HD>
        struct BwdSmem
        {
            static constexpr uint32_t TILE_BYTES = HD / 64 * BOX_BYTES;
            static constexpr uint32_t OWN  = 0; // the two tiles of the block itself
            static constexpr uint32_t RING = 2 * TILE_BYTES; // two stages of each of the two tiles that are walked
            static constexpr uint32_t LIST = RING + 4 * TILE_BYTES;
            static constexpr uint32_t RAW  = LIST + SEG * 4;
            static constexpr uint32_t STAT = RAW + SEG; // dkv: two stages of 128 lse and 128 delta
            static constexpr uint32_t BARS = STAT + 4 * TILE * 4;
            static constexpr uint32_t OWN_FULL = BARS, FULL = OWN_FULL + 8, EMPTY = FULL + 32, // [2 tiles][2 stages]
                                      S_FULL = EMPTY + 32, DP_FULL = S_FULL + 8, P_FULL = DP_FULL + 16, DS_FULL = P_FULL + 8,
                                      DONE = DS_FULL + 16;
            static constexpr uint32_t MISC  = DONE + 8;
            static constexpr uint32_t BYTES = MISC + 16 + 1024;
        };
        enum BwdRole : uint32_t
        {
            DKV_PRODUCER = 0x41,
            DKV_MMA      = 0x42,
            DKV_COMPUTE  = 0x43,
            DQ_PRODUCER  = 0x51,
            DQ_MMA       = 0x52,
            DQ_COMPUTE   = 0x53
        };

        // delta = rowsum(dout * o) and the row statistics in units of log 2, rows padded to whole tiles.  Rows that see nothing
        // and rows behind the last one get lse = +infinity, so that every P of theirs is 0.  16 lanes to a row.
        template <typename T>
        __global__ void __launch_bounds__(256)
            bwd_rows_kernel(const __grid_constant__ Params p, const T* __restrict__ o, const T* __restrict__ dout, const float* __restrict__ lse,
                            float* __restrict__ lse2, float* __restrict__ delta, uint32_t padded, uint32_t total)
        {
            ptx::grid_dep_launch_dependents();
            const uint32_t at = blockIdx.x * 16 + (threadIdx.x >> 4), lane = threadIdx.x & 15u;
            const uint32_t i = at % padded, bh = at / padded, h = bh % p.heads_q, b = bh / p.heads_q;
            float          sum = 0.0f, s = -INFINITY;
            if(at < total && i < p.len_q)
            {
                s = lse[size_t(bh) * p.len_q + i];
                if(s != -INFINITY && lane * 8 < p.dim)
                {
                    const uint4 x = *reinterpret_cast<const uint4*>(o + int64_t(b) * p.o.batch + int64_t(i) * p.o.token + int64_t(h) * p.o.head + lane * 8);
                    const uint4 y = *reinterpret_cast<const uint4*>(dout + int64_t(b) * p.dout.batch + int64_t(i) * p.dout.token
                                                                    + int64_t(h) * p.dout.head + lane * 8);
                    const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                    for(int j = 0; j < 4; ++j)
                    {
                        const float2 u = tc05::Pack16<T>::widen(xs[j]), v = tc05::Pack16<T>::widen(ys[j]);
                        sum = fmaf(u.x, v.x, sum);
                        sum = fmaf(u.y, v.y, sum);
                    }
                }
            }
#pragma unroll
            for(int d = 8; d > 0; d >>= 1)
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
            if(at < total && lane == 0)
            {
                lse2[at]  = s == -INFINITY ? INFINITY : s * LOG2E;
                delta[at] = sum;
            }
        }

        __device__ __forceinline__ void store_columns(uint32_t taddr, const uint32_t (&r)[16])
        {
            tmem_st_32x32b_x16(taddr, r);
        }
        __device__ __forceinline__ void store_columns(uint32_t taddr, const uint32_t (&r)[32])
        {
            tmem_st_32x32b_x32(taddr, r);
        }
        // D (+)= A B over 128 tokens; the left operand's parts of COLS tokens start COLS columns apart
        template <typename T, uint32_t HD, uint32_t COLS>
        __device__ __forceinline__ void mma_over_tokens_parts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_smem, bool accumulate)
        {
            constexpr uint32_t idesc = tc05::make_idesc<kind_of<T>, TILE, HD, false, true>();
            const uint64_t     b     = ptx::make_mnmajor_sw128_desc(b_smem, BOX_BYTES);
#pragma unroll
            for(uint32_t k = 0; k < TILE / 16; ++k)
                mma_f16_ts(d_tmem, a_tmem + k * 16 / COLS * COLS + k * 16 % COLS / 2, b + k * (2048u >> 4), idesc, (accumulate || k != 0) ? 1u : 0u);
        }

        // ---------------------------------------------------------------------------------------------------------------
        template <typename T, uint32_t HD, bool CAP, bool BIAS>
        __global__ void __launch_bounds__(BwdWarps<CAP>::THREADS, 1)
            bwd_dkv_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                           const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do,
                           const __grid_constant__ CUtensorMap map_dk, const __grid_constant__ CUtensorMap map_dv, const __grid_constant__ Params p,
                           const float* __restrict__ lse2, const float* __restrict__ delta, const DocTile* __restrict__ doc_tiles_q,
                           const DocTile* __restrict__ doc_tiles_kv, uint32_t splits, float* __restrict__ partial, unsigned* status)
        {
            using L = BwdSmem<HD>;
            using W = BwdWarps<CAP>;
            extern __shared__ uint8_t smem_raw[];
            const uint32_t            base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
            uint8_t*                  smem = smem_raw + (base - ptx::smem_u32(smem_raw));
            uint32_t*                 list = reinterpret_cast<uint32_t*>(smem + L::LIST);
            uint32_t*                 misc = reinterpret_cast<uint32_t*>(smem + L::MISC);
            volatile uint32_t*        cta_abort = misc + 1;

            const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
            const uint32_t split = blockIdx.x % splits, block = blockIdx.x / splits;
            const uint32_t bg = block % (p.batch * p.heads_kv), kv_tile = block / (p.batch * p.heads_kv);
            const uint32_t g = bg % p.heads_kv, b = bg / p.heads_kv, share = p.heads_q / p.heads_kv;
            const uint32_t c0 = kv_tile * TILE, q_tiles = (p.len_q + TILE - 1) / TILE, kv_tiles = (p.len_kv + TILE - 1) / TILE;
            const int32_t  prefix = p.prefix ? p.prefix[b] : 0;
            const bool     docs   = p.doc_q != nullptr;

            if(threadIdx.x == 0)
            {
                ptx::prefetch_tensormap(&map_q);
                ptx::prefetch_tensormap(&map_k);
                ptx::prefetch_tensormap(&map_v);
                ptx::prefetch_tensormap(&map_do);
                ptx::mbar_init(base + L::OWN_FULL, 1);
                for(uint32_t s = 0; s < 4; ++s)
                {
                    ptx::mbar_init(base + L::FULL + 8 * s, 1);
                    ptx::mbar_init(base + L::EMPTY + 8 * s, 1);
                }
                ptx::mbar_init(base + L::S_FULL, 1);
                ptx::mbar_init(base + L::DP_FULL, 1);
                ptx::mbar_init(base + L::P_FULL, W::COMPUTE); // warps
                ptx::mbar_init(base + L::DS_FULL, W::COMPUTE);
                ptx::mbar_init(base + L::DONE, 1);
                *cta_abort = 0u;
                ptx::fence_barrier_init();
                ptx::fence_proxy_async_smem();
            }
            if(warp == W::MMA)
            {
                ptx::tmem_alloc(base + L::MISC, 512);
                ptx::tmem_relinquish();
            }
            ptx::tc_fence_before_sync();
            __syncthreads();
            ptx::tc_fence_after_sync();
            ptx::grid_dep_wait(); // the row statistics are there
            const uint32_t tmem = misc[0], s_tmem = tmem, dp_tmem = tmem + TILE, dv_tmem = tmem + 2 * TILE, dk_tmem = dv_tmem + HD;

            const uint32_t   n_stat = q_tiles * TILE; // padded rows of a head
            uint32_t         it = 0; // pairs (head, query tile) so far, in every role
            bool             ok = true;
            const uint32_t   part = warp >> 2, quad = warp & 3u; // compute: columns [COLS part, COLS part + COLS) of lane 32 quad + lane
            const uint32_t   col = c0 + quad * 32u + lane; // its key
            const uint32_t   lane_tmem = ((quad * 32u) << 16) + part * W::COLS;
            const int32_t    doc = (docs && col < p.len_kv) ? p.doc_kv[size_t(b) * p.len_kv + col] : 0;

            for(uint32_t seg = 0; seg < q_tiles; seg += SEG)
            {
                const uint32_t entries
                    = list_tiles<W::THREADS>(seg, min(SEG, q_tiles - seg), list, smem + L::RAW, misc + 2, [&](uint32_t tile) {
                          const DocTile* dq = docs ? doc_tiles_q + size_t(b) * q_tiles + tile : nullptr;
                          const uint32_t f  = tile_flags(p, tile * TILE, c0, prefix, dq, docs ? doc_tiles_kv + size_t(b) * kv_tiles + kv_tile : nullptr);
                          return f && docs && dq->neg ? f | TILE_DIRTY : f;
                      });
                // all tiles of one head, then those of the next; this block takes steps n0 .. n1 - 1 of them
                const uint64_t steps = uint64_t(entries) * share;
                const uint32_t n0 = uint32_t(steps * split / splits), n1 = uint32_t(steps * (split + 1) / splits);
                if(warp == W::TMA)
                {
                    // ------------------------------ TMA producer ------------------------------
                    if(lane == 0 && ok && n0 < n1)
                    {
                        if(it == 0)
                        {
                            ptx::mbar_arrive_expect_tx(base + L::OWN_FULL, 2 * L::TILE_BYTES);
                            load_tile<HD>(base + L::OWN, &map_k, c0, g, b, base + L::OWN_FULL);
                            load_tile<HD>(base + L::OWN + L::TILE_BYTES, &map_v, c0, g, b, base + L::OWN_FULL);
                        }
                        for(uint32_t n = n0; ok && n < n1; ++n, ++it)
                        {
                            const uint32_t h = g * share + n / entries, r0 = (list[n % entries] & 0xFFFFFFu) * TILE;
                            const uint32_t st = it & 1u, ph = (it >> 1) & 1u;
                            const size_t   stat = (size_t(b) * p.heads_q + h) * n_stat + r0;
                            for(uint32_t what = 0; ok && what < 2; ++what) // q with the row statistics (read until dS), dout
                            {
                                const uint32_t full = base + L::FULL + 16 * what + 8 * st;
                                ok = ptx::mbar_wait_bounded(base + L::EMPTY + 16 * what + 8 * st, ph ^ 1u, cta_abort, status,
                                                            DKV_PRODUCER << 24 | (blockIdx.x & 0xFFFFFFu), tc05::WAIT_TIMEOUT_NS);
                                if(!ok)
                                    break;
                                ptx::mbar_arrive_expect_tx(full, L::TILE_BYTES + (what ? 0u : 2 * TILE * 4));
                                load_tile<HD>(base + L::RING + (2 * what + st) * L::TILE_BYTES, what ? &map_do : &map_q, r0, h, b, full);
                                if(what == 0)
                                {
                                    ptx::bulk_load_1d(base + L::STAT + st * TILE * 4, lse2 + stat, TILE * 4, full);
                                    ptx::bulk_load_1d(base + L::STAT + (2 + st) * TILE * 4, delta + stat, TILE * 4, full);
                                }
                            }
                        }
                    }
                    __syncwarp();
                }
                else if(warp == W::MMA)
                {
                    // ------------------------------- MMA issuer -------------------------------
                    const auto wait = [&](uint32_t bar, uint32_t parity, uint32_t what) {
                        ok = ok
                             && wait_bounded_warp(bar, parity, cta_abort, status,
                                                            DKV_MMA << 24 | what << 20 | (blockIdx.x & 0xFFFFFu));
                        ptx::tc_fence_after_sync();
                        return ok;
                    };
                    // waits for tile `what` (0 q, 1 dout) of step n and clears its rows of padding
                    const auto arrive = [&](uint32_t what, uint32_t at, uint32_t n) {
                        if(!wait(base + L::FULL + 16 * what + 8 * (at & 1u), (at >> 1) & 1u, what))
                            return false;
                        const uint32_t e = list[n % entries];
                        if(e >> 24 & TILE_DIRTY)
                        {
                            const uint32_t r0 = (e & 0xFFFFFFu) * TILE;
                            clear_padding<HD>(smem + L::RING + (2 * what + (at & 1u)) * L::TILE_BYTES, p.doc_q + size_t(b) * p.len_q + r0,
                                              min(TILE, p.len_q - r0), lane);
                        }
                        return true;
                    };
                    const auto scores = [&](uint32_t at) {
                        if(elect_one())
                        {
                            mma_over_head<T, HD>(s_tmem, base + L::OWN, base + L::RING + (at & 1u) * L::TILE_BYTES);
                            ptx::tc_commit(base + L::S_FULL);
                        }
                    };
                    const auto grads = [&](uint32_t at) {
                        if(elect_one())
                        {
                            mma_over_head<T, HD>(dp_tmem, base + L::OWN + L::TILE_BYTES, base + L::RING + (2 + (at & 1u)) * L::TILE_BYTES);
                            ptx::tc_commit(base + L::DP_FULL);
                        }
                    };
                    if(n0 < n1 && ok)
                    {
                        if(it == 0)
                            wait(base + L::OWN_FULL, 0, 2);
                        if(ok && arrive(0, it, n0))
                            scores(it);
                        if(ok && arrive(1, it, n0))
                            grads(it);
                        for(uint32_t n = n0; ok && n < n1; ++n, ++it)
                        {
                            const bool more = n + 1 < n1;
                            if(!wait(base + L::P_FULL, it & 1u, 3))
                                break;
                            if(elect_one())
                            {
                                mma_over_tokens_parts<T, HD, W::COLS>(dv_tmem, s_tmem, base + L::RING + (2 + (it & 1u)) * L::TILE_BYTES, it != 0);
                                ptx::tc_commit(base + L::EMPTY + 16 + 8 * (it & 1u));
                            }
                            if(more)
                            {
                                if(!arrive(0, it + 1, n + 1))
                                    break;
                                scores(it + 1);
                            }
                            if(!wait(base + L::DS_FULL, it & 1u, 4))
                                break;
                            if(elect_one())
                            {
                                mma_over_tokens_parts<T, HD, W::COLS>(dk_tmem, dp_tmem, base + L::RING + (it & 1u) * L::TILE_BYTES, it != 0);
                                ptx::tc_commit(base + L::EMPTY + 8 * (it & 1u));
                            }
                            if(more)
                            {
                                if(!arrive(1, it + 1, n + 1))
                                    break;
                                grads(it + 1);
                            }
                        }
                    }
                    __syncwarp();
                }
                else
                {
                    // --------------------------------- compute --------------------------------
                    for(uint32_t n = n0; ok && n < n1; ++n, ++it)
                    {
                        const uint32_t e = list[n % entries], r0 = (e & 0xFFFFFFu) * TILE, st = it & 1u;
                        const auto     wait = [&](uint32_t bar, uint32_t what) {
                            ok = wait_bounded_warp(bar, it & 1u, cta_abort, status,
                                                                 DKV_COMPUTE << 24 | what << 20 | (blockIdx.x & 0xFFFFFu));
                            ptx::tc_fence_after_sync();
                            return ok;
                        };
                        const ScoreConst sc = score_const(p, g * share + n / entries);
                        const uint32_t   row0 = r0 + part * W::COLS;
                        int32_t          query_docs[W::CHUNKS]; // on their way while the product is
                        if(docs && (e >> 24 & TILE_MASK))
#pragma unroll
                            for(uint32_t i = 0; i < W::CHUNKS; ++i)
                                query_docs[i] = row0 + 32 * i + lane < p.len_q ? __ldg(p.doc_q + size_t(b) * p.len_q + row0 + 32 * i + lane) : -1;
                        // the statistics came with the tiles: an acquire of the same barriers
                        ok = wait_bounded_warp(base + L::FULL + 8 * st, (it >> 1) & 1u, cta_abort, status,
                                                         DKV_COMPUTE << 24 | 2u << 20 | (blockIdx.x & 0xFFFFFu));
                        if(!ok || !wait(base + L::S_FULL, 0))
                            break;
                        uint32_t v[W::CHUNKS][32];
#pragma unroll
                        for(uint32_t i = 0; i < W::CHUNKS; ++i)
                            ptx::tmem_ld_32x32b_x32(s_tmem + lane_tmem + 32 * i, v[i]);
                        ptx::tmem_ld_wait();
                        // v becomes P, and then P (1 - tanh^2)
                        const float4* ls   = reinterpret_cast<const float4*>(smem + L::STAT + st * TILE * 4) + part * (W::COLS / 4);
                        const float   from = static_cast<float>(int32_t(row0) + p.off - int32_t(col));
                        uint32_t seen[W::CHUNKS]; // bit j of word i: this key is visible to query 32 i + j of the part
#pragma unroll
                        for(uint32_t i = 0; i < W::CHUNKS; ++i)
                            seen[i] = ~0u;
                        if(e >> 24 & TILE_MASK)
                        {
                            const int32_t first = col >= p.len_kv                           ? int32_t(W::COLS)
                                                  : (p.causal && int32_t(col) >= prefix) ? int32_t(col) - p.off - int32_t(row0)
                                                                                         : 0;
                            uint32_t same[W::CHUNKS] = {};
                            if(docs)
                                same_docs(query_docs, doc, same);
#pragma unroll
                            for(uint32_t i = 0; i < W::CHUNKS; ++i)
                            {
                                seen[i] = ~below(first, i);
                                if(docs)
                                    seen[i] = doc < 0 ? 0u : seen[i] & same[i];
                            }
                        }
                        const auto weights = [&](auto masked, auto how) {
#pragma unroll
                            for(uint32_t i = 0; i < W::CHUNKS; ++i)
                            {
                                uint32_t w[16];
#pragma unroll
                                for(int j4 = 0; j4 < 8; ++j4)
                                {
                                    const float4 s4    = ls[i * 8 + j4];
                                    const float  sv[4] = {s4.x, s4.y, s4.z, s4.w};
                                    float        pr[4];
#pragma unroll
                                    for(int k = 0; k < 4; k += 2)
                                    {
                                        const int      j   = j4 * 4 + k;
                                        const uint64_t dot = pair(__uint_as_float(v[i][j]), __uint_as_float(v[i][j + 1]));
                                        const uint64_t sub = pair(-sv[k], -sv[k + 1]);
                                        uint64_t       slip2 = pair(1.0f, 1.0f);
                                        float          x[2], slip[2];
                                        if constexpr(CAP || BIAS)
                                            unpair(add2(score2<CAP, BIAS, decltype(how)::value>(sc, dot, from + static_cast<float>(32 * i + j), 1.0f, slip2), sub),
                                                   x[0], x[1]);
                                        else
                                            unpair(fma2(dot, pair(sc.c, sc.c), sub), x[0], x[1]);
                                        unpair(slip2, slip[0], slip[1]);
#pragma unroll
                                        for(int u = 0; u < 2; ++u)
                                        {
                                            if constexpr(decltype(masked)::value)
                                                if(!(seen[i] >> (j + u) & 1u))
                                                    x[u] = -INFINITY, slip[u] = 0.0f; // the product may be NaN
                                            pr[k + u] = ex2(x[u]);
                                            v[i][j + u]  = __float_as_uint(CAP ? pr[k + u] * slip[u] : pr[k + u]);
                                        }
                                    }
                                    w[2 * j4] = pack2<T>(pr[0], pr[1]), w[2 * j4 + 1] = pack2<T>(pr[2], pr[3]);
                                }
                                tmem_st_32x32b_x16(s_tmem + lane_tmem + 16 * i, w);
                            }
                        };
                        bool small = true;
#pragma unroll
                        for(uint32_t i = 0; i < W::CHUNKS; ++i)
                            small = small && tame<CAP>(sc, v[i]);
                        if(!small || (e >> 24 & TILE_MASK))
                            bend<CAP>(sc, small, [&](auto how) { weights(std::true_type{}, how); });
                        else
                            weights(std::false_type{}, Bent<TAME>{});
                        tmem_st_wait();
                        ptx::tc_fence_before_sync();
                        __syncwarp();
                        if(lane == 0)
                            ptx::mbar_arrive(base + L::P_FULL);

                        if(!wait(base + L::DP_FULL, 1))
                            break;
                        const float4* de = reinterpret_cast<const float4*>(smem + L::STAT + (2 + st) * TILE * 4) + part * (W::COLS / 4);
                        uint32_t ds[W::COLS / 2];
#pragma unroll
                        for(uint32_t i = 0; i < W::COLS / 16; ++i)
                        {
                            uint32_t u[16];
                            ptx::tmem_ld_32x32b_x16(dp_tmem + lane_tmem + 16 * i, u);
                            ptx::tmem_ld_wait();
#pragma unroll
                            for(int j4 = 0; j4 < 4; ++j4)
                            {
                                const float4 d4    = de[i * 4 + j4];
                                const float  dl[4] = {d4.x, d4.y, d4.z, d4.w};
                                float        x[4];
#pragma unroll
                                for(int k = 0; k < 4; ++k)
                                {
                                    const float pr = __uint_as_float(v[i / 2][i % 2 * 16 + j4 * 4 + k]);
                                    x[k]           = pr * (__uint_as_float(u[j4 * 4 + k]) - dl[k]);
                                    if(e >> 24 & TILE_MASK) // a row of padding may have made the product NaN
                                        x[k] = pr == 0.0f ? 0.0f : x[k];
                                }
                                ds[i * 8 + 2 * j4] = pack2<T>(x[0], x[1]), ds[i * 8 + 2 * j4 + 1] = pack2<T>(x[2], x[3]);
                            }
                        }
                        store_columns(dp_tmem + lane_tmem, ds);
                        tmem_st_wait();
                        ptx::tc_fence_before_sync();
                        __syncwarp();
                        if(lane == 0)
                            ptx::mbar_arrive(base + L::DS_FULL);
                    }
                }
                if(seg + SEG < q_tiles)
                    __syncthreads();
            }

            // ---- results: dv by the first half of the threads, dk by the other ----
            if(warp == W::MMA && ok && elect_one())
                ptx::tc_commit(base + L::DONE);
            if(warp < W::COMPUTE)
            {
                constexpr uint32_t HALF = W::PARTS / 2; // parts to each
                const uint32_t     is_dk = part / HALF;
                if(ok)
                    ok = wait_bounded_warp(base + L::DONE, 0, cta_abort, status, DKV_COMPUTE << 24 | 4u << 20 | (blockIdx.x & 0xFFFFFu));
                const uint32_t acc = (is_dk ? dk_tmem : dv_tmem) + ((quad * 32u) << 16), from = part % HALF * (HD / HALF), to = from + HD / HALF;
                ptx::tc_fence_after_sync();
                if(ok && splits > 1)
                {
                    float* out = partial + ((size_t(split * 2 + is_dk) * (gridDim.x / splits) + block) * TILE + (threadIdx.x & 127u)) * HD;
#pragma unroll 1
                    for(uint32_t c = from; c < to; c += 32)
                    {
                        uint32_t w[32];
                        ptx::tmem_ld_32x32b_x32(acc + c, w);
                        ptx::tmem_ld_wait();
#pragma unroll
                        for(int i = 0; i < 8; ++i)
                            *reinterpret_cast<uint4*>(out + c + 4 * i)
                                = it != 0 ? make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]) : make_uint4(0, 0, 0, 0);
                    }
                }
                else if(ok)
                {
                    // every product is done: the tiles of K and V make room
                    stage_row<T>(smem + L::OWN + is_dk * L::TILE_BYTES, threadIdx.x & 127u, acc, from, to, it == 0 ? 0.0f : is_dk ? p.scale : 1.0f);
                    ptx::fence_proxy_async_smem();
                }
                ptx::named_bar_sync(1 + is_dk, HALF * TILE); // warps that gave up come here too
                if(threadIdx.x % (HALF * TILE) == 0 && splits == 1 && !*cta_abort)
                    store_tile<HD>(is_dk ? &map_dk : &map_dv, base + L::OWN + is_dk * L::TILE_BYTES, c0, g, b);
            }
            ptx::tc_fence_before_sync();
            __syncthreads();
            if(*cta_abort)
            {
                // A wait was abandoned: give copies and products in flight a bounded grace period before memory is released.
                const uint64_t t0 = ptx::globaltimer_ns();
                while(ptx::globaltimer_ns() - t0 < 2000000ull)
                    __nanosleep(1000);
                __syncthreads();
            }
            if(warp == W::MMA)
            {
                ptx::tc_fence_after_sync();
                ptx::tmem_dealloc(tmem, 512);
            }
        }

        // Sums the partial dk and dv of a tile's splits, in order: four elements to a thread.
        template <typename T, uint32_t HD>
        __global__ void __launch_bounds__(256)
            bwd_join_kernel(const __grid_constant__ Params p, const float* __restrict__ partial, uint32_t splits, uint32_t blocks, T* __restrict__ dk,
                            T* __restrict__ dv)
        {
            const size_t   at = (size_t(blockIdx.x) * 256 + threadIdx.x) * 4, tile = size_t(TILE) * HD;
            const uint32_t d = at % HD, row = at / HD % TILE, block = uint32_t(at / tile % blocks), is_dk = uint32_t(at / tile / blocks);
            const uint32_t bg = block % (p.batch * p.heads_kv), token = block / (p.batch * p.heads_kv) * TILE + row;
            if(is_dk > 1 || token >= p.len_kv || d >= p.dim)
                return;
            float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
            for(uint32_t s = 0; s < splits; ++s)
            {
                const float4 x = *reinterpret_cast<const float4*>(partial + at + size_t(s) * 2 * blocks * tile);
                y.x += x.x, y.y += x.y, y.z += x.z, y.w += x.w;
            }
            const float    by = is_dk ? p.scale : 1.0f;
            const Strides& st = is_dk ? p.dk : p.dv;
            T* out = (is_dk ? dk : dv) + int64_t(bg / p.heads_kv) * st.batch + int64_t(token) * st.token + int64_t(bg % p.heads_kv) * st.head + d;
            *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(y.x * by, y.y * by), pack2<T>(y.z * by, y.w * by));
        }

        // ---------------------------------------------------------------------------------------------------------------
        // delta from an o in 16 bits is off by e_i, which moves dQ_i by e_i (P K)_i: as much as the rounding of dS does where a
        // query sees few keys.  sum_j P (dP - delta) is that error, so this kernel adds it up, adds up P K next to dQ, takes the
        // product off at the end and leaves the right delta for the dkv kernel.  The steps are interleaved as there.
        template <typename T, uint32_t HD, bool CAP, bool BIAS>
        __global__ void __launch_bounds__(BwdWarps<CAP>::THREADS, 1)
            bwd_dq_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                          const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do,
                          const __grid_constant__ CUtensorMap map_dq, const __grid_constant__ Params p, const float* __restrict__ lse2,
                          float* __restrict__ delta, const DocTile* __restrict__ doc_tiles_q, const DocTile* __restrict__ doc_tiles_kv,
                          unsigned* status)
        {
            using L = BwdSmem<HD>;
            using W = BwdWarps<CAP>;
            extern __shared__ uint8_t smem_raw[];
            const uint32_t            base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
            uint8_t*                  smem = smem_raw + (base - ptx::smem_u32(smem_raw));
            uint32_t*                 list = reinterpret_cast<uint32_t*>(smem + L::LIST);
            uint32_t*                 misc = reinterpret_cast<uint32_t*>(smem + L::MISC);
            volatile uint32_t*        cta_abort = misc + 1;

            const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
            const uint32_t q_tiles = (p.len_q + TILE - 1) / TILE, kv_tiles = (p.len_kv + TILE - 1) / TILE;
            const uint32_t bh = blockIdx.x % (p.batch * p.heads_q), q_tile = q_tiles - 1 - blockIdx.x / (p.batch * p.heads_q);
            const uint32_t h = bh % p.heads_q, b = bh / p.heads_q, g = h / (p.heads_q / p.heads_kv);
            const uint32_t row0   = q_tile * TILE;
            const int32_t  prefix = p.prefix ? p.prefix[b] : 0;
            const bool     docs   = p.doc_q != nullptr;

            if(threadIdx.x == 0)
            {
                ptx::prefetch_tensormap(&map_q);
                ptx::prefetch_tensormap(&map_k);
                ptx::prefetch_tensormap(&map_v);
                ptx::prefetch_tensormap(&map_do);
                ptx::mbar_init(base + L::OWN_FULL, 1);
                for(uint32_t s = 0; s < 4; ++s)
                {
                    ptx::mbar_init(base + L::FULL + 8 * s, 1);
                    ptx::mbar_init(base + L::EMPTY + 8 * s, 1);
                }
                ptx::mbar_init(base + L::S_FULL, 1);
                ptx::mbar_init(base + L::DP_FULL, 1);
                ptx::mbar_init(base + L::P_FULL, W::COMPUTE); // warps
                ptx::mbar_init(base + L::DS_FULL, W::COMPUTE);
                ptx::mbar_init(base + L::DONE, 1);
                *cta_abort = 0u;
                ptx::fence_barrier_init();
                ptx::fence_proxy_async_smem();
            }
            if(warp == W::MMA)
            {
                ptx::tmem_alloc(base + L::MISC, 512);
                ptx::tmem_relinquish();
            }
            ptx::tc_fence_before_sync();
            __syncthreads();
            ptx::tc_fence_after_sync();
            ptx::grid_dep_wait(); // the row statistics are there
            ptx::grid_dep_launch_dependents();
            const uint32_t tmem = misc[0], s_tmem = tmem, dp_tmem = tmem + TILE, dq_tmem = tmem + 2 * TILE, pk_tmem = dq_tmem + HD;

            uint32_t         it = 0;
            bool             ok = true;
            const uint32_t   part = warp >> 2, quad = warp & 3u;
            const uint32_t   row = row0 + quad * 32u + lane, lane_tmem = ((quad * 32u) << 16) + part * W::COLS;
            const int32_t    at  = int32_t(row) + p.off;
            const int32_t    doc = (docs && row < p.len_q) ? p.doc_q[size_t(b) * p.len_q + row] : 0;
            const int32_t    lim = (row >= p.len_q || doc < 0) ? 0 : (p.causal ? min(max(at + 1, prefix), int32_t(p.len_kv)) : int32_t(p.len_kv));
            const ScoreConst sc  = score_const(p, h);
            float            ls = 0.0f, de = 0.0f, rest = 0.0f; // rest: sum of P (dP - delta)
            if(warp < W::COMPUTE)
            {
                const size_t stat = (size_t(b) * p.heads_q + h) * (q_tiles * TILE) + row;
                ls = __ldcg(lse2 + stat), de = __ldcg(delta + stat);
            }

            for(uint32_t seg = 0; seg < kv_tiles; seg += SEG)
            {
                const uint32_t entries
                    = list_tiles<W::THREADS>(seg, min(SEG, kv_tiles - seg), list, smem + L::RAW, misc + 2, [&](uint32_t tile) {
                          const DocTile* dk = docs ? doc_tiles_kv + size_t(b) * kv_tiles + tile : nullptr;
                          const uint32_t f  = tile_flags(p, row0, tile * TILE, prefix, docs ? doc_tiles_q + size_t(b) * q_tiles + q_tile : nullptr, dk);
                          return f && docs && dk->neg ? f | TILE_DIRTY : f;
                      });
                if(warp == W::TMA)
                {
                    if(lane == 0 && ok && entries)
                    {
                        if(it == 0)
                        {
                            ptx::mbar_arrive_expect_tx(base + L::OWN_FULL, 2 * L::TILE_BYTES);
                            load_tile<HD>(base + L::OWN, &map_q, row0, h, b, base + L::OWN_FULL);
                            load_tile<HD>(base + L::OWN + L::TILE_BYTES, &map_do, row0, h, b, base + L::OWN_FULL);
                        }
                        for(uint32_t n = 0; ok && n < entries; ++n, ++it)
                            for(uint32_t what = 0; ok && what < 2; ++what) // k, v
                            {
                                const uint32_t st = it & 1u, full = base + L::FULL + 16 * what + 8 * st;
                                ok = ptx::mbar_wait_bounded(base + L::EMPTY + 16 * what + 8 * st, ((it >> 1) & 1u) ^ 1u, cta_abort, status,
                                                            DQ_PRODUCER << 24 | (blockIdx.x & 0xFFFFFFu), tc05::WAIT_TIMEOUT_NS);
                                if(!ok)
                                    break;
                                ptx::mbar_arrive_expect_tx(full, L::TILE_BYTES);
                                load_tile<HD>(base + L::RING + (2 * what + st) * L::TILE_BYTES, what ? &map_v : &map_k, (list[n] & 0xFFFFFFu) * TILE, g,
                                              b, full);
                            }
                    }
                    __syncwarp();
                }
                else if(warp == W::MMA)
                {
                    const auto wait = [&](uint32_t bar, uint32_t parity, uint32_t what) {
                        ok = ok
                             && wait_bounded_warp(bar, parity, cta_abort, status, DQ_MMA << 24 | what << 20 | (blockIdx.x & 0xFFFFFu));
                        ptx::tc_fence_after_sync();
                        return ok;
                    };
                    const auto scores = [&](uint32_t a, uint32_t n) { // S of step n (number `a` over all segments)
                        const uint32_t st = a & 1u;
                        if(!wait(base + L::FULL + 8 * st, (a >> 1) & 1u, 0))
                            return;
                        if(list[n] >> 24 & TILE_DIRTY) // the keys are contracted over; the values' rows only reach their own columns
                        {
                            const uint32_t c0 = (list[n] & 0xFFFFFFu) * TILE;
                            clear_padding<HD>(smem + L::RING + st * L::TILE_BYTES, p.doc_kv + size_t(b) * p.len_kv + c0, min(TILE, p.len_kv - c0), lane);
                        }
                        if(elect_one())
                        {
                            mma_over_head<T, HD>(s_tmem, base + L::OWN, base + L::RING + st * L::TILE_BYTES);
                            ptx::tc_commit(base + L::S_FULL);
                        }
                    };
                    const auto grads = [&](uint32_t a) { // dP
                        const uint32_t st = a & 1u;
                        if(!wait(base + L::FULL + 16 + 8 * st, (a >> 1) & 1u, 2))
                            return;
                        if(elect_one())
                        {
                            mma_over_head<T, HD>(dp_tmem, base + L::OWN + L::TILE_BYTES, base + L::RING + (2 + st) * L::TILE_BYTES);
                            ptx::tc_commit(base + L::DP_FULL);
                            ptx::tc_commit(base + L::EMPTY + 16 + 8 * st);
                        }
                    };
                    if(entries && ok)
                    {
                        if(it == 0)
                            wait(base + L::OWN_FULL, 0, 3);
                        if(ok)
                            scores(it, 0);
                        if(ok)
                            grads(it);
                        for(uint32_t n = 0; ok && n < entries; ++n, ++it)
                        {
                            const uint32_t k_smem = base + L::RING + (it & 1u) * L::TILE_BYTES;
                            if(!wait(base + L::P_FULL, it & 1u, 1))
                                break;
                            if(elect_one())
                                mma_over_tokens_parts<T, HD, W::COLS>(pk_tmem, s_tmem, k_smem, it != 0);
                            if(n + 1 < entries)
                                scores(it + 1, n + 1);
                            if(!ok || !wait(base + L::DS_FULL, it & 1u, 4))
                                break;
                            if(elect_one())
                            {
                                mma_over_tokens_parts<T, HD, W::COLS>(dq_tmem, dp_tmem, k_smem, it != 0);
                                ptx::tc_commit(base + L::EMPTY + 8 * (it & 1u));
                            }
                            if(n + 1 < entries)
                                grads(it + 1);
                        }
                    }
                    __syncwarp();
                }
                else
                {
                    for(uint32_t n = 0; ok && n < entries; ++n, ++it)
                    {
                        const uint32_t e = list[n], c0 = (e & 0xFFFFFFu) * TILE + part * W::COLS;
                        int32_t        key_docs[W::CHUNKS]; // on their way while the product is
                        if(docs && (e >> 24 & TILE_MASK))
#pragma unroll
                            for(uint32_t i = 0; i < W::CHUNKS; ++i)
                                key_docs[i] = c0 + 32 * i + lane < p.len_kv ? __ldg(p.doc_kv + size_t(b) * p.len_kv + c0 + 32 * i + lane) : -1;
                        ok = wait_bounded_warp(base + L::S_FULL, it & 1u, cta_abort, status, DQ_COMPUTE << 24 | (blockIdx.x & 0xFFFFFFu));
                        if(!ok)
                            break;
                        ptx::tc_fence_after_sync();
                        uint32_t v[W::CHUNKS][32];
#pragma unroll
                        for(uint32_t i = 0; i < W::CHUNKS; ++i)
                            ptx::tmem_ld_32x32b_x32(s_tmem + lane_tmem + 32 * i, v[i]);
                        ptx::tmem_ld_wait();
                        uint32_t seen[W::CHUNKS]; // bit j of word i: key 32 i + j of the part is visible to this query
#pragma unroll
                        for(uint32_t i = 0; i < W::CHUNKS; ++i)
                            seen[i] = ~0u;
                        if(e >> 24 & TILE_MASK)
                        {
                            uint32_t same[W::CHUNKS] = {};
                            if(docs)
                                same_docs(key_docs, doc, same);
#pragma unroll
                            for(uint32_t i = 0; i < W::CHUNKS; ++i)
                            {
                                seen[i] = below(lim - int32_t(c0), i);
                                if(docs)
                                    seen[i] &= same[i];
                            }
                        }
                        const float from    = static_cast<float>(at - int32_t(c0));
                        // v becomes P, or under a cap the tanh, from which P and the cap's derivative come again below (registers for both
                        // would not do, and from a weight a tanh comes back only as well as the cap is large); P (1 - tanh^2) goes over
                        // the scores.  -infinity stands for pairs that are not visible.
                        const auto weights = [&](auto masked, auto how) {
#pragma unroll
                            for(uint32_t i = 0; i < W::CHUNKS; ++i)
                            {
                                uint32_t w[16];
#pragma unroll
                                for(int j = 0; j < 32; j += 2)
                                {
                                    const uint64_t dot = pair(__uint_as_float(v[i][j]), __uint_as_float(v[i][j + 1])), sub = pair(-ls, -ls);
                                    [[maybe_unused]] const float dist = from - static_cast<float>(32 * i + j);
                                    float                        x[2], tanh[2], slip[2] = {1.0f, 1.0f};
                                    if constexpr(CAP)
                                    {
                                        const uint64_t t = tanh2<decltype(how)::value>(sc, dot);
                                        unpair(t, tanh[0], tanh[1]);
                                        unpair(slip_of(t), slip[0], slip[1]);
                                        unpair(add2(capped<BIAS>(sc, t, dist, -1.0f), sub), x[0], x[1]);
                                    }
                                    else if constexpr(BIAS)
                                        unpair(add2(biased<BIAS>(sc, mul2(dot, pair(sc.c, sc.c)), dist, -1.0f), sub), x[0], x[1]);
                                    else
                                        unpair(fma2(dot, pair(sc.c, sc.c), sub), x[0], x[1]);
#pragma unroll
                                    for(int u = 0; u < 2; ++u)
                                    {
                                        if constexpr(decltype(masked)::value)
                                            if(!(seen[i] >> (j + u) & 1u))
                                                x[u] = tanh[u] = -INFINITY, slip[u] = 0.0f; // the product may be NaN
                                        x[u]        = ex2(x[u]);
                                        v[i][j + u] = __float_as_uint(CAP ? tanh[u] : x[u]);
                                        if(CAP)
                                            x[u] *= slip[u];
                                    }
                                    w[j / 2] = pack2<T>(x[0], x[1]);
                                }
                                tmem_st_32x32b_x16(s_tmem + lane_tmem + 16 * i, w);
                            }
                        };
                        bool small = true;
#pragma unroll
                        for(uint32_t i = 0; i < W::CHUNKS; ++i)
                            small = small && tame<CAP>(sc, v[i]);
                        if(!small || (e >> 24 & TILE_MASK))
                            bend<CAP>(sc, small, [&](auto how) { weights(std::true_type{}, how); });
                        else
                            weights(std::false_type{}, Bent<TAME>{});
                        tmem_st_wait();
                        ptx::tc_fence_before_sync();
                        __syncwarp();
                        if(lane == 0)
                            ptx::mbar_arrive(base + L::P_FULL);

                        ok = wait_bounded_warp(base + L::DP_FULL, it & 1u, cta_abort, status, DQ_COMPUTE << 24 | 1u << 20 | (blockIdx.x & 0xFFFFFu));
                        if(!ok)
                            break;
                        ptx::tc_fence_after_sync();
                        uint32_t ds[W::COLS / 2];
#pragma unroll
                        for(uint32_t i = 0; i < W::COLS / 16; ++i)
                        {
                            uint32_t u[16];
                            ptx::tmem_ld_32x32b_x16(dp_tmem + lane_tmem + 16 * i, u);
                            ptx::tmem_ld_wait();
#pragma unroll
                            for(int j = 0; j < 8; ++j)
                            {
                                const uint32_t c = 16 * i + 2 * j;
                                float          x[2], pr[2] = {__uint_as_float(v[c / 32][c % 32]), __uint_as_float(v[c / 32][c % 32 + 1])}, slip[2];
                                if constexpr(CAP)
                                {
                                    const uint64_t t = pair(pr[0], pr[1]);
                                    unpair(slip_of(t), slip[0], slip[1]);
                                    unpair(add2(capped<BIAS>(sc, t, from - static_cast<float>(c), -1.0f), pair(-ls, -ls)), pr[0], pr[1]);
                                    pr[0] = ex2(pr[0]), pr[1] = ex2(pr[1]);
                                }
#pragma unroll
                                for(int k = 0; k < 2; ++k)
                                {
                                    x[k] = pr[k] * (__uint_as_float(u[2 * j + k]) - de);
                                    if(e >> 24 & TILE_MASK) // a row of padding may have made the product NaN
                                        x[k] = pr[k] == 0.0f ? 0.0f : x[k];
                                    rest += x[k];
                                    if constexpr(CAP)
                                        x[k] = pr[k] == 0.0f ? 0.0f : x[k] * slip[k];
                                }
                                ds[i * 8 + j] = pack2<T>(x[0], x[1]);
                            }
                        }
                        store_columns(dp_tmem + lane_tmem, ds);
                        tmem_st_wait();
                        ptx::tc_fence_before_sync();
                        __syncwarp();
                        if(lane == 0)
                            ptx::mbar_arrive(base + L::DS_FULL);
                    }
                }
                if(seg + SEG < kv_tiles)
                    __syncthreads();
            }

            if(warp == W::MMA && ok && elect_one())
                ptx::tc_commit(base + L::DONE);
            if(warp < W::COMPUTE)
            {
                if(ok)
                    ok = wait_bounded_warp(base + L::DONE, 0, cta_abort, status, DQ_COMPUTE << 24 | 2u << 20 | (blockIdx.x & 0xFFFFFu));
                float* rests       = reinterpret_cast<float*>(smem + L::STAT);
                rests[threadIdx.x] = rest;
                ptx::named_bar_sync(1, W::PARTS * TILE); // warps that gave up come here too
                if(ok)
                {
                    ptx::tc_fence_after_sync();
                    const uint32_t i = threadIdx.x & 127u;
                    rest = rests[i];
#pragma unroll
                    for(uint32_t k = 1; k < W::PARTS; ++k)
                        rest += rests[k * TILE + i];
                    if(part == 0 && row < p.len_q)
                        delta[(size_t(b) * p.heads_q + h) * (q_tiles * TILE) + row] = de + rest;
                    // every product is done: the tile of Q makes room; the parts share its columns, at least 32 to each
                    constexpr uint32_t SHARE = HD / W::PARTS < 32 ? 32 : HD / W::PARTS;
                    if(part * SHARE < HD)
                        stage_row<T>(smem + L::OWN, threadIdx.x & 127u, dq_tmem + ((quad * 32u) << 16), part * SHARE, (part + 1) * SHARE,
                                     it != 0 ? p.scale : 0.0f, pk_tmem + ((quad * 32u) << 16), it != 0 ? -rest * p.scale : 0.0f);
                    ptx::fence_proxy_async_smem();
                }
                ptx::named_bar_sync(1, W::PARTS * TILE);
                if(threadIdx.x == 0 && !*cta_abort)
                    store_tile<HD>(&map_dq, base + L::OWN, row0, h, b);
            }
            ptx::tc_fence_before_sync();
            __syncthreads();
            if(*cta_abort)
            {
                // A wait was abandoned: give copies and products in flight a bounded grace period before memory is released.
                const uint64_t t0 = ptx::globaltimer_ns();
                while(ptx::globaltimer_ns() - t0 < 2000000ull)
                    __nanosleep(1000);
                __syncthreads();
            }
            if(warp == W::MMA)
            {
                ptx::tc_fence_after_sync();
                ptx::tmem_dealloc(tmem, 512);
            }
        }
    } // namespace attn
} // namespace b200wmma
