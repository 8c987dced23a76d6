// Attention of many drafted rows over a paged cache, on tcgen05: the form that attn_tree.cu takes where the rows that share a
// key head are too many for its warp-level products.
//
// A block owns 128 rows of one key head and the tokens of one split, in tiles of 128 tokens that two groups of 128 threads
// (one to a row) take in turn, each with its own scores, maximum, sum and accumulator in tensor memory:
//   S = Q K^T, P = 2^(x - m) in 16 bits over S, O += P V
// so that the tensor cores work on one tile while the other one's softmax runs; the two accumulators meet at the end.
// Measured, bf16: 128 rows (16 drafted tokens x 8 heads), 16 sequences of 8000 tokens x 4 key heads x 128: 56 us (4.7 TB/s, 605
// TFLOP/s), about 1 us a tile; a block takes 10 us before its second tile (page table, copies, first softmax, joining).
#pragma once
#include "attn_tc05.cuh"

namespace b200wmma
{
    namespace attn_tree
    {
        constexpr uint32_t TC_THREADS = 320; // warps 0-3: even tiles, 4-7: odd tiles, 8: copies, 9: products
        using attn::TILE;

        template <uint32_t HD>
        struct TcSmem
        {
            static constexpr uint32_t TILE_BYTES = HD / 64 * attn::BOX_BYTES;
            static constexpr uint32_t STAGES     = HD == 128 ? 5 : 8; // tiles of keys and of values
            static constexpr uint32_t Q          = 0;
            static constexpr uint32_t KV         = TILE_BYTES;
            static constexpr uint32_t VALID      = KV + STAGES * TILE_BYTES; // 8 x 4 words: tokens of a tile that are there
            static constexpr uint32_t TABLE      = VALID + 128; // 4 x 128 {page, row in it}
            static constexpr uint32_t STATS      = TABLE + 4 * TILE * 8; // 2 x 128: maximum and sum of the odd tiles
            static constexpr uint32_t BARS       = STATS + 2 * TILE * 4;
            static constexpr uint32_t FULL = BARS, EMPTY = FULL + 8 * STAGES, S_FULL = EMPTY + 8 * STAGES, P_FULL = S_FULL + 16, O_DONE = P_FULL + 16, Q_FULL = O_DONE + 16;
            static constexpr uint32_t MISC  = Q_FULL + 8;
            static constexpr uint32_t BYTES = MISC + 16 + 1024;
            static_assert(STAGES * TILE_BYTES >= TILE * HD * 4, "an accumulator passes through the ring");
        };
        enum TcRole : uint32_t
        {
            TREE_TC_PRODUCER = 0x71,
            TREE_TC_MMA      = 0x72,
            TREE_TC_SOFTMAX  = 0x73
        };

        template <typename T, uint32_t HD, bool CAP, bool BIAS>
        __global__ void __launch_bounds__(TC_THREADS, 1)
            tree_tc05_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ Params p,
                             const T* __restrict__ q, T* __restrict__ o)
        {
            using L = TcSmem<HD>;
            using attn::ex2;
            extern __shared__ uint8_t smem_raw[];
            const uint32_t     base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
            uint8_t*           smem = smem_raw + (base - ptx::smem_u32(smem_raw));
            uint32_t*          misc = reinterpret_cast<uint32_t*>(smem + L::MISC);
            volatile uint32_t* cta_abort = misc + 1;
            const uint32_t     tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;

            uint32_t       x     = blockIdx.x;
            const uint32_t split = x % p.splits;
            x /= p.splits;
            const uint32_t row_tile = x % p.tiles;
            x /= p.tiles;
            const uint32_t head = x % p.heads_kv, b = x / p.heads_kv, rows = p.share * p.drafts;
            const uint32_t n_drafts = drafts_of(p, b);
            const int64_t  len      = max(__ldg(p.lens + b), 0);
            const uint32_t end      = n_drafts ? uint32_t(min(len + n_drafts, int64_t(p.ld_table) * p.page_size)) : 0u;
            const uint32_t all = (end + TILE - 1) / TILE, from = uint32_t(uint64_t(all) * split / p.splits);
            const uint32_t steps = uint32_t(uint64_t(all) * (split + 1) / p.splits) - from;

            if(tid == 0)
            {
                ptx::prefetch_tensormap(&map_k);
                ptx::prefetch_tensormap(&map_v);
                for(uint32_t s = 0; s < L::STAGES; ++s)
                {
                    ptx::mbar_init(base + L::FULL + 8 * s, 1);
                    ptx::mbar_init(base + L::EMPTY + 8 * s, 1);
                }
                for(uint32_t u = 0; u < 2; ++u)
                {
                    ptx::mbar_init(base + L::S_FULL + 8 * u, 1);
                    ptx::mbar_init(base + L::P_FULL + 8 * u, 4); // warps
                    ptx::mbar_init(base + L::O_DONE + 8 * u, 1);
                }
                ptx::mbar_init(base + L::Q_FULL, 256);
                *cta_abort = 0u;
                ptx::fence_barrier_init();
            }
            if(warp == 9)
            {
                ptx::tmem_alloc(base + L::MISC, 512);
                ptx::tmem_relinquish();
            }
            ptx::tc_fence_before_sync();
            __syncthreads();
            ptx::tc_fence_after_sync();
            if(warp < 8)
            {
                // the rows of Q as a K-major tile with the 128-byte swizzle
                constexpr uint32_t N = TILE * (HD / 8) / 256;
                uint4              w[N];
#pragma unroll
                for(uint32_t i = 0; i < N; ++i)
                {
                    const uint32_t e = tid + i * 256, c = e % (HD / 8), qr = row_tile * TILE + e / (HD / 8), draft = qr / p.share;
                    w[i] = make_uint4(0, 0, 0, 0);
                    if(qr < rows && draft < n_drafts && c * 8 < p.dim)
                        w[i] = *reinterpret_cast<const uint4*>(q + row_of(p.q, b, draft, head * p.share + qr - draft * p.share) + c * 8);
                }
#pragma unroll
                for(uint32_t i = 0; i < N; ++i)
                {
                    const uint32_t e = tid + i * 256, c = e % (HD / 8), row = e / (HD / 8);
                    *reinterpret_cast<uint4*>(smem + L::Q + (c / 8) * attn::BOX_BYTES + row * 128 + (((c % 8) ^ (row & 7u)) << 4)) = w[i];
                }
                ptx::fence_proxy_async_smem();
                ptx::mbar_arrive(base + L::Q_FULL);
            }
            ptx::grid_dep_launch_dependents();
            const uint32_t tmem = misc[0], s_tmem = tmem, o_tmem = tmem + 2 * TILE; // tile u: + u * TILE, + u * HD
            bool           ok = true;
            const uint32_t u = warp >> 2, quad = warp & 3u, lane_tmem = (quad * 32u) << 16, r = row_tile * TILE + (tid & 127u);
            const bool     live = warp < 8 && r < rows && r / p.share < n_drafts;
            float          m = -INFINITY, l = 0.0f;
            uint32_t       mine = 0; // tiles that this thread's group has had

            if(warp == 8)
            {
                // The pages of a tile are asked for one tile ahead and put down, with the tokens that are there, in a table of
                // four tiles: a tile's values are copied two steps after its keys.
                const uint32_t boxes = TILE / p.box; // a lane takes boxes lane, lane + 32, ...
                int2*          table = reinterpret_cast<int2*>(smem + L::TABLE);
                int32_t        page[4], slot[4];
                uint32_t       c = 0; // place in the ring
                const auto     ask = [&](uint32_t n) {
#pragma unroll
                    for(int i = 0; i < 4; ++i)
                    {
                        const uint32_t box = lane + 32 * i, j = (from + n) * TILE + box * p.box;
                        page[i] = -1, slot[i] = 0;
                        if(box < boxes && n < steps && j < end)
                        {
                            const uint32_t at = p.page_shift < 32 ? j >> p.page_shift : j / p.page_size;
                            slot[i]           = int32_t(j - at * p.page_size);
                            page[i]           = __ldg(p.block_table + size_t(b) * p.ld_table + at);
                        }
                    }
                };
                const auto note = [&](uint32_t n) {
                    int2*          to   = table + (n & 3u) * TILE;
                    const uint32_t left = end - min(end, (from + n) * TILE);
                    bool           all_there = left >= TILE;
#pragma unroll
                    for(int i = 0; i < 4; ++i)
                        if(lane + 32 * i < boxes)
                        {
                            const bool there = uint32_t(page[i]) < p.num_pages;
                            all_there &= there; // a page that is not there: one behind the last, which reads as zeros
                            to[lane + 32 * i] = make_int2(there ? page[i] : int32_t(p.num_pages), slot[i]);
                        }
                    uint4* valid = reinterpret_cast<uint4*>(smem + L::VALID) + (n & 7u);
                    if(__all_sync(0xFFFFFFFFu, all_there))
                    {
                        if(lane == 0)
                            *valid = make_uint4(0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu);
                    }
                    else // four tokens to a lane
                    {
                        __syncwarp();
                        uint32_t four = 0;
#pragma unroll
                        for(uint32_t k = 0; k < 4; ++k)
                            if(lane * 4 + k < left && uint32_t(to[(lane * 4 + k) / p.box].x) < p.num_pages)
                                four |= 1u << k;
                        four <<= lane * 4 & 31u;
#pragma unroll
                        for(uint32_t w = 0; w < 4; ++w)
                        {
                            const uint32_t word = __reduce_or_sync(0xFFFFFFFFu, lane / 8 == w ? four : 0u);
                            if(lane == 0)
                                reinterpret_cast<uint32_t*>(valid)[w] = word;
                        }
                    }
                };
                const auto load = [&](uint32_t n, bool values) {
                    const uint32_t st = c % L::STAGES, full = base + L::FULL + 8 * st, stage = base + L::KV + st * L::TILE_BYTES;
                    ok = ok
                         && attn::wait_bounded_warp(base + L::EMPTY + 8 * st, (c / L::STAGES & 1u) ^ 1u, cta_abort, p.status,
                                                        TREE_TC_PRODUCER << 24 | (blockIdx.x & 0xFFFFFFu));
                    if(!ok)
                        return;
                    ++c;
                    if(!values)
                    {
                        note(n);
                        ask(n + 1);
                    }
                    if(lane == 0)
                        ptx::mbar_arrive_expect_tx(full, L::TILE_BYTES);
                    __syncwarp();
                    for(uint32_t box = lane; box < boxes; box += 32)
                    {
                        const int2 at = table[(n & 3u) * TILE + box];
#pragma unroll
                        for(uint32_t h = 0; h < HD / 64; ++h)
                            attn::tma_load_4d(stage + h * attn::BOX_BYTES + box * p.box * 128, values ? &map_v : &map_k, h * 64, at.y, head, at.x, full);
                    }
                };
                // in the order of their use: K0 K1 | V0 K2 | V1 K3 | ...
                ask(0);
                for(uint32_t n = 0; ok && n < min(steps, 2u); ++n)
                    load(n, false);
                for(uint32_t n = 0; ok && n < steps; ++n)
                {
                    load(n, true);
                    if(ok && n + 2 < steps)
                        load(n + 2, false);
                }
            }
            else if(warp == 9)
            {
                uint32_t   c = 0;
                const auto wait = [&](uint32_t bar, uint32_t parity, uint32_t what) {
                    ok = ok
                         && attn::wait_bounded_warp(bar, parity, cta_abort, p.status, TREE_TC_MMA << 24 | what << 20 | (blockIdx.x & 0xFFFFFu));
                    ptx::tc_fence_after_sync();
                    return ok;
                };
                const auto scores = [&](uint32_t n) {
                    const uint32_t st = c % L::STAGES;
                    if(!wait(base + L::FULL + 8 * st, c / L::STAGES & 1u, 0))
                        return;
                    ++c;
                    if(attn::elect_one())
                    {
                        attn::mma_over_head<T, HD>(s_tmem + (n & 1u) * TILE, base + L::Q, base + L::KV + st * L::TILE_BYTES);
                        ptx::tc_commit(base + L::S_FULL + 8 * (n & 1u));
                        ptx::tc_commit(base + L::EMPTY + 8 * st);
                    }
                };
                wait(base + L::Q_FULL, 0, 3);
                for(uint32_t n = 0; ok && n < min(steps, 2u); ++n)
                    scores(n);
                for(uint32_t n = 0; ok && n < steps; ++n)
                {
                    const uint32_t st = c % L::STAGES;
                    if(!wait(base + L::FULL + 8 * st, c / L::STAGES & 1u, 1))
                        break;
                    ++c;
                    if((from + n + 1) * TILE > end)
                    {
                        // rows behind the last token may hold anything: they are contracted over
                        for(uint32_t e = lane; e < TILE * (HD / 8); e += 32)
                        {
                            const uint32_t key = e / (HD / 8), piece = e % (HD / 8);
                            if((from + n) * TILE + key >= end)
                                *reinterpret_cast<uint4*>(smem + L::KV + st * L::TILE_BYTES + (piece / 8) * attn::BOX_BYTES + key * 128 + piece % 8 * 16)
                                    = make_uint4(0, 0, 0, 0);
                        }
                        ptx::fence_proxy_async_smem();
                        __syncwarp();
                    }
                    if(!wait(base + L::P_FULL + 8 * (n & 1u), n >> 1 & 1u, 2))
                        break;
                    if(attn::elect_one())
                    {
                        attn::mma_over_tokens<T, HD>(o_tmem + (n & 1u) * HD, s_tmem + (n & 1u) * TILE, base + L::KV + st * L::TILE_BYTES, n >= 2);
                        ptx::tc_commit(base + L::O_DONE + 8 * (n & 1u));
                        ptx::tc_commit(base + L::EMPTY + 8 * st);
                    }
                    if(n + 2 < steps)
                        scores(n + 2);
                }
                __syncwarp();
            }
            else
            {
                const uint32_t draft = live ? r / p.share : 0;
                const uint64_t bits  = !live ? 0 : p.tree ? __ldg(p.tree + size_t(b) * p.drafts + draft) : (uint64_t(2) << draft) - 1;
                attn::ScoreConst sc;
                sc.c = p.scale * LOG2E, sc.k2 = CAP ? p.scale / p.cap : 0.0f, sc.k1 = 2.0f * LOG2E * sc.k2, sc.cap2 = p.cap * LOG2E;
                sc.slope = BIAS && live ? __ldg(p.slopes + head * p.share + r % p.share) * LOG2E : 0.0f;
                // distances are taken from token `len`, so that they stay small and exact
                const int32_t at = BIAS && live ? (p.depths ? __ldg(p.depths + size_t(b) * p.drafts + draft) : int32_t(draft)) : 0;
                for(uint32_t n = u; ok && n < steps; n += 2, ++mine)
                {
                    ok = attn::wait_bounded_warp(base + L::S_FULL + 8 * u, mine & 1u, cta_abort, p.status,
                                                     TREE_TC_SOFTMAX << 24 | (blockIdx.x & 0xFFFFFFu));
                    if(!ok)
                        break;
                    ptx::tc_fence_after_sync();
                    const uint32_t  j0    = (from + n) * TILE;
                    const uint32_t* valid = reinterpret_cast<const uint32_t*>(smem + L::VALID) + (n & 7u) * 4;
                    const int32_t   rel0  = int32_t(int64_t(j0) - len); // place of the tile's first token behind the cached ones
                    const bool      masked = (valid[0] & valid[1] & valid[2] & valid[3]) != 0xFFFFFFFFu || rel0 + int32_t(TILE) > 0;
                    const uint32_t  s_row  = s_tmem + u * TILE + lane_tmem;
                    const auto      scores = [&](auto mask) {
                        return attn::row_max<true>(s_row, [&](int at_col, uint32_t(&v)[32]) {
                            const int  i      = at_col / 32;
                            const auto change = [&](auto how) {
                                constexpr bool MASK = decltype(mask)::value;
                                const uint32_t see  = MASK ? valid[i] & seen_of(bits, rel0 + 32 * i) : 0u;
#pragma unroll
                                for(int k = 0; k < 32; k += 2)
                                {
                                    uint64_t unused;
                                    float    dist = 0.0f, step = -1.0f, y[2];
                                    if constexpr(BIAS)
                                    {
                                        dist = static_cast<float>(at - rel0) - static_cast<float>(i * 32 + k);
                                        if constexpr(MASK)
                                            if(p.depths && rel0 + i * 32 + k + 1 >= 0) // drafted tokens stand at their depths
                                            {
                                                const int32_t rel = rel0 + i * 32 + k;
                                                const auto    d   = [&](int32_t to) {
                                                    return static_cast<float>(
                                                        at - (to >= 0 && to < int32_t(n_drafts) ? __ldg(p.depths + size_t(b) * p.drafts + to) : to));
                                                };
                                                dist = d(rel);
                                                step = d(rel + 1) - dist;
                                            }
                                    }
                                    attn::unpair(attn::score2<CAP, BIAS, decltype(how)::value>(sc, attn::pair(__uint_as_float(v[k]), __uint_as_float(v[k + 1])), dist, step, unused),
                                                 y[0], y[1]);
#pragma unroll
                                    for(int e = 0; e < 2; ++e)
                                    {
                                        if constexpr(MASK)
                                            if(!(see >> (k + e) & 1u))
                                                y[e] = -INFINITY;
                                        v[k + e] = __float_as_uint(y[e]);
                                    }
                                }
                            };
                            attn::bend<CAP>(sc, attn::tame<CAP>(sc, v), change);
                        });
                    };
                    const float top = masked ? scores(std::true_type{}) : scores(std::false_type{});
                    if(__any_sync(0xFFFFFFFFu, top > m + attn::RESCALE_STEP))
                    {
                        const float m2 = fmaxf(m, top), by = m2 == -INFINITY ? 1.0f : ex2(m - m2);
                        l *= by;
                        m = m2;
                        if(mine != 0)
                        {
                            ok = attn::wait_bounded_warp(base + L::O_DONE + 8 * u, (mine - 1) & 1u, cta_abort, p.status,
                                                             TREE_TC_SOFTMAX << 24 | 1u << 20 | (blockIdx.x & 0xFFFFFu));
                            if(!ok)
                                break;
                            ptx::tc_fence_after_sync();
#pragma unroll 1
                            for(uint32_t c = 0; c < HD; c += 32)
                            {
                                uint32_t w[32];
                                ptx::tmem_ld_32x32b_x32(o_tmem + u * HD + lane_tmem + c, w);
                                ptx::tmem_ld_wait();
#pragma unroll
                                for(int i = 0; i < 32; ++i)
                                    w[i] = __float_as_uint(__uint_as_float(w[i]) * by);
                                attn::tmem_st_32x32b_x32(o_tmem + u * HD + lane_tmem + c, w);
                            }
                        }
                    }
                    const float sub = m == -INFINITY ? 0.0f : m;
                    l += attn::weights<T>(s_row, 1.0f, -sub);
                    attn::tmem_st_wait();
                    ptx::tc_fence_before_sync();
                    __syncwarp();
                    if(lane == 0)
                        ptx::mbar_arrive(base + L::P_FULL + 8 * u);
                }
                if(ok && mine != 0)
                {
                    ok = attn::wait_bounded_warp(base + L::O_DONE + 8 * u, (mine - 1) & 1u, cta_abort, p.status,
                                                     TREE_TC_SOFTMAX << 24 | 2u << 20 | (blockIdx.x & 0xFFFFFu));
                    ptx::tc_fence_after_sync();
                }
            }
            if(m == -INFINITY && l != 0.0f)
                m = 0.0f; // nothing but NaN was seen, which is not the same as nothing
            __syncthreads(); // every product is done (or the block gives up): the ring is free
            if(!*cta_abort)
            {
                // the odd tiles' accumulator through shared memory, column by column: neighbouring rows lie next to one another
                float *other = reinterpret_cast<float*>(smem + L::KV) + (tid & 127u), *stats = reinterpret_cast<float*>(smem + L::STATS);
                if(u == 1 && warp < 8)
                {
                    stats[tid & 127u] = m, stats[TILE + (tid & 127u)] = l;
                    if(mine != 0)
#pragma unroll 1
                        for(uint32_t c = 0; c < HD; c += 32)
                        {
                            uint32_t w[32];
                            ptx::tmem_ld_32x32b_x32(o_tmem + HD + lane_tmem + c, w);
                            ptx::tmem_ld_wait();
#pragma unroll
                            for(int i = 0; i < 32; ++i)
                                other[(c + i) * TILE] = __uint_as_float(w[i]);
                        }
                }
                __syncthreads();
                if(u == 0)
                {
                    const float m1 = stats[tid], l1 = stats[TILE + tid], mx = fmaxf(m, m1);
                    const float by0 = m == -INFINITY ? 0.0f : ex2(m - mx), by1 = m1 == -INFINITY ? 0.0f : ex2(m1 - mx);
                    const float sum = by0 * l + by1 * l1;
                    const bool  one = p.splits == 1, two = steps > 1;
                    const float inv = !one ? 1.0f : sum > 0.0f ? 1.0f / sum : sum; // nothing visible: 0; NaN stays NaN
                    const size_t all_rows = size_t(p.batch) * p.heads_kv * rows;
                    const size_t part     = split * all_rows + (size_t(b) * p.heads_kv + head) * rows + r;
                    if(live && !one)
                        *reinterpret_cast<float2*>(p.part_ml + part * 2) = make_float2(mx, sum);
                    T* out = live ? o + row_of(p.o, b, r / p.share, head * p.share + r % p.share) : nullptr;
#pragma unroll 1
                    for(uint32_t c = 0; c < HD; c += 32)
                    {
                        uint32_t w[32];
                        __syncwarp();
                        if(steps != 0)
                        {
                            ptx::tmem_ld_32x32b_x32(o_tmem + lane_tmem + c, w);
                            ptx::tmem_ld_wait();
                        }
                        if(!live || (mx == -INFINITY && !one))
                            continue;
#pragma unroll
                        for(int i = 0; i < 32; ++i)
                        {
                            float y = by0 != 0.0f ? by0 * __uint_as_float(w[i]) : 0.0f; // accumulators that were not written are not used
                            if(two && by1 != 0.0f)
                                y = fmaf(by1, other[(c + i) * TILE], y);
                            w[i] = __float_as_uint(y * inv);
                        }
#pragma unroll
                        for(int i = 0; i < 8; ++i)
                            if(!one)
                                *reinterpret_cast<uint4*>(p.part_o + part * HD + c + 4 * i) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                            else if(i < 4 && c + 8 * i < p.dim)
                            {
                                uint32_t z[4];
#pragma unroll
                                for(int k = 0; k < 4; ++k)
                                    z[k] = attn::pack2<T>(__uint_as_float(w[8 * (i & 3) + 2 * k]), __uint_as_float(w[8 * (i & 3) + 2 * k + 1]));
                                *reinterpret_cast<uint4*>(out + c + 8 * i) = make_uint4(z[0], z[1], z[2], z[3]);
                            }
                    }
                }
            }
            ptx::tc_fence_before_sync();
            __syncthreads();
            if(*cta_abort)
            {
                // A wait was abandoned: copies or products may still be in flight.  Give them a bounded grace period.
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
    } // namespace attn_tree
} // namespace b200wmma
