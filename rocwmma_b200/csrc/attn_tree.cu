// Attention of drafted tokens over a paged cache: the entry point b200wmma_attn_tree.
//
// Bound: keys and values are read once.  Rows that share a key head (its query heads times the drafted tokens) are the rows of
// one product, so a block reads 64 tokens of the cache at a time into shared memory and every row uses them.  One warp walks the
// page table and issues the copies (TMA boxes of as many tokens as surely lie in one page; a page number outside the cache
// reads as zeros), the others wait for a stage and never for one another.  With up to 32 rows a token's 2 x head_dim values meet
// 4 x 32 x head_dim flops, which warp-level matrix instructions keep up with; tcgen05 tiles are 128 rows high and would be mostly
// empty (more rows take them: attn_tree_tc05.cuh).  One pass: running maximum and sum per row, the weights go from accumulators
// to operands in registers.
// The tokens are split over blocks where rows, heads and sequences alone do not fill the machine; a second kernel joins the
// parts in a fixed order.
// Measured, bf16, 32/8 heads x 128, one token each: 32 sequences of 4500 tokens 89 us (6.6 TB/s), of 3094 to 6000 tokens 94 us
// (6.4 TB/s; a copy, which also writes, reaches 6.5, the dgemv kernel, which only reads, 7.3); 8 drafted tokens each, 16 sequences
// of 8000: 89 us (5.9 TB/s); 5 drafted tokens, 8/2 heads x 64, one sequence of 120000, fp16 with slopes: 19-21 us (3.0-3.2 TB/s;
// 13 stages to a block, latency); one token after 8192: 13 us.
#include "attn_tc05.cuh"

namespace b200wmma
{
    namespace attn_tree
    {
        using attn::ex2;
        using attn::LOG2E;
        constexpr uint32_t MAX_DRAFTS = 64;
        constexpr uint32_t KEYS       = 64; // tokens of a stage
        constexpr uint32_t THREADS    = 160; // warps 0-3 compute, warp 4 copies
        constexpr uint32_t MAX_SPLITS = 256; // what 16 warps join

        struct Params
        {
            uint32_t batch, heads_q, heads_kv, share, dim, drafts, num_pages, page_size, ld_table, splits, tiles;
            uint32_t page_shift; // log2 of page_size, 32 where it is no power of two
            uint32_t box; // tokens of a copy: a power of two that divides page_size, at most 64
            unsigned* status;
            float    scale, cap;
            const float*    slopes;
            const int32_t * block_table, *lens, *n_drafts, *depths;
            const uint64_t* tree;
            attn::Strides   q, k, v, o;
            float *         part_o, *part_ml; // [split][row][HD], [split][row][2]; rows: batch x heads_kv x share x drafts
        };

        __device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at)
        {
            asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                         : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                         : "r"(at)
                         : "memory");
        }
        __device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t at)
        {
            asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                         : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                         : "r"(at)
                         : "memory");
        }
        template <typename T>
        __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
        {
            if constexpr(std::is_same<T, __half>::value)
                asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                             : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                             : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
            else
                asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                             : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                             : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
        }
        __device__ __forceinline__ uint32_t drafts_of(const Params& p, uint32_t b)
        {
            return p.n_drafts ? min(uint32_t(max(__ldg(p.n_drafts + b), 0)), p.drafts) : p.drafts;
        }
        // Bit i: a row whose tree word is `bits` sees the token that stands `rel` + i behind the cached ones (before them: rel < 0).
        __device__ __forceinline__ uint32_t seen_of(uint64_t bits, int32_t rel)
        {
            if(rel >= 64)
                return 0;
            if(rel >= 0)
                return uint32_t(bits >> rel);
            return rel <= -32 ? 0xFFFFFFFFu : uint32_t(bits << -rel) | ((1u << -rel) - 1u);
        }
        __device__ __forceinline__ int64_t row_of(const attn::Strides& s, uint32_t b, uint32_t t, uint32_t h)
        {
            return int64_t(b) * s.batch + int64_t(t) * s.token + int64_t(h) * s.head;
        }

    } // namespace attn_tree
} // namespace b200wmma

#include "attn_tree_tc05.cuh"

namespace b200wmma
{
    namespace attn_tree
    {
        enum Role : uint32_t
        {
            TREE_PRODUCER = 0x61,
            TREE_COMPUTE  = 0x62
        };
        template <uint32_t HD>
        struct Smem
        {
            static constexpr uint32_t HALF   = KEYS * 128; // 64 tokens x 64 elements, rows of 128 bytes with the 128-byte swizzle
            static constexpr uint32_t TILE   = HD / 64 * HALF; // a stage is a tile of keys and one of values
            static constexpr uint32_t STAGES = HD == 128 ? 3 : 4;
            static constexpr uint32_t SUMS = 4 * 16 * (HD + 2) * 4, RING = STAGES * 2 * TILE; // sums of the warps reuse the ring
            static constexpr uint32_t BARS  = RING;
            static constexpr uint32_t VALID = BARS + 16 * STAGES; // STAGES words of 64 bits: tokens that are there
            static constexpr uint32_t ABORT = VALID + 8 * STAGES;
            static constexpr uint32_t BYTES = ABORT + 16 + 1024;
            static_assert(RING >= SUMS, "");
        };

        // A block: 16 WM rows of one key head and the tokens of one split.  4 warps: WM along the rows, 4 / WM along the 64
        // tokens of a stage, each with its own running maximum.
        template <typename T, uint32_t HD, uint32_t WM, bool CAP, bool BIAS>
        __global__ void __launch_bounds__(THREADS, 2)
            tree_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ Params p,
                        const T* __restrict__ q, T* __restrict__ o)
        {
            using L               = Smem<HD>;
            constexpr uint32_t WN = 4 / WM, MINE = KEYS / WN, STAGES = L::STAGES; // tokens of a warp
            extern __shared__ uint8_t smem_raw[];
            const uint32_t     base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
            uint8_t*           smem = smem_raw + (base - ptx::smem_u32(smem_raw));
            const uint32_t     tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, g = lane >> 2, t = lane & 3u;
            const uint32_t     wm = warp % WM, wn = (warp & 3u) / WM;
            uint32_t*          valid     = reinterpret_cast<uint32_t*>(smem + L::VALID);
            volatile uint32_t* cta_abort = reinterpret_cast<uint32_t*>(smem + L::ABORT);
            if(tid == 0)
            {
                ptx::prefetch_tensormap(&map_k);
                ptx::prefetch_tensormap(&map_v);
                for(uint32_t s = 0; s < STAGES; ++s)
                {
                    ptx::mbar_init(base + L::BARS + 16 * s, 1); // full
                    ptx::mbar_init(base + L::BARS + 16 * s + 8, 4); // empty
                }
                *cta_abort = 0u;
                ptx::fence_barrier_init();
                ptx::fence_proxy_async_smem();
            }

            uint32_t       x     = blockIdx.x;
            const uint32_t split = x % p.splits;
            x /= p.splits;
            const uint32_t tile = x % p.tiles;
            x /= p.tiles;
            const uint32_t head = x % p.heads_kv, b = x / p.heads_kv, rows = p.share * p.drafts;
            const uint32_t n_drafts = drafts_of(p, b);
            const int64_t  len      = max(__ldg(p.lens + b), 0);
            const uint32_t end      = n_drafts ? uint32_t(min(len + n_drafts, int64_t(p.ld_table) * p.page_size)) : 0u;
            const uint32_t stages = (end + KEYS - 1) / KEYS, from = uint32_t(uint64_t(stages) * split / p.splits);
            const uint32_t steps = uint32_t(uint64_t(stages) * (split + 1) / p.splits) - from;
            const size_t   all_rows = size_t(p.batch) * p.heads_kv * rows, row_base = (size_t(b) * p.heads_kv + head) * rows;

            // this lane's rows: g and g + 8 of the warp's 16; row r is drafted token r / share of query head head * share + r % share
            uint32_t r[2], draft[2];
            bool     live[2];
            float    slope[2];
            int32_t  at[2];
            uint64_t bits[2];
#pragma unroll
            for(int i = 0; i < 2; ++i)
            {
                r[i]     = tile * 16 * WM + wm * 16 + g + 8 * i;
                draft[i] = r[i] / p.share;
                live[i]  = r[i] < rows && draft[i] < n_drafts;
                bits[i]  = !live[i] ? 0 : p.tree ? __ldg(p.tree + size_t(b) * p.drafts + draft[i]) : (uint64_t(2) << draft[i]) - 1;
                slope[i] = BIAS && live[i] ? __ldg(p.slopes + head * p.share + r[i] % p.share) * LOG2E : 0.0f;
                // distances are taken from token `len`, so that they stay small and exact
                at[i] = BIAS && live[i] ? (p.depths ? __ldg(p.depths + size_t(b) * p.drafts + draft[i]) : int32_t(draft[i])) : 0;
            }
            attn::ScoreConst sc;
            sc.c = p.scale * LOG2E, sc.k2 = CAP ? p.scale / p.cap : 0.0f, sc.k1 = 2.0f * LOG2E * sc.k2, sc.cap2 = p.cap * LOG2E, sc.slope = 0.0f;

            uint32_t qf[HD / 16][4];
#pragma unroll
            for(uint32_t c = 0; c < HD / 16; ++c)
#pragma unroll
                for(int i = 0; i < 4; ++i)
                {
                    const uint32_t d = c * 16 + t * 2 + 8 * (i >> 1);
                    qf[c][i]         = live[i & 1] && d < p.dim
                                           ? *reinterpret_cast<const uint32_t*>(q + row_of(p.q, b, draft[i & 1], head * p.share + r[i & 1] % p.share) + d)
                                           : 0u;
                }

            __syncthreads();
            ptx::grid_dep_launch_dependents();
            bool ok = true;
            if(warp == 4)
            {
                const uint32_t boxes = KEYS / p.box; // a lane takes boxes lane, lane + 32
                int32_t        page[2], slot[2];
                const auto     ask = [&](uint32_t i) { // starts the loads of the pages of step i
#pragma unroll
                    for(int u = 0; u < 2; ++u)
                    {
                        const uint32_t at_box = lane + 32 * u, j = (from + i) * KEYS + at_box * p.box;
                        page[u] = -1, slot[u] = 0;
                        if(at_box < boxes && i < steps && j < end)
                        {
                            const uint32_t n = p.page_shift < 32 ? j >> p.page_shift : j / p.page_size;
                            slot[u]          = int32_t(j - n * p.page_size);
                            page[u]          = __ldg(p.block_table + size_t(b) * p.ld_table + n);
                        }
                    }
                };
                ask(0);
                for(uint32_t i = 0; i < steps; ++i)
                {
                    const uint32_t st = i % STAGES, full = base + L::BARS + 16 * st, stage = base + st * 2 * L::TILE;
                    const int32_t  pg[2] = {page[0], page[1]}, sl[2] = {slot[0], slot[1]};
                    ask(i + 1);
                    ok = attn::wait_bounded_warp(full + 8, (i / STAGES & 1u) ^ 1u, cta_abort, p.status,
                                                     TREE_PRODUCER << 24 | (blockIdx.x & 0xFFFFFFu));
                    if(!ok)
                        break;
                    // which of the 64 tokens are there: their box's page is, and they lie before the end
                    const uint64_t box_bits = p.box < 64 ? (uint64_t(1) << p.box) - 1 : ~uint64_t(0);
                    uint64_t       there    = 0;
#pragma unroll
                    for(int u = 0; u < 2; ++u)
                        if(uint32_t(pg[u]) < p.num_pages && lane + 32 * u < boxes)
                            there |= box_bits << ((lane + 32 * u) * p.box);
                    const uint32_t left = end - (from + i) * KEYS;
                    uint32_t       lo = __reduce_or_sync(0xFFFFFFFFu, uint32_t(there)), hi = __reduce_or_sync(0xFFFFFFFFu, uint32_t(there >> 32));
                    if(left < 64)
                    {
                        lo &= left < 32 ? (1u << left) - 1u : 0xFFFFFFFFu;
                        hi &= left <= 32 ? 0u : (1u << (left - 32)) - 1u;
                    }
                    if(lane == 0)
                    {
                        valid[2 * st] = lo, valid[2 * st + 1] = hi;
                        ptx::mbar_arrive_expect_tx(full, 2 * L::TILE);
                    }
                    __syncwarp();
#pragma unroll
                    for(int u = 0; u < 2; ++u)
                    {
                        const uint32_t at_box = lane + 32 * u;
                        if(at_box < boxes)
                        {
                            // a page that is not there: one behind the last, which reads as zeros
                            const int32_t c3 = uint32_t(pg[u]) < p.num_pages ? pg[u] : int32_t(p.num_pages);
#pragma unroll
                            for(uint32_t h = 0; h < HD / 64; ++h)
                            {
                                const uint32_t to = stage + h * L::HALF + at_box * p.box * 128;
                                attn::tma_load_4d(to, &map_k, h * 64, sl[u], head, c3, full);
                                attn::tma_load_4d(to + L::TILE, &map_v, h * 64, sl[u], head, c3, full);
                            }
                        }
                    }
                }
            }
            float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, acc[HD / 8][4];
#pragma unroll
            for(uint32_t i = 0; i < HD / 8; ++i)
                acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;

            for(uint32_t i = 0; warp < 4 && i < steps; ++i)
            {
                const uint32_t st = i % STAGES;
                ok = attn::wait_bounded_warp(base + L::BARS + 16 * st, i / STAGES & 1u, cta_abort, p.status,
                                                 TREE_COMPUTE << 24 | (blockIdx.x & 0xFFFFFFu));
                if(!ok)
                    break;
                const uint32_t keys_at = base + st * 2 * L::TILE + wn * MINE * 128, values_at = keys_at + L::TILE;
                float          s[MINE / 8][4];
#pragma unroll
                for(uint32_t n = 0; n < MINE / 8; ++n)
                {
                    s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
                    // 8 tokens x 32 elements at a time: lanes 8j .. 8j + 7 give the rows of piece j
                    const uint32_t key = n * 8 + (lane & 7u), piece = lane >> 3;
#pragma unroll
                    for(uint32_t c = 0; c < HD / 32; ++c)
                    {
                        uint32_t f[4];
                        ldmatrix4(f, keys_at + (c / 2) * L::HALF + key * 128 + ((((c % 2) * 4 + piece) ^ (key & 7u)) << 4));
                        mma<T>(s[n], qf[2 * c], f[0], f[1]);
                        mma<T>(s[n], qf[2 * c + 1], f[2], f[3]);
                    }
                }
                // scores in units of log 2, masked
                const uint32_t j0 = (from + i) * KEYS + wn * MINE;
                const uint32_t v0 = valid[2 * st], v1 = valid[2 * st + 1];
                const bool     masked = (v0 & v1) != 0xFFFFFFFFu || (from + i + 1) * KEYS > len;
                const int32_t  rel0   = int32_t(int64_t(j0) - len); // place of the warp's first token behind the cached ones
                float          top[2] = {-INFINITY, -INFINITY};
                const auto     scores = [&](auto mask, auto how) {
                    constexpr bool MASK = decltype(mask)::value;
                    uint32_t       see[2][(MINE + 31) / 32]; // of this lane's first token on
                    if constexpr(MASK)
                    {
#pragma unroll
                        for(uint32_t w = 0; w < (MINE + 31) / 32; ++w)
                        {
                            const uint32_t bit = wn * MINE + 32 * w, there = (bit < 32 ? v0 : v1) >> (bit & 31u);
                            see[0][w] = (there & seen_of(bits[0], rel0 + int32_t(32 * w))) >> (t * 2);
                            see[1][w] = (there & seen_of(bits[1], rel0 + int32_t(32 * w))) >> (t * 2);
                        }
                    }
#pragma unroll
                    for(uint32_t n = 0; n < MINE / 8; ++n)
#pragma unroll
                        for(int h = 0; h < 2; ++h)
                        {
                            const uint32_t off  = n * 8; // and t * 2: the first of two tokens
                            float          dist = 0.0f, step = -1.0f, y[2];
                            if constexpr(BIAS)
                            {
                                dist = static_cast<float>(at[h] - rel0 - int32_t(t * 2)) - static_cast<float>(off);
                                if constexpr(MASK)
                                {
                                    const int32_t rel = rel0 + int32_t(off + t * 2);
                                    if(rel + 1 >= 0 && p.depths) // drafted tokens stand at their depths
                                    {
                                        const auto d = [&](uint32_t e) {
                                            const int32_t to = rel + int32_t(e);
                                            return static_cast<float>(
                                                at[h] - (to >= 0 && j0 + off + t * 2 + e < end ? __ldg(p.depths + size_t(b) * p.drafts + to) : to));
                                        };
                                        dist = d(0);
                                        step = d(1) - dist;
                                    }
                                }
                            }
                            sc.slope = slope[h];
                            uint64_t unused;
                            attn::unpair(attn::score2<CAP, BIAS, decltype(how)::value>(sc, attn::pair(s[n][2 * h], s[n][2 * h + 1]), dist, step, unused),
                                         y[0], y[1]);
#pragma unroll
                            for(int e = 0; e < 2; ++e)
                            {
                                if constexpr(MASK)
                                    if(!(see[h][off / 32] >> ((off & 31u) + e) & 1u))
                                        y[e] = -INFINITY;
                                s[n][2 * h + e] = y[e];
                                top[h]          = fmaxf(top[h], y[e]);
                            }
                        }
                };
                float largest = 0.0f;
                if constexpr(CAP)
#pragma unroll
                    for(uint32_t n = 0; n < MINE / 8; ++n)
#pragma unroll
                        for(int e = 0; e < 4; ++e)
                            largest = fmaxf(largest, fabsf(s[n][e]));
                const auto masked_scores = [&](auto mask) {
                    attn::bend<CAP>(sc, attn::tame<CAP>(sc, largest), [&](auto how) { scores(mask, how); });
                };
                if(masked)
                    masked_scores(std::true_type{});
                else
                    masked_scores(std::false_type{});
#pragma unroll
                for(int h = 0; h < 2; ++h)
                {
                    top[h] = fmaxf(top[h], __shfl_xor_sync(0xFFFFFFFFu, top[h], 1));
                    top[h] = fmaxf(top[h], __shfl_xor_sync(0xFFFFFFFFu, top[h], 2));
                }
                if(__any_sync(0xFFFFFFFFu, top[0] > m[0] + attn::RESCALE_STEP || top[1] > m[1] + attn::RESCALE_STEP))
                {
                    float by[2];
#pragma unroll
                    for(int h = 0; h < 2; ++h)
                    {
                        const float m2 = fmaxf(m[h], top[h]);
                        by[h]          = m2 == -INFINITY ? 1.0f : ex2(m[h] - m2);
                        m[h]           = m2;
                        l[h] *= by[h];
                    }
#pragma unroll
                    for(uint32_t c = 0; c < HD / 8; ++c)
                        acc[c][0] *= by[0], acc[c][1] *= by[0], acc[c][2] *= by[1], acc[c][3] *= by[1];
                }
                const float sub[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
                uint32_t    pf[MINE / 16][4];
#pragma unroll
                for(uint32_t n = 0; n < MINE / 8; ++n)
                {
                    float w[4];
#pragma unroll
                    for(int e = 0; e < 4; ++e)
                        w[e] = ex2(s[n][e] - sub[e >> 1]);
                    l[0] += w[0] + w[1], l[1] += w[2] + w[3];
                    pf[n / 2][2 * (n & 1)] = attn::pack2<T>(w[0], w[1]), pf[n / 2][2 * (n & 1) + 1] = attn::pack2<T>(w[2], w[3]);
                }
                // rows behind the last token hold anything; only the last step has them, whose stage is not filled again
                if((from + i + 1) * KEYS > end)
                {
                    for(uint32_t e = lane; e < MINE * (HD / 8); e += 32)
                    {
                        const uint32_t key = e / (HD / 8), c = e % (HD / 8);
                        if(j0 + key >= end)
                            *reinterpret_cast<uint4*>(smem + (values_at - base) + (c / 8) * L::HALF + key * 128 + c % 8 * 16) = make_uint4(0, 0, 0, 0);
                    }
                    __syncwarp();
                }
#pragma unroll
                for(uint32_t n = 0; n < MINE / 16; ++n)
                {
                    // 16 tokens x 16 elements at a time: lanes 0-15 give the tokens of the first 8 elements, 16-31 of the next
                    const uint32_t key = n * 16 + (lane & 15u);
#pragma unroll
                    for(uint32_t c = 0; c < HD / 16; ++c)
                    {
                        uint32_t f[4];
                        ldmatrix4_trans(f, values_at + (c / 4) * L::HALF + key * 128 + ((((c % 4) * 2 + (lane >> 4)) ^ (key & 7u)) << 4));
                        mma<T>(acc[2 * c], pf[n], f[0], f[1]);
                        mma<T>(acc[2 * c + 1], pf[n], f[2], f[3]);
                    }
                }
                __syncwarp();
                if(lane == 0)
                    ptx::mbar_arrive(base + L::BARS + 16 * st + 8);
            }
#pragma unroll
            for(int h = 0; h < 2; ++h)
            {
                l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], 1);
                l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], 2);
                if(m[h] == -INFINITY && l[h] != 0.0f)
                    m[h] = 0.0f; // nothing but NaN was seen, which is not the same as nothing
            }
            // join the warps that share the rows: [warp][16 rows][HD] sums, [warp][16 rows] maximum and sum of weights
            __syncthreads();
            if(*cta_abort)
            {
                // A wait was abandoned: copies may still be in flight.  Give them a bounded grace period, then leave.
                const uint64_t t0 = ptx::globaltimer_ns();
                while(ptx::globaltimer_ns() - t0 < 2000000ull)
                    __nanosleep(1000);
                return;
            }
            float *sums = reinterpret_cast<float*>(smem), *stats = sums + 4 * 16 * HD;
            if(warp < 4)
            {
#pragma unroll
                for(uint32_t c = 0; c < HD / 8; ++c)
#pragma unroll
                    for(int h = 0; h < 2; ++h)
                        *reinterpret_cast<float2*>(sums + (warp * 16 + g + 8 * h) * HD + c * 8 + t * 2) = make_float2(acc[c][2 * h], acc[c][2 * h + 1]);
                if(t == 0)
#pragma unroll
                    for(int h = 0; h < 2; ++h)
                        stats[(warp * 16 + g + 8 * h) * 2] = m[h], stats[(warp * 16 + g + 8 * h) * 2 + 1] = l[h];
            }
            __syncthreads();
            // four elements of a row to a thread
            for(uint32_t e = tid; e < 16 * WM * (HD / 4); e += THREADS)
            {
                const uint32_t row = e / (HD / 4), d = e % (HD / 4) * 4, rr = tile * 16 * WM + row;
                if(rr >= rows || rr / p.share >= n_drafts)
                    continue;
                float mx = -INFINITY;
#pragma unroll
                for(uint32_t w = 0; w < WN; ++w)
                    mx = fmaxf(mx, stats[((w * WM + row / 16) * 16 + row % 16) * 2]);
                float  sum = 0.0f;
                float4 y   = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if(mx != -INFINITY)
#pragma unroll
                    for(uint32_t w = 0; w < WN; ++w)
                    {
                        const uint32_t at_w = (w * WM + row / 16) * 16 + row % 16;
                        const float    by   = ex2(stats[at_w * 2] - mx);
                        const float4   z    = *reinterpret_cast<const float4*>(sums + at_w * HD + d);
                        sum += by * stats[at_w * 2 + 1];
                        y.x += by * z.x, y.y += by * z.y, y.z += by * z.z, y.w += by * z.w;
                    }
                if(p.splits == 1)
                {
                    const float inv = sum > 0.0f ? 1.0f / sum : sum; // nothing visible: 0; NaN stays NaN
                    if(d < p.dim)
                        *reinterpret_cast<uint2*>(o + row_of(p.o, b, rr / p.share, head * p.share + rr % p.share) + d)
                            = make_uint2(attn::pack2<T>(y.x * inv, y.y * inv), attn::pack2<T>(y.z * inv, y.w * inv));
                }
                else
                {
                    const size_t part = split * all_rows + row_base + rr;
                    *reinterpret_cast<float4*>(p.part_o + part * HD + d) = y;
                    if(d == 0)
                        *reinterpret_cast<float2*>(p.part_ml + part * 2) = make_float2(mx, sum);
                }
            }
        }

        // Joins the splits of a row: W warps with up to PER splits each, whose parts are all on their way before the first maximum is
        // known (148 splits of 8 rows: 2.6 us behind the first kernel, 6.8 with a few loads at a time); HD / 32 elements to a lane;
        // everything in a fixed order.
        template <uint32_t W>
        struct Join
        {
            static constexpr uint32_t PER = W == 16 ? 16 : 8, ROWS = W == 16 ? 1 : 8 / W, THREADS = 32 * W * ROWS; // rows of a block
        };
        template <typename T, uint32_t HD, uint32_t W>
        __global__ void __launch_bounds__(Join<W>::THREADS) join_kernel(const __grid_constant__ Params p, T* __restrict__ o)
        {
            constexpr uint32_t E = HD / 32, PER = Join<W>::PER, ROWS = Join<W>::ROWS;
            using Piece          = std::conditional_t<E == 4, float4, float2>;
            __shared__ float   red[ROWS][W][HD], stats[ROWS][W][2];
            const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, slot = warp / W, w = warp % W;
            const uint32_t rows = p.share * p.drafts, row = blockIdx.x * ROWS + slot, all_rows = p.batch * p.heads_kv * rows;
            const uint32_t r = row % rows, head = row / rows % p.heads_kv, b = row / rows / p.heads_kv, draft = r / p.share;
            const bool     live = row < all_rows && draft < drafts_of(p, b);
            const uint32_t first = w * PER, mine = live && first < p.splits ? min(PER, p.splits - first) : 0;
            ptx::grid_dep_wait(); // before anything leaves: the kernel may not end before the one it follows
            float2 ml = make_float2(-INFINITY, 0.0f);
            if(lane < mine)
                ml = *reinterpret_cast<const float2*>(p.part_ml + (size_t(first + lane) * all_rows + row) * 2);
            Piece part[PER];
#pragma unroll
            for(uint32_t k = 0; k < PER; ++k)
                if(k < mine)
                    part[k] = *reinterpret_cast<const Piece*>(p.part_o + (size_t(first + k) * all_rows + row) * HD + lane * E);
            float mx = ml.x;
#pragma unroll
            for(int d = 16; d > 0; d >>= 1)
                mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, d));
            const float by  = ml.x == -INFINITY ? 0.0f : ex2(ml.x - mx); // splits without a visible token have written no sums
            float       sum = ml.x == -INFINITY ? 0.0f : by * ml.y, y[E] = {};
#pragma unroll
            for(int d = 16; d > 0; d >>= 1)
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
#pragma unroll
            for(uint32_t k = 0; k < PER; ++k)
            {
                const float f = __shfl_sync(0xFFFFFFFFu, by, k);
                if(k < mine && f != 0.0f) // NaN counts
                {
                    const float* from = reinterpret_cast<const float*>(&part[k]);
#pragma unroll
                    for(uint32_t e = 0; e < E; ++e)
                        y[e] = fmaf(f, from[e], y[e]);
                }
            }
            if constexpr(W > 1)
            {
#pragma unroll
                for(uint32_t e = 0; e < E; ++e)
                    red[slot][w][lane * E + e] = y[e], y[e] = 0.0f;
                if(lane == 0)
                    stats[slot][w][0] = mx, stats[slot][w][1] = sum;
                __syncthreads();
                if(w != 0)
                    return;
                mx = -INFINITY, sum = 0.0f;
#pragma unroll
                for(uint32_t i = 0; i < W; ++i)
                    mx = fmaxf(mx, stats[slot][i][0]);
#pragma unroll
                for(uint32_t i = 0; i < W; ++i)
                {
                    const float f = stats[slot][i][0] == -INFINITY ? 0.0f : ex2(stats[slot][i][0] - mx);
                    if(f != 0.0f)
                    {
                        sum = fmaf(f, stats[slot][i][1], sum);
#pragma unroll
                        for(uint32_t e = 0; e < E; ++e)
                            y[e] = fmaf(f, red[slot][i][lane * E + e], y[e]);
                    }
                }
            }
            const float inv = sum > 0.0f ? 1.0f / sum : sum;
            if(live && lane * E < p.dim)
            {
                uint32_t* out = reinterpret_cast<uint32_t*>(o + row_of(p.o, b, draft, head * p.share + r % p.share) + lane * E);
#pragma unroll
                for(uint32_t e = 0; e < E; e += 2)
                    out[e / 2] = attn::pack2<T>(y[e] * inv, y[e + 1] * inv);
            }
        }
        template <typename T, uint32_t HD, uint32_t W>
        static int launch_join(const Params& p, void* o, cudaStream_t stream)
        {
            const uint32_t     rows = p.batch * p.heads_kv * p.share * p.drafts;
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3(ceil_div(rows, Join<W>::ROWS)), cfg.blockDim = dim3(Join<W>::THREADS), cfg.stream = stream;
            // launched while the last blocks of the kernel before it still run; it waits for them before it reads
            cudaLaunchAttribute attr{};
            attr.id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
            attr.val.programmaticStreamSerializationAllowed = 1;
            cfg.attrs = &attr, cfg.numAttrs = 1;
            B200_CHECK_CUDA(cudaLaunchKernelEx(&cfg, join_kernel<T, HD, W>, p, static_cast<T*>(o)));
            return B200WMMA_OK;
        }

        // More rows than 32 take the tcgen05 form: 8 drafted tokens x 4 heads (32 rows) over 16 x 8000 tokens take 92 us with
        // warp-level products and 145 us with tiles of 128 rows that are mostly empty; 128 rows took 212 us and 69 us
        // when this was chosen (32 rows now 89 us).
        constexpr uint32_t WARP_ROWS = 32;
        static bool many_rows(uint32_t rows)
        {
            return rows > WARP_ROWS;
        }
        static uint32_t rows_of_block(uint32_t rows)
        {
            return many_rows(rows) ? TILE : rows <= 16 ? 16 : 32;
        }
        // Splits of the tokens: what fills one round of blocks (two per SM, or one of the tcgen05 form), but at least 256 (512)
        // tokens to a block if a sequence is as long as its table allows.  Two rounds measured 8 % slower for 32 equal sequences,
        // 3 % faster for lengths between half and all of the longest; a block costs 10 us before its second tile.
        static uint32_t splits_of(uint32_t batch, uint32_t heads_kv, uint32_t rows, uint32_t max_tokens)
        {
            const uint64_t blocks = uint64_t(batch) * heads_kv * ceil_div(rows, rows_of_block(rows));
            const uint64_t slots = many_rows(rows) ? 148 : 2 * 148, least = many_rows(rows) ? 4 * TILE : 4 * KEYS;
            const uint64_t want = slots / blocks, most = (uint64_t(max_tokens) + least - 1) / least;
            const uint64_t n = want < most ? want : most;
            return n < 1 ? 1u : n > MAX_SPLITS ? MAX_SPLITS : uint32_t(n);
        }
        // batch x heads_q x drafts (at most 64) counts in 31 bits
        static bool few_rows(uint32_t batch, uint32_t drafts, uint32_t heads_q)
        {
            const uint64_t most = uint64_t(1) << 31, rows = uint64_t(batch) * heads_q;
            return rows < most && rows * drafts < most;
        }
        static uint32_t padded_dim(uint32_t dim)
        {
            return dim <= 64 ? 64 : 128;
        }

        // WM: rows of a block of the warp-level kernel in units of 16; 0: the tcgen05 kernel
        template <typename T, uint32_t HD, uint32_t WM, bool CAP, bool BIAS>
        static int launch(const Params& p, const CUtensorMap (&maps)[2], const void* q, void* o, cudaStream_t stream)
        {
            const uint32_t grid = p.batch * p.heads_kv * p.tiles * p.splits;
            static attn::Allowed allowed;
            if constexpr(WM == 0)
            {
                auto kern = tree_tc05_kernel<T, HD, CAP, BIAS>;
                if(int e = attn::allow_smem(reinterpret_cast<const void*>(kern), TcSmem<HD>::BYTES, allowed))
                    return e;
                kern<<<grid, TC_THREADS, TcSmem<HD>::BYTES, stream>>>(maps[0], maps[1], p, static_cast<const T*>(q), static_cast<T*>(o));
            }
            else
            {
                auto kern = tree_kernel<T, HD, WM, CAP, BIAS>;
                if(int e = attn::allow_smem(reinterpret_cast<const void*>(kern), Smem<HD>::BYTES, allowed))
                    return e;
                kern<<<grid, THREADS, Smem<HD>::BYTES, stream>>>(maps[0], maps[1], p, static_cast<const T*>(q), static_cast<T*>(o));
            }
            B200_CHECK_CUDA(cudaGetLastError());
            if(p.splits == 1)
                return B200WMMA_OK;
            return p.splits <= Join<1>::PER       ? launch_join<T, HD, 1>(p, o, stream)
                   : p.splits <= 4 * Join<4>::PER ? launch_join<T, HD, 4>(p, o, stream) : launch_join<T, HD, 16>(p, o, stream);
        }
        template <typename T, uint32_t HD, uint32_t WM>
        static int launch_scores(const Params& p, const CUtensorMap (&maps)[2], const void* q, void* o, cudaStream_t stream)
        {
            if(p.cap > 0.0f)
                return p.slopes ? launch<T, HD, WM, true, true>(p, maps, q, o, stream) : launch<T, HD, WM, true, false>(p, maps, q, o, stream);
            return p.slopes ? launch<T, HD, WM, false, true>(p, maps, q, o, stream) : launch<T, HD, WM, false, false>(p, maps, q, o, stream);
        }
        template <typename T, uint32_t HD>
        static int launch_rows(const Params& p, const CUtensorMap (&maps)[2], const void* q, void* o, cudaStream_t stream)
        {
            const uint32_t rows = p.share * p.drafts;
            return many_rows(rows) ? launch_scores<T, HD, 0>(p, maps, q, o, stream)
                   : rows <= 16    ? launch_scores<T, HD, 1>(p, maps, q, o, stream) : launch_scores<T, HD, 2>(p, maps, q, o, stream);
        }
        template <typename T>
        static int launch_dim(const Params& p, const CUtensorMap (&maps)[2], const void* q, void* o, cudaStream_t stream)
        {
            return p.dim <= 64 ? launch_rows<T, 64>(p, maps, q, o, stream) : launch_rows<T, 128>(p, maps, q, o, stream);
        }
    } // namespace attn_tree
} // namespace b200wmma

using namespace b200wmma;

extern "C" size_t b200wmma_attn_tree_workspace_bytes(uint32_t batch, uint32_t drafts, uint32_t heads_q, uint32_t heads_kv,
                                                     uint32_t head_dim, uint32_t max_tokens)
{
    // shapes that the call refuses need nothing
    if(!batch || !drafts || drafts > attn_tree::MAX_DRAFTS || !heads_q || !heads_kv || heads_q % heads_kv != 0
       || !attn_tree::few_rows(batch, drafts, heads_q))
        return 0;
    const uint32_t rows = heads_q / heads_kv * drafts, splits = attn_tree::splits_of(batch, heads_kv, rows, max_tokens);
    return splits == 1 ? 0 : size_t(splits) * batch * heads_kv * rows * (attn_tree::padded_dim(head_dim) + 2) * sizeof(float);
}

extern "C" int b200wmma_attn_tree(const b200wmma_attn_args* a, uint32_t drafts, const void* q, const void* k_cache, const void* v_cache,
                                  uint32_t num_pages, uint32_t page_size, const int32_t* block_table, uint32_t ld_table,
                                  const int32_t* lens, const int32_t* n_drafts, const uint64_t* tree, const int32_t* depths, void* o,
                                  void* workspace, size_t workspace_bytes, void* stream)
{
    clear_error();
    static const char* const who = "attn_tree";
    if(int e = attn::check_common(who, a))
        return e;
    B200_REQUIRE(!a->len_q && !a->len_kv && !a->causal && !a->prefix && !a->doc_q && !a->doc_kv, B200WMMA_ERR_INVALID_ARG,
                 "%s: len_q, len_kv, causal, prefix and documents belong to attn_fwd and must be zero", who);
    B200_REQUIRE(drafts >= 1 && drafts <= attn_tree::MAX_DRAFTS, B200WMMA_ERR_UNSUPPORTED, "%s: drafts must be 1 to %u", who,
                 attn_tree::MAX_DRAFTS);
    B200_REQUIRE(num_pages && page_size && ld_table, B200WMMA_ERR_INVALID_ARG, "%s: num_pages, page_size and ld_table must be non-zero", who);
    B200_REQUIRE(num_pages < (1u << 31) && uint64_t(ld_table) * page_size < (uint64_t(1) << 31), B200WMMA_ERR_UNSUPPORTED,
                 "%s: num_pages and ld_table x page_size must be below 2^31", who);
    B200_REQUIRE(block_table && lens, B200WMMA_ERR_INVALID_ARG, "%s: block_table and lens must be non-null", who);
    B200_REQUIRE(attn_tree::few_rows(a->batch, drafts, a->heads_q), B200WMMA_ERR_UNSUPPORTED,
                 "%s: batch x heads_q x drafts must be below 2^31", who);
    attn_tree::Params p{};
    if(int e = attn::check_strides(who, "q", q, a->q, a->batch, drafts, a->heads_q, &p.q))
        return e;
    if(int e = attn::check_strides(who, "k_cache", k_cache, a->k, num_pages, page_size, a->heads_kv, &p.k))
        return e;
    if(int e = attn::check_strides(who, "v_cache", v_cache, a->v, num_pages, page_size, a->heads_kv, &p.v))
        return e;
    if(int e = attn::check_strides(who, "o", o, a->o, a->batch, drafts, a->heads_q, &p.o))
        return e;
    B200_REQUIRE(attn::disjoint(p.o, a->batch, drafts, a->heads_q, a->head_dim), B200WMMA_ERR_INVALID_ARG, "%s: rows of o overlap", who);
    const uint32_t max_tokens = ld_table * page_size;
    const size_t   need       = b200wmma_attn_tree_workspace_bytes(a->batch, drafts, a->heads_q, a->heads_kv, a->head_dim, max_tokens);
    B200_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), B200WMMA_ERR_INVALID_ARG, "%s: workspace of %zu bytes needed, %zu given",
                 who, need, workspace ? workspace_bytes : size_t(0));
    B200_REQUIRE(need == 0 || aligned16(workspace), B200WMMA_ERR_ALIGNMENT, "%s: workspace must be 16-byte aligned", who);
    if(int e = require_sm100())
        return e;
    p.batch = a->batch, p.heads_q = a->heads_q, p.heads_kv = a->heads_kv, p.share = a->heads_q / a->heads_kv, p.dim = a->head_dim;
    p.page_shift = 32;
    for(uint32_t i = 0; i < 32; ++i)
        if(page_size == 1u << i)
            p.page_shift = i;
    p.drafts = drafts, p.num_pages = num_pages, p.page_size = page_size, p.ld_table = ld_table, p.scale = a->scale, p.cap = a->cap;
    p.slopes = a->slopes, p.block_table = block_table, p.lens = lens, p.n_drafts = n_drafts, p.depths = depths, p.tree = tree;
    const uint32_t rows = p.share * drafts;
    p.splits  = attn_tree::splits_of(p.batch, p.heads_kv, rows, max_tokens);
    p.tiles   = ceil_div(rows, attn_tree::rows_of_block(rows));
    p.part_o  = static_cast<float*>(workspace);
    p.part_ml = p.part_o + size_t(p.splits) * p.batch * p.heads_kv * rows * attn_tree::padded_dim(p.dim);
    p.box = 64;
    while(page_size % p.box != 0)
        p.box /= 2;
    if(int e = status_word_ptr(&p.status))
        return e;
    CUtensorMap maps[2];
    if(int e = attn::make_map(&maps[0], a->data_type, k_cache, p.dim, page_size, p.heads_kv, num_pages, p.k, p.box))
        return e;
    if(int e = attn::make_map(&maps[1], a->data_type, v_cache, p.dim, page_size, p.heads_kv, num_pages, p.v, p.box))
        return e;
    return a->data_type == B200WMMA_OUT_F16 ? attn_tree::launch_dim<__half>(p, maps, q, o, as_stream(stream))
                                            : attn_tree::launch_dim<__nv_bfloat16>(p, maps, q, o, as_stream(stream));
}
