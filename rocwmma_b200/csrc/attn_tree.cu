// Attention of drafted tokens over a paged cache: the entry point b200wmma_attn_tree.
//
// Bound: keys and values are read once.  Rows that share a key head (its query heads times the drafted tokens) are the rows of
// one product, so a block reads 64 tokens of the cache at a time into shared memory (a ring of asynchronous copies, 16 bytes
// each, rows found through the page table) and every row uses them.  With up to 64 rows a token's 2 x head_dim values meet
// 4 x 64 x head_dim flops, which warp-level matrix instructions keep up with; tcgen05 tiles would be 128 rows high and mostly
// empty.  One pass: running maximum and sum per row, the weights go from accumulators to operands in registers.
// The tokens are split over blocks where rows, heads and sequences alone do not fill the machine; a second kernel joins the
// parts in a fixed order.
#include "attn_tc05.cuh"

namespace b200wmma
{
    namespace attn_tree
    {
        using attn::ex2;
        using attn::LOG2E;
        constexpr uint32_t MAX_DRAFTS = 64;
        constexpr uint32_t KEYS       = 64; // tokens of a stage
        constexpr uint32_t STAGES     = 3;
        constexpr uint32_t THREADS    = 128;
        constexpr uint32_t MAX_SPLITS = 256;

        struct Params
        {
            uint32_t batch, heads_q, heads_kv, share, dim, drafts, num_pages, page_size, ld_table, splits, tiles;
            float    scale, cap;
            const float*    slopes;
            const int32_t * block_table, *lens, *n_drafts, *depths;
            const uint64_t* tree;
            attn::Strides   q, k, v, o;
            float *         part_o, *part_ml; // [split][row][HD], [split][row][2]; rows: batch x heads_kv x share x drafts
        };

        __device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there)
        {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
        }
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
        __device__ __forceinline__ int64_t row_of(const attn::Strides& s, uint32_t b, uint32_t t, uint32_t h)
        {
            return int64_t(b) * s.batch + int64_t(t) * s.token + int64_t(h) * s.head;
        }

        template <uint32_t HD>
        struct Smem
        {
            static constexpr uint32_t ROW = HD * 2, TILE = KEYS * ROW; // a stage is a tile of keys and one of values
            static constexpr uint32_t TABLE = STAGES * 2 * TILE; // 2 x 64 {page, row in it}; page -1: not there
            static constexpr uint32_t VALID = TABLE + 2 * KEYS * 8; // STAGES words of 64 bits
            static constexpr uint32_t BYTES = VALID + 8 * (STAGES + 1);
            static_assert(STAGES * 2 * TILE >= 4 * 16 * (HD + 2) * 4, "sums of the warps reuse the ring");
        };

        // A block: 16 WM rows of one key head and the tokens of one split.  4 warps: WM along the rows, 4 / WM along the 64
        // tokens of a stage, each with its own running maximum.
        template <typename T, uint32_t HD, uint32_t WM, bool CAP, bool BIAS>
        __global__ void __launch_bounds__(THREADS) tree_kernel(const __grid_constant__ Params p, const T* __restrict__ q, const T* __restrict__ k,
                                                               const T* __restrict__ v, T* __restrict__ o)
        {
            using L                   = Smem<HD>;
            constexpr uint32_t WN     = 4 / WM, MINE = KEYS / WN, CHUNKS = HD / 8; // tokens of a warp, 16-byte pieces of a row
            extern __shared__ __align__(1024) uint8_t smem[];
            const uint32_t base = ptx::smem_u32(smem), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, g = lane >> 2, t = lane & 3u;
            const uint32_t wm = warp % WM, wn = warp / WM;
            int2*          table = reinterpret_cast<int2*>(smem + L::TABLE);
            uint32_t*      valid = reinterpret_cast<uint32_t*>(smem + L::VALID);

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
            sc.c = p.scale * LOG2E, sc.k1 = CAP ? 2.0f * LOG2E * (p.scale / p.cap) : 0.0f, sc.cap2 = p.cap * LOG2E, sc.slope = 0.0f;

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

            // where the tokens of step i are, for the copies of the step after the next barrier
            const auto look_up = [&](uint32_t i) {
                if(tid < KEYS)
                {
                    const uint32_t j = (from + i) * KEYS + tid;
                    int2           e = make_int2(-1, 0);
                    if(i < steps && j < end)
                    {
                        const uint32_t n = j / p.page_size;
                        e                = make_int2(__ldg(p.block_table + size_t(b) * p.ld_table + n), int32_t(j - n * p.page_size));
                        if(uint32_t(e.x) >= p.num_pages)
                            e.x = -1;
                    }
                    table[(i & 1u) * KEYS + tid] = e;
                    const uint32_t there = __ballot_sync(0xFFFFFFFFu, e.x >= 0);
                    if(lane == 0)
                        valid[2 * (i % (STAGES + 1)) + warp] = there;
                }
            };
            const auto fetch = [&](uint32_t i) {
                const uint32_t stage = base + (i % STAGES) * 2 * L::TILE, c = tid % CHUNKS;
                const T *      kh = k + int64_t(head) * p.k.head, *vh = v + int64_t(head) * p.v.head;
#pragma unroll 4
                for(uint32_t key = tid / CHUNKS; key < KEYS; key += THREADS / CHUNKS)
                {
                    const int2     e     = table[(i & 1u) * KEYS + key];
                    const bool     there = e.x >= 0 && c * 8 < p.dim;
                    const uint32_t to    = stage + key * L::ROW + ((c ^ (key & 7u)) << 4);
                    copy16(to, there ? kh + int64_t(e.x) * p.k.batch + int64_t(e.y) * p.k.token + c * 8 : k, there);
                    copy16(to + L::TILE, there ? vh + int64_t(e.x) * p.v.batch + int64_t(e.y) * p.v.token + c * 8 : v, there);
                }
            };
            float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, acc[HD / 8][4];
#pragma unroll
            for(uint32_t i = 0; i < HD / 8; ++i)
                acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;

#pragma unroll
            for(uint32_t i = 0; i < STAGES - 1; ++i)
            {
                look_up(i);
                __syncthreads();
                if(i < steps)
                    fetch(i);
                asm volatile("cp.async.commit_group;" ::: "memory");
            }
            look_up(STAGES - 1);
            for(uint32_t i = 0; i < steps; ++i)
            {
                asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
                __syncthreads(); // the stage is there for everyone, as is the table; the stage that is fetched into has been read
                if(i + STAGES - 1 < steps)
                    fetch(i + STAGES - 1);
                asm volatile("cp.async.commit_group;" ::: "memory");

                const uint32_t keys_at = base + (i % STAGES) * 2 * L::TILE + wn * MINE * L::ROW, values_at = keys_at + L::TILE;
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
                        ldmatrix4(f, keys_at + key * L::ROW + (((c * 4 + piece) ^ (key & 7u)) << 4));
                        mma<T>(s[n], qf[2 * c], f[0], f[1]);
                        mma<T>(s[n], qf[2 * c + 1], f[2], f[3]);
                    }
                }
                // scores in units of log 2, masked
                const uint32_t j0 = (from + i) * KEYS + wn * MINE;
                const uint32_t v0 = valid[2 * (i % (STAGES + 1))], v1 = valid[2 * (i % (STAGES + 1)) + 1];
                const bool     masked = (v0 & v1) != 0xFFFFFFFFu || (from + i + 1) * KEYS > len;
                const uint64_t there  = (uint64_t(v1) << 32 | v0) >> (wn * MINE);
                float          top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for(uint32_t n = 0; n < MINE / 8; ++n)
#pragma unroll
                    for(int e = 0; e < 4; ++e)
                    {
                        const uint32_t off = n * 8 + t * 2 + (e & 1), j = j0 + off;
                        const int32_t  rel = int32_t(int64_t(j) - len); // place behind the cached tokens
                        float          dist = 0.0f, unused;
                        if constexpr(BIAS)
                        {
                            int32_t where = rel;
                            if(rel >= 0 && p.depths && j < end)
                                where = __ldg(p.depths + size_t(b) * p.drafts + rel);
                            dist = static_cast<float>(at[e >> 1] - where);
                        }
                        sc.slope = slope[e >> 1];
                        float y  = attn::score<CAP, BIAS>(sc, s[n][e], dist, unused);
                        if(masked)
                            if(!(there >> off & 1u) || (rel >= 0 && !(bits[e >> 1] >> (rel & 63) & 1u)))
                                y = -INFINITY;
                        s[n][e]     = y;
                        top[e >> 1] = fmaxf(top[e >> 1], y);
                    }
#pragma unroll
                for(int h = 0; h < 2; ++h)
                {
                    top[h] = fmaxf(top[h], __shfl_xor_sync(0xFFFFFFFFu, top[h], 1));
                    top[h] = fmaxf(top[h], __shfl_xor_sync(0xFFFFFFFFu, top[h], 2));
                }
                // the maximum moves only where a score passes it by more than 2^8: until then weights grow up to 256
                if(__any_sync(0xFFFFFFFFu, top[0] > m[0] + 8.0f || top[1] > m[1] + 8.0f))
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
#pragma unroll
                for(uint32_t n = 0; n < MINE / 16; ++n)
                {
                    // 16 tokens x 16 elements at a time: lanes 0-15 give the tokens of the first 8 elements, 16-31 of the next
                    const uint32_t key = n * 16 + (lane & 15u);
#pragma unroll
                    for(uint32_t c = 0; c < HD / 16; ++c)
                    {
                        uint32_t f[4];
                        ldmatrix4_trans(f, values_at + key * L::ROW + (((c * 2 + (lane >> 4)) ^ (key & 7u)) << 4));
                        mma<T>(acc[2 * c], pf[n], f[0], f[1]);
                        mma<T>(acc[2 * c + 1], pf[n], f[2], f[3]);
                    }
                }
                look_up(i + STAGES); // into the half of the table that the copies above have left
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
            for(int h = 0; h < 2; ++h)
            {
                l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], 1);
                l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], 2);
            }
            // join the warps that share the rows: [warp][16 rows][HD] sums, [warp][16 rows] maximum and sum of weights
            __syncthreads();
            float *sums = reinterpret_cast<float*>(smem), *stats = sums + 4 * 16 * HD;
#pragma unroll
            for(uint32_t c = 0; c < HD / 8; ++c)
#pragma unroll
                for(int h = 0; h < 2; ++h)
                    *reinterpret_cast<float2*>(sums + (warp * 16 + g + 8 * h) * HD + c * 8 + t * 2) = make_float2(acc[c][2 * h], acc[c][2 * h + 1]);
            if(t == 0)
#pragma unroll
                for(int h = 0; h < 2; ++h)
                    stats[(warp * 16 + g + 8 * h) * 2] = m[h], stats[(warp * 16 + g + 8 * h) * 2 + 1] = l[h];
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
            ptx::grid_dep_launch_dependents();
        }

        // Joins the splits: one warp to a row, four (HD = 128) or two elements to a lane, splits in order.
        template <typename T, uint32_t HD>
        __global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ Params p, T* __restrict__ o)
        {
            constexpr uint32_t E = HD / 32;
            ptx::grid_dep_wait();
            const uint32_t rows = p.share * p.drafts, row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31u;
            const uint32_t all_rows = p.batch * p.heads_kv * rows;
            if(row >= all_rows)
                return;
            const uint32_t r = row % rows, head = row / rows % p.heads_kv, b = row / rows / p.heads_kv, draft = r / p.share;
            if(draft >= drafts_of(p, b))
                return;
            float mx = -INFINITY;
            for(uint32_t s = lane; s < p.splits; s += 32)
                mx = fmaxf(mx, p.part_ml[(size_t(s) * all_rows + row) * 2]);
#pragma unroll
            for(int d = 16; d > 0; d >>= 1)
                mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, d));
            float sum = 0.0f, y[E] = {};
            if(mx != -INFINITY)
                for(uint32_t s = 0; s < p.splits; ++s)
                {
                    const size_t part = size_t(s) * all_rows + row;
                    const float2 ml   = *reinterpret_cast<const float2*>(p.part_ml + part * 2);
                    if(ml.x == -INFINITY)
                        continue;
                    const float by = ex2(ml.x - mx);
                    sum += by * ml.y;
#pragma unroll
                    for(uint32_t e = 0; e < E; ++e)
                        y[e] = fmaf(by, p.part_o[part * HD + lane * E + e], y[e]);
                }
            const float inv = sum > 0.0f ? 1.0f / sum : sum;
            if(lane * E < p.dim)
            {
                uint32_t* out = reinterpret_cast<uint32_t*>(o + row_of(p.o, b, draft, head * p.share + r % p.share) + lane * E);
#pragma unroll
                for(uint32_t e = 0; e < E; e += 2)
                    out[e / 2] = attn::pack2<T>(y[e] * inv, y[e + 1] * inv);
            }
        }

        // Rows of a block in units of 16: 1, 2 or 4.
        static uint32_t rows_of_block(uint32_t rows)
        {
            return rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
        }
        // Splits of the tokens: enough blocks for two to four rounds of two per SM, but at least 8 stages (512 tokens) to a
        // block if a sequence is as long as its table allows.
        static uint32_t splits_of(uint32_t batch, uint32_t heads_kv, uint32_t rows, uint32_t max_tokens)
        {
            const uint64_t blocks = uint64_t(batch) * heads_kv * ceil_div(rows, 16 * rows_of_block(rows));
            const uint64_t want = (4 * 148 + blocks - 1) / blocks, most = (uint64_t(max_tokens) + 8 * KEYS - 1) / (8 * KEYS);
            const uint64_t n = want < most ? want : most;
            return n < 1 ? 1u : n > MAX_SPLITS ? MAX_SPLITS : uint32_t(n);
        }
        static uint32_t padded_dim(uint32_t dim)
        {
            return dim <= 64 ? 64 : 128;
        }

        template <typename T, uint32_t HD, uint32_t WM, bool CAP, bool BIAS>
        static int launch(const Params& p, const void* q, const void* k, const void* v, void* o, cudaStream_t stream)
        {
            auto kern = tree_kernel<T, HD, WM, CAP, BIAS>;
            B200_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<HD>::BYTES));
            kern<<<p.batch * p.heads_kv * p.tiles * p.splits, THREADS, Smem<HD>::BYTES, stream>>>(p, static_cast<const T*>(q), static_cast<const T*>(k),
                                                                                             static_cast<const T*>(v), static_cast<T*>(o));
            B200_CHECK_CUDA(cudaGetLastError());
            if(p.splits > 1)
            {
                cudaLaunchConfig_t cfg{};
                cfg.gridDim = dim3(ceil_div(p.batch * p.heads_kv * p.share * p.drafts, 4)), cfg.blockDim = dim3(128), cfg.stream = stream;
                cudaLaunchAttribute attr{};
                attr.id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
                attr.val.programmaticStreamSerializationAllowed = 1;
                cfg.attrs = &attr, cfg.numAttrs = 1;
                B200_CHECK_CUDA(cudaLaunchKernelEx(&cfg, join_kernel<T, HD>, p, static_cast<T*>(o)));
            }
            return B200WMMA_OK;
        }
        template <typename T, uint32_t HD, uint32_t WM>
        static int launch_scores(const Params& p, const void* q, const void* k, const void* v, void* o, cudaStream_t stream)
        {
            if(p.cap > 0.0f)
                return p.slopes ? launch<T, HD, WM, true, true>(p, q, k, v, o, stream) : launch<T, HD, WM, true, false>(p, q, k, v, o, stream);
            return p.slopes ? launch<T, HD, WM, false, true>(p, q, k, v, o, stream) : launch<T, HD, WM, false, false>(p, q, k, v, o, stream);
        }
        template <typename T, uint32_t HD>
        static int launch_rows(const Params& p, const void* q, const void* k, const void* v, void* o, cudaStream_t stream)
        {
            const uint32_t wm = rows_of_block(p.share * p.drafts);
            return wm == 1   ? launch_scores<T, HD, 1>(p, q, k, v, o, stream)
                   : wm == 2 ? launch_scores<T, HD, 2>(p, q, k, v, o, stream) : launch_scores<T, HD, 4>(p, q, k, v, o, stream);
        }
        template <typename T>
        static int launch_dim(const Params& p, const void* q, const void* k, const void* v, void* o, cudaStream_t stream)
        {
            return p.dim <= 64 ? launch_rows<T, 64>(p, q, k, v, o, stream) : launch_rows<T, 128>(p, q, k, v, o, stream);
        }
    } // namespace attn_tree
} // namespace b200wmma

using namespace b200wmma;

extern "C" size_t b200wmma_attn_tree_workspace_bytes(uint32_t batch, uint32_t drafts, uint32_t heads_q, uint32_t heads_kv,
                                                     uint32_t head_dim, uint32_t max_tokens)
{
    if(!batch || !drafts || !heads_q || !heads_kv)
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
    B200_REQUIRE(uint64_t(a->batch) * a->heads_q * drafts < (uint64_t(1) << 31), B200WMMA_ERR_UNSUPPORTED,
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
    p.drafts = drafts, p.num_pages = num_pages, p.page_size = page_size, p.ld_table = ld_table, p.scale = a->scale, p.cap = a->cap;
    p.slopes = a->slopes, p.block_table = block_table, p.lens = lens, p.n_drafts = n_drafts, p.depths = depths, p.tree = tree;
    const uint32_t rows = p.share * drafts;
    p.splits  = attn_tree::splits_of(p.batch, p.heads_kv, rows, max_tokens);
    p.tiles   = ceil_div(rows, 16 * attn_tree::rows_of_block(rows));
    p.part_o  = static_cast<float*>(workspace);
    p.part_ml = p.part_o + size_t(p.splits) * p.batch * p.heads_kv * rows * attn_tree::padded_dim(p.dim);
    return a->data_type == B200WMMA_OUT_F16 ? attn_tree::launch_dim<__half>(p, q, k_cache, v_cache, o, as_stream(stream))
                                            : attn_tree::launch_dim<__nv_bfloat16>(p, q, k_cache, v_cache, o, as_stream(stream));
}
