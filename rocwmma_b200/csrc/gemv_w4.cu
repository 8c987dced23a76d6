// Matrix-vector products with 4-bit weights and group scales: the entry point b200wmma_gemv_w4.
//   y[r][i] = alpha * sum_k x[r][k] * s[i][k / G] * (q[i][k] - z[i][k / G]) + beta * y[r][i]
//
// Bound: the packed weights, m * n / 2 bytes, are read once.  What competes is the arithmetic on each weight, so
//  - values become 16-bit numbers two at a time, by putting the nibble into the mantissa of 1024 (fp16) or 128 (bf16) and
//    subtracting that with the zero point: exact, since |q - z| <= 15 (published for fp16 by Kim, Henry, Fahim and Hassan Awadalla,
//    "Who Says Elephants Can't Run: Bringing Large Scale MoE Models into Cloud Scale Production", 2022);
//  - the products are warp-level matrix instructions (16 outputs x 8 vectors x 16 columns, fp32 sums) even for one vector:
//    a fused multiply-add per weight and vector would take the issue slots that the conversion needs.  Beyond 8 vectors
//    tcgen05 takes over (gemv_w4_tc05.cuh);
//  - sums of a group are scaled in fp32, so nothing is rounded before y.
// The columns' order inside a group of 32 is free as long as weights and x agree: lane t of four takes word t of each 16-byte
// piece (8 weights), whose nibbles i and i + 4 come out as one pair, and x is permuted to that by four byte selections.
// Measured (replayed graph, weights from memory): 1 x 16384 x 8192 fp16, groups of 128 with zero points: 21-23 us (3.0-3.2 TB/s);
// 1 x 2048 x 2048: 3.1 us; 7 x 5003 x 4128 bf16, groups of 32: 11.6 us; 8 x 14336 x 4096 bf16, groups of 64: 17 us; on tcgen05 9 to
// 32 vectors of that 25-28 us (32 of them warp-level: 36 us), 64 vectors, groups of 128: 29 us (50 us); groups of 64 take 64 vectors
// in two passes, 52 us.
// What bounds one vector is latency: a warp has four stretches behind a ring of two, 27 of an SM's 64 warps are there (shared memory
// for four blocks; 1024 blocks are 1.73 rounds), and waiting for memory is the largest part of the 12.6 cycles between two
// instructions of a warp (4.0), with 55 % of the issue slots and 36 % of the memory's rate in use.
#include "attn_common.cuh"
#include "gemm_tc05_common.cuh"

namespace b200wmma
{
    namespace gemv_w4
    {
        constexpr uint32_t FEW_VECTORS = 8; // the warp-level kernel's; more take the tcgen05 form

        struct Args
        {
            uint32_t       m, n, rows;
            const uint8_t* a;
            uint32_t       lda;
            const void*    scales;
            uint32_t       ld_scales;
            const uint8_t* zeros;
            uint32_t       ld_zeros, group, groups;
            const void*    x;
            uint32_t       ldx;
            void*          y;
            uint32_t       ldy;
            float          alpha, beta;
            bool           y_f32;
        };

        __device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there)
        {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
        }
        __device__ __forceinline__ void copy_commit()
        {
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        template <int N>
        __device__ __forceinline__ void copy_wait()
        {
            asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
        }
        // Plain loads from shared memory at a byte address of the shared window: unlike volatile assembly they may be scheduled
        // ahead of the products before them.
        __device__ __forceinline__ uint32_t lds32(uint32_t at)
        {
            return *static_cast<const uint32_t*>(__cvta_shared_to_generic(at));
        }
        __device__ __forceinline__ uint4 lds128(uint32_t at)
        {
            return *static_cast<const uint4*>(__cvta_shared_to_generic(at));
        }
        __device__ __forceinline__ void sts128(uint32_t at, const uint4& v)
        {
            *static_cast<uint4*>(__cvta_shared_to_generic(at)) = v;
        }
        // c = a b + d: `d` is c, or 0 for the first product of a sum
        template <typename T>
        __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, bool fresh)
        {
            const float d0 = fresh ? 0.0f : c[0], d1 = fresh ? 0.0f : c[1], d2 = fresh ? 0.0f : c[2], d3 = fresh ? 0.0f : c[3];
            if constexpr(std::is_same<T, __half>::value)
                asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
                             : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                             : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(d0), "f"(d1), "f"(d2), "f"(d3));
            else
                asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
                             : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                             : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(d0), "f"(d1), "f"(d2), "f"(d3));
        }

        // What a group subtracts: 1024 + z and 64 + z as fp16 pairs, 128 + z as a bf16 pair (z = 8 for signed values).
        template <typename T>
        struct Offset
        {
            uint32_t low, high;
            __device__ __forceinline__ void set(uint32_t z)
            {
                if constexpr(std::is_same<T, __half>::value)
                {
                    low  = (0x6400u + z) * 0x10001u; // 1024 + z
                    high = (0x5400u + (z << 4)) * 0x10001u; // 64 + z: a step there is 1/16
                }
                else
                    low = (0x4300u + z) * 0x10001u; // 128 + z
            }
        };
        // (w & mask) ^ flip in one instruction: 1 x 16384 x 8192 22 us, 26 us with the expression in C, at that step
        __device__ __forceinline__ uint32_t and_xor(uint32_t w, uint32_t mask, uint32_t flip)
        {
            uint32_t r;
            asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(r) : "r"(w), "r"(mask), "r"(flip));
            return r;
        }
        // Eight weights of a word as pairs (0, 4), (1, 5), (2, 6), (3, 7).  flip = 8 turns signed nibbles into unsigned ones.
        template <typename T, bool SIGNED>
        __device__ __forceinline__ void unpack(uint32_t w, const Offset<T>& z, uint32_t (&p)[4])
        {
            if constexpr(std::is_same<T, __half>::value)
            {
                constexpr uint32_t LOW = SIGNED ? 0x64086408u : 0x64006400u, HIGH = SIGNED ? 0x64806480u : 0x64006400u;
                const __half2      zl = *reinterpret_cast<const __half2*>(&z.low), zh = *reinterpret_cast<const __half2*>(&z.high);
                const uint32_t     w8 = w >> 8;
                uint32_t           u[4] = {and_xor(w, 0x000F000Fu, LOW), and_xor(w, 0x00F000F0u, HIGH), and_xor(w8, 0x000F000Fu, LOW),
                                               and_xor(w8, 0x00F000F0u, HIGH)};
#pragma unroll
                for(int i = 0; i < 4; ++i)
                {
                    const __half2 h = *reinterpret_cast<const __half2*>(&u[i]);
                    // 1024 + 16 q comes down to 64 + q exactly
                    const __half2 r = (i & 1) ? __hfma2(h, __float2half2_rn(0.0625f), __hneg2(zh)) : __hsub2(h, zl);
                    p[i]            = *reinterpret_cast<const uint32_t*>(&r);
                }
            }
            else
            {
                constexpr uint32_t   BASE = SIGNED ? 0x43084308u : 0x43004300u;
                const __nv_bfloat162 zl   = *reinterpret_cast<const __nv_bfloat162*>(&z.low);
#pragma unroll
                for(int i = 0; i < 4; ++i)
                {
                    const uint32_t       u = and_xor(w >> (4 * i), 0x000F000Fu, BASE);
                    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), zl);
                    p[i]                   = *reinterpret_cast<const uint32_t*>(&r);
                }
            }
        }

        // Scales (and zero points) of the groups that a stretch of columns touches, for the two rows of a lane: lane t of four
        // holds groups t, t + 4, ...; the upper half belongs to the second row.
        template <typename T, bool SIGNED, int N>
        struct GroupInfo
        {
            uint32_t scale[N], zero[N];
            __device__ __forceinline__ void load(const Args& p, uint32_t row0, uint32_t row1, uint32_t first, uint32_t last)
            {
                const uint16_t* s0 = static_cast<const uint16_t*>(p.scales) + size_t(row0) * p.ld_scales;
                const uint16_t* s1 = static_cast<const uint16_t*>(p.scales) + size_t(row1) * p.ld_scales;
                const uint8_t*  z0 = SIGNED ? nullptr : p.zeros + size_t(row0) * p.ld_zeros;
                const uint8_t*  z1 = SIGNED ? nullptr : p.zeros + size_t(row1) * p.ld_zeros;
#pragma unroll
                for(int i = 0; i < N; ++i)
                {
                    const uint32_t g = first + 4 * i;
                    scale[i] = zero[i] = 0;
                    if(g <= last)
                    {
                        scale[i] = __ldg(s0 + g) | uint32_t(__ldg(s1 + g)) << 16;
                        if constexpr(!SIGNED)
                            zero[i] = (__ldg(z0 + g) | uint32_t(__ldg(z1 + g)) << 16) & 0xF000Fu;
                    }
                }
            }
            __device__ __forceinline__ uint32_t pick(const uint32_t (&from)[N], uint32_t i, uint32_t lane) const
            {
                uint32_t v = from[0];
                if constexpr(N == 2)
                    v = i >= 4 ? from[1] : from[0];
                return __shfl_sync(0xFFFFFFFFu, v, (lane & ~3u) | (i & 3u));
            }
            __device__ __forceinline__ void offsets(uint32_t i, uint32_t lane, Offset<T> (&z)[2]) const
            {
                if constexpr(SIGNED)
                    z[0].set(8), z[1].set(8);
                else
                {
                    const uint32_t v = pick(zero, i, lane);
                    z[0].set(v & 0xFFFFu), z[1].set(v >> 16);
                }
            }
            // sum += scale * part
            template <int NT>
            __device__ __forceinline__ void flush(uint32_t i, uint32_t lane, float (&sum)[NT][4], float (&part)[NT][4]) const
            {
                const float2 s = tc05::Pack16<T>::widen(pick(scale, i, lane));
#pragma unroll
                for(int c = 0; c < NT; ++c)
#pragma unroll
                    for(int j = 0; j < 4; ++j)
                    {
                        sum[c][j] = fmaf(j < 2 ? s.x : s.y, part[c][j], sum[c][j]);
                    }
            }
        };

        // The order that unpack gives its pairs in, for 8 elements of x.
        __device__ __forceinline__ uint4 pair_up(const uint4& x)
        {
            return make_uint4(__byte_perm(x.x, x.z, 0x5410), __byte_perm(x.x, x.z, 0x7632), __byte_perm(x.y, x.w, 0x5410),
                              __byte_perm(x.y, x.w, 0x7632));
        }
        // 32 columns: words of the two rows, 8 paired elements of x for each block of 8 vectors
        template <typename T, bool SIGNED, int NT>
        __device__ __forceinline__ void step(uint32_t w0, uint32_t w1, const uint4 (&x)[NT], const Offset<T> (&z)[2], float (&part)[NT][4], bool fresh)
        {
            uint32_t p[4], q[4];
            unpack<T, SIGNED>(w0, z[0], p);
            unpack<T, SIGNED>(w1, z[1], q);
#pragma unroll
            for(int c = 0; c < NT; ++c)
            {
                mma<T>(part[c], p[0], q[0], p[1], q[1], x[c].x, x[c].y, fresh);
                mma<T>(part[c], p[2], q[2], p[3], q[3], x[c].z, x[c].w, false);
            }
        }

        // Sum of the same place in the shared memory of a cluster's first `parts` (at most 8) blocks, in order; the loads are all
        // on their way before the first is added.
        __device__ __forceinline__ float cluster_sum(const float* at, uint32_t parts)
        {
            uint32_t v[8];
#pragma unroll
            for(uint32_t c = 0; c < 8; ++c)
                v[c] = c < parts ? ptx::ld_shared_cluster_u32(ptx::mapa(ptx::smem_u32(at), c)) : 0u;
            float s = __uint_as_float(v[0]);
#pragma unroll
            for(uint32_t c = 1; c < 8; ++c)
                s += __uint_as_float(v[c]);
            return s;
        }
        template <typename T>
        __device__ __forceinline__ void put(const Args& p, uint32_t r, uint32_t i, float s)
        {
            const size_t at = size_t(r) * p.ldy + i;
            s *= p.alpha;
            if(p.y_f32)
            {
                float* out = static_cast<float*>(p.y) + at;
                *out       = p.beta != 0.0f ? fmaf(p.beta, *out, s) : s;
            }
            else
            {
                T* out = static_cast<T*>(p.y) + at;
                *out   = attn::from_f32<T>(p.beta != 0.0f ? fmaf(p.beta, attn::to_f32(*out), s) : s);
            }
        }

    } // namespace gemv_w4
} // namespace b200wmma

#include "gemv_w4_tc05.cuh"

namespace b200wmma
{
    namespace gemv_w4
    {
        // Up to 8 vectors.  A block owns 16 outputs; its W warps share the columns in stretches of 256, each through a ring of its
        // own in shared memory (128 bytes of each row, and the x that belongs to them), so warps never wait for one another
        // before the sums meet.  Few outputs: a cluster of blocks shares the columns too and the sums meet in the first
        // block's shared memory.
        // STEPS: pieces of 32 columns to a group inside a stretch, where groups and stretches are aligned (groups of 32, 64,
        // 128 and multiples of 256); 0: counted at run time.
        // ONE: a single vector.  Each warp pairs up its part of x once, before the weights are there.
        constexpr uint32_t FEW_K = 256, FEW_STAGES = 2, FEW_ROWS = 16;
        struct Few
        {
            static constexpr uint32_t W_STAGE = FEW_ROWS * FEW_K / 2, ZERO = 512; // zeros: the x of vectors that do not exist
            uint32_t x_warp, bytes; // bytes of a warp's x
            // one vector, kept whole
            __host__ __device__ Few(uint32_t w, uint32_t n, uint32_t parts)
            {
                const uint32_t stretches = (n + FEW_K - 1) / FEW_K;
                x_warp = (stretches + w * parts - 1) / (w * parts) * FEW_K * 2;
                bytes  = total(w, x_warp);
            }
            // x in rings
            static constexpr __host__ __device__ uint32_t ring_x(uint32_t rows)
            {
                return FEW_STAGES * rows * FEW_K * 2;
            }
            static constexpr __host__ __device__ uint32_t ring_bytes(uint32_t w, uint32_t rows)
            {
                return total(w, ring_x(rows));
            }
            static constexpr __host__ __device__ uint32_t total(uint32_t w, uint32_t x)
            {
                const uint32_t ring = w * (FEW_STAGES * W_STAGE + x), red = w * 128 * 4; // the sums reuse the ring
                return ZERO + (ring > red ? ring : red);
            }
        };
        template <typename T, bool SIGNED, int W, int STEPS, bool ONE>
        __global__ void __launch_bounds__(32 * W) few_kernel(const __grid_constant__ Args p, uint32_t parts)
        {
            constexpr int GROUPS = STEPS == 0 ? 8 : 8 / STEPS, INFO = GROUPS > 4 ? 2 : 1;
            extern __shared__ __align__(1024) uint8_t smem[];
            const uint32_t x_warp = ONE ? Few(W, p.n, parts).x_warp : Few::ring_x(p.rows);
            const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
            const uint32_t part_id = parts > 1 ? blockIdx.x % parts : 0, row0 = (parts > 1 ? blockIdx.x / parts : blockIdx.x) * FEW_ROWS;
            const uint32_t zero = ptx::smem_u32(smem), ring = zero + Few::ZERO + warp * (FEW_STAGES * Few::W_STAGE + x_warp);
            const uint32_t ring_x = ring + FEW_STAGES * Few::W_STAGE, x_stage = x_warp / FEW_STAGES;
            const uint32_t stretches = (p.n + FEW_K - 1) / FEW_K, stride = W * parts, first = part_id * W + warp;
            const uint32_t mine = first < stretches ? (stretches - first - 1) / stride + 1 : 0;
            const bool     rows_full = row0 + FEW_ROWS <= p.m;

            // a lane copies piece lane % 8 of rows lane / 8, lane / 8 + 4, ... and piece `lane` of each vector
            const uint8_t* src_a = p.a + size_t(row0 + (lane >> 3)) * p.lda + (lane & 7u) * 16 + size_t(first) * (FEW_K / 2);
            const T*       src_x = static_cast<const T*>(p.x) + size_t(first) * FEW_K + lane * 8;
            const uint32_t place[2] = {ring + (lane >> 3) * 128 + (((lane & 7u) ^ (lane >> 3)) << 4),
                                       ring + (lane >> 3) * 128 + (((lane & 7u) ^ ((lane >> 3) + 4)) << 4)};
            const size_t   rows4    = size_t(p.lda) * 4;
            uint32_t       k_next   = first * FEW_K;
            const auto     fetch    = [&](uint32_t slot) {
                const uint8_t* from = src_a;
                if(rows_full && k_next + FEW_K <= p.n)
                {
#pragma unroll
                    for(uint32_t j = 0; j < 4; ++j, from += rows4)
                        copy16(place[j & 1u] + slot * Few::W_STAGE + j * 512, from, true);
                }
                else
#pragma unroll
                    for(uint32_t j = 0; j < 4; ++j, from += rows4)
                    {
                        const bool there = row0 + (lane >> 3) + j * 4 < p.m && k_next + (lane & 7u) * 32 < p.n;
                        copy16(place[j & 1u] + slot * Few::W_STAGE + j * 512, there ? from : p.a, there);
                    }
                if constexpr(!ONE)
                {
                    const bool there = k_next + lane * 8 < p.n;
                    for(uint32_t r = 0; r < p.rows; ++r)
                        copy16(ring_x + slot * x_stage + r * 512 + ((lane ^ ((r & 1u) << 2)) << 4),
                               there ? src_x + size_t(r) * p.ldx : static_cast<const T*>(p.x), there);
                    src_x += size_t(stride) * FEW_K;
                }
                src_a += size_t(stride) * (FEW_K / 2), k_next += stride * FEW_K;
            };
            float                      sum[1][4] = {}, part[1][4] = {};
            GroupInfo<T, SIGNED, INFO> info, next;
            const uint32_t             ra = min(row0 + g, p.m - 1), rb = min(row0 + g + 8, p.m - 1);
            uint32_t                   k_info = first * FEW_K, g_info = k_info / p.group; // first group of the stretch
            const auto                 groups = [&]() {
                if constexpr(STEPS == 0 || STEPS == 8)
                    g_info = k_info / p.group;
                const uint32_t last = STEPS == 8 ? g_info : STEPS == 0 ? min(p.groups - 1, (k_info + FEW_K - 1) / p.group) : p.groups - 1;
                next.load(p, ra, rb, g_info + t, min(last, g_info + GROUPS - 1));
                k_info += stride * FEW_K, g_info += stride * GROUPS;
            };
#pragma unroll
            for(uint32_t i = 0; i < FEW_STAGES; ++i)
            {
                if(i < mine)
                    fetch(i);
                copy_commit();
            }
            if(mine)
                groups();
            if constexpr(ONE)
            {
#pragma unroll 4
                for(uint32_t i = 0; i < mine; ++i)
                {
                    uint4 x = make_uint4(0, 0, 0, 0);
                    if((first + i * stride) * FEW_K + lane * 8 < p.n)
                        x = __ldg(reinterpret_cast<const uint4*>(src_x + size_t(i) * stride * FEW_K));
                    sts128(ring_x + i * 512 + lane * 16, pair_up(x));
                }
            }
            if(threadIdx.x < Few::ZERO / 16)
                sts128(zero + threadIdx.x * 16, make_uint4(0, 0, 0, 0));
            __syncthreads();
            uint32_t       slot = 0, k0 = first * FEW_K;
            const uint32_t wa = ring + g * 128 + (g << 4) + t * 4; // pieces are 16 bytes apart and swizzled by their row
            // lanes of vectors that do not exist read zeros
            uint32_t xa = g >= p.rows ? zero + t * 16 : ring_x + t * 16 + (ONE ? 0u : g * 512 + ((g & 1u) << 6));
            for(uint32_t i = 0; i < mine; ++i)
            {
                info = next;
                if(i + 1 < mine)
                    groups();
                copy_wait<FEW_STAGES - 1>();
                __syncwarp();
                const uint32_t ws = wa + slot * Few::W_STAGE, xs = ONE || g >= p.rows ? xa : xa + slot * x_stage;
                uint32_t       grp = 0, left = STEPS == 0 ? p.group - k0 % p.group : 0; // columns left of the current group
                bool           fresh = true;
                Offset<T>      z[2];
                info.offsets(0, lane, z);
#pragma unroll
                for(uint32_t c = 0; c < 8; ++c)
                {
                    uint4 x[1];
                    if constexpr(ONE)
                        x[0] = lds128(xs + c * 64);
                    else
                        x[0] = pair_up(lds128(xs ^ (c << 6)));
                    if constexpr(STEPS != 0)
                        fresh = c % STEPS == 0;
                    step<T, SIGNED, 1>(lds32(ws ^ (c << 4)), lds32((ws ^ (c << 4)) + 1024), x, z, part, fresh);
                    fresh    = false;
                    bool end = c == 7;
                    if constexpr(STEPS == 0)
                    {
                        left -= 32;
                        end |= left == 0;
                    }
                    else
                        end |= (c + 1) % STEPS == 0;
                    if(end)
                    {
                        info.template flush<1>(grp, lane, sum, part);
                        fresh = true;
                        if(STEPS != 0 || left == 0)
                        {
                            left = p.group;
                            ++grp;
                            if(!SIGNED && c != 7)
                                info.offsets(grp, lane, z);
                        }
                    }
                }
                __syncwarp(); // everyone has read the stage
                if(i + FEW_STAGES < mine)
                    fetch(slot);
                copy_commit();
                slot ^= 1u;
                k0 += stride * FEW_K;
                if(ONE && g == 0)
                    xa += 512;
            }
            copy_wait<0>();
            __syncthreads();
            // sums of the warps, [warp][vector][output]
            float* red = reinterpret_cast<float*>(smem + Few::ZERO);
#pragma unroll
            for(int j = 0; j < 4; ++j)
                if(!ONE || (t == 0 && (j & 1) == 0))
                    red[warp * 128 + (t * 2 + (j & 1)) * FEW_ROWS + g + 8 * (j >> 1)] = sum[0][j];
            __syncthreads();
            const uint32_t outs = (ONE ? 1 : p.rows) * FEW_ROWS;
            for(uint32_t e = threadIdx.x; e < outs; e += 32 * W)
            {
                float s = 0.0f;
#pragma unroll
                for(uint32_t w = 0; w < W; ++w)
                    s += red[w * 128 + e];
                if(parts > 1)
                    red[e] = s; // no other thread reads or writes the place
                else if(row0 + e % FEW_ROWS < p.m)
                    put<T>(p, e / FEW_ROWS, row0 + e % FEW_ROWS, s);
            }
            if(parts > 1)
            {
                ptx::cluster_sync();
                if(part_id == 0)
                    for(uint32_t e = threadIdx.x; e < outs; e += 32 * W)
                    {
                        const float s = cluster_sum(red + e, parts);
                        if(row0 + e % FEW_ROWS < p.m)
                            put<T>(p, e / FEW_ROWS, row0 + e % FEW_ROWS, s);
                    }
                ptx::cluster_sync(); // no block leaves while another reads its sums
            }
        }

        // MOST: what any call of KERN asks for.
        template <auto KERN, uint32_t MOST, typename... More>
        static int launch_clusters(const Args& p, uint32_t blocks, uint32_t blocks_y, uint32_t parts, uint32_t smem,
                                   uint32_t threads, cudaStream_t stream, More... more)
        {
            static attn::Allowed allowed;
            if(int e = attn::allow_smem(reinterpret_cast<const void*>(KERN), MOST, allowed))
                return e;
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3(blocks * parts, blocks_y), cfg.blockDim = dim3(threads), cfg.dynamicSmemBytes = smem, cfg.stream = stream;
            cudaLaunchAttribute attr{};
            attr.id               = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = parts, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
            cfg.attrs = &attr, cfg.numAttrs = parts > 1 ? 1 : 0;
            B200_CHECK_CUDA(cudaLaunchKernelEx(&cfg, KERN, p, parts, more...));
            return B200WMMA_OK;
        }
        // Blocks of a cluster: a power of two, up to 8, to `most` (parts with work enough) and to per_sm blocks on an SM.
        static uint32_t parts_of(uint64_t blocks, uint32_t most, uint32_t per_sm)
        {
            uint32_t parts = 1;
            while(parts < 8 && 2 * parts <= most && blocks * parts * 2 <= per_sm * 148)
                parts *= 2;
            return parts;
        }
        // Warps of a block: 8 for one vector (16384 x 8192 fp16: 21 us, 24 with 4), 4 for more, whose rings would leave room for
        // one or two blocks on an SM (7 x 5003 x 4128 bf16, groups of 32: 12 us, 14 with 8).  One vector that is too long to lie in
        // shared memory next to the rings goes through them like several.
        constexpr uint32_t ONE_BYTES = 100 * 1024, RING_BYTES = Few::ring_bytes(4, FEW_VECTORS);
        template <typename T, bool SIGNED, int STEPS>
        static int launch_few(const Args& p, cudaStream_t stream)
        {
            const uint32_t blocks = ceil_div(p.m, FEW_ROWS);
            if(p.rows == 1)
            {
                const uint32_t parts = parts_of(blocks, ceil_div(p.n, 8 * FEW_K), 2);
                const Few      f(8, p.n, parts);
                if(f.bytes <= ONE_BYTES)
                    return launch_clusters<few_kernel<T, SIGNED, 8, STEPS, true>, ONE_BYTES>(p, blocks, 1, parts, f.bytes, 256, stream);
            }
            const uint32_t parts = parts_of(blocks, ceil_div(p.n, 4 * FEW_K), 2);
            return launch_clusters<few_kernel<T, SIGNED, 4, STEPS, false>, RING_BYTES>(p, blocks, 1, parts, Few::ring_bytes(4, p.rows), 128, stream);
        }
        template <typename T, bool SIGNED, int N, int SETS>
        static int launch_tc(const Args& p, cudaStream_t stream)
        {
            unsigned* status = nullptr;
            if(int e = status_word_ptr(&status))
                return e;
            using L = TcSmem<N, SETS>;
            const uint32_t blocks = ceil_div(p.m, TC_M), blocks_y = ceil_div(p.rows, uint32_t(N));
            const uint32_t parts = parts_of(uint64_t(blocks) * blocks_y, ceil_div(p.n, 2 * TC_K), 1);
            CUtensorMap    map;
            if(int e = tc05::make_kmajor_tmap(&map, std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                                              p.x, p.rows, p.n, p.ldx, N))
                return e;
            return launch_clusters<tc_kernel<T, SIGNED, N, SETS>, L::BYTES>(p, blocks, blocks_y, parts, L::BYTES, TC_THREADS, stream, status, map);
        }
        template <typename T, bool SIGNED, int SETS>
        static int launch_tc_rows(const Args& p, cudaStream_t stream)
        {
            if constexpr(SETS == 1)
                if(p.rows > 32)
                    return launch_tc<T, SIGNED, 64, SETS>(p, stream);
            if constexpr(SETS <= 2)
                if(p.rows > 16)
                    return launch_tc<T, SIGNED, 32, SETS>(p, stream);
            return launch_tc<T, SIGNED, 16, SETS>(p, stream);
        }
        template <typename T, bool SIGNED>
        static int launch(const Args& p, cudaStream_t stream)
        {
            if(p.rows > FEW_VECTORS)
                return p.group % TC_K == 0 ? launch_tc_rows<T, SIGNED, 1>(p, stream)
                       : p.group == 64     ? launch_tc_rows<T, SIGNED, 2>(p, stream) : launch_tc_rows<T, SIGNED, 4>(p, stream);

            if(p.group % FEW_K == 0)
                return launch_few<T, SIGNED, 8>(p, stream);
            return p.group == 128 ? launch_few<T, SIGNED, 4>(p, stream)
                   : p.group == 64 ? launch_few<T, SIGNED, 2>(p, stream)
                   : p.group == 32 ? launch_few<T, SIGNED, 1>(p, stream) : launch_few<T, SIGNED, 0>(p, stream);
        }
    } // namespace gemv_w4
} // namespace b200wmma

extern "C" int b200wmma_gemv_w4(uint32_t m, uint32_t n, uint32_t rows, const uint8_t* a, uint32_t lda_bytes, const void* scales,
                                uint32_t ld_scales, const uint8_t* zeros, uint32_t ld_zeros, uint32_t group, const void* x, uint32_t ldx,
                                void* y, uint32_t ldy, float alpha, float beta, int data_type, int out_type, void* stream)
{
    using namespace b200wmma;
    clear_error();
    B200_REQUIRE(m && n && rows && group, B200WMMA_ERR_INVALID_ARG, "gemv_w4: m, n, rows and group must be non-zero");
    B200_REQUIRE(a && scales && x && y, B200WMMA_ERR_INVALID_ARG, "gemv_w4: a, scales, x and y must be non-null");
    B200_REQUIRE(data_type == B200WMMA_OUT_F16 || data_type == B200WMMA_OUT_BF16, B200WMMA_ERR_INVALID_ARG,
                 "gemv_w4: data_type must be B200WMMA_OUT_F16 or B200WMMA_OUT_BF16");
    B200_REQUIRE(out_type == data_type || out_type == B200WMMA_OUT_F32, B200WMMA_ERR_INVALID_ARG,
                 "gemv_w4: out_type must be data_type or B200WMMA_OUT_F32");
    B200_REQUIRE(n % 32 == 0 && group % 32 == 0, B200WMMA_ERR_UNSUPPORTED, "gemv_w4: n and group must be multiples of 32");
    B200_REQUIRE(m < (1u << 30) && n < (1u << 30) && rows < 65536u, B200WMMA_ERR_UNSUPPORTED,
                 "gemv_w4: m and n must be below 2^30 and rows below 65536");
    const uint32_t groups = (n - 1) / group + 1;
    B200_REQUIRE(lda_bytes >= n / 2 && ldx >= n && ldy >= m && ld_scales >= groups && (!zeros || ld_zeros >= groups),
                 B200WMMA_ERR_INVALID_ARG, "gemv_w4: a leading dimension is smaller than its row");
    B200_REQUIRE(aligned16(a) && lda_bytes % 16 == 0 && aligned16(x) && ldx % 8 == 0, B200WMMA_ERR_ALIGNMENT,
                 "gemv_w4: a, x and their leading dimensions must be multiples of 16 bytes");
    if(int e = require_sm100())
        return e;
    // a group that outlasts the row is the row: what is left of it never runs out
    const gemv_w4::Args p{m, n, rows, a, lda_bytes, scales, ld_scales, zeros, ld_zeros, group, groups, x, ldx, y, ldy, alpha, beta,
                          out_type == B200WMMA_OUT_F32};
    const cudaStream_t  s = as_stream(stream);
    if(data_type == B200WMMA_OUT_F16)
        return zeros ? gemv_w4::launch<__half, false>(p, s) : gemv_w4::launch<__half, true>(p, s);
    return zeros ? gemv_w4::launch<__nv_bfloat16, false>(p, s) : gemv_w4::launch<__nv_bfloat16, true>(p, s);
}
