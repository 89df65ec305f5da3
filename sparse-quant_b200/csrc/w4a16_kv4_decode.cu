// Decode attention over the paged 4-bit cache: one new token per row, appended and attended to in one launch.
//
// Mathematics.  With codes n, steps s and minima m per group g of a head row, a score is
//     k . q = sum_g  s_g (sum_{d in g} n_d q_d) + m_g (sum_{d in g} q_d)
// and the output
//     sum_t p_t v_t[d] = sum_t (p_t s_{t,g}) n_{t,d} + sum_t p_t m_{t,g}         (g the group of d)
// so that both products run over the codes themselves: a nibble is only masked in place, which leaves a subnormal fp16 bit pattern
// (q 2^-24 or q 2^-20) that the tensor core multiplies exactly, and is never rounded.  What is rounded to fp16: the rotated query
// (as the cache's own keys are), scaled by a power of two of its head's largest element, which is exact; and the weight p s of a
// (token, group), 2^-11 of it, scaled by a power of two that follows the largest step seen, so that values near fp16's smallest keep
// their precision.  Scores, maxima, sums and the minima's part of the output are fp32.
//
// A warp owns tiles of 16 tokens of one (row, key/value head), with a ring of tiles of its own in shared memory, filled by the copy
// engine (a tile is one contiguous run, also where pages are small), and a softmax of its own: running maximum and sum, rescaled
// only when a score exceeds the maximum by 2^8.  Queries that share the key/value head are the 8 columns of mma.m16n8k16:
//     scores  A = keys (16 tokens x 16 dims), B = queries;   output  A = values^T (16 dims x 16 tokens), B = weights
// and the accumulator of the first is the layout the second needs after an 8x8 transpose (movmatrix).  Warps, and the S CTAs that
// split a row's tiles, meet in shared memory, through the cluster's for S <= 8, or through a workspace and a second launch.
#include <cooperative_groups.h>

#include "w4a16_kv4.cuh"
#include "w4a16_sm100.cuh"

namespace cg = cooperative_groups;

namespace w4a16 {
namespace kv4 {
namespace {

using namespace sm100;

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kCols = 8;                          // query heads of one pass
constexpr uint64_t kWaitNs = 400000000ull;        // a copy that has not arrived by then never will: error word 1

struct DecodeArgs {
    Cache c;
    const __half* qkv;
    __half* out;
    const int* pos;
    const __half* cos;
    const __half* sin;
    int* error;
    float* part;                  // split over the grid: [batch][heads][splits][D + 2]
    int heads, share;             // share: query heads of a key/value head
    int blocks;                   // passes of 8 query heads over a key/value head
    int splits, rope_rows;
    long long stride;
    float scale_log2;             // scale * log2(e)
};

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v)
{
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t pack2(float a, float b)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }        // -126 <= e <= 127

// which token of a tile stands in row i (of 8) of a fragment; rows 8 to 15 are the tokens 8 further on.  The order spreads the rows
// that one load instruction touches over the shared-memory banks, for keys (two or four rows at a time) and values (every other).
__device__ __forceinline__ int token_of(int i) { return i ^ ((i >> 2) & 1); }

template <class F, int D>
struct Smem {
    static constexpr int kStages = F::kBytes > 2304 ? 5 : F::kBytes > 1280 ? 6 : 10;      // four CTAs an SM
    alignas(128) unsigned char ring[kWarps][kStages][F::kBytes];
    uint64_t full[kWarps][kStages];
    float m[kWarps + 1][kCols], l[kWarps + 1][kCols];                                      // [kWarps]: of the whole CTA
    int abort_flag[kWarps];
};

template <class F, int D>
__global__ void __launch_bounds__(kThreads, 4) decode_kernel(const DecodeArgs a)
{
    constexpr int J = F::J, NG = F::NG, kStages = Smem<F, D>::kStages, kPitch = D + 4;
    static_assert(sizeof(float) * kCols * kPitch <= sizeof(Smem<F, D>::ring[0]), "a warp's output takes the place of its ring");
    extern __shared__ __align__(128) unsigned char raw[];
    Smem<F, D>& sm = *reinterpret_cast<Smem<F, D>*>(raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = lane >> 2, c4 = lane & 3;
    const int split = blockIdx.x, kvh = blockIdx.y / a.blocks, hb = blockIdx.y % a.blocks, b = blockIdx.z;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (lane < kStages) mbar_init(smem_u32(&sm.full[warp][lane]), 1);
    if (lane == 0) sm.abort_flag[warp] = 0;
    mbar_fence_init();
    __syncwarp();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int pos = a.pos[b];
    if (pos < 0) return;                                                        // (uniform over the cluster: nobody waits)
    if (pos >= a.c.capacity() || (a.cos && pos >= a.rope_rows)) {
        if (threadIdx.x == 0) atomicExch(a.error, kErrPosition);
        return;
    }
    const int tiles = (pos >> 4) + 1;
    const int lo = (int)((long long)tiles * split / a.splits), hi = (int)((long long)tiles * (split + 1) / a.splits);
    const int mine = hi - lo > warp ? (hi - lo - warp + kWarps - 1) / kWarps : 0;  // tiles lo + warp, lo + warp + kWarps, ...

    // ---- the ring: page numbers 32 tiles at a time, one batch ahead
    const int* table = a.c.table + (size_t)b * a.c.width;
    const int tshift = a.c.page_shift - 4;
    auto page_of = [&](int i) {
        const int t = lo + warp + i * kWarps;
        return t < hi ? table[t >> tshift] : -1;
    };
    int ids0 = page_of(lane), ids1 = mine > 32 ? page_of(32 + lane) : -1, batch = 0;
    auto id_at = [&](int i) { return __shfl_sync(0xffffffffu, (i >> 5) == batch ? ids0 : ids1, i & 31); };
    auto tile_at = [&](int i, int page) {
        const int t = lo + warp + i * kWarps;
        return a.c.pool + ((((size_t)page * a.c.kv_heads + kvh) << tshift) + (t & ((1 << tshift) - 1))) * (size_t)F::kBytes;
    };
    auto fetch = [&](int i) {
        const int page = id_at(i);
        if (lane == 0 && (unsigned)page < (unsigned)a.c.pages) {
            const uint32_t bar = smem_u32(&sm.full[warp][i % kStages]);
            mbar_arrive_expect_tx(bar, F::kBytes);
            bulk_load(smem_u32(sm.ring[warp][i % kStages]), tile_at(i, page), F::kBytes, bar);
        } else if (lane == 0) {
            mbar_arrive(smem_u32(&sm.full[warp][i % kStages]));                 // no page: the phase passes, the tile is left out
        }
    };
    for (int i = 0; i < kStages && i < mine; ++i) fetch(i);

    // ---- queries: column n = lane / 4, dims 32 j + 8 c .. + 7 (the key word the same lane reads)
    uint32_t qf[J][4];                                                          // low nibbles' dims (0,4)(2,6), high nibbles' (1,5)(3,7) / 16
    float qsum[NG][2], unit[2];
    {
        const int h = hb * kCols + row;
        float q[J][8], top = 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j) {
#pragma unroll
            for (int i = 0; i < 8; ++i) q[j][i] = 0.f;
            if (h < a.share) load_rotated<D>(a.qkv + b * a.stride + (kvh * a.share + h) * D, 4 * j + c4, a.cos, a.sin, pos, q[j]);
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(q[j][i]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // largest element into [2^14, 2^15): then a sixteenth of an element is exact down to 2^-39 of the largest
        const int e = top > 0.f ? max(14 - ((__float_as_int(top) >> 23) - 127), -2) : 0;      // (-2: infinities)
        const float up = pow2(e);
        float sums[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) sums[g] = 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                q[j][i] *= up;
                sums[32 * j * NG / D] += q[j][i];
            }
            qf[j][0] = pack2(q[j][0], q[j][4]);
            qf[j][1] = pack2(q[j][2], q[j][6]);
            qf[j][2] = pack2(q[j][1] * 0.0625f, q[j][5] * 0.0625f);
            qf[j][3] = pack2(q[j][3] * 0.0625f, q[j][7] * 0.0625f);
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            sums[g] += __shfl_xor_sync(0xffffffffu, sums[g], 1);
            sums[g] += __shfl_xor_sync(0xffffffffu, sums[g], 2);
            sums[g] *= 5.9604644775390625e-08f;                                 // 2^-24, as the codes' products carry it
#pragma unroll
            for (int k = 0; k < 2; ++k) qsum[g][k] = __shfl_sync(0xffffffffu, sums[g], 4 * (2 * c4 + k));
        }
        const float mul = a.scale_log2 * pow2(24 - e);
#pragma unroll
        for (int k = 0; k < 2; ++k) unit[k] = __shfl_sync(0xffffffffu, mul, 4 * (2 * c4 + k));
    }

    float acc[J][2][4];                                                         // [32 dims][pair of dims of a half-word][fragment]
    float off[NG][2];                                                           // the minima's part
    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
    float vinv = 16777216.f;                                                    // power of two: steps times it are at most 32
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[j][e][i] = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) off[g][0] = off[g][1] = 0.f;

    const int t0 = token_of(row);
    bool gave_up = false;
    int issued = mine < kStages ? mine : kStages;
    for (int i = 0; i < mine && i < issued; ++i) {
        if ((i >> 5) != batch) {
            ids0 = ids1;
            ++batch;
            ids1 = page_of(32 * (batch + 1) + lane);
        }
        const int page = id_at(i);
        unsigned char* tile = sm.ring[warp][i % kStages];
        if (!mbar_wait(smem_u32(&sm.full[warp][i % kStages]), (i / kStages) & 1, &sm.abort_flag[warp], kWaitNs)) gave_up = true;
        gave_up = __any_sync(0xffffffffu, gave_up);
        const bool there = (unsigned)page < (unsigned)a.c.pages;
        if (!there && lane == 0) atomicExch(a.error, kErrPage);
        if (there && !gave_up) {
            const bool last = lo + warp + i * kWarps == tiles - 1;
            if (last) {
                // the new token's row: quantised here, into this tile and (by the first pass) into the cache
                const bool value = (lane / F::NW) & 1;
                const int w = lane % F::NW, r = pos & 15;
                constexpr int kLanes = D / NG / 8;
                float x[8];
                load_rotated<D>(a.qkv + b * a.stride + (a.heads + (value ? a.c.kv_heads : 0) + kvh) * D, w, value ? nullptr : a.cos, a.sin, pos, x);
                __half2 par;
                const uint32_t word = quantize8(x, kLanes, par);
                auto put = [&](unsigned char* to) {
                    if (!value) {
                        *reinterpret_cast<uint32_t*>(to + F::key_word(r, w)) = word;
                    } else {
                        *reinterpret_cast<uint16_t*>(to + F::val_half(r, 2 * w)) = (uint16_t)word;
                        *reinterpret_cast<uint16_t*>(to + F::val_half(r, 2 * w + 1)) = (uint16_t)(word >> 16);
                    }
                    if (w % kLanes == 0) *reinterpret_cast<__half2*>(to + (value ? F::val_par(r, w / kLanes) : F::key_par(r, w / kLanes))) = par;
                };
                if (lane < 2 * F::NW) {
                    put(tile);
                    if (hb == 0) put(tile_at(i, page));
                }
                __syncwarp();
            }
            // scores: fragment rows are the tokens t0 and t0 + 8, columns the heads 2 c and 2 c + 1
            float x[4] = {0.f, 0.f, 0.f, 0.f};
            {
                uint32_t ka[J], kb[J];
                if constexpr (J == 4) {
                    *reinterpret_cast<uint4*>(ka) = *reinterpret_cast<const uint4*>(tile + t0 * (D / 2) + 16 * c4);
                    *reinterpret_cast<uint4*>(kb) = *reinterpret_cast<const uint4*>(tile + (t0 + 8) * (D / 2) + 16 * c4);
                } else {
                    *reinterpret_cast<uint2*>(ka) = *reinterpret_cast<const uint2*>(tile + t0 * (D / 2) + 8 * c4);
                    *reinterpret_cast<uint2*>(kb) = *reinterpret_cast<const uint2*>(tile + (t0 + 8) * (D / 2) + 8 * c4);
                }
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int j = g * J / NG; j < (g + 1) * J / NG; ++j) {
                        uint32_t ha[4], hc[4];
                        unpack_s4x8_denorm(ka[j], ha);
                        unpack_s4x8_denorm(kb[j], hc);
                        const uint32_t lowf[4] = {ha[0], hc[0], ha[2], hc[2]}, highf[4] = {ha[1], hc[1], ha[3], hc[3]};
                        mma_m16n8k16(s4, lowf, qf[j][0], qf[j][1]);
                        mma_m16n8k16(s4, highf, qf[j][2], qf[j][3]);
                    }
                    const float2 pa = __half22float2(*reinterpret_cast<const __half2*>(tile + F::key_par(t0, g)));
                    const float2 pb = __half22float2(*reinterpret_cast<const __half2*>(tile + F::key_par(t0 + 8, g)));
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        x[k] = fmaf(pa.x, s4[k], fmaf(pa.y, qsum[g][k], x[k]));
                        x[2 + k] = fmaf(pb.x, s4[2 + k], fmaf(pb.y, qsum[g][k], x[2 + k]));
                    }
                }
            }
            float2 va[NG], vb[NG];                                              // (step, minimum) of the two tokens' values
            float smax = 0.f;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                va[g] = __half22float2(*reinterpret_cast<const __half2*>(tile + F::val_par(t0, g)));
                vb[g] = __half22float2(*reinterpret_cast<const __half2*>(tile + F::val_par(t0 + 8, g)));
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                x[k] *= unit[k];
                x[2 + k] *= unit[k];
            }
            if (last) {                                                         // tokens behind the new one: whatever the page holds there
                const int left = pos & 15;
                if (t0 > left) {
                    x[0] = x[1] = -INFINITY;
#pragma unroll
                    for (int g = 0; g < NG; ++g) va[g] = make_float2(0.f, 0.f);
                }
                if (t0 + 8 > left) {
                    x[2] = x[3] = -INFINITY;
#pragma unroll
                    for (int g = 0; g < NG; ++g) vb[g] = make_float2(0.f, 0.f);
                }
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) smax = fmaxf(smax, fmaxf(va[g].x, vb[g].x));
            const float m0 = fmaxf(x[0], x[2]), m1 = fmaxf(x[1], x[3]);
            if (__any_sync(0xffffffffu, m0 > top[0] + 8.f || m1 > top[1] + 8.f || smax * vinv > 32.f)) {
                float n0 = fmaxf(m0, top[0]), n1 = fmaxf(m1, top[1]);
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) {
                    n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, o));
                    n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, o));
                    smax = fmaxf(smax, __shfl_xor_sync(0xffffffffu, smax, o));
                }
                // steps up to the largest fp16, 2^16, down to 2^-24
                const float vnew = smax * vinv > 32.f ? pow2(-((__float_as_int(fminf(smax, 65504.f)) >> 23) - 127)) : vinv;
                const float keep[2] = {top[0] == -INFINITY ? 0.f : ex2(top[0] - n0), top[1] == -INFINITY ? 0.f : ex2(top[1] - n1)};
                const float turn = vnew / vinv;
                top[0] = n0;
                top[1] = n1;
                vinv = vnew;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    sum[k] *= keep[k];
#pragma unroll
                    for (int g = 0; g < NG; ++g) off[g][k] *= keep[k];
#pragma unroll
                    for (int j = 0; j < J; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            acc[j][e][k] *= keep[k] * turn;
                            acc[j][e][2 + k] *= keep[k] * turn;
                        }
                }
            }
            const float p[4] = {ex2(x[0] - top[0]), ex2(x[1] - top[1]), ex2(x[2] - top[0]), ex2(x[3] - top[1])};
            sum[0] += p[0] + p[2];
            sum[1] += p[1] + p[3];
            uint32_t wf[NG][2];                                                 // B fragments: tokens 2c, 2c+1 (+ 8) of column lane / 4
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const float sa = va[g].x * vinv, sb = vb[g].x * vinv;
                wf[g][0] = transpose8x8(pack2(p[0] * sa, p[1] * sa));
                wf[g][1] = transpose8x8(pack2(p[2] * sb, p[3] * sb));
#pragma unroll
                for (int k = 0; k < 2; ++k) off[g][k] = fmaf(p[k], va[g].y, fmaf(p[2 + k], vb[g].y, off[g][k]));
            }
            // output: fragment rows are dims 32 j + 4 row + 2 e and the next one
            uint32_t v[4][J / 2];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int t = token_of(2 * c4 + (k & 1)) + 8 * (k >> 1);
                const unsigned char* at = tile + F::kVal + t * (D / 2) + (D == 128 ? (8 * row) ^ (((t >> 1) & 1) << 5) : 4 * row);
                if constexpr (J == 4) *reinterpret_cast<uint2*>(v[k]) = *reinterpret_cast<const uint2*>(at);
                else v[k][0] = *reinterpret_cast<const uint32_t*>(at);
            }
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const uint32_t u0 = __byte_perm(v[0][j / 2], v[1][j / 2], j & 1 ? 0x7632 : 0x5410);
                const uint32_t u1 = __byte_perm(v[2][j / 2], v[3][j / 2], j & 1 ? 0x7632 : 0x5410);
                uint32_t h0[4], h1[4];
                unpack_s4x8_denorm(u0, h0);
                unpack_s4x8_denorm(u1, h1);
                const uint32_t f0[4] = {h0[0], h0[1], h1[0], h1[1]}, f1[4] = {h0[2], h0[3], h1[2], h1[3]};
                constexpr int per = D / NG;
                mma_m16n8k16(acc[j][0], f0, wf[32 * j / per][0], wf[32 * j / per][1]);
                mma_m16n8k16(acc[j][1], f1, wf[32 * j / per][0], wf[32 * j / per][1]);
            }
        }
        __syncwarp();                                                           // everybody has read the tile
        if (!gave_up && issued < mine) {
            fetch(issued);
            ++issued;
        }
    }
    if (gave_up && lane == 0) atomicExch(a.error, 1);

    // ---- the warp's result takes the place of its ring: [column][D], maxima and sums beside it
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
            sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], o);
#pragma unroll
            for (int g = 0; g < NG; ++g) off[g][k] += __shfl_xor_sync(0xffffffffu, off[g][k], o);
        }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
        if (sum[k] != sum[k]) top[k] = sum[k];                                  // NaN scores: not to be taken for "no tiles"
    __syncwarp();
    float* o_s = reinterpret_cast<float*>(sm.ring[warp]);
    const float back = 1.f / vinv;                                              // (exact: a power of two)
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                float* at = o_s + (2 * c4 + k) * kPitch + 32 * j + 4 * row + 2 * e;
                at[0] = fmaf(acc[j][e][k] * kDenormScaleLo, back, off[32 * j * NG / D][k]);
                at[1] = fmaf(acc[j][e][2 + k] * kDenormScaleHi, back, off[32 * j * NG / D][k]);
            }
    if (row == 0) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            sm.m[warp][2 * c4 + k] = top[k];
            sm.l[warp][2 * c4 + k] = sum[k];
        }
    }
    __syncthreads();
    const int cols = min(kCols, a.share - hb * kCols);
    if (threadIdx.x < kCols) {
        float m = -INFINITY, l = 0.f;
        for (int w = 0; w < kWarps; ++w) m = fmaxf(m, sm.m[w][threadIdx.x]);
        for (int w = 0; w < kWarps; ++w) {
            const float f = sm.m[w][threadIdx.x] == -INFINITY ? 0.f : ex2(sm.m[w][threadIdx.x] - m);
            l = fmaf(sm.l[w][threadIdx.x], f, l);
            sm.m[w][threadIdx.x] = f;                                           // from here on: the warp's factor
        }
        sm.m[kWarps][threadIdx.x] = m;
        sm.l[kWarps][threadIdx.x] = l;
    }
    __syncthreads();
    auto merged = [&](int col, int d) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = sm.m[w][col];
            if (f != 0.f) v = fmaf(reinterpret_cast<const float*>(sm.ring[w])[col * kPitch + d], f, v);
        }
        return v;
    };
    const int head0 = kvh * a.share + hb * kCols;
    if (a.splits == 1) {
        for (int i = threadIdx.x; i < cols * D; i += kThreads) {
            const float l = sm.l[kWarps][i / D];
            a.out[((size_t)b * a.heads + head0) * D + i] = __float2half_rn(l == 0.f ? 0.f : merged(i / D, i % D) / l);
        }
        return;
    }
    if (a.part) {                                                               // joined by join_kernel
        for (int i = threadIdx.x; i < cols * D; i += kThreads)
            a.part[(((size_t)b * a.heads + head0 + i / D) * a.splits + split) * (D + 2) + i % D] = merged(i / D, i % D);
        if (threadIdx.x < cols) {
            float* at = a.part + (((size_t)b * a.heads + head0 + threadIdx.x) * a.splits + split) * (D + 2) + D;
            at[0] = sm.m[kWarps][threadIdx.x];
            at[1] = sm.l[kWarps][threadIdx.x];
        }
        return;
    }
    // the cluster: every CTA leaves its merged output in place of warp 0's, and joins its share of the elements
    {
        float* o0 = reinterpret_cast<float*>(sm.ring[0]);
        for (int i = threadIdx.x; i < cols * D; i += kThreads) o0[(i / D) * kPitch + i % D] = merged(i / D, i % D);
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        for (int i = threadIdx.x + split * kThreads; i < cols * D; i += kThreads * a.splits) {
            const int col = i / D;
            float m = -INFINITY, num = 0.f, den = 0.f;
            for (int r = 0; r < a.splits; ++r) m = fmaxf(m, *cluster.map_shared_rank(&sm.m[kWarps][col], r));
            for (int r = 0; r < a.splits; ++r) {
                const float mr = *cluster.map_shared_rank(&sm.m[kWarps][col], r);
                if (mr == -INFINITY) continue;                                  // no tiles of its own
                const float f = ex2(mr - m);
                num = fmaf(*cluster.map_shared_rank(o0 + col * kPitch + i % D, r), f, num);
                den = fmaf(*cluster.map_shared_rank(&sm.l[kWarps][col], r), f, den);
            }
            a.out[((size_t)b * a.heads + head0) * D + i] = __float2half_rn(den == 0.f ? 0.f : num / den);
        }
        cluster.sync();                                                         // others may still be reading this CTA's
    }
}

// Joins the partial outputs of a row's splits: grid (heads, batch), a thread per dim.
template <int D>
__global__ void __launch_bounds__(D) join_kernel(const DecodeArgs a)
{
    const int head = blockIdx.x, b = blockIdx.y, pos = a.pos[b];
    if (pos < 0 || pos >= a.c.capacity() || (a.cos && pos >= a.rope_rows)) return;
    const float* part = a.part + ((size_t)b * a.heads + head) * a.splits * (D + 2);
    float m = -INFINITY, num = 0.f, den = 0.f;
    for (int r = 0; r < a.splits; ++r) m = fmaxf(m, part[r * (D + 2) + D]);
    for (int r = 0; r < a.splits; ++r) {
        const float mr = part[r * (D + 2) + D];
        if (mr == -INFINITY) continue;
        const float f = ex2(mr - m);
        num = fmaf(part[r * (D + 2) + threadIdx.x], f, num);
        den = fmaf(part[r * (D + 2) + D + 1], f, den);
    }
    a.out[((size_t)b * a.heads + head) * D + threadIdx.x] = __float2half_rn(den == 0.f ? 0.f : num / den);
}

int g_force_split = 0;

}  // namespace

// CTAs that share a row's tiles.  Up to 8 meet in a cluster, more go through the workspace.
int decode_splits(int batch, int heads, int kv_heads, int page_size, int width)
{
    if (g_force_split) return g_force_split;
    const int share = heads / kv_heads, blocks = (share + kCols - 1) / kCols;
    const long long units = (long long)batch * kv_heads * blocks, slots = 4ll * device_sm_count();
    const long long tiles = (long long)width * page_size / kTile;              // of the longest row the table can hold
    int s = 1;
    while (s < 8 && units * s * 2 <= slots && tiles >= 2ll * kWarps * s * 2) s *= 2;
    if (s == 8 && units * 16 <= slots && tiles >= 16ll * kWarps * 8) {
        s = (int)(slots / units);
        while (s > 16 && tiles < (long long)s * kWarps * 4) --s;
        if (s > 128) s = 128;
    }
    return s;
}

template <class F, int D>
static int launch_decode_as(const DecodeArgs& a, int batch, cudaStream_t st)
{
    using S = Smem<F, D>;
    static int configured[64] = {0};   // benign race: the attribute call is idempotent
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return record_cuda_error(e);
    if (dev >= 64 || !configured[dev]) {
        e = cudaFuncSetAttribute(decode_kernel<F, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(S));
        if (e != cudaSuccess) return record_cuda_error(e);
        if (dev < 64) configured[dev] = 1;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.splits, a.c.kv_heads * a.blocks, batch);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = sizeof(S);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (a.splits > 1 && !a.part) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = a.splits;
        attr[n].val.clusterDim.y = 1;
        attr[n++].val.clusterDim.z = 1;
    }
    if (aux_programmatic_launch()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    e = cudaLaunchKernelEx(&cfg, decode_kernel<F, D>, a);
    if (e != cudaSuccess) return record_cuda_error(e);
    count_launch();
    if (a.part) {
        join_kernel<D><<<dim3(a.heads, batch), D, 0, st>>>(a);
        count_launch();
        e = cudaGetLastError();
        if (e != cudaSuccess) return record_cuda_error(e);
    }
    return W4A16_OK;
}

}  // namespace kv4
}  // namespace w4a16

using namespace w4a16;
using namespace w4a16::kv4;

// Tuning hook for tests and benchmarks: CTAs per (row, head), 0 = automatic.  Not part of the drop-in surface.
extern "C" void w4a16_tune_kv4(int splits)
{
    const bool ok = splits == 1 || splits == 2 || splits == 4 || splits == 8 || (splits > 8 && splits <= 128);
    w4a16::kv4::g_force_split = ok ? splits : 0;
}

extern "C" size_t w4a16_kv4_decode_workspace(int batch, int heads, int kv_heads, int head_dim, int page_size, int width)
{
    if (batch <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || head_dim <= 0 || page_size <= 0 || width <= 0) return 0;
    const int s = decode_splits(batch, heads, kv_heads, page_size, width);
    return s <= 8 ? 0 : (size_t)batch * heads * s * (head_dim + 2) * sizeof(float);
}

extern "C" int w4a16_kv4_decode_attention(const void* qkv, void* pool, const void* table, const void* pos, const void* rope_cos,
                                          const void* rope_sin, void* out, void* workspace, size_t workspace_bytes, int batch, int heads,
                                          int kv_heads, int head_dim, int group, int page_size, int pages, int width, long long qkv_stride,
                                          int rope_rows, float scale, void* stream)
{
    DecodeArgs a;
    if (!qkv || !pos || !out || ((rope_cos == nullptr) != (rope_sin == nullptr))) return W4A16_ERR_NULL_POINTER;
    int s = check_cache(a.c, pool, table, pages, width, page_size, kv_heads, head_dim, group);
    if (s != W4A16_OK) return s;
    if (batch < 0 || heads <= 0 || heads % kv_heads || qkv_stride < (heads + 2ll * kv_heads) * head_dim || (qkv_stride % 8) ||
        (rope_cos && rope_rows <= 0))
        return W4A16_ERR_BAD_SHAPE;
    if (((uintptr_t)qkv | (uintptr_t)out | (uintptr_t)rope_cos | (uintptr_t)rope_sin) & 15 || ((uintptr_t)pos | (uintptr_t)workspace) & 3)
        return W4A16_ERR_MISALIGNED;
    if ((heads + 2ll * kv_heads) * head_dim >= (1ll << 30) || batch > 65535) return W4A16_ERR_TOO_LARGE;
    a.share = heads / kv_heads;
    a.blocks = (a.share + kCols - 1) / kCols;
    if ((long long)kv_heads * a.blocks > 65535) return W4A16_ERR_TOO_LARGE;
    if (batch == 0) return W4A16_OK;
    a.splits = decode_splits(batch, heads, kv_heads, page_size, width);
    a.part = nullptr;
    if (a.splits > 8) {
        if (!workspace || workspace_bytes < w4a16_kv4_decode_workspace(batch, heads, kv_heads, head_dim, page_size, width)) return W4A16_ERR_WORKSPACE;
        a.part = (float*)workspace;
    }
    a.qkv = (const __half*)qkv; a.out = (__half*)out; a.pos = (const int*)pos;
    a.cos = (const __half*)rope_cos; a.sin = (const __half*)rope_sin;
    a.heads = heads; a.rope_rows = rope_rows; a.stride = qkv_stride;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.error = device_error_word();
    if (!a.error) return W4A16_ERR_CUDA;
    return with_format(head_dim, group, [&](auto f) {
        using F = decltype(f);
        return launch_decode_as<F, F::NW * 8>(a, batch, (cudaStream_t)stream);
    });
}
