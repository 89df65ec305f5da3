// Attention of a chunk of queries over the paged 4-bit cache, on the 5th-generation tensor cores.
//
// A CTA takes 128 rows of one (batch row, key/value head): row f of the chunk's S x R is query f / R of head f % R of the R that share the
// key/value head.  It walks over tiles of 128 cached tokens, up to its last query's position:
//     S = Q K^T     128 x 128, Q and K in shared memory, S in tensor memory
//     P = 2^(S scale - ref), rounded to fp16, over S's place in tensor memory; ref follows the row's maximum by steps of 2^8 and more
//     O += P V      P in tensor memory, V^T in shared memory, O in tensor memory
// K and V come as codes: all eight warps turn m + n s into fp16 (one rounding, 2^-11 of the value) while the matrix products of the step
// before run, and write the 128-byte swizzled layouts the products read - keys by tokens (dims of a word of 8 in the order 0 4 1 5 2 6
// 3 7 that the codes unpack in; the queries are stored in the same order), values by dims (pairs of tokens unpack side by side).  Codes
// travel from global memory through registers, one tile ahead.  256 threads, two for each row in the softmax, and two CTAs an SM: what
// one of them waits for - S, then P V, one after the other, since P stands where S stood - is time for the other's arithmetic.
//
// A value whose group is not finite is multiplied as 0, so that rows that must not see its token stay clean, and the rows that do see it
// get NaN for that group's dims at the end.
#include "w4a16_kv4.cuh"
#include "w4a16_sm100.cuh"

namespace w4a16 {
namespace kv4 {
namespace {

using namespace sm100;

constexpr int kRows = 128, kTokens = 128, kThreads = 256;
constexpr int kTilesOf = kTokens / kTile;         // 16-token tiles of a step
constexpr uint64_t kWaitNs = 400000000ull;        // a product that has not finished by then never will: error word 1
constexpr uint32_t kTmemCols = 256;               // S (then P) in columns 0 .. 127, O behind it: two CTAs an SM

struct PromptArgs {
    Cache c;
    const __half* qkv;            // [batch][seq] rows of `stride` elements; the queries of all heads stand first
    __half* out;                  // [batch][seq][heads * D]
    const int* pos;
    const int* counts;            // null: seq queries in every row
    const __half* cos;
    const __half* sin;
    int* error;
    int seq, heads, share;        // share: query heads of a key/value head
    int blocks;                   // of 128 rows
    int rope_rows;
    long long stride, page_bytes;
    float scale_log2;             // scale * log2(e)
};

template <int D>
struct Smem {
    alignas(1024) unsigned char q[kRows * D * 2], k[kTokens * D * 2], v[kTokens * D * 2];
    uint64_t s_done, pv_done;
    uint32_t tmem;
    int abort_flag;
    unsigned char page_ok[2][kTilesOf];           // 1: the tile's page is one of the pool
    int bad[kTokens];                             // groups of a token's value that are not finite
    float swap[2][kRows];                         // what the two threads of a row tell each other
    int swap_bad[kRows];
};

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ __half2 h2_of(uint32_t b) { return *reinterpret_cast<const __half2*>(&b); }

// Codes of a word as half2: dims (0,4), (1,5), (2,6), (3,7).
__device__ __forceinline__ void codes8(uint32_t w, __half2 (&n)[4])
{
    const uint32_t top = w >> 8;
    const __half2 k1024 = h2_of(0x64006400u), k16th = h2_of(0x2c002c00u), k64 = h2_of(0xd400d400u);   // 1024, 1/16, -64
    n[0] = __hsub2(h2_of(lop3_and_or(w, 0x000f000fu, 0x64006400u)), k1024);
    n[1] = __hfma2(h2_of(lop3_and_or(w, 0x00f000f0u, 0x64006400u)), k16th, k64);
    n[2] = __hsub2(h2_of(lop3_and_or(top, 0x000f000fu, 0x64006400u)), k1024);
    n[3] = __hfma2(h2_of(lop3_and_or(top, 0x00f000f0u, 0x64006400u)), k16th, k64);
}
__device__ __forceinline__ bool finite2(__half2 p) { return (h2_bits(p) & 0x7c00u) != 0x7c00u && (h2_bits(p) & 0x7c000000u) != 0x7c000000u; }

// D[tmem] (+)= A[smem] * B[smem], both K-major fp16
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
          "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void smem_for_mma() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// byte of 16-byte chunk `c` (8 halves) of row r in an operand of `rows` rows, 64 halves a sub-tile, 128-byte swizzle
__device__ __forceinline__ int operand_at(int rows, int r, int c) { return (c >> 3) * rows * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4); }

template <class F, int D>
__global__ void __launch_bounds__(kThreads, 2) prompt_kernel(const PromptArgs a)
{
    constexpr int J = F::J, NG = F::NG, kBytes = F::kBytes;
    extern __shared__ unsigned char raw[];
    Smem<D>& sm = *reinterpret_cast<Smem<D>*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int block = a.blocks - 1 - (int)blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;         // the longest rows first
    const int pos = a.pos[b], count = a.counts ? min(a.counts[b], a.seq) : a.seq;
    if (pos < 0 || count <= 0) return;
    const int room = min(a.c.capacity(), a.cos ? a.rope_rows : 0x7fffffff);
    const int fit = pos >= room ? 0 : min(count, room - pos);                                    // queries that can be served
    if (fit < count && block == 0 && kvh == 0 && tid == 0) atomicExch(a.error, kErrPosition);
    const long long rows = (long long)fit * a.share;
    if ((long long)block * kRows >= rows) return;
    const int first_i = (int)((long long)block * kRows / a.share);
    const int last_i = (int)(min((long long)(block + 1) * kRows, rows) - 1) / a.share;
    const int last = pos + last_i;                                                               // the last token anybody here sees
    const int steps = last / kTokens + 1;

    if (warp == 0) {
        tmem_alloc(smem_u32(&sm.tmem), kTmemCols);
        tmem_relinquish();
    }
    if (tid == 0) {
        mbar_init(smem_u32(&sm.s_done), 1);
        mbar_init(smem_u32(&sm.pv_done), 1);
        sm.abort_flag = 0;
    }
    mbar_fence_init();
    if (tid < kTokens) sm.bad[tid] = 0;

    // ---- codes on their way: what a thread turns into K and V of a step, in registers from one step to the next
    const int tshift = a.c.page_shift - 4, per1 = (1 << tshift) - 1;
    const int* ids = a.c.table + (size_t)b * a.c.width;
    const unsigned char* head = a.c.pool + ((size_t)kvh << tshift) * kBytes;
    auto tile_at = [&](int t16) -> const unsigned char* {                                       // null: behind the last token, or no page
        if (t16 > last >> 4) return nullptr;
        const int page = ids[t16 >> tshift];
        if ((unsigned)page >= (unsigned)a.c.pages) return nullptr;
        return head + page * a.page_bytes + (t16 & per1) * kBytes;
    };
    // keys: 16-byte pieces (4 words of 8 dims) of rows kt0 and, at D = 128, kt0 + 64; eight lanes take eight rows, so that their stores
    // fall on different banks
    constexpr int kPieces = D / 64;
    const int kt0 = D == 128 ? 8 * warp + (lane & 7) : 8 * (2 * warp + (lane >> 4)) + (lane & 7), kc = D == 128 ? lane >> 3 : (lane >> 3) & 1;
    // values: 8 tokens (group vt) by the half-words vh0 .. of lane-row vr; the lanes of a store fall on different banks as well
    constexpr int kHalves = J / 2;
    const int vt = 4 * (warp >> 1) + (lane & 3), vr = ((lane >> 2) & 1) | ((lane >> 3) << 1), vh0 = (warp & 1) * kHalves;
    constexpr int kVGroups = D / NG == 32 && kHalves == 2 ? 2 : 1;
    uint4 kw[kPieces];
    __half2 kp[kPieces][NG], vp[8][kVGroups];
    uint32_t vw[8];
    auto load_k = [&](int step) {
        if (tid < kTilesOf) {                                                                    // which tiles of the step have a page
            const int t16 = step * kTilesOf + tid;
            const bool ok = t16 > last >> 4 || tile_at(t16) != nullptr;
            sm.page_ok[step & 1][tid] = ok;
            if (!ok) atomicExch(a.error, kErrPage);
        }
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
            const int t = step * kTokens + kt0 + 64 * k, r = t & 15;
            const unsigned char* tile = tile_at(t >> 4);
            kw[k] = make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int g = 0; g < NG; ++g) kp[k][g] = h2_of(0);
            if (tile && t <= last) {
                kw[k] = *reinterpret_cast<const uint4*>(tile + r * (D / 2) + 16 * kc);
#pragma unroll
                for (int g = 0; g < NG; ++g) kp[k][g] = *reinterpret_cast<const __half2*>(tile + F::key_par(r, g));
            }
        }
    };
    auto put_k = [&]() {
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
            const uint32_t w4[4] = {kw[k].x, kw[k].y, kw[k].z, kw[k].w};
            __half2 s[NG], m[NG];
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                s[g] = __low2half2(kp[k][g]);
                m[g] = __high2half2(kp[k][g]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // stored word 4 kc + i is word w of the row; its group is known here where a piece holds one word of each 32 dims
                const int j = D == 128 ? i : i & 1, w = D == 128 ? 4 * i + kc : 4 * (i & 1) + 2 * kc + (i >> 1);
                const int g = 32 * j * NG / D;
                __half2 n[4];
                codes8(w4[i], n);
                uint4 o;
                o.x = h2_bits(__hfma2(n[0], s[g], m[g]));
                o.y = h2_bits(__hfma2(n[1], s[g], m[g]));
                o.z = h2_bits(__hfma2(n[2], s[g], m[g]));
                o.w = h2_bits(__hfma2(n[3], s[g], m[g]));
                *reinterpret_cast<uint4*>(sm.k + operand_at(kTokens, kt0 + 64 * k, w)) = o;
            }
        }
    };
    auto load_v = [&](int step) {
        const int t = step * kTokens + 8 * vt, r0 = t & 15;
        const unsigned char* tile = tile_at(t >> 4);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            vw[k] = 0;
#pragma unroll
            for (int g = 0; g < kVGroups; ++g) vp[k][g] = h2_of(0);
            if (tile && t + k <= last) {
                const int at = 2 * (vr * J + vh0);
                const unsigned char* from = tile + F::kVal + (r0 + k) * (D / 2) + (D == 128 ? at ^ (((k >> 1) & 1) << 5) : at);
                if constexpr (kHalves == 2) vw[k] = *reinterpret_cast<const uint32_t*>(from);
                else vw[k] = *reinterpret_cast<const uint16_t*>(from);
#pragma unroll
                for (int g = 0; g < kVGroups; ++g)
                    vp[k][g] = *reinterpret_cast<const __half2*>(tile + F::val_par(r0 + k, 32 * (vh0 + g) * NG / D));
            }
        }
    };
    auto put_v = [&]() {                                                                         // true: some value is not finite
        bool found = false;
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int g = 0; g < kVGroups; ++g)
                if (!finite2(vp[k][g])) {
                    vp[k][g] = h2_of(0);
                    atomicOr(&sm.bad[8 * vt + k], 1 << (32 * (vh0 + g) * NG / D));
                    found = true;
                }
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
            constexpr int last_group = kVGroups - 1;
            const int g = h < last_group ? h : last_group;
            uint32_t o[4][4];                                                                    // [dim of the half-word][pair of tokens]
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t pa = h2_bits(vp[2 * k][g]), pb = h2_bits(vp[2 * k + 1][g]);
                const __half2 s = h2_of(__byte_perm(pa, pb, 0x5410)), m = h2_of(__byte_perm(pa, pb, 0x7632));
                __half2 n[4];
                codes8(__byte_perm(vw[2 * k], vw[2 * k + 1], h ? 0x7632 : 0x5410), n);
#pragma unroll
                for (int d = 0; d < 4; ++d) o[d][k] = h2_bits(__hfma2(n[d], s, m));
            }
#pragma unroll
            for (int d = 0; d < 4; ++d)
                *reinterpret_cast<uint4*>(sm.v + operand_at(D, 32 * (vh0 + h) + 4 * vr + d, vt)) = make_uint4(o[d][0], o[d][1], o[d][2], o[d][3]);
        }
        return found;
    };
    load_k(0);
    load_v(0);

    // ---- queries: two threads a row, rotated as the decode kernel does, in the order of the keys' dims
    {
        const int r = tid >> 1;
        const long long f = (long long)block * kRows + r;
        const int i = (int)(f / a.share), h = (int)(f % a.share);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
            const int w = (tid & 1) * (D / 16) + k;
            float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (f < rows) load_rotated<D>(a.qkv + ((long long)b * a.seq + i) * a.stride + (kvh * a.share + h) * D, w, a.cos, a.sin, pos + i, x);
            uint4 o;
            o.x = h2_bits(__floats2half2_rn(x[0], x[4]));
            o.y = h2_bits(__floats2half2_rn(x[1], x[5]));
            o.z = h2_bits(__floats2half2_rn(x[2], x[6]));
            o.w = h2_bits(__floats2half2_rn(x[3], x[7]));
            *reinterpret_cast<uint4*>(sm.q + operand_at(kRows, r, w)) = o;
        }
    }
    put_k();
    smem_for_mma();
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = sm.tmem, lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t s_bar = smem_u32(&sm.s_done), pv_bar = smem_u32(&sm.pv_done);
    const uint64_t q_desc = smem_desc_sw128(smem_u32(sm.q)), k_desc = smem_desc_sw128(smem_u32(sm.k)), v_desc = smem_desc_sw128(smem_u32(sm.v));
    auto issue_s = [&]() {                                                                       // warp 0
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
            const uint64_t at = (uint64_t)((kk >> 2) * (kRows * 128 / 16) + 2 * (kk & 3));
            if (elect_one()) mma_f16_ss(tmem, q_desc + at, k_desc + at, idesc_f16_m128(kTokens), kk > 0);
        }
        if (elect_one()) tc_commit(s_bar);
        __syncwarp();
    };
    auto issue_pv = [&](bool first) {
#pragma unroll
        for (int kk = 0; kk < kTokens / 16; ++kk) {
            // P of tokens 0 .. 63 stands in columns 0 .. 31, of tokens 64 .. 127 in columns 64 .. 95
            const uint32_t p = tmem + (kk >> 2) * 64 + (kk & 3) * 8;
            const uint64_t at = (uint64_t)((kk >> 2) * (D * 128 / 16) + 2 * (kk & 3));
            if (elect_one()) mma_f16_ts(tmem + kTokens, p, v_desc + at, idesc_f16_m128(D), !first || kk > 0);
        }
        if (elect_one()) tc_commit(pv_bar);
        __syncwarp();
    };
    if (warp == 0) issue_s();

    // ---- the row of this thread in the softmax, and its half of the columns
    const int row = 32 * (warp & 3) + lane, half = warp >> 2;
    const int sees = pos + min((int)(((long long)block * kRows + row) / a.share), last_i);      // last token it sees (rows behind the last: as that one)
    const int first_sees = pos + first_i;
    // (the sign of a negative scale goes into the scores, so that `unit` is positive; a scale of zero makes them zero)
    const float unit = a.scale_log2 == 0.f ? 1.f : fabsf(a.scale_log2), sign = a.scale_log2 == 0.f ? 0.f : a.scale_log2 < 0.f ? -1.f : 1.f;
    float ref = -INFINITY, sum = 0.f;
    int nan_groups = 0;
    bool ok = true;
    for (int step = 0; step < steps; ++step) {
        const bool found = put_v();                                                              // (P V of the step before is over)
        smem_for_mma();
        if (step + 1 < steps) load_k(step + 1);
        ok = ok && mbar_wait(s_bar, step & 1, &sm.abort_flag, kWaitNs);
        tc_fence_after_sync();
        const uint64_t pages = *reinterpret_cast<const uint64_t*>(sm.page_ok[step & 1]);
        const bool masked = (step + 1) * kTokens - 1 > first_sees || pages != 0x0101010101010101ull;
        const int from = step * kTokens + 64 * half;                                             // the thread's first token
        uint32_t s[32];
        float top = -INFINITY;
        auto hide = [&](int c0) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const int t = from + c0 + i;
                const bool seen = t <= sees && (pages >> (8 * ((64 * half + c0 + i) >> 4)) & 1);
                if (!seen) s[i] = 0xff800000u;
            }
        };
        auto fetch = [&](int c0) {
            tmem_ld_32x32b_x32(tmem + lanes + 64 * half + c0, s);
            tmem_wait_ld();
            if (sign != 1.f) {
#pragma unroll
                for (int i = 0; i < 32; ++i) s[i] = __float_as_uint(__uint_as_float(s[i]) * sign);
            }
            if (masked) hide(c0);
        };
#pragma unroll
        for (int c = 1; c >= 0; --c) {
            fetch(32 * c);
#pragma unroll
            for (int i = 0; i < 32; ++i) top = fmaxf(top, __uint_as_float(s[i]));
        }
        // both threads of a row move the reference alike
        sm.swap[half][row] = top;
        asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory");
        top = fmaxf(top, sm.swap[half ^ 1][row]) * unit;
        bool move = top - ref > 8.f;                                                             // (from minus infinity as well; not with nothing seen)
        if (__any_sync(0xffffffffu, move)) {
            const float to = move ? top : ref, keep = ref == -INFINITY ? 0.f : ex2(ref - to);
            ref = to;
            sum *= keep;
            if (step > 0) {
                uint32_t o[16];
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    const uint32_t at = tmem + lanes + kTokens + half * (D / 2) + 16 * c;
                    tmem_ld_32x32b_x16(at, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
                    tmem_st_32x32b_x16(at, o);
                }
            }
        }
        const float shift = ref == -INFINITY ? 0.f : ref;                                        // nothing seen yet: weights 0
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            if (c == 1) fetch(32);
            uint32_t p[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float p0 = ex2(fmaf(__uint_as_float(s[2 * i]), unit, -shift)), p1 = ex2(fmaf(__uint_as_float(s[2 * i + 1]), unit, -shift));
                sum += p0 + p1;
                p[i] = h2_bits(__floats2half2_rn(p0, p1));
            }
            // over columns of S that this thread has read (its tokens 32 .. 63 are read again)
            tmem_st_32x32b_x16(tmem + lanes + 64 * half + 16 * c, p);
        }
        tmem_wait_st();
        tc_fence_before_sync();
        if (__syncthreads_or(found)) {
            // rows that see a value that is not finite
#pragma unroll 1
            for (int i = 0; i < 64; ++i) {
                const int t = from + i;
                if (t <= sees && (pages >> (8 * ((64 * half + i) >> 4)) & 1)) nan_groups |= sm.bad[64 * half + i];
            }
            __syncthreads();
            if (tid < kTokens) sm.bad[tid] = 0;
        }
        if (warp == 0) {
            tc_fence_after_sync();
            issue_pv(step == 0);
        }
        if (step + 1 < steps) {
            put_k();                                                                             // (S of this step is over)
            smem_for_mma();
            load_v(step + 1);
            ok = ok && mbar_wait(pv_bar, step & 1, &sm.abort_flag, kWaitNs);
            tc_fence_after_sync();
            tc_fence_before_sync();
            __syncthreads();
            if (warp == 0) {
                tc_fence_after_sync();
                issue_s();
            }
        }
    }
    ok = ok && mbar_wait(pv_bar, (steps - 1) & 1, &sm.abort_flag, kWaitNs);
    tc_fence_after_sync();
    if (!ok && lane == 0) atomicExch(a.error, 1);

    // ---- out = O / sum
    sm.swap[half][row] = sum;
    if (half) sm.swap_bad[row] = nan_groups;
    __syncthreads();
    sum += sm.swap[half ^ 1][row];
    if (!half) {
        nan_groups |= sm.swap_bad[row];
        sm.swap_bad[row] = nan_groups;
    }
    __syncthreads();
    nan_groups = sm.swap_bad[row];
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const long long f = (long long)block * kRows + row;
    __half* to = a.out + ((long long)b * a.seq + (int)(f / a.share)) * a.heads * D + (kvh * a.share + (int)(f % a.share)) * D + half * (D / 2);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
        uint32_t o[16];
        tmem_ld_32x32b_x16(tmem + lanes + kTokens + half * (D / 2) + 16 * c, o);
        tmem_wait_ld();
        if (f >= rows) continue;
        const int g = (half * (D / 2) + 16 * c) * NG / D;
        const float mul = nan_groups >> g & 1 ? __int_as_float(0x7fffffff) : inv;
        uint32_t h[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = h2_bits(__floats2half2_rn(__uint_as_float(o[2 * i]) * mul, __uint_as_float(o[2 * i + 1]) * mul));
        *reinterpret_cast<uint4*>(to + 16 * c) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(to + 16 * c + 8) = make_uint4(h[4], h[5], h[6], h[7]);
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem, kTmemCols);
}

template <class F, int D>
int launch_prompt_as(const PromptArgs& a, int batch, cudaStream_t st)
{
    static int configured[64] = {0};   // benign race: the attribute call is idempotent
    const int smem = (int)sizeof(Smem<D>) + 1024;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return record_cuda_error(e);
    if (dev >= 64 || !configured[dev]) {
        e = cudaFuncSetAttribute(prompt_kernel<F, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return record_cuda_error(e);
        if (dev < 64) configured[dev] = 1;
    }
    prompt_kernel<F, D><<<dim3(a.blocks, a.c.kv_heads, batch), kThreads, smem, st>>>(a);
    count_launch();
    e = cudaGetLastError();
    return e == cudaSuccess ? W4A16_OK : record_cuda_error(e);
}

}  // namespace
}  // namespace kv4
}  // namespace w4a16

using namespace w4a16;
using namespace w4a16::kv4;

extern "C" int w4a16_kv4_attention(const void* qkv, const void* pool, const void* table, const void* pos, const void* counts,
                                   const void* rope_cos, const void* rope_sin, void* out, int batch, int seq, int heads, int kv_heads,
                                   int head_dim, int group, int page_size, int pages, int width, long long qkv_stride, int rope_rows,
                                   float scale, void* stream)
{
    PromptArgs a;
    if (!qkv || !pos || !out || ((rope_cos == nullptr) != (rope_sin == nullptr))) return W4A16_ERR_NULL_POINTER;
    int s = check_cache(a.c, pool, table, pages, width, page_size, kv_heads, head_dim, group);
    if (s != W4A16_OK) return s;
    if (batch < 0 || seq < 0 || heads <= 0 || heads % kv_heads || qkv_stride < (long long)heads * head_dim || (qkv_stride % 8) ||
        (rope_cos && rope_rows <= 0))
        return W4A16_ERR_BAD_SHAPE;
    if (((uintptr_t)qkv | (uintptr_t)out | (uintptr_t)rope_cos | (uintptr_t)rope_sin) & 15 || ((uintptr_t)pos | (uintptr_t)counts) & 3)
        return W4A16_ERR_MISALIGNED;
    if ((heads + 2ll * kv_heads) * head_dim >= (1ll << 30) || batch > 65535 || kv_heads > 65535 || seq >= (1 << 30)) return W4A16_ERR_TOO_LARGE;
    a.share = heads / kv_heads;
    const long long blocks = ((long long)seq * a.share + kRows - 1) / kRows;
    if (blocks >= (1ll << 31)) return W4A16_ERR_TOO_LARGE;
    if (batch == 0 || seq == 0) return W4A16_OK;
    a.qkv = (const __half*)qkv; a.out = (__half*)out; a.pos = (const int*)pos; a.counts = (const int*)counts;
    a.cos = (const __half*)rope_cos; a.sin = (const __half*)rope_sin;
    a.seq = seq; a.heads = heads; a.blocks = (int)blocks; a.rope_rows = rope_rows; a.stride = qkv_stride;
    a.page_bytes = (long long)kv_heads * (page_size / kTile) * tile_bytes(head_dim, group);
    a.scale_log2 = scale * 1.4426950408889634f;
    a.error = device_error_word();
    if (!a.error) return W4A16_ERR_CUDA;
    return with_format(head_dim, group, [&](auto f) {
        using F = decltype(f);
        return launch_prompt_as<F, F::NW * 8>(a, batch, (cudaStream_t)stream);
    });
}
