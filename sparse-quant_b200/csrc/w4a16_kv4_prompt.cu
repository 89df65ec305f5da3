// Attention of a chunk of queries over the paged 4-bit cache, on the 5th-generation tensor cores.
//
// A CTA takes T x 128 rows of one (batch row, key/value head): row f of the chunk's S x R is query f / R of head f % R of the R that share
// the key/value head.  It walks over tiles of 128 cached tokens, up to its last query's position, for each of its T row tiles:
//     S = Q K^T     128 x 128, Q and K in shared memory, S in tensor memory
//     P = 2^(S scale - ref), rounded to fp16, over S's place in tensor memory; ref follows the row's maximum by steps of 2^8 and more
//     O += P V      P in tensor memory, V^T in shared memory, O in tensor memory
// K and V come as codes: the worker warps turn m + n s into fp16 (one rounding, 2^-11 of the value) while the products run, and write the
// 128-byte swizzled layouts the products read - keys by tokens (dims of a word of 8 in the order 0 4 1 5 2 6 3 7 that the codes unpack
// in; the queries are stored in the same order), values by dims: a transposing matrix load gives a lane the same four dims of two tokens,
// which unpack side by side.  The rows of V^T, and with them the columns of O, stand in the order 8 n + h + 32 p of dim n of the half-word
// 8 p + h that the cache stores, which puts the eight rows that one store instruction touches on different banks.  The codes of the next step are on
// their way to shared memory meanwhile, and where its tiles stand is looked up two steps ahead.  Two threads a row in the softmax, eight
// warps a row tile, and one warp that issues the products (issuing eight takes as long as they run).
//
// What bounds it is what the workers can issue: a tile of K and V costs them as much as its softmax.  So T = 2 (one CTA an SM) for more
// than 128 rows of 128 dims, which halves that cost; otherwise T = 1, two CTAs an SM.
//
// A value whose group is not finite is multiplied as 0, so that rows that must not see its token stay clean, and the rows that do see it
// get NaN for that group's dims at the end.
#include "w4a16_kv4.cuh"
#include "w4a16_sm100.cuh"

namespace w4a16 {
namespace kv4 {
namespace {

using namespace sm100;

constexpr int kRows = 128, kTokens = 128;
constexpr int kTilesOf = kTokens / kTile;         // 16-token tiles of a step
constexpr uint64_t kWaitNs = 400000000ull;        // a product that has not finished by then never will: error word 1

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
    int blocks;                   // of T x 128 rows
    int rope_rows;
    long long stride, page_bytes;
    float scale_log2;             // scale * log2(e)
};

template <int D, int half_tile, int T>
struct Smem {
    alignas(1024) unsigned char q[T][kRows * D * 2], k[kTokens * D * 2], v[kTokens * D * 2];
    // codes of the next step, with steps and minima (T = 1: the keys' come through registers, or two CTAs would not fit)
    alignas(16) unsigned char v_codes[kTilesOf][half_tile], k_codes[T == 1 ? 1 : kTilesOf][half_tile];
    const unsigned char* tile[4][kTilesOf];       // by step modulo 4: where its tiles stand; null: behind the last token, or no page
    unsigned char page_ok[4][kTilesOf];           // 0: a page is needed and is none of the pool
    uint64_t s_done[T], pv_done[T];               // products over
    uint64_t k_ready, v_ready, p_ready[T];        // operands written
    uint32_t tmem;
    int abort_flag;
    int bad[kTokens];                             // groups of a token's value that are not finite
    float swap[2][T * kRows];                     // what the two threads of a row tell each other
    int swap_bad[T * kRows];
};

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// two fp32 operations in one instruction
__device__ __forceinline__ uint64_t pair(float a, float b)
{
    uint64_t p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
    return p;
}
__device__ __forceinline__ float2 unpair(uint64_t p)
{
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
    return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
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
template <int N>
__device__ __forceinline__ void load_params(const unsigned char* at, __half2 (&p)[N])
{
    if constexpr (N == 4) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(at);
    else if constexpr (N == 2) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(at);
    else p[0] = *reinterpret_cast<const __half2*>(at);
}

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
__device__ __forceinline__ void copies_landed() { asm volatile("cp.async.wait_all;" ::: "memory"); }      // this thread's
// barriers of the worker warps
template <int N>
__device__ __forceinline__ void workers_sync() { asm volatile("bar.sync 9, %0;" ::"n"(N) : "memory"); }
template <int N>
__device__ __forceinline__ bool workers_any(bool mine)
{
    int any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.s32 p, %1, 0;\n\tbarrier.cta.red.or.aligned.pred q, 10, %2, p;\n\tselp.s32 %0, 1, 0, q;\n\t}"
                 : "=r"(any) : "r"((int)mine), "n"(N) : "memory");
    return any != 0;
}
// the warp's operand writes of either kind, made visible to the products, and its arrival
__device__ __forceinline__ void written(uint32_t bar, int lane)
{
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc_fence_before_sync();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
}

// byte of 16-byte chunk `c` (8 halves) of row r in an operand of `rows` rows, 64 halves a sub-tile, 128-byte swizzle
__device__ __forceinline__ int operand_at(int rows, int r, int c) { return (c >> 3) * rows * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4); }

template <class F, int D, int T>
__global__ void __launch_bounds__(256 * T + 32, T == 1 ? 2 : 1) prompt_kernel(const PromptArgs a)
{
    constexpr int J = F::J, NG = F::NG, kBytes = F::kBytes, kHalf = kBytes / 2, kWorkers = 256 * T, kWarps = 8 * T;
    constexpr uint32_t kTmemCols = 256 * T;       // a row tile's S (then P) in 128 columns, O in the 128 behind them
    static_assert(F::kVal == kHalf, "keys and values are halves of a tile");
    extern __shared__ unsigned char raw[];
    using S = Smem<D, kHalf, T>;
    S& sm = *reinterpret_cast<S*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int block = a.blocks - 1 - (int)blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;         // the longest rows first
    const int pos = a.pos[b], count = a.counts ? min(a.counts[b], a.seq) : a.seq;
    if (pos < 0 || count <= 0) return;
    const int room = min(a.c.capacity(), a.cos ? a.rope_rows : 0x7fffffff);
    const int fit = pos >= room ? 0 : min(count, room - pos);                                    // queries that can be served
    if (fit < count && block == 0 && kvh == 0 && tid == 0) atomicExch(a.error, kErrPosition);
    const long long rows = (long long)fit * a.share, row0 = (long long)block * (T * kRows);
    if (row0 >= rows) return;
    const int first_i = (int)(row0 / a.share), last_i = (int)(min(row0 + T * kRows, rows) - 1) / a.share;
    const int last = pos + last_i;                                                               // the last token anybody here sees
    const int steps = last / kTokens + 1;

    if (warp == kWarps) {
        tmem_alloc(smem_u32(&sm.tmem), kTmemCols);
        tmem_relinquish();
    }
    if (tid == 0) {
#pragma unroll
        for (int t = 0; t < T; ++t) {
            mbar_init(smem_u32(&sm.s_done[t]), 1);
            mbar_init(smem_u32(&sm.pv_done[t]), 1);
            mbar_init(smem_u32(&sm.p_ready[t]), 8);
        }
        mbar_init(smem_u32(&sm.k_ready), kWarps);
        mbar_init(smem_u32(&sm.v_ready), kWarps);
        sm.abort_flag = 0;
    }
    mbar_fence_init();
    if (tid < kTokens) sm.bad[tid] = 0;

    // ---- where the tiles of a step stand (threads 0 .. 7)
    const int tshift = a.c.page_shift - 4, per1 = (1 << tshift) - 1;
    const int* ids = a.c.table + (size_t)b * a.c.width;
    const unsigned char* head = a.c.pool + ((size_t)kvh << tshift) * kBytes;
    int next_id = -1;
    auto look = [&](int step) {
        const int t16 = step * kTilesOf + tid;
        next_id = t16 <= last >> 4 ? ids[t16 >> tshift] : -1;
    };
    auto note = [&](int step) {
        const int t16 = step * kTilesOf + tid;
        const bool needed = t16 <= last >> 4, there = needed && (unsigned)next_id < (unsigned)a.c.pages;
        sm.tile[step & 3][tid] = there ? head + next_id * a.page_bytes + (t16 & per1) * kBytes : nullptr;
        sm.page_ok[step & 3][tid] = there || !needed;
        if (needed && !there) atomicExch(a.error, kErrPage);
    };
    if (tid < kTilesOf) {
        look(0);
        note(0);
        look(1);
        note(1);
    }
    __syncthreads();
    const uint32_t tmem = sm.tmem;
    const uint32_t k_bar = smem_u32(&sm.k_ready), v_bar = smem_u32(&sm.v_ready);
    bool ok = true;

    if (warp == kWarps) {
        // ---- the products.  P stands where S stood: S of a step is issued when P V of the step before is over
        const uint64_t k_desc = smem_desc_sw128(smem_u32(sm.k)), v_desc = smem_desc_sw128(smem_u32(sm.v));
        for (int step = 0; step < steps; ++step) {
            ok = ok && mbar_wait(k_bar, step & 1, &sm.abort_flag, kWaitNs);                      // (the queries, at the first step)
#pragma unroll
            for (int t = 0; t < T; ++t) {
                if (step > 0) ok = ok && mbar_wait(smem_u32(&sm.pv_done[t]), (step - 1) & 1, &sm.abort_flag, kWaitNs);
                tc_fence_after_sync();
                __syncwarp();
                const uint64_t q_desc = smem_desc_sw128(smem_u32(sm.q[t]));
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    const uint64_t at = (uint64_t)((kk >> 2) * (kRows * 128 / 16) + 2 * (kk & 3));
                    if (elect_one()) mma_f16_ss(tmem + 256 * t, q_desc + at, k_desc + at, idesc_f16_m128(kTokens), kk > 0);
                }
                if (elect_one()) tc_commit(smem_u32(&sm.s_done[t]));
                __syncwarp();
            }
            ok = ok && mbar_wait(v_bar, step & 1, &sm.abort_flag, kWaitNs);
#pragma unroll
            for (int t = 0; t < T; ++t) {
                ok = ok && mbar_wait(smem_u32(&sm.p_ready[t]), step & 1, &sm.abort_flag, kWaitNs);
                tc_fence_after_sync();
                __syncwarp();
#pragma unroll
                for (int kk = 0; kk < kTokens / 16; ++kk) {
                    // P of tokens 0 .. 63 stands in columns 0 .. 31, of tokens 64 .. 127 in columns 64 .. 95
                    const uint32_t p = tmem + 256 * t + (kk >> 2) * 64 + (kk & 3) * 8;
                    const uint64_t at = (uint64_t)((kk >> 2) * (D * 128 / 16) + 2 * (kk & 3));
                    if (elect_one()) mma_f16_ts(tmem + 256 * t + kTokens, p, v_desc + at, idesc_f16_m128(D), step > 0 || kk > 0);
                }
                if (elect_one()) tc_commit(smem_u32(&sm.pv_done[t]));
                __syncwarp();
            }
        }
#pragma unroll
        for (int t = 0; t < T; ++t) ok = ok && mbar_wait(smem_u32(&sm.pv_done[t]), (steps - 1) & 1, &sm.abort_flag, kWaitNs);
        if (!ok && lane == 0) atomicExch(a.error, 1);
        __syncthreads();                                                                         // the workers have read O
        tmem_dealloc(tmem, kTmemCols);
        return;
    }

    // ---- codes of a step to shared memory, keys or values: tiles are contiguous halves of 16-byte pieces.  A code row's pieces change
    // places, so that the eight rows that are read together stand on different banks: by rows' bits 1 and 2 (keys; values stand
    // exchanged by bit 1 already), at D = 64 by bit 2.
    auto piece_of = [&](int row, int piece, bool values) {
        return D == 128 ? piece ^ (values ? (row >> 2) & 1 : (row >> 1) & 3) : piece ^ ((row >> 2) & 1);
    };
    auto load_codes = [&](unsigned char* to, int step, int half_at) {
        constexpr int kPieces = kHalf / 16, kRowPieces = D / 32;                                 // of a tile, of a code row
#pragma unroll
        for (int i = 0; i < (kTilesOf * kPieces + kWorkers - 1) / kWorkers; ++i) {
            const int at = tid + i * kWorkers;
            if (at >= kTilesOf * kPieces) break;
            const unsigned char* tile = sm.tile[step & 3][at / kPieces];
            const int piece = at % kPieces, row = piece / kRowPieces;
            const int there = row < kTile ? row * kRowPieces + piece_of(row, piece % kRowPieces, half_at != 0) : piece;
            // (a tile that is none is filled with zeros: its values are 0, its keys are hidden)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                         ::"r"(smem_u32(to) + (at - piece + there) * 16), "l"(tile ? tile + half_at + piece * 16 : a.c.pool), "r"(tile ? 16 : 0) : "memory");
        }
    };
    // keys: 16-byte pieces (4 words of 8 dims); eight lanes take eight rows, so that their stores fall on different banks
    constexpr int kPieces = kTokens * D / 32 / kWorkers < 1 ? 1 : kTokens * D / 32 / kWorkers;  // of a thread
    const int kp = lane >> 3, kt0 = D == 128 ? 8 * warp + (lane & 7) : 8 * (2 * warp + (kp >> 1)) + (lane & 7), kc = D == 128 ? kp : kp & 1;
    const bool has_k = kt0 < kTokens;                                                            // (D = 64, T = 2: half of the threads)
    uint4 kreg[T == 1 ? kPieces : 1];
    __half2 kpar[T == 1 ? kPieces : 1][NG];
    auto fetch_k = [&](int step) {
        if constexpr (T == 2) {
            load_codes(sm.k_codes[0], step, 0);
        } else {
#pragma unroll
            for (int k = 0; k < kPieces; ++k) {
                const int row = kt0 + 8 * kWarps * k;
                const unsigned char* tile = sm.tile[step & 3][row >> 4];
                kreg[k] = make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int g = 0; g < NG; ++g) kpar[k][g] = h2_of(0);
                if (tile) {
                    kreg[k] = *reinterpret_cast<const uint4*>(tile + (row & 15) * (D / 2) + 16 * kc);
                    load_params<NG>(tile + F::key_par(row & 15, 0), kpar[k]);
                }
            }
        }
    };
    auto put_k = [&]() {
        if (!has_k) return;
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
            const int row = kt0 + 8 * kWarps * k;
            uint4 kw;
            __half2 par[NG], s[NG], m[NG];
            if constexpr (T == 2) {
                const unsigned char* tile = sm.k_codes[row >> 4];
                kw = *reinterpret_cast<const uint4*>(tile + (row & 15) * (D / 2) + 16 * piece_of(row & 15, kc, false));
                load_params<NG>(tile + F::key_par(row & 15, 0), par);
            } else {
                kw = kreg[k];
#pragma unroll
                for (int g = 0; g < NG; ++g) par[g] = kpar[k][g];
            }
            const uint32_t w4[4] = {kw.x, kw.y, kw.z, kw.w};
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                s[g] = __low2half2(par[g]);
                m[g] = __high2half2(par[g]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // stored word 4 kc + i is word w of the row
                const int j = D == 128 ? i : i & 1, w = D == 128 ? 4 * i + kc : 4 * (i & 1) + 2 * kc + (i >> 1);
                const int g = 32 * j * NG / D;
                __half2 n[4];
                codes8(w4[i], n);
                uint4 o;
                o.x = h2_bits(__hfma2(n[0], s[g], m[g]));
                o.y = h2_bits(__hfma2(n[1], s[g], m[g]));
                o.z = h2_bits(__hfma2(n[2], s[g], m[g]));
                o.w = h2_bits(__hfma2(n[3], s[g], m[g]));
                *reinterpret_cast<uint4*>(sm.k + operand_at(kTokens, row, w)) = o;
            }
        }
    };
    // values: a warp takes groups of 8 tokens.  Matrix p of the load is the 16-byte piece p of the tokens' rows: the lane gets half-word
    // 8 p + lane / 4 of tokens 2 (lane % 4) and the next one, all of one group of dims.
    const int vh = lane >> 2, vp2 = 2 * (lane & 3), vgroup = 32 * (vh % J) * NG / D;
    auto put_v = [&](int step) {                                                                 // true: some value is not finite
        bool found = false;
#pragma unroll
        for (int i = 0; i < kTokens / 8 / kWarps; ++i) {
            const int vt = warp + i * kWarps, r0 = 8 * (vt & 1);
            const unsigned char* tile = sm.v_codes[vt >> 1];
            const int left = last - (step * kTokens + 8 * vt) - vp2;                             // tokens behind the lane's first
            // lane l gives the address of row l % 8 of matrix l / 8 (at D = 64, two matrices: lanes 16 .. 31 repeat)
            const int lr = r0 + (lane & 7), lp = (lane >> 3) & (J - 1);
            const int stored = D == 128 ? lp ^ (((lr >> 1) & 1) << 1) : lp;
            const uint32_t from = smem_u32(tile + lr * (D / 2) + 16 * piece_of(lr, stored, true));
            uint32_t w[J];
            if constexpr (J == 4)
                asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                             : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(from) : "memory");
            else
                asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(from) : "memory");
            __half2 pa = *reinterpret_cast<const __half2*>(tile + F::val_par(r0 + vp2, vgroup) - F::kVal);
            __half2 pb = *reinterpret_cast<const __half2*>(tile + F::val_par(r0 + vp2 + 1, vgroup) - F::kVal);
            if (left < 0) pa = h2_of(0);                                                         // behind the last token: whatever the page holds
            if (left < 1) pb = h2_of(0);
            const __half2 zero = __hfma2(pa, h2_of(0), __hmul2(pb, h2_of(0)));                   // NaN if one of them is not finite
            if (!__hbeq2(zero, zero)) {
                found = true;
                if (!finite2(pa)) {
                    pa = h2_of(0);
                    atomicOr(&sm.bad[8 * vt + vp2], 1 << vgroup);
                }
                if (!finite2(pb)) {
                    pb = h2_of(0);
                    atomicOr(&sm.bad[8 * vt + vp2 + 1], 1 << vgroup);
                }
            }
            const __half2 s = __lows2half2(pa, pb), m = __highs2half2(pa, pb);
#pragma unroll
            for (int q = 0; q < J; ++q) {
                __half2 n[4];
                codes8(w[q], n);
#pragma unroll
                for (int d = 0; d < 4; ++d)
                    *reinterpret_cast<__half2*>(sm.v + operand_at(D, 32 * q + 8 * d + vh, vt) + 2 * vp2) = __hfma2(n[d], s, m);
            }
        }
        return found;
    };

    fetch_k(0);
    load_codes(sm.v_codes[0], 0, kHalf);
    // ---- queries: two threads a row, rotated as the decode kernel does, in the order of the keys' dims
    const int mine = warp >> 3;                                                                  // the thread's row tile
    {
        const int r = (tid & 255) >> 1;
        const long long f = row0 + mine * kRows + r;
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
            *reinterpret_cast<uint4*>(sm.q[mine] + operand_at(kRows, r, w)) = o;
        }
    }
    copies_landed();
    workers_sync<kWorkers>();
    put_k();
    written(k_bar, lane);
    workers_sync<kWorkers>();                                                                    // the keys' codes have been read
    if (T == 2 && steps > 1) fetch_k(1);

    // ---- the row of this thread in the softmax, and its half of the columns
    const int row = 32 * (warp & 3) + lane, half = (warp >> 2) & 1, slot = mine * kRows + row;
    const uint32_t at_s = tmem + 256 * mine + ((uint32_t)(32 * (warp & 3)) << 16), at_o = at_s + kTokens + half * (D / 2);
    const uint32_t s_bar = smem_u32(&sm.s_done[mine]), p_bar = smem_u32(&sm.p_ready[mine]);
    const int sees = pos + min((int)((row0 + slot) / a.share), last_i);                         // last token it sees (rows behind the last: as that one)
    const int first_sees = pos + first_i;
    // (the sign of a negative scale goes into the scores, so that `unit` is positive; a scale of zero makes them zero)
    const float unit = a.scale_log2 == 0.f ? 1.f : fabsf(a.scale_log2), sign = a.scale_log2 == 0.f ? 0.f : a.scale_log2 < 0.f ? -1.f : 1.f;
    const uint64_t unit2 = pair(unit, unit);
    float ref = -INFINITY;
    uint64_t sum2 = pair(0.f, 0.f);
    int nan_groups = 0;
    for (int step = 0; step < steps; ++step) {
        const bool found = put_v(step);                                                          // (P V of the step before is over)
        written(v_bar, lane);
        if (T == 1 && step + 1 < steps) fetch_k(step + 1);
        if (tid < kTilesOf) look(step + 2);
        ok = ok && mbar_wait(s_bar, step & 1, &sm.abort_flag, kWaitNs);
        tc_fence_after_sync();
        const uint64_t pages = *reinterpret_cast<const uint64_t*>(sm.page_ok[step & 3]);
        const bool masked = (step + 1) * kTokens - 1 > first_sees || pages != 0x0101010101010101ull;
        const int from = step * kTokens + 64 * half;                                             // the thread's first token
        uint32_t s[32];
        auto fetch = [&](int c) {                                                                // scores of 32 tokens
            tmem_ld_32x32b_x32(at_s + 64 * half + 32 * c, s);
            tmem_wait_ld();
            if (sign != 1.f) {
#pragma unroll
                for (int i = 0; i < 32; ++i) s[i] = __float_as_uint(__uint_as_float(s[i]) * sign);
            }
            if (masked) {
                const int seen = sees - (from + 32 * c);
                const uint32_t p0 = (uint32_t)(pages >> (8 * (4 * half + 2 * c))) & 1, p1 = (uint32_t)(pages >> (8 * (4 * half + 2 * c + 1))) & 1;
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (i > seen || !(i < 16 ? p0 : p1)) s[i] = 0xff800000u;
            }
        };
        float top = -INFINITY;
#pragma unroll
        for (int c = 1; c >= 0; --c) {
            fetch(c);
            float t0 = top, t1 = -INFINITY;
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
                t0 = max3(t0, __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
                t1 = max3(t1, __uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]));
            }
            top = fmaxf(t0, t1);
        }
        // both threads of a row move the reference alike
        sm.swap[half][slot] = top;
        asm volatile("bar.sync %0, 64;" ::"r"(1 + mine * 4 + (warp & 3)) : "memory");
        top = fmaxf(top, sm.swap[half ^ 1][slot]) * unit;
        const bool move = top - ref > 8.f;                                                       // (from minus infinity as well; not with nothing seen)
        if (__any_sync(0xffffffffu, move)) {
            const float to = move ? top : ref, keep = ref == -INFINITY ? 0.f : ex2(ref - to);
            ref = to;
            const float2 f = unpair(sum2);
            sum2 = pair(f.x * keep, f.y * keep);
            if (step > 0) {
                uint32_t o[16];
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    tmem_ld_32x32b_x16(at_o + 16 * c, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
                    tmem_st_32x32b_x16(at_o + 16 * c, o);
                }
            }
        }
        const float shift = ref == -INFINITY ? 0.f : -ref;                                       // nothing seen yet: weights 0
        const uint64_t shift2 = pair(shift, shift);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            if (c == 1) fetch(1);                                                                // (again: 64 at a time are too many registers)
            uint32_t p[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float2 x = unpair(fma2(pair(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), unit2, shift2));
                const float p0 = ex2(x.x), p1 = ex2(x.y);
                sum2 = add2(sum2, pair(p0, p1));
                p[i] = h2_bits(__floats2half2_rn(p0, p1));
            }
            tmem_st_32x32b_x16(at_s + 64 * half + 16 * c, p);                                    // over columns that this thread has read
        }
        tmem_wait_st();
        written(p_bar, lane);
        copies_landed();
        if (workers_any<kWorkers>(found)) {
            // rows that see a value that is not finite
#pragma unroll 1
            for (int i = 0; i < 64; ++i) {
                const int t = from + i;
                if (t <= sees && (pages >> (8 * ((64 * half + i) >> 4)) & 1)) nan_groups |= sm.bad[64 * half + i];
            }
            workers_sync<kWorkers>();
            if (tid < kTokens) sm.bad[tid] = 0;
        }
        if (step + 1 < steps) {
            load_codes(sm.v_codes[0], step + 1, kHalf);                                             // (everybody has read the codes of this step)
            put_k();                                                                             // (S of this step is over in all row tiles)
            written(k_bar, lane);
            if (tid < kTilesOf) note(step + 2);
            copies_landed();
            workers_sync<kWorkers>();
            if (T == 2 && step + 2 < steps) fetch_k(step + 2);
#pragma unroll
            for (int t = 0; t < T; ++t) ok = ok && mbar_wait(smem_u32(&sm.pv_done[t]), step & 1, &sm.abort_flag, kWaitNs);
            tc_fence_after_sync();
        }
    }
    ok = ok && mbar_wait(smem_u32(&sm.pv_done[mine]), (steps - 1) & 1, &sm.abort_flag, kWaitNs);
    tc_fence_after_sync();
    if (!ok && lane == 0) atomicExch(a.error, 1);

    // ---- out = O / sum
    const float2 sums = unpair(sum2);
    float sum = sums.x + sums.y;
    sm.swap[half][slot] = sum;
    if (half) sm.swap_bad[slot] = nan_groups;
    workers_sync<kWorkers>();
    sum += sm.swap[half ^ 1][slot];
    if (!half) {
        nan_groups |= sm.swap_bad[slot];
        sm.swap_bad[slot] = nan_groups;
    }
    workers_sync<kWorkers>();
    nan_groups = sm.swap_bad[slot];
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const long long f = row0 + slot;
    __half* to = a.out + ((long long)b * a.seq + (int)(f / a.share)) * a.heads * D + (kvh * a.share + (int)(f % a.share)) * D;
    // columns of this half: pieces p = half D/64 .. of half-words, 32 columns each; 32/J adjacent dims of each 32 stand in a piece
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
        uint32_t o[32];
        tmem_ld_32x32b_x32(at_o + 32 * c, o);
        tmem_wait_ld();
        if (f >= rows) continue;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const float mul = nan_groups >> (32 * j * NG / D) & 1 ? __int_as_float(0x7fffffff) : inv;
            __half* dims = to + 32 * j + (half * (D / 64) + c) * (32 / J);
#pragma unroll
            for (int r = 0; r < 8 / J; r += 2) {                                                 // half-words r J + j of the piece: four dims each
                uint32_t h[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int at = (r + i / 2) * J + j + 16 * (i % 2);
                    h[i] = h2_bits(__floats2half2_rn(__uint_as_float(o[at]) * mul, __uint_as_float(o[at + 8]) * mul));
                }
                *reinterpret_cast<uint4*>(dims + 4 * r) = make_uint4(h[0], h[1], h[2], h[3]);
            }
        }
    }
    tc_fence_before_sync();
    __syncthreads();
}

template <class F, int D, int T>
int launch_prompt_as(PromptArgs& a, long long rows, int batch, cudaStream_t st)
{
    static int configured[64] = {0};   // benign race: the attribute call is idempotent
    const int smem = (int)sizeof(Smem<D, F::kBytes / 2, T>) + 1024;
    static_assert(sizeof(Smem<D, F::kBytes / 2, T>) + 1024 <= (T == 1 ? 115712 : 232448), "fits the SM");
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return record_cuda_error(e);
    if (dev >= 64 || !configured[dev]) {
        e = cudaFuncSetAttribute(prompt_kernel<F, D, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return record_cuda_error(e);
        if (dev < 64) configured[dev] = 1;
    }
    a.blocks = (int)((rows + T * kRows - 1) / (T * kRows));
    prompt_kernel<F, D, T><<<dim3(a.blocks, a.c.kv_heads, batch), 256 * T + 32, smem, st>>>(a);
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
    const long long rows = (long long)seq * a.share;
    if (rows >= (1ll << 37)) return W4A16_ERR_TOO_LARGE;
    if (batch == 0 || seq == 0) return W4A16_OK;
    a.qkv = (const __half*)qkv; a.out = (__half*)out; a.pos = (const int*)pos; a.counts = (const int*)counts;
    a.cos = (const __half*)rope_cos; a.sin = (const __half*)rope_sin;
    a.seq = seq; a.heads = heads; a.rope_rows = rope_rows; a.stride = qkv_stride;
    a.page_bytes = (long long)kv_heads * (page_size / kTile) * tile_bytes(head_dim, group);
    a.scale_log2 = scale * 1.4426950408889634f;
    a.error = device_error_word();
    if (!a.error) return W4A16_ERR_CUDA;
    return with_format(head_dim, group, [&](auto f) {
        using F = decltype(f);
        // (at 64 dims a tile of K and V costs half as much, and two CTAs that wait for each other's products do better: 243 / 265 us for
        // 2 x 2048 queries behind 1000 tokens, 32 heads on 8; at 128 dims 1014 / 788 us for 4096 behind 4096)
        if constexpr (F::NW == 16) {
            if (rows > kRows) return launch_prompt_as<F, 128, 2>(a, rows, batch, (cudaStream_t)stream);
        }
        return launch_prompt_as<F, F::NW * 8, 1>(a, rows, batch, (cudaStream_t)stream);
    });
}
