// Attention over the paged 4-bit key/value cache.
#include "w4a16_kv4.cuh"

namespace w4a16 {
namespace kv4 {
namespace {

struct AttnArgs {
    Cache c;
    const __half* qkv;            // [batch][seq] rows of `stride` elements; the queries of all heads stand first
    __half* out;                  // [batch][seq][heads * D]
    const int* pos;
    const int* counts;            // null: seq queries in every row
    const __half* cos;
    const __half* sin;
    int* error;
    int seq, heads, group_heads;  // group_heads: query heads that share a key/value head
    int rope_rows;
    long long stride;
    float scale;
};

// One CTA per query and head, D/8 lanes per cached position, running maximum and sum per lane group, fp32 throughout.
template <class F, int D>
__global__ void __launch_bounds__(128) attention_kernel(const AttnArgs a)
{
    constexpr int kLanes = F::NW, kSub = 128 / kLanes;
    __shared__ float part[kSub][D + 2];
    const int head = blockIdx.x, s = blockIdx.y, b = blockIdx.z;
    const int sub = threadIdx.x / kLanes, w = threadIdx.x % kLanes;
    const int p = a.pos[b];
    if (p < 0 || (a.counts && s >= a.counts[b])) return;
    if (p > a.c.capacity() || p + s >= a.c.capacity() || (a.cos && p + s >= a.rope_rows)) {
        if (threadIdx.x == 0) atomicExch(a.error, kErrPosition);
        return;
    }
    const int n = p + s + 1, kv = head / a.group_heads;
    float q[8];
    load_rotated<D>(a.qkv + ((long long)b * a.seq + s) * a.stride + head * D, w, a.cos, a.sin, p + s, q);
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
    const int g = w * 8 * F::NG / D;
    for (int t0 = 0; t0 < n; t0 += kSub) {
        const int t = t0 + sub;
        const unsigned char* tile = t < n ? a.c.tile(b, kv, t, F::kBytes) : nullptr;
        if (t < n && !tile && w == 0) atomicExch(a.error, kErrPage);
        const int r = t & 15;
        float dot = 0.f;
        if (tile) {
            const uint32_t k = *reinterpret_cast<const uint32_t*>(tile + F::key_word(r, w));
            const float2 par = __half22float2(*reinterpret_cast<const __half2*>(tile + F::key_par(r, g)));
#pragma unroll
            for (int i = 0; i < 8; ++i) dot = fmaf(fmaf((float)((k >> (4 * i)) & 15), par.x, par.y), q[i], dot);
        }
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        if (tile) {
            dot *= a.scale;
            const float top = fmaxf(m, dot);
            const float keep = __expf(m - top), e = __expf(dot - top);
            const uint32_t v = *reinterpret_cast<const uint16_t*>(tile + F::val_half(r, 2 * w)) |
                               (uint32_t)*reinterpret_cast<const uint16_t*>(tile + F::val_half(r, 2 * w + 1)) << 16;
            const float2 par = __half22float2(*reinterpret_cast<const __half2*>(tile + F::val_par(r, g)));
            l = fmaf(l, keep, e);
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] = fmaf(acc[i], keep, e * fmaf((float)((v >> (4 * i)) & 15), par.x, par.y));
            m = top;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) part[sub][8 * w + i] = acc[i];
    if (w == 0) {
        part[sub][D] = m;
        part[sub][D + 1] = l;
    }
    __syncthreads();
    if (threadIdx.x < D) {
        float top = -INFINITY;
        for (int i = 0; i < kSub; ++i) top = fmaxf(top, part[i][D]);
        float num = 0.f, den = 0.f;
        for (int i = 0; i < kSub; ++i) {
            if (part[i][D + 1] == 0.f) continue;                                 // no position of its own
            const float e = __expf(part[i][D] - top);
            num = fmaf(part[i][threadIdx.x], e, num);
            den = fmaf(part[i][D + 1], e, den);
        }
        a.out[((long long)b * a.seq + s) * a.heads * D + head * D + threadIdx.x] = __float2half_rn(den == 0.f ? 0.f : num / den);
    }
}

int check_attention(AttnArgs& a, const void* qkv, const void* pool, const void* table, const void* pos, const void* counts,
                    const void* rope_cos, const void* rope_sin, void* out, int batch, int seq, int heads, int kv_heads, int head_dim,
                    int group, int page_size, int pages, int width, long long qkv_stride, int rope_rows, float scale, long long need)
{
    if (!qkv || !pos || !out || ((rope_cos == nullptr) != (rope_sin == nullptr))) return W4A16_ERR_NULL_POINTER;
    int s = check_cache(a.c, pool, table, pages, width, page_size, kv_heads, head_dim, group);
    if (s != W4A16_OK) return s;
    if (batch < 0 || seq < 0 || heads <= 0 || heads % kv_heads || qkv_stride < need || (qkv_stride % 8) || (rope_cos && rope_rows <= 0))
        return W4A16_ERR_BAD_SHAPE;
    if (((uintptr_t)qkv | (uintptr_t)out | (uintptr_t)rope_cos | (uintptr_t)rope_sin) & 15 || ((uintptr_t)pos | (uintptr_t)counts) & 3)
        return W4A16_ERR_MISALIGNED;
    if ((heads + 2ll * kv_heads) * head_dim >= (1ll << 30) || batch > 65535) return W4A16_ERR_TOO_LARGE;
    a.qkv = (const __half*)qkv; a.out = (__half*)out; a.pos = (const int*)pos; a.counts = (const int*)counts;
    a.cos = (const __half*)rope_cos; a.sin = (const __half*)rope_sin;
    a.seq = seq; a.heads = heads; a.group_heads = heads / kv_heads; a.rope_rows = rope_rows; a.stride = qkv_stride; a.scale = scale;
    a.error = batch && seq ? device_error_word() : nullptr;
    return a.error || !batch || !seq ? W4A16_OK : W4A16_ERR_CUDA;
}

int launch_simple(const AttnArgs& a, int batch, int head_dim, int group, cudaStream_t st)
{
    return with_format(head_dim, group, [&](auto f) {
        using F = decltype(f);
        attention_kernel<F, F::NW * 8><<<dim3(a.heads, a.seq, batch), 128, 0, st>>>(a);
        count_launch();
        const cudaError_t e = cudaGetLastError();
        return e == cudaSuccess ? (int)W4A16_OK : record_cuda_error(e);
    });
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
    AttnArgs a;
    const int s = check_attention(a, qkv, pool, table, pos, counts, rope_cos, rope_sin, out, batch, seq, heads, kv_heads, head_dim, group,
                                  page_size, pages, width, qkv_stride, rope_rows, scale, (long long)heads * head_dim);
    if (s != W4A16_OK) return s;
    if (seq > 65535) return W4A16_ERR_TOO_LARGE;
    if (batch == 0 || seq == 0) return W4A16_OK;
    return launch_simple(a, batch, head_dim, group, (cudaStream_t)stream);
}
