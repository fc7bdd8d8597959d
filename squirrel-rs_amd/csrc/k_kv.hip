// Kernels of the paged 8-bit key/value cache (kv.h): the rotation table of a
// step, appending and reading back.
//
// Everything that decides a stored integer is computed in 64 bits: the angle
// position * inv_freq (in f32 it is off by 2^-24 of itself, 4e-3 radians at
// position 65536), the rotated key, the page's maximum and x / scale.  A
// stored integer is then the definition's wherever that does not lie within
// 1e-15 of a rounding border, where f32 steps give another integer for one
// element in about 1e5.
#include <algorithm>

#include "kv.h"

namespace sq {
namespace {

inline int check_launch(const char* what) {
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return set_error(SQ_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
    return 0;
}

__global__ __launch_bounds__(64) void kv_rope_kernel(const KvSeq* __restrict__ seqs, int half,
                                                     const float* __restrict__ inv_freq, double2* __restrict__ out,
                                                     float2* __restrict__ out32) {
    const KvSeq s = seqs[blockIdx.y];
    for (int i = blockIdx.x; i < s.n_new; i += gridDim.x)
        for (int j = threadIdx.x; j < half; j += 64) {
            double sn, cs;
            sincos((double)(s.past + i) * (double)inv_freq[j], &sn, &cs);
            out[(size_t)(s.row0 + i) * half + j] = double2{cs, sn};
            out32[(size_t)(s.row0 + i) * half + j] = make_float2((float)cs, (float)sn);
        }
}

__device__ __forceinline__ double wave_max64(double v) {
#pragma unroll
    for (int m = 1; m < 64; m *= 2) v = fmax(v, __shfl_xor(v, m, 64));
    return v;
}

// x / s rounded as a division is, from r = 1 / s: the product is off by its last
// bits, and the remainder, which is exact, corrects it (a quotient that is a
// whole and a half comes out as that, so ties go where a division's go).
__device__ __forceinline__ double divide(double x, double s, double r) {
    const double y = x * r;
    return fma(fma(-y, s, x), r, y);
}
// rint(x / s) as the stored byte; r = 0: a scale of 0, whose values are zeros
__device__ __forceinline__ uint32_t quant(double x, double s, double r) {
    return (uint32_t)((int)fmin(fmax(rint(divide(x, s, r)), -127.0), 127.0) + 128);
}
// a stored byte in the steps of a larger scale
__device__ __forceinline__ uint32_t requant(uint32_t b, double from, double s, double r) {
    return (uint32_t)((int)rint(divide((double)((int)b - 128) * from, s, r)) + 128);
}
__device__ __forceinline__ double reciprocal(double s) { return s > 0.0 ? 1.0 / s : 0.0; }

constexpr int kFewTokens = 16;

// One workgroup per (written page, KV head) and one of keys and values.  A
// wavefront's lanes have pairs of dimensions, HD / 2 threads a position and
// eight positions at a time, so a single decoded token is one load of each.
// The page's maximum first (the values stay in registers), then:
//   few new rows and no scale that grows: their bytes go where they belong (2
//   bytes of keys a lane, or two single ones of values);
//   otherwise through an image of the page in LDS, written out 16 bytes a
//   thread; earlier rows of the page are in it, in the steps of the new scale.
// Bound by latency for single tokens (one: 3.4 us, 96 sequences with one each:
// 5.6), by the chain read - maximum - quantize - write for whole pages: 2011 rows
// of 8 x 128 are 20.6 MB in 10.2 us, two workgroups a CU.
template <int HD, bool VALUES>
__device__ __forceinline__ void append_page(const KvView& kv, const KvItem& it, int head,
                                            const double2* __restrict__ rope, int half, const float* __restrict__ in,
                                            size_t stride, uint32_t* bad, double* s_max, uint8_t* s_img) {
    constexpr int NT = HD * 4, PAIRS = HD / 2, PASSES = kPage / 8, BYTES = kPage * HD;
    const size_t cell = (size_t)it.page * kv.kv_heads + head;
    uint8_t* page = kv.bytes + (cell * 2 + VALUES) * BYTES;
    float* scale = (float*)(kv.scales + cell) + VALUES;
    const float old = it.tok0 ? *scale : 0.0f;
    const int d = 2 * (threadIdx.x % PAIRS), first = threadIdx.x / PAIRS;
    const bool vec = (((uintptr_t)in | (stride * 4)) & 7) == 0;
    double x[PASSES][2];
    double top = 0.0;
    bool ok = true;
#pragma unroll
    for (int p = 0; p < PASSES; p++) {
        const int i = first + 8 * p;  // the new row
        float a = 0.0f, b = 0.0f;
        double2 cs{1.0, 0.0};
        if (i < it.n) {
            const size_t row = (size_t)it.row0 + i;
            const float* r = in + row * stride + (size_t)head * HD + d;
            if (vec) {
                const float2 t = *(const float2*)r;
                a = t.x, b = t.y;
            } else {
                a = r[0], b = r[1];
            }
            if (!VALUES && rope && d / 2 < half) cs = rope[row * half + d / 2];
        }
        // values that are not finite are reported and stored as zero: in the
        // page's scale they would take the other positions with them
        if (!(fabsf(a) < INFINITY)) a = 0.0f, b = VALUES ? b : 0.0f, ok = false;
        if (!(fabsf(b) < INFINITY)) b = 0.0f, a = VALUES ? a : 0.0f, ok = false;
        if constexpr (VALUES) {
            x[p][0] = a, x[p][1] = b;
        } else {
            x[p][0] = (double)a * cs.x - (double)b * cs.y;
            x[p][1] = (double)a * cs.y + (double)b * cs.x;
        }
        top = fmax(top, fmax(fabs(x[p][0]), fabs(x[p][1])));
    }
    if (!ok) *bad = 1u;
    top = wave_max64(top);
    if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; w++) top = fmax(top, s_max[w]);
    const float s = fmaxf(old, (float)(top / 127.0));
    const double r = reciprocal(s);
    const bool grown = it.tok0 && s > old;
    if (threadIdx.x == 0) *scale = s;
    auto put = [&](uint8_t* to, int tok, const double* v) {
        const uint32_t b0 = quant(v[0], s, r), b1 = quant(v[1], s, r);
        if constexpr (VALUES) {
            to[kv_v_off(tok, d)] = (uint8_t)b0;
            to[kv_v_off(tok, d + 1)] = (uint8_t)b1;
        } else {
            *(uint16_t*)&to[kv_k_off(tok, d, HD)] = (uint16_t)(b0 | b1 << 8);
        }
    };
    if (it.n <= kFewTokens && !grown) {
#pragma unroll
        for (int p = 0; p < kFewTokens / 8; p++)
            if (first + 8 * p < it.n) put(page, it.tok0 + first + 8 * p, x[p]);
        return;
    }
    // the image's 16-byte pieces: the page's as they are where it has earlier rows
    constexpr int PIECES = BYTES / 16;
    if (it.tok0) {
        for (int e = threadIdx.x; e < PIECES; e += NT) ((uint4*)s_img)[e] = ((const uint4*)page)[e];
        __syncthreads();
        if (grown)
            for (int e = threadIdx.x; e < it.tok0 * HD; e += NT) {
                uint8_t* b = &s_img[VALUES ? kv_v_off(e / HD, e % HD) : kv_k_off(e / HD, e % HD, HD)];
                *b = (uint8_t)requant(*b, old, s, r);
            }
    }
#pragma unroll
    for (int p = 0; p < PASSES; p++)
        if (first + 8 * p < it.n) put(s_img, it.tok0 + first + 8 * p, x[p]);
    __syncthreads();
    // (positions behind the new rows are nobody's: what the image holds there goes along)
    for (int e = threadIdx.x; e < PIECES; e += NT) ((uint4*)page)[e] = ((const uint4*)s_img)[e];
}

template <int HD>
__global__ __launch_bounds__(HD * 4) void kv_append_kernel(KvView kv, const KvItem* __restrict__ items,
                                                           const double2* __restrict__ rope, int half,
                                                           const float* __restrict__ k, size_t k_stride,
                                                           const float* __restrict__ v, size_t v_stride,
                                                           uint32_t* bad) {
    __shared__ double s_max[HD * 4 / 64];
    __shared__ __attribute__((aligned(16))) uint8_t s_img[kPage * HD];
    const int at = blockIdx.x / kv.kv_heads, head = blockIdx.x - at * kv.kv_heads;
    const KvItem it = items[at];
    if (blockIdx.y == 0)
        append_page<HD, false>(kv, it, head, rope, half, k, k_stride, bad, s_max, s_img);
    else
        append_page<HD, true>(kv, it, head, rope, half, v, v_stride, bad, s_max, s_img);
}

// One workgroup per (sequence, page of its last positions, KV head) and one of
// keys and values: the page's bytes through LDS, four dimensions a thread on the
// way out.  Bound by the writes: 2048 rows of 8 x 128 (21 MB) in 8.6 us.
template <int HD>
__global__ __launch_bounds__(HD * 4) void kv_read_kernel(KvView kv, KvPlanView p, int last, float* __restrict__ k_out,
                                                         float* __restrict__ v_out) {
    constexpr int NT = HD * 4, BYTES = kPage * HD, PIECES = BYTES / 16, Q = HD / 4;
    __shared__ __attribute__((aligned(16))) uint8_t s_img[BYTES];
    __shared__ int s_row;
    const int j = blockIdx.x / kv.kv_heads, head = blockIdx.x - j * kv.kv_heads, seq = blockIdx.y, which = blockIdx.z;
    float* out = which ? v_out : k_out;
    const KvSeq s = p.seqs[seq];
    const int len = s.past + s.n_new, first = len > last ? len - last : 0;
    const int page = first / kPage + j;
    if (!out || page * kPage >= len) return;
    const size_t cell = (size_t)p.pages[s.table0 + page] * kv.kv_heads + head;
    const float scale = which ? kv.scales[cell].y : kv.scales[cell].x;
    const uint4* from = (const uint4*)(kv.bytes + (cell * 2 + which) * BYTES);
    for (int e = threadIdx.x; e < PIECES; e += NT) ((uint4*)s_img)[e] = from[e];
    if (threadIdx.x == 0) s_row = 0;
    __syncthreads();
    // rows of the sequences before this one
    int before = 0;
    for (int i = threadIdx.x; i < seq; i += NT) {
        const int l = p.seqs[i].past + p.seqs[i].n_new;
        before += l < last ? l : last;
    }
    if (before) atomicAdd(&s_row, before);
    __syncthreads();
    const size_t width = (size_t)kv.kv_heads * HD;
    out += ((size_t)s_row + page * kPage - first) * width + (size_t)head * HD;
    const int lo = max(first - page * kPage, 0), hi = min(len - page * kPage, kPage);
    const bool vec = ((uintptr_t)out & 15) == 0;
    for (int e = lo * Q + threadIdx.x; e < hi * Q; e += NT) {
        const int tok = e / Q, d = e % Q * 4;
        float w[4];
#pragma unroll
        for (int c = 0; c < 4; c++)
            w[c] = (float)((int)s_img[which ? kv_v_off(tok, d + c) : kv_k_off(tok, d + c, HD)] - 128) * scale;
        float* o = out + tok * width + d;
        if (vec) {
            *(float4*)o = make_float4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int c = 0; c < 4; c++) o[c] = w[c];
        }
    }
}

}  // namespace

int launch_kv_rope(hipStream_t s, const KvPlanView& p, const float* inv_freq, int rows, double2* out, float2* out32) {
    hipLaunchKernelGGL(kv_rope_kernel, dim3(std::min(rows, 1024), p.n_seqs), dim3(64), 0, s, p.seqs, p.half, inv_freq,
                       out, out32);
    return check_launch("kv_rope");
}

int launch_kv_append(hipStream_t s, const KvView& kv, const KvPlanView& p, const float* k, size_t k_stride,
                     const float* v, size_t v_stride, uint32_t* bad) {
    const size_t grid = (size_t)p.n_items * kv.kv_heads;
    if (!grid_fits(grid, 4 * kv.head_dim)) return set_error(SQ_ERR_SHAPE, "kv_append: ShapeMismatch (too many pages)");
    if (kv.head_dim == 64)
        hipLaunchKernelGGL(kv_append_kernel<64>, dim3((unsigned)grid, 2), dim3(256), 0, s, kv, p.items, p.rope,
                           p.half, k, k_stride, v, v_stride, bad);
    else
        hipLaunchKernelGGL(kv_append_kernel<128>, dim3((unsigned)grid, 2), dim3(512), 0, s, kv, p.items, p.rope,
                           p.half, k, k_stride, v, v_stride, bad);
    return check_launch("kv_append");
}

int launch_kv_read(hipStream_t s, const KvView& kv, const KvPlanView& p, int last, int max_pages, float* k_out,
                   float* v_out) {
    const size_t grid = (size_t)max_pages * kv.kv_heads;
    if (!grid_fits(grid, 4 * kv.head_dim)) return set_error(SQ_ERR_SHAPE, "kv_read: ShapeMismatch (too many pages)");
    auto kernel = kv.head_dim == 64 ? kv_read_kernel<64> : kv_read_kernel<128>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid, p.n_seqs, 2), dim3(4 * kv.head_dim), 0, s, kv, p, last, k_out,
                       v_out);
    return check_launch("kv_read");
}

}  // namespace sq
