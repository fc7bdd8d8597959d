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

constexpr int kBlock = 256;

inline int check_launch(const char* what) {
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return set_error(SQ_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
    return 0;
}

__global__ __launch_bounds__(64) void kv_rope_kernel(const KvSeq* __restrict__ seqs, int half,
                                                     const float* __restrict__ inv_freq, double2* __restrict__ out) {
    const KvSeq s = seqs[blockIdx.y];
    for (int i = blockIdx.x; i < s.n_new; i += gridDim.x)
        for (int j = threadIdx.x; j < half; j += 64) {
            double sn, cs;
            sincos((double)(s.past + i) * (double)inv_freq[j], &sn, &cs);
            out[(size_t)(s.row0 + i) * half + j] = double2{cs, sn};
        }
}

__device__ __forceinline__ double wave_max64(double v) {
#pragma unroll
    for (int m = 1; m < 64; m *= 2) v = fmax(v, __shfl_xor(v, m, 64));
    return v;
}

// rint(x / scale) as the stored byte
__device__ __forceinline__ uint32_t quant(double x, double scale) {
    double q = scale > 0.0 ? rint(x / scale) : 0.0;
    q = fmin(fmax(q, -127.0), 127.0);
    return (uint32_t)((int)q + 128);
}
// a stored byte in the steps of a larger scale
__device__ __forceinline__ uint32_t requant(uint32_t b, double from, double to) {
    return (uint32_t)((int)rint((double)((int)b - 128) * from / to) + 128);
}

// One workgroup per (written page, KV head).  Thread t has position t / 4 of
// the page and dimensions 16 (t % 4) .. + 15 of each 64: one 16-byte piece of
// the keys' order.
template <int HD>
__global__ __launch_bounds__(kBlock) void kv_append_kernel(KvView kv, const KvItem* __restrict__ items,
                                                           const double2* __restrict__ rope, int half,
                                                           const float* __restrict__ k, size_t k_stride,
                                                           const float* __restrict__ v, size_t v_stride,
                                                           uint32_t* bad) {
    constexpr int C = HD / 64;
    __shared__ double s_max[2][kBlock / 64];
    const KvItem it = items[blockIdx.x / kv.kv_heads];
    const int head = blockIdx.x % kv.kv_heads;
    const size_t cell = (size_t)it.page * kv.kv_heads + head;
    uint8_t* kb = kv.bytes + cell * 2 * kPage * HD;
    uint8_t* vb = kb + kPage * HD;
    const int tok = threadIdx.x >> 2, g = threadIdx.x & 3;
    const int i = tok - it.tok0;
    const bool mine = i >= 0 && i < it.n;
    double x[C][16], y[C][16];
    double kmax = 0.0, vmax = 0.0;
    bool ok = true;
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
            const int d = 64 * c + 16 * g + e;
            double a = 0.0, b = 0.0, p = 0.0, q = 0.0;
            if (mine) {
                const size_t row = it.row0 + i;
                const float* kr = k + row * k_stride + (size_t)head * HD + d;
                const float* vr = v + row * v_stride + (size_t)head * HD + d;
                a = kr[0], b = kr[1], p = vr[0], q = vr[1];
                // values that are not finite are reported and stored as zero: in
                // the page's scale they would take the other positions with them
                if (!(fabs(a) < INFINITY && fabs(b) < INFINITY)) a = b = 0.0, ok = false;
                if (!(fabs(p) < INFINITY)) p = 0.0, ok = false;
                if (!(fabs(q) < INFINITY)) q = 0.0, ok = false;
                if (rope && d / 2 < half) {
                    const double2 cs = rope[row * half + d / 2];
                    const double t = a * cs.x - b * cs.y;
                    b = a * cs.y + b * cs.x;
                    a = t;
                }
            }
            x[c][e] = a, x[c][e + 1] = b, y[c][e] = p, y[c][e + 1] = q;
            kmax = fmax(kmax, fmax(fabs(a), fabs(b)));
            vmax = fmax(vmax, fmax(fabs(p), fabs(q)));
        }
    if (!ok) *bad = 1u;
    kmax = wave_max64(kmax);
    vmax = wave_max64(vmax);
    if ((threadIdx.x & 63) == 0) s_max[0][threadIdx.x >> 6] = kmax, s_max[1][threadIdx.x >> 6] = vmax;
    const float2 old = it.tok0 ? kv.scales[cell] : make_float2(0.0f, 0.0f);
    __syncthreads();
    for (int w = 0; w < kBlock / 64; w++) kmax = fmax(kmax, s_max[0][w]), vmax = fmax(vmax, s_max[1][w]);
    const float ks = fmaxf(old.x, (float)(kmax / 127.0)), vs = fmaxf(old.y, (float)(vmax / 127.0));
    if (it.tok0 && (ks > old.x || vs > old.y)) {
        // earlier rows of the page, in the steps of the larger scales
        for (int e = threadIdx.x; e < it.tok0 * HD; e += kBlock) {
            const int t = e / HD, d = e % HD;
            uint8_t* pk = kb + kv_k_off(t, d, HD);
            uint8_t* pv = vb + kv_v_off(t, d);
            if (ks > old.x) *pk = (uint8_t)requant(*pk, old.x, ks);
            if (vs > old.y) *pv = (uint8_t)requant(*pv, old.y, vs);
        }
    }
    if (threadIdx.x == 0) kv.scales[cell] = make_float2(ks, vs);
    if (!mine) return;
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const int d = 64 * c + 16 * g + e;
            kb[kv_k_off(tok, d, HD)] = (uint8_t)quant(x[c][e], ks);
            vb[kv_v_off(tok, d)] = (uint8_t)quant(y[c][e], vs);
        }
}

// One workgroup per (sequence, page of its last positions, KV head).
__global__ __launch_bounds__(kBlock) void kv_read_kernel(KvView kv, KvPlanView p, int last, float* __restrict__ k_out,
                                                         float* __restrict__ v_out) {
    __shared__ int s_row;
    const int head = blockIdx.x % kv.kv_heads, j = blockIdx.x / kv.kv_heads, seq = blockIdx.y;
    const KvSeq s = p.seqs[seq];
    const int len = s.past + s.n_new, first = len > last ? len - last : 0;
    const int page = first / kPage + j;
    if (page * kPage >= len) return;
    if (threadIdx.x == 0) s_row = 0;
    __syncthreads();
    // rows of the sequences before this one
    int before = 0;
    for (int i = threadIdx.x; i < seq; i += kBlock) {
        const int l = p.seqs[i].past + p.seqs[i].n_new;
        before += l < last ? l : last;
    }
    if (before) atomicAdd(&s_row, before);
    __syncthreads();
    const size_t row0 = (size_t)s_row, width = (size_t)kv.kv_heads * kv.head_dim;
    const size_t cell = (size_t)p.pages[s.table0 + page] * kv.kv_heads + head;
    const float2 scale = kv.scales[cell];
    const uint8_t* kb = kv.bytes + cell * 2 * kPage * kv.head_dim;
    const uint8_t* vb = kb + kPage * kv.head_dim;
    for (int e = threadIdx.x; e < kPage * kv.head_dim; e += kBlock) {
        const int tok = e / kv.head_dim, d = e % kv.head_dim, pos = page * kPage + tok;
        if (pos < first || pos >= len) continue;
        const size_t o = (row0 + pos - first) * width + (size_t)head * kv.head_dim + d;
        if (k_out) k_out[o] = (float)((int)kb[kv_k_off(tok, d, kv.head_dim)] - 128) * scale.x;
        if (v_out) v_out[o] = (float)((int)vb[kv_v_off(tok, d)] - 128) * scale.y;
    }
}

}  // namespace

int launch_kv_rope(hipStream_t s, const KvPlanView& p, const float* inv_freq, int rows, double2* out) {
    hipLaunchKernelGGL(kv_rope_kernel, dim3(std::min(rows, 1024), p.n_seqs), dim3(64), 0, s, p.seqs, p.half, inv_freq,
                       out);
    return check_launch("kv_rope");
}

int launch_kv_append(hipStream_t s, const KvView& kv, const KvPlanView& p, const float* k, size_t k_stride,
                     const float* v, size_t v_stride, uint32_t* bad) {
    const size_t grid = (size_t)p.n_items * kv.kv_heads;
    if (grid > (size_t)INT32_MAX) return set_error(SQ_ERR_SHAPE, "kv_append: ShapeMismatch (too many pages)");
    if (kv.head_dim == 64)
        hipLaunchKernelGGL(kv_append_kernel<64>, dim3((unsigned)grid), dim3(kBlock), 0, s, kv, p.items,
                           p.rope, p.half, k, k_stride, v, v_stride, bad);
    else
        hipLaunchKernelGGL(kv_append_kernel<128>, dim3((unsigned)grid), dim3(kBlock), 0, s, kv, p.items,
                           p.rope, p.half, k, k_stride, v, v_stride, bad);
    return check_launch("kv_append");
}

int launch_kv_read(hipStream_t s, const KvView& kv, const KvPlanView& p, int last, int max_pages, float* k_out,
                   float* v_out) {
    const size_t grid = (size_t)max_pages * kv.kv_heads;
    if (grid > (size_t)INT32_MAX) return set_error(SQ_ERR_SHAPE, "kv_read: ShapeMismatch (too many pages)");
    hipLaunchKernelGGL(kv_read_kernel, dim3((unsigned)grid, p.n_seqs), dim3(kBlock), 0, s, kv, p, last, k_out, v_out);
    return check_launch("kv_read");
}

}  // namespace sq
