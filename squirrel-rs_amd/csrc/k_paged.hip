// Attention over the paged 8-bit key/value cache (kv.h).
//
// Row r of the batch, at position p of its sequence, head h of KV head
// h / (heads / kv_heads):  o = sum_j softmax_j(q . k_j / sqrt(d)) v_j  over the
// positions j <= p, with a window only those with j > p - window or
// j < sinks.
#include <algorithm>

#include "kv.h"

namespace sq {
namespace {

inline int check_launch(const char* what) {
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return set_error(SQ_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
    return 0;
}

// One wavefront per (row, head): a lane per position for the scores, a lane
// per dimension for the output.
__global__ __launch_bounds__(64) void sdpa_paged_kernel(KvView kv, KvPlanView pl, PagedArgs a, float scale) {
    __shared__ float s_q[128], s_p[kPage];
    const KvSeq s = pl.seqs[blockIdx.z];
    const int i = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, D = kv.head_dim;
    if (i >= s.n_new) return;
    const size_t row = (size_t)s.row0 + i;
    const float* q = a.q + row * a.q_stride + (size_t)h * D;
    for (int j = lane; j < D / 2; j += 64) {
        double x = q[2 * j], y = q[2 * j + 1];
        if (pl.rope && j < pl.half) {
            const double2 cs = pl.rope[row * pl.half + j];
            const double t = x * cs.x - y * cs.y;
            y = x * cs.y + y * cs.x;
            x = t;
        }
        s_q[2 * j] = (float)x, s_q[2 * j + 1] = (float)y;
    }
    __syncthreads();
    const int pos = s.past + i, head = h / (a.heads / kv.kv_heads);
    const int w0 = a.window && a.window <= pos ? pos - a.window + 1 : 0;  // first position of the window
    float m = -INFINITY, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int page = 0; page * kPage <= pos; page++) {
        if ((page + 1) * kPage <= w0 && page * kPage >= a.sinks) continue;
        const size_t cell = (size_t)pl.pages[s.table0 + page] * kv.kv_heads + head;
        const float2 sc = kv.scales[cell];
        const uint8_t* kb = kv.bytes + cell * 2 * kPage * D;
        const uint8_t* vb = kb + kPage * D;
        const int at = page * kPage + lane;
        float x = -INFINITY;
        if (at <= pos && (at >= w0 || at < a.sinks)) {
            x = 0.0f;
            for (int d = 0; d < D; d++) x += s_q[d] * (float)((int)kb[kv_k_off(lane, d, D)] - 128);
            x *= sc.x * scale;
        }
        const float mn = fmaxf(m, sq_wave_max(x));
        const float e = x == -INFINITY ? 0.0f : expf(x - mn), alpha = m == -INFINITY ? 0.0f : expf(m - mn);
        m = mn;
        l = l * alpha + sq_wave_sum(e);
        s_p[lane] = e * sc.y;
        __syncthreads();
        o0 *= alpha, o1 *= alpha;
        for (int t = 0; t < kPage; t++) {
            o0 += s_p[t] * (float)((int)vb[kv_v_off(t, lane)] - 128);
            if (D > 64) o1 += s_p[t] * (float)((int)vb[kv_v_off(t, 64 + lane)] - 128);
        }
        __syncthreads();
    }
    float* out = a.out + row * a.out_stride + (size_t)h * D;
    out[lane] = o0 / l;
    if (D > 64) out[64 + lane] = o1 / l;
}

}  // namespace

size_t sdpa_paged_floats(const std::vector<KvSeq>&, const KvView&, const PagedArgs&) { return 0; }

int launch_sdpa_paged(hipStream_t s, const std::vector<KvSeq>& seqs, const KvView& kv, const KvPlanView& p,
                      const PagedArgs& a, float*) {
    int most = 0;
    for (const KvSeq& q : seqs) most = std::max(most, q.n_new);
    const float scale = 1.0f / sqrtf((float)kv.head_dim);
    hipLaunchKernelGGL(sdpa_paged_kernel, dim3(most, a.heads, p.n_seqs), dim3(64), 0, s, kv, p, a, scale);
    return check_launch("sdpa_paged");
}

}  // namespace sq
