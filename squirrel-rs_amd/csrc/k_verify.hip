// Verification of drafted tokens against the target's probabilities, from
// given random numbers.
//
// p = softmax(target / T), q = softmax(draft / T).  Draft x_i is accepted while
// u_i q_i(x_i) < p_i(x_i); the next token is drawn from max(p_i - q_i, 0) at
// the first rejection, from p_n behind the last draft: the smallest t whose
// running sum of weights exceeds u_n times their total.
//
// The token is an integer, so sums decide which one it is: an error of 1e-7 in
// the running sum (f32) would give another token in about one draw in a
// hundred with a vocabulary of 128256.  Exponentials and sums are in 64 bits.
#include <algorithm>

#include "verify.h"

namespace sq {
namespace {

constexpr int kBlock = 256;
constexpr int kPer = 16;                    // logits of one thread
constexpr int kChunk = kBlock * kPer;       // logits of one workgroup

inline int check_launch(const char* what) {
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return set_error(SQ_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
    return 0;
}

// A row's part: its maximum, the sum of 2^((l - max) inv_t) and the last index
// of the maximum.  sum < 0: a value that is NaN or +inf is among them.
struct Part {
    double sum;
    float max;
    uint32_t at;
};

// 2^x, x <= 0, to about 1e-14: Taylor's polynomial of 2^r on |r| <= 1/2.
__device__ __forceinline__ double exp2_64(double x) {
    if (x < -1060.0) return 0.0;  // (also -inf)
    const double n = rint(x), r = (x - n) * 0.69314718055994530942;
    double p = 1.0 / 6227020800.0;
    p = fma(p, r, 1.0 / 479001600.0);
    p = fma(p, r, 1.0 / 39916800.0);
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return ldexp(p, (int)n);
}

__device__ __forceinline__ double weight(float l, float m, double inv_t) {
    return exp2_64(((double)l - (double)m) * inv_t);
}

__device__ __forceinline__ void merge(Part& a, const Part& b, double inv_t) {
    if (a.sum < 0.0 || b.sum < 0.0) {
        a.sum = -1.0;
        return;
    }
    if (b.max > a.max || (b.max == a.max && b.at > a.at)) a.at = b.at;
    const float m = fmaxf(a.max, b.max);
    if (m != -INFINITY && inv_t > 0.0) a.sum = a.sum * weight(a.max, m, inv_t) + b.sum * weight(b.max, m, inv_t);
    a.max = m;
}

__device__ __forceinline__ Part shuffled(const Part& p, int mask) {
    return Part{__shfl_xor(p.sum, mask, 64), __shfl_xor(p.max, mask, 64), __shfl_xor(p.at, mask, 64)};
}

// Every lane of the wavefront: the merge of all 64 parts.
__device__ __forceinline__ Part wave_merge(Part p, double inv_t) {
    for (int m = 1; m < 64; m *= 2) merge(p, shuffled(p, m), inv_t);
    return p;
}

// One workgroup per (chunk of a row, row): target rows, then draft rows.
__global__ __launch_bounds__(kBlock) void verify_parts_kernel(VerifyArgs a, int target_rows, int chunks,
                                                              Part* __restrict__ parts) {
    __shared__ Part s_part[kBlock / 64];
    const int r = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
    const float* row = r < target_rows ? a.target + (size_t)r * a.target_stride
                                       : a.draft + (size_t)(r - target_rows) * a.draft_stride;
    float x[kPer];
    float m = -INFINITY;
    uint32_t at = 0;
    bool ok = true;
    const int base = chunk * kChunk + threadIdx.x;
#pragma unroll
    for (int e = 0; e < kPer; e++) {
        const int i = base + e * kBlock;
        x[e] = i < a.vocab ? row[i] : -INFINITY;
        ok = ok && x[e] < INFINITY;
        if (i < a.vocab && x[e] >= m) m = x[e], at = i;
    }
    double sum = 0.0;
    if (m != -INFINITY && a.inv_t > 0.0)
#pragma unroll
        for (int e = 0; e < kPer; e++) sum += weight(x[e], m, a.inv_t);
    Part p = wave_merge(Part{ok ? sum : -1.0, m, at}, a.inv_t);
    if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = p;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kBlock / 64; w++) merge(p, s_part[w], a.inv_t);
        parts[blockIdx.x] = p;
    }
}

// What a sequence's decision needs of its rows.
struct Choice {
    uint32_t accepted, bad;
    uint32_t t_row, d_row;  // the rows whose difference is drawn from
    float t_max, d_max;
    double t_inv, d_inv;    // 1 / sums; d_inv = 0: nothing is taken off
    uint32_t off;           // a draft without probabilities: the token left out (else 0xffffffff)
    uint32_t greedy;
};

__device__ __forceinline__ Part row_part(const Part* parts, size_t row, int chunks, double inv_t) {
    Part p{0.0, -INFINITY, 0};
    for (int c = threadIdx.x & 63; c < chunks; c += 64) merge(p, parts[row * chunks + c], inv_t);
    return wave_merge(p, inv_t);
}

// One wavefront: the drafts of sequence s in order, until one is rejected.
__device__ __forceinline__ Choice choose(const VerifyBatch& b, const VerifyArgs& a, int target_rows, int s, int chunks,
                                         const Part* parts) {
    const int n = b.n[s];
    const size_t t0 = b.target0[s], d0 = t0 - s;
    Choice c{};
    c.off = 0xffffffffu;
    for (int i = 0; i <= n; i++) {
        const Part t = row_part(parts, t0 + i, chunks, a.inv_t);
        c.accepted = i;
        c.t_row = (uint32_t)(t0 + i);
        c.t_max = t.max;
        c.t_inv = 1.0 / t.sum;
        c.greedy = t.at;
        if (t.sum < 0.0 || t.max == -INFINITY) {
            c.bad = 1;
            return c;
        }
        if (i == n) return c;
        const uint32_t x = a.tokens[d0 + i];
        if (x >= (uint32_t)a.vocab) {
            c.bad = 2;
            return c;
        }
        if (a.inv_t == 0.0) {
            if (x != t.at) return c;
            continue;
        }
        const double px = weight(a.target[(t0 + i) * a.target_stride + x], t.max, a.inv_t) * c.t_inv;
        double qx = 1.0;
        Part d{1.0, 0.0f, 0};
        if (a.draft) {
            d = row_part(parts, target_rows + d0 + i, chunks, a.inv_t);
            if (d.sum < 0.0 || d.max == -INFINITY) {
                c.bad = 1;
                return c;
            }
            qx = weight(a.draft[(d0 + i) * a.draft_stride + x], d.max, a.inv_t) / d.sum;
        }
        if ((double)a.u[t0 + i] * qx < px) continue;
        c.d_row = (uint32_t)(d0 + i);
        c.d_max = d.max;
        c.d_inv = a.draft ? 1.0 / d.sum : 0.0;
        c.off = a.draft ? 0xffffffffu : x;
        return c;
    }
    return c;
}

__device__ __forceinline__ double drawn_weight(const VerifyArgs& a, const Choice& c, int i) {
    double w = weight(a.target[(size_t)c.t_row * a.target_stride + i], c.t_max, a.inv_t) * c.t_inv;
    if (c.d_inv > 0.0)
        w = fmax(w - weight(a.draft[(size_t)c.d_row * a.draft_stride + i], c.d_max, a.inv_t) * c.d_inv, 0.0);
    return (uint32_t)i == c.off ? 0.0 : w;
}

__device__ __forceinline__ double wave_sum64(double v) {
    for (int m = 1; m < 64; m *= 2) v += __shfl_xor(v, m, 64);
    return v;
}

// One workgroup per (chunk, sequence): the sum of the chunk's weights.
__global__ __launch_bounds__(kBlock) void verify_sums_kernel(VerifyBatch b, VerifyArgs a, int target_rows,
                                                             const Part* __restrict__ parts, double* __restrict__ sums,
                                                             Choice* __restrict__ choices) {
    __shared__ Choice s_c;
    __shared__ double s_sum[kBlock / 64];
    const int s = blockIdx.y;
    if (threadIdx.x < 64) {
        const Choice c = choose(b, a, target_rows, s, gridDim.x, parts);
        if (threadIdx.x == 0) s_c = c;
    }
    __syncthreads();
    const Choice c = s_c;
    if (blockIdx.x == 0 && threadIdx.x == 0) choices[s] = c;
    if (c.bad || a.inv_t == 0.0) return;
    double sum = 0.0;
    for (int e = 0; e < kPer; e++) {
        const int i = blockIdx.x * kChunk + e * kBlock + threadIdx.x;
        if (i < a.vocab) sum += drawn_weight(a, c, i);
    }
    sum = wave_sum64(sum);
    if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kBlock / 64; w++) sum += s_sum[w];
        sums[(size_t)s * gridDim.x + blockIdx.x] = sum;
    }
}

// One workgroup per sequence: the chunk that holds the drawn point, and the
// token in it.
__global__ __launch_bounds__(kBlock) void verify_draw_kernel(VerifyBatch b, VerifyArgs a, int chunks,
                                                             const double* __restrict__ sums,
                                                             const Choice* __restrict__ choices,
                                                             VerifyResult* __restrict__ results) {
    __shared__ double s_sum[kBlock], s_at, s_total;
    __shared__ int s_chunk, s_found, s_last;
    const int s = blockIdx.x;
    Choice c = choices[s];
    VerifyResult& out = results[s];
    if (c.bad || a.inv_t == 0.0) {
        if (threadIdx.x == 0) out = VerifyResult{c.accepted, c.greedy, c.bad, 0};
        return;
    }
    const double u = (double)a.u[b.target0[s] + b.n[s]];
    if (threadIdx.x == 0) {
        double total = 0.0;
        for (int i = 0; i < chunks; i++) total += sums[(size_t)s * chunks + i];
        s_total = total;
    }
    __syncthreads();
    // (p <= q everywhere, by rounding: p and q agree and the draft had neither's
    // probability; drawn from p)
    const bool equal = !(s_total > 0.0);
    if (equal) c.d_inv = 0.0, c.off = 0xffffffffu;
    auto chunk_sum = [&](int chunk) {  // of thread t: kPer consecutive logits
        double sum = 0.0;
        for (int e = 0; e < kPer; e++) {
            const int i = chunk * kChunk + (int)threadIdx.x * kPer + e;
            if (i < a.vocab) sum += drawn_weight(a, c, i);
        }
        return sum;
    };
    if (threadIdx.x == 0) {
        double total = s_total, run = 0.0;
        int chunk = 0, last = -1;
        if (equal) total = 1.0;
        const double at = u * total;
        if (!equal) {
            for (chunk = 0; chunk < chunks; chunk++) {
                const double w = sums[(size_t)s * chunks + chunk];
                if (w > 0.0) last = chunk;
                if (run + w > at) break;
                run += w;
            }
            // (u near 1 and the order of the sums: the last chunk with any weight)
            if (chunk == chunks) {
                chunk = last;
                run = 0.0;
                for (int i = 0; i < chunk; i++) run += sums[(size_t)s * chunks + i];
            }
        }
        s_chunk = chunk;
        s_at = at - run;
        s_found = 0x7fffffff;
        s_last = -1;
    }
    __syncthreads();
    double at = s_at;
    for (int chunk = s_chunk; chunk < chunks; chunk++) {
        const double mine = chunk_sum(chunk);
        s_sum[threadIdx.x] = mine;
        __syncthreads();
        double before = 0.0, all = 0.0;
        for (int t = 0; t < kBlock; t++) {
            if (t < (int)threadIdx.x) before += s_sum[t];
            all += s_sum[t];
        }
        double run = before;
        for (int e = 0; e < kPer; e++) {
            const int i = chunk * kChunk + (int)threadIdx.x * kPer + e;
            const double w = i < a.vocab ? drawn_weight(a, c, i) : 0.0;
            run += w;
            if (w > 0.0) {
                atomicMax(&s_last, i);
                if (run > at) {
                    atomicMin(&s_found, i);
                    break;
                }
            }
        }
        __syncthreads();
        const bool done = s_found != 0x7fffffff || (!equal && s_last >= 0);
        if (done) break;
        at -= all;
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        const int t = s_found != 0x7fffffff ? s_found : s_last;
        out = VerifyResult{c.accepted, (uint32_t)(t < 0 ? c.greedy : t), 0, 0};
    }
}

size_t align16(size_t n) { return (n + 15) & ~(size_t)15; }

}  // namespace

size_t verify_ws_bytes(size_t rows, size_t n_seqs, int vocab) {
    const size_t chunks = ((size_t)vocab + kChunk - 1) / kChunk;
    return align16(rows * chunks * sizeof(Part)) + align16(n_seqs * chunks * sizeof(double)) + n_seqs * sizeof(Choice);
}

int launch_verify(hipStream_t s, const VerifyBatch& b, const VerifyArgs& a, size_t target_rows, size_t draft_rows,
                  void* ws, VerifyResult* results) {
    const int chunks = (a.vocab + kChunk - 1) / kChunk;
    const size_t rows = target_rows + draft_rows;
    Part* parts = (Part*)ws;
    double* sums = (double*)((char*)ws + align16(rows * chunks * sizeof(Part)));
    Choice* choices = (Choice*)((char*)sums + align16((size_t)b.n_seqs * chunks * sizeof(double)));
    hipLaunchKernelGGL(verify_parts_kernel, dim3((unsigned)(rows * chunks)), dim3(kBlock), 0, s, a, (int)target_rows,
                       chunks, parts);
    hipLaunchKernelGGL(verify_sums_kernel, dim3(chunks, b.n_seqs), dim3(kBlock), 0, s, b, a, (int)target_rows,
                       (const Part*)parts, sums, choices);
    hipLaunchKernelGGL(verify_draw_kernel, dim3(b.n_seqs), dim3(kBlock), 0, s, b, a, chunks, (const double*)sums,
                       (const Choice*)choices, results);
    return check_launch("verify");
}

}  // namespace sq
