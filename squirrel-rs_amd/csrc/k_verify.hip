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

constexpr int kBlock = 512;
constexpr int kPer = 8;                // logits of one thread, next to each other
constexpr int kChunk = kBlock * kPer;  // logits of one workgroup
constexpr int kWaves = kBlock / 64;

inline int check_launch(const char* what) {
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return set_error(SQ_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
    return 0;
}

// A chunk of a row: its maximum, the sum of 2^((l - max) inv_t) over it and the
// last index of the maximum.  max = +inf: a value that is NaN or +inf is in it.
struct Part {
    double sum;
    float max;
    uint32_t at;
};

// 2^((l - m) inv_t) for l <= m to 1.1e-12 of itself: 2^n times the polynomial
// that meets 2^r at nine Chebyshev points of |r| <= 1/2.
__device__ __forceinline__ double weight(float l, float m, double inv_t) {
    const double x = fmax(((double)l - (double)m) * inv_t, -1100.0);  // (2^-1100 is 0; also for -inf)
    const double n = rint(x), r = x - n;
    double p = 1.3255224884796412e-06;
    p = fma(p, r, 1.5310079402334074e-05);
    p = fma(p, r, 0.00015403455852418322);
    p = fma(p, r, 0.0013333450568000249);
    p = fma(p, r, 0.009618129159402623);
    p = fma(p, r, 0.055504109412059334);
    p = fma(p, r, 0.2402265069581299);
    p = fma(p, r, 0.6931471805459335);
    p = fma(p, r, 1.0);
    return ldexp(p, (int)n);
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int m = 1; m < 64; m *= 2) v += __shfl_xor(v, m, 64);
    return v;
}

// Sums up to and including each lane's.
__device__ __forceinline__ double wave_scan64(double v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int k = 1; k < 64; k *= 2) {
        const double up = __shfl_up(v, k, 64);
        v += lane >= k ? up : 0.0;
    }
    return v;
}

// kPer logits from `i` on, -inf past the row.
__device__ __forceinline__ void load_logits(const float* row, int i, int vocab, bool vec, float* x) {
    if (vec && i + kPer <= vocab) {
#pragma unroll
        for (int e = 0; e < kPer; e += 4) {
            const float4 f = *(const float4*)(row + i + e);
            x[e] = f.x, x[e + 1] = f.y, x[e + 2] = f.z, x[e + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < kPer; e++) x[e] = i + e < vocab ? row[i + e] : -INFINITY;
    }
}
__device__ __forceinline__ bool aligned(const float* row) { return ((uintptr_t)row & 15) == 0; }

// One workgroup per (chunk of a row, row): target rows, then draft rows.  The
// chunk's maximum first, then one sum against it.  Bound by the read of the
// logits: 192 MB in 42.5 us, 4.5 TB/s, with 17 f64 instructions each beside it;
// 256 threads with sixteen logits each keep twice the loads in flight of 512 with
// eight (51 us).
constexpr int kPartBlock = 256, kPartWaves = kPartBlock / 64, kPartPer = kChunk / kPartBlock;
template <bool GREEDY>
__global__ __launch_bounds__(kPartBlock) void verify_parts_kernel(VerifyArgs a, int target_rows, int chunks,
                                                                  Part* __restrict__ parts) {
    __shared__ float s_max[kPartWaves];
    __shared__ double s_sum[kPartWaves];
    __shared__ int s_at[kPartWaves];
    const int r = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
    const float* row = r < target_rows ? a.target + (size_t)r * a.target_stride
                                       : a.draft + (size_t)(r - target_rows) * a.draft_stride;
    const int i0 = chunk * kChunk, wave = threadIdx.x >> 6;
    // logits 4 (t + 256 j) .. + 3 of the chunk
    float x[kPartPer];
    if (aligned(row) && i0 + kChunk <= a.vocab) {
#pragma unroll
        for (int j = 0; j < kPartPer; j += 4) {
            const float4 f = *(const float4*)(row + i0 + 4 * threadIdx.x + j * kPartBlock);
            x[j] = f.x, x[j + 1] = f.y, x[j + 2] = f.z, x[j + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < kPartPer; j++) {
            const int i = i0 + 4 * (int)threadIdx.x + (j & ~3) * kPartBlock + (j & 3);
            x[j] = i < a.vocab ? row[i] : -INFINITY;
        }
    }
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < kPartPer; j++) m = fmaxf(m, x[j] < INFINITY ? x[j] : INFINITY);
    m = sq_wave_max(m);
    if ((threadIdx.x & 63) == 0) s_max[wave] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kPartWaves; w++) m = fmaxf(m, s_max[w]);
    double sum = 0.0;
    int at = 0;
    if constexpr (GREEDY) {
#pragma unroll
        for (int j = 0; j < kPartPer; j++) {
            const int i = i0 + 4 * (int)threadIdx.x + (j & ~3) * kPartBlock + (j & 3);
            if (i < a.vocab && x[j] == m) at = max(at, i);
        }
#pragma unroll
        for (int k = 1; k < 64; k *= 2) at = max(at, __shfl_xor(at, k, 64));
        if ((threadIdx.x & 63) == 0) s_at[wave] = at;
    } else {
        if (m > -INFINITY && m < INFINITY) {
#pragma unroll
            for (int j = 0; j < kPartPer; j++) sum += weight(x[j], m, a.inv_t);
        }
        sum = wave_sum64(sum);
        if ((threadIdx.x & 63) == 0) s_sum[wave] = sum;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int w = 1; w < kPartWaves; w++) {
            if constexpr (GREEDY)
                at = max(at, s_at[w]);
            else
                sum += s_sum[w];
        }
        parts[blockIdx.x] = Part{sum, m, (uint32_t)at};
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

// Every lane of the wavefront: a row's maximum, sum and last index of the maximum.
__device__ __forceinline__ Part row_part(const Part* parts, size_t row, int chunks, double inv_t) {
    const int lane = threadIdx.x & 63;
    float m = -INFINITY;
    for (int c = lane; c < chunks; c += 64) m = fmaxf(m, parts[row * chunks + c].max);
    m = sq_wave_max(m);
    Part r{0.0, m, 0};
    if (inv_t == 0.0) {
        int at = 0;
        for (int c = lane; c < chunks; c += 64)
            if (parts[row * chunks + c].max == m) at = max(at, (int)parts[row * chunks + c].at);
#pragma unroll
        for (int k = 1; k < 64; k *= 2) at = max(at, __shfl_xor(at, k, 64));
        r.at = (uint32_t)at;
    } else if (m > -INFINITY && m < INFINITY) {
        for (int c = lane; c < chunks; c += 64) {
            const Part p = parts[row * chunks + c];
            r.sum += p.sum * weight(p.max, m, inv_t);
        }
        r.sum = wave_sum64(r.sum);
    }
    return r;
}

// One wavefront: draft i of sequence s (i = n: the row behind the last).
// `stop`: the sequence ends here, rejected, ill or at its end.
__device__ __forceinline__ Choice examine(const VerifyArgs& a, int target_rows, int chunks, const Part* parts, size_t t,
                                          size_t d, bool last, int i, bool& stop) {
    Choice c{};
    c.accepted = i;
    c.off = 0xffffffffu;
    c.t_row = (uint32_t)t;
    stop = true;
    const uint32_t x = last ? 0u : a.tokens[d];
    const bool there = x < (uint32_t)a.vocab;
    const float lt = there ? a.target[t * a.target_stride + x] : 0.0f;
    const bool sampled = a.draft && !last;
    const float ld = sampled && there ? a.draft[d * a.draft_stride + x] : 0.0f;
    const float u = last ? 0.0f : a.u[t];
    const Part pt = row_part(parts, t, chunks, a.inv_t);
    Part pd{1.0, 0.0f, 0};
    if (sampled) pd = row_part(parts, target_rows + d, chunks, a.inv_t);
    c.t_max = pt.max;
    c.t_inv = 1.0 / pt.sum;
    c.greedy = pt.at;
    if (!(pt.max > -INFINITY && pt.max < INFINITY)) {
        c.bad = 1;
    } else if (!there) {
        c.bad = 2;
    } else if (last) {
    } else if (a.inv_t == 0.0) {
        stop = x != pt.at;
    } else if (!(pd.max > -INFINITY && pd.max < INFINITY)) {
        c.bad = 1;
    } else {
        c.d_row = (uint32_t)d;
        c.d_max = pd.max;
        c.d_inv = sampled ? 1.0 / pd.sum : 0.0;
        c.off = sampled ? 0xffffffffu : x;
        const double px = weight(lt, pt.max, a.inv_t) * c.t_inv;
        const double qx = sampled ? weight(ld, pd.max, a.inv_t) * c.d_inv : 1.0;
        stop = !((double)u * qx < px);
    }
    return c;
}

// The whole workgroup: the drafts of sequence s, one wavefront each, until one
// ends the sequence.
__device__ __forceinline__ Choice choose(const VerifyBatch& b, const VerifyArgs& a, int target_rows, int s, int chunks,
                                         const Part* parts, Choice* s_c, int* s_stop) {
    const int n = b.n[s], wave = threadIdx.x >> 6;
    const size_t t0 = b.target0[s], d0 = t0 - s;
    for (int i0 = 0;; i0 += kWaves) {
        const int i = i0 + wave;
        bool stop = false;
        Choice c{};
        if (i <= n) c = examine(a, target_rows, chunks, parts, t0 + i, d0 + min(i, n - 1), i == n, i, stop);
        if ((threadIdx.x & 63) == 0) s_c[wave] = c, s_stop[wave] = stop;
        __syncthreads();
        // (the row behind the last draft always stops)
        for (int w = 0; w < kWaves; w++)
            if (s_stop[w]) return s_c[w];
        __syncthreads();
    }
}

// Weights of the kPer logits from i on: max(p - q, 0), or p.
__device__ __forceinline__ void drawn_weights(const VerifyArgs& a, const Choice& c, int i, double* w) {
#pragma clang fp contract(off)
    float x[kPer];
    const float* t = a.target + (size_t)c.t_row * a.target_stride;
    load_logits(t, i, a.vocab, aligned(t), x);
#pragma unroll
    for (int e = 0; e < kPer; e++) w[e] = weight(x[e], c.t_max, a.inv_t) * c.t_inv;
    if (c.d_inv > 0.0) {
        const float* d = a.draft + (size_t)c.d_row * a.draft_stride;
        load_logits(d, i, a.vocab, aligned(d), x);
        // (products rounded before the difference: equal rows leave exact zeros)
#pragma unroll
        for (int e = 0; e < kPer; e++) {
            const double q = weight(x[e], c.d_max, a.inv_t) * c.d_inv;
            w[e] = fmax(w[e] - q, 0.0);
        }
    }
#pragma unroll
    for (int e = 0; e < kPer; e++)
        if ((uint32_t)(i + e) == c.off || i + e >= a.vocab) w[e] = 0.0;
}

// The sums of the chunks' weights: a sequence's chunks dealt over the
// workgroups of one grid row, each of which makes the sequence's decision for
// itself (from parts that the L2 holds; handing it over would be a launch).  The
// decision is a chain of dependent loads, 5 of one sequence's 7 us; with 25
// workgroups a sequence instead of 12 its reads cost 40 sequences 20.5 us
// instead of 17.
__global__ __launch_bounds__(kBlock) void verify_sums_kernel(VerifyBatch b, VerifyArgs a, int target_rows, int chunks,
                                                             const Part* __restrict__ parts, double* __restrict__ sums,
                                                             Choice* __restrict__ choices) {
    __shared__ Choice s_c[kWaves];
    __shared__ int s_stop[kWaves];
    __shared__ double s_sum[2][kWaves];
    const int s = blockIdx.y;
    const Choice c = choose(b, a, target_rows, s, chunks, parts, s_c, s_stop);
    if (blockIdx.x == 0 && threadIdx.x == 0) choices[s] = c;
    if (c.bad || a.inv_t == 0.0) return;
    int turn = 0;
    for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x, turn ^= 1) {
        double w[kPer], sum = 0.0;
        drawn_weights(a, c, chunk * kChunk + (int)threadIdx.x * kPer, w);
#pragma unroll
        for (int e = 0; e < kPer; e++) sum += w[e];
        sum = wave_sum64(sum);
        if ((threadIdx.x & 63) == 0) s_sum[turn][threadIdx.x >> 6] = sum;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int k = 1; k < kWaves; k++) sum += s_sum[turn][k];
            sums[(size_t)s * chunks + chunk] = sum;
        }
    }
}

// One workgroup per sequence: the chunk that holds the drawn point, and the
// token in it.  Latency: 5.5 us.  (Done by the sums' last workgroup to finish it
// was no faster: 12.2 us for both against 7.0 + 5.5.)
__global__ __launch_bounds__(kBlock) void verify_draw_kernel(VerifyBatch b, VerifyArgs a, int chunks,
                                                             const double* __restrict__ sums,
                                                             const Choice* __restrict__ choices,
                                                             VerifyResult* __restrict__ results) {
    __shared__ double s_sum[kWaves], s_at;
    __shared__ int s_chunk, s_found[kWaves], s_last[kWaves];
    const int s = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Choice c = choices[s];
    VerifyResult& out = results[s];
    if (c.bad || a.inv_t == 0.0) {
        if (threadIdx.x == 0) out = VerifyResult{c.accepted, c.greedy, c.bad, 0};
        return;
    }
    const double u = (double)a.u[b.target0[s] + b.n[s]];
    const double* mine = sums + (size_t)s * chunks;
    if (wave == 0) {
        double total = 0.0;
        for (int i = lane; i < chunks; i += 64) total += mine[i];
        total = wave_sum64(total);
        const double at = u * total;
        double run = 0.0, before = 0.0, last_before = 0.0;
        int chunk = -1, last = -1;
        for (int i0 = 0; i0 < chunks && chunk < 0; i0 += 64) {
            const double w = i0 + lane < chunks ? mine[i0 + lane] : 0.0;
            const double upto = run + wave_scan64(w);
            const unsigned long long over = __ballot(w > 0.0 && upto > at), some = __ballot(w > 0.0);
            if (over) {
                const int k = __builtin_ctzll(over);
                chunk = i0 + k;
                before = __shfl(upto - w, k, 64);
            } else if (some) {
                const int k = 63 - __builtin_clzll(some);
                last = i0 + k;
                last_before = __shfl(upto - w, k, 64);
            }
            run = __shfl(upto, 63, 64);
        }
        // (u near 1 and the order of the sums: the last chunk with any weight)
        if (chunk < 0) chunk = last, before = last_before;
        if (lane == 0) {
            s_chunk = total > 0.0 ? chunk : -1;
            s_at = total > 0.0 ? at - before : u;
        }
    }
    __syncthreads();
    // (no weight anywhere: p and q agree, and neither had the draft; drawn from p, whose sum is 1)
    const bool equal = s_chunk < 0;
    if (equal) c.d_inv = 0.0, c.off = 0xffffffffu;
    double at = s_at;
    int token = 0;
    for (int chunk = max(s_chunk, 0); chunk < chunks; chunk++) {
        const int i = chunk * kChunk + (int)threadIdx.x * kPer;
        double w[kPer], sum = 0.0;
        drawn_weights(a, c, i, w);
#pragma unroll
        for (int e = 0; e < kPer; e++) sum += w[e];
        // the sums before this thread's: whole wavefronts', then its own wavefront's
        const double upto = wave_scan64(sum);
        if (lane == 63) s_sum[wave] = upto;
        __syncthreads();
        double run = upto - sum, all = 0.0;
        for (int k = 0; k < kWaves; k++) {
            if (k == wave) run += all;
            all += s_sum[k];
        }
        int first = 0x7fffffff, last = -1;
#pragma unroll
        for (int e = kPer - 1; e >= 0; e--) last = last < 0 && w[e] > 0.0 ? i + e : last;
#pragma unroll
        for (int e = 0; e < kPer; e++) {
            run += w[e];
            if (w[e] > 0.0 && run > at) first = min(first, i + e);
        }
#pragma unroll
        for (int k = 1; k < 64; k *= 2) {
            first = min(first, __shfl_xor(first, k, 64));
            last = max(last, __shfl_xor(last, k, 64));
        }
        if (lane == 0) s_found[wave] = first, s_last[wave] = last;
        __syncthreads();
        for (int k = 0; k < kWaves; k++) first = min(first, s_found[k]), last = max(last, s_last[k]);
        if (last >= 0) token = last;
        if (first != 0x7fffffff) token = first;
        if (first != 0x7fffffff || (!equal && last >= 0)) break;
        at -= all;
        __syncthreads();
    }
    if (threadIdx.x == 0) out = VerifyResult{c.accepted, (uint32_t)token, 0, 0};
}

constexpr int kSumGroups = 512;  // workgroups of the sums' launch, about two a CU

size_t align16(size_t n) { return (n + 15) & ~(size_t)15; }

}  // namespace

bool verify_fits(size_t rows, int vocab) {
    return grid_fits(rows * (((size_t)vocab + kChunk - 1) / kChunk), kPartBlock);
}

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
    if (!verify_fits(rows, a.vocab)) return set_error(SQ_ERR_SHAPE, "verify_draft: ShapeMismatch (too many logits)");
    auto kernel = a.inv_t == 0.0 ? verify_parts_kernel<true> : verify_parts_kernel<false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(rows * chunks)), dim3(kPartBlock), 0, s, a, (int)target_rows, chunks,
                       parts);
    hipLaunchKernelGGL(verify_sums_kernel, dim3(std::min(chunks, std::max(1, kSumGroups / (int)b.n_seqs)), b.n_seqs),
                       dim3(kBlock), 0, s, b, a, (int)target_rows, chunks, (const Part*)parts, sums, choices);
    hipLaunchKernelGGL(verify_draw_kernel, dim3(b.n_seqs), dim3(kBlock), 0, s, b, a, chunks, (const double*)sums,
                       (const Choice*)choices, results);
    return check_launch("verify");
}

}  // namespace sq
