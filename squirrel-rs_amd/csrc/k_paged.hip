// Attention over the paged 8-bit key/value cache (kv.h).
//
// Row r of the batch, at position p of its sequence, head h of KV head
// h / (heads / kv_heads):  o = sum_j softmax_j(q . k_j / sqrt(d)) v_j  over the
// positions j <= p, with a window only those with j > p - window or
// j < sinks.
#include <algorithm>
#include <cmath>

#include "kv.h"

namespace sq {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

inline int check_launch(const char* what) {
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return set_error(SQ_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
    return 0;
}

// The query rows of one KV head of a sequence are its n_new * G (position,
// head) pairs, row r = i * G + (head in the group).
//
// The pages that the rows of a tile see, as one list: first those of the
// sinks, then those from the first page of the tile's windows to its last
// position's.
struct Span {
    int sink_pages, first, count;
    __host__ __device__ int page(int i) const { return i < sink_pages ? i : first + i - sink_pages; }
};
__host__ __device__ inline Span tile_span(int pos_lo, int pos_hi, int window, int sinks) {
    Span s{0, 0, pos_hi / kPage + 1};
    if (window > 0 && pos_lo >= window) {
        s.first = (pos_lo - window + 1) / kPage;
        s.sink_pages = (sinks + kPage - 1) / kPage;
        if (s.sink_pages > s.first) s.sink_pages = s.first;
        s.count = s.sink_pages + pos_hi / kPage - s.first + 1;
    }
    return s;
}

// What a launch covers: the sequences with rows_lo <= n_new * G <= rows_hi,
// their pages cut into parts of `chunk`.  The parts' sums stand in the
// workspace at slot (table0 / chunk + sequence + part): a sequence has at
// most pages / chunk + 1 parts, so slots do not overlap.
struct Cut {
    int rows_lo, rows_hi, chunk, tiles, splits;
    float* ws;
    __host__ __device__ size_t slot(const KvSeq& s, int seq, int part) const {
        return (size_t)(s.table0 / chunk) + seq + part;
    }
};

// Eight stored bytes as f16, exactly: 0x64uu is 1024 + u, u = q + 128.
__device__ __forceinline__ v8h unpack8(uint32_t a, uint32_t b) {
    const uint32_t w[4] = {
        __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u),
        __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)};
    v8h r;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const v2h x = __builtin_bit_cast(v2h, w[i]) - (v2h){(_Float16)1152.0f, (_Float16)1152.0f};
        r[2 * i] = x[0], r[2 * i + 1] = x[1];
    }
    return r;
}

// Maximum / sum over the four lanes that share a query (l % 16).
__device__ __forceinline__ float groups_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float groups_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

// Scores are formed transposed, K Q^T, so that a lane holds one query's
// probabilities of sixteen positions, in the order of the stored values: they
// are the second product's operand as they stand (V^T P^T), and its results,
// dimensions of the same query, are scaled lane by lane.
//
// The cached integers are exact in f16.  A query's elements, scaled by a power
// of two to at most 2^14, and a page's probabilities, times 2^14, are split into
// two f16 halves each (x = hi + lo to 2^-22 of x): two products on the matrix
// pipe give what one in f32 would, four times as fast.
//
// PAGES: the four wavefronts take pages in turn for the same 16 R rows and meet in
// LDS; otherwise each has its own 16 R rows and all walk the same pages.
template <int HD, int R, bool PAGES>
__global__ __launch_bounds__(256) void sdpa_paged_kernel(KvView kv, KvPlanView pl, PagedArgs a, Cut cut, float scale) {
    constexpr int C = HD / 64, DT = HD / 16, TR = PAGES ? 16 * R : 64 * R;
    __shared__ float s_o[PAGES ? 4 * 16 * R * (HD + 4) : 1];
    __shared__ float s_m[PAGES ? 4 * 16 * R : 1], s_l[PAGES ? 4 * 16 * R : 1];
    int b = blockIdx.x;
    const int head = b % kv.kv_heads;
    b /= kv.kv_heads;
    const int part = b % cut.splits;
    b /= cut.splits;
    const int tile = b % cut.tiles, seq = b / cut.tiles;
    const KvSeq s = pl.seqs[seq];
    const int G = a.heads / kv.kv_heads, rows = s.n_new * G;
    if (rows < cut.rows_lo || rows > cut.rows_hi || tile * TR >= rows) return;
    const int row_end = min(rows, (tile + 1) * TR);
    const Span span = tile_span(s.past + tile * TR / G, s.past + (row_end - 1) / G, a.window, a.sinks);
    const int i_end = min(span.count, (part + 1) * cut.chunk);
    if (part * cut.chunk >= i_end) return;
    const bool whole = span.count <= cut.chunk;

    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, q16 = lane & 15, g = lane >> 4;
    const int row0 = tile * TR + (PAGES ? 0 : wave * 16 * R);  // the wavefront's first row

    // queries: halves [chunk of 64][half of a lane's 16 dimensions]
    v8h qh[R][C][2], ql[R][C][2];
    float cq[R];
    int pos[R], w0[R];
#pragma unroll
    for (int t = 0; t < R; t++) {
        const int r = min(row0 + 16 * t + q16, rows - 1), i = r / G;
        pos[t] = s.past + i;
        w0[t] = a.window && a.window <= pos[t] ? pos[t] - a.window + 1 : 0;
        const size_t row = (size_t)s.row0 + i;
        const float* q = a.q + row * a.q_stride + (size_t)(head * G + r % G) * HD;
        float x[C][16];
        float amax = 0.0f;
        bool ok = true;
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                const int d = 64 * c + 16 * g + e;
                float u = q[d], v = q[d + 1];
                ok = ok && fabsf(u) < INFINITY && fabsf(v) < INFINITY;
                if (pl.rope && d / 2 < pl.half) {
                    const double2 cs = pl.rope[row * pl.half + d / 2];
                    const double p = (double)u * cs.x - (double)v * cs.y;
                    v = (float)((double)u * cs.y + (double)v * cs.x);
                    u = (float)p;
                }
                x[c][e] = u, x[c][e + 1] = v;
                amax = fmaxf(amax, fmaxf(fabsf(u), fabsf(v)));
            }
        // (a row that is not finite, or leaves f32 by its rotation: NaN scores for it alone)
        amax = groups_max(ok ? amax : INFINITY);
        const int shift = amax < INFINITY ? min(13 - (int)((__builtin_bit_cast(uint32_t, amax) >> 23) & 255) + 127, 100) : 0;
        cq[t] = amax < INFINITY ? ldexpf(scale, -shift) : NAN;
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const float y = amax < INFINITY ? ldexpf(x[c][e], shift) : 0.0f;
                const _Float16 h = (_Float16)y;
                qh[t][c][e / 8][e % 8] = h;
                ql[t][c][e / 8][e % 8] = (_Float16)(y - (float)h);
            }
    }

    v4f o[R][DT];
    float m[R], l[R];
#pragma unroll
    for (int t = 0; t < R; t++) {
        m[t] = -INFINITY, l[t] = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; d++) o[t][d] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // rows between the tile's first and last position see a page whole where both do
    const int pos_lo = s.past + row0 / G, pos_hi = s.past + (min(rows, row0 + 16 * R) - 1) / G;
    const int w0_hi = a.window && a.window <= pos_hi ? pos_hi - a.window + 1 : 0;

    const int step = PAGES ? 4 : 1;
    for (int i = part * cut.chunk + (PAGES ? wave : 0); i < i_end; i += step) {
        const int page = span.page(i);
        const size_t cell = (size_t)pl.pages[s.table0 + page] * kv.kv_heads + head;
        const float2 sc = kv.scales[cell];
        const uint4* kb = (const uint4*)(kv.bytes + cell * 2 * kPage * HD) + lane;
        uint4 kw[4][C], vw[DT];
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int c = 0; c < C; c++) kw[t][c] = kb[(t * C + c) * 64];
#pragma unroll
        for (int d = 0; d < DT; d++) vw[d] = kb[(4 * C + d) * 64];
        // scores [tile of 16 positions][position 4 g + r]
        v4f x[R][4];
#pragma unroll
        for (int t = 0; t < 4; t++) {
#pragma unroll
            for (int u = 0; u < R; u++) x[u][t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < C; c++) {
                const v8h k0 = unpack8(kw[t][c].x, kw[t][c].y), k1 = unpack8(kw[t][c].z, kw[t][c].w);
#pragma unroll
                for (int u = 0; u < R; u++) {
                    x[u][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, ql[u][c][0], x[u][t], 0, 0, 0);
                    x[u][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, ql[u][c][1], x[u][t], 0, 0, 0);
                    x[u][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qh[u][c][0], x[u][t], 0, 0, 0);
                    x[u][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qh[u][c][1], x[u][t], 0, 0, 0);
                }
            }
        }
        const bool full = (page + 1) * kPage - 1 <= pos_lo && (page * kPage >= w0_hi || (page + 1) * kPage <= a.sinks);
        v8h ph[R][2], plo[R][2];
        float alpha[R];
#pragma unroll
        for (int u = 0; u < R; u++) {
            const float cs = cq[u] * sc.x;
            float mx = -INFINITY;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float y = x[u][t][r] * cs;
                    if (!full) {
                        const int at = page * kPage + 16 * t + 4 * g + r;
                        if (at > pos[u] || (at < w0[u] && at >= a.sinks)) y = -INFINITY;
                    }
                    x[u][t][r] = y;
                    mx = fmaxf(mx, y);
                }
            const float mn = fmaxf(m[u], groups_max(mx));
            const float base = mn == -INFINITY ? 0.0f : mn;
            alpha[u] = __builtin_amdgcn_exp2f(m[u] - base);
            m[u] = mn;
            float sum = 0.0f;
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const float p = __builtin_amdgcn_exp2f(x[u][t][r] - base + 14.0f);
                    sum += p;
                    const _Float16 h = (_Float16)p;
                    const int j = 4 * r + t;
                    ph[u][j / 8][j % 8] = h;
                    plo[u][j / 8][j % 8] = (_Float16)(p - (float)h);
                }
            l[u] = l[u] * alpha[u] + sum;
        }
#pragma unroll
        for (int d = 0; d < DT; d++) {
            const v8h v0 = unpack8(vw[d].x, vw[d].y), v1 = unpack8(vw[d].z, vw[d].w);
#pragma unroll
            for (int u = 0; u < R; u++) {
                v4f y = {0.0f, 0.0f, 0.0f, 0.0f};
                y = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, plo[u][0], y, 0, 0, 0);
                y = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, plo[u][1], y, 0, 0, 0);
                y = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, ph[u][0], y, 0, 0, 0);
                y = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, ph[u][1], y, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; r++) o[u][d][r] = o[u][d][r] * alpha[u] + y[r] * sc.y;
            }
        }
    }
#pragma unroll
    for (int u = 0; u < R; u++) l[u] = groups_sum(l[u]);

    // where row r's sums go: its output, or its part of the workspace
    auto emit = [&](int r, int d, float v, float mm, float ll) {
        if (whole) {
            a.out[((size_t)s.row0 + r / G) * a.out_stride + (size_t)(head * G + r % G) * HD + d] = v / ll;
        } else {
            const size_t at = (cut.slot(s, seq, part) * kv.kv_heads + head) * cut.rows_hi + r;
            float* w = cut.ws + at * (HD + 2);
            w[d] = v;
            if (d == 0) w[HD] = mm, w[HD + 1] = ll;
        }
    };
    if constexpr (PAGES) {
#pragma unroll
        for (int u = 0; u < R; u++) {
            const int r = wave * 16 * R + 16 * u + q16;
            if (g == 0) s_m[r] = m[u], s_l[r] = l[u];
#pragma unroll
            for (int d = 0; d < DT; d++) *(v4f*)&s_o[r * (HD + 4) + 16 * d + 4 * g] = o[u][d];
        }
        __syncthreads();
        for (int e = threadIdx.x; e < 16 * R * HD; e += 256) {
            const int r = e / HD, d = e % HD;
            if (row0 + r >= rows) break;
            float mm = -INFINITY, ll = 0.0f, v = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; w++) mm = fmaxf(mm, s_m[w * 16 * R + r]);
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const int k = w * 16 * R + r;
                // (no page, or none visible: nothing; NaN scores keep their NaN)
                const float f = s_m[k] == -INFINITY && s_l[k] == 0.0f ? 0.0f
                                : __builtin_amdgcn_exp2f((s_m[k] == -INFINITY ? 0.0f : s_m[k]) - (mm == -INFINITY ? 0.0f : mm));
                ll += s_l[k] * f;
                v += s_o[k * (HD + 4) + d] * f;
            }
            emit(row0 + r, d, v, mm, ll);
        }
    } else {
#pragma unroll
        for (int u = 0; u < R; u++) {
            const int r = row0 + 16 * u + q16;
            if (r >= rows) continue;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int k = 0; k < 4; k++) emit(r, 16 * d + 4 * g + k, o[u][d][k], m[u], l[u]);
        }
    }
}

// The parts of the rows whose pages were cut: one workgroup per (sequence,
// KV head, row), a wavefront per quarter of the parts.
template <int HD>
__global__ __launch_bounds__(256) void sdpa_merge_kernel(KvView kv, KvPlanView pl, PagedArgs a, Cut cut, int tile_rows) {
    __shared__ float s_o[4][HD], s_m[4], s_l[4];
    const int seq = blockIdx.y, head = blockIdx.x % kv.kv_heads, r = blockIdx.x / kv.kv_heads;
    const KvSeq s = pl.seqs[seq];
    const int G = a.heads / kv.kv_heads, rows = s.n_new * G;
    if (rows < cut.rows_lo || rows > cut.rows_hi || r >= rows) return;
    const int tile = r / tile_rows, row_end = min(rows, (tile + 1) * tile_rows);
    const Span span = tile_span(s.past + tile * tile_rows / G, s.past + (row_end - 1) / G, a.window, a.sinks);
    if (span.count <= cut.chunk) return;
    const int parts = (span.count + cut.chunk - 1) / cut.chunk;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const size_t stride = (size_t)kv.kv_heads * cut.rows_hi * (HD + 2);
    const float* w = cut.ws + ((cut.slot(s, seq, 0) * kv.kv_heads + head) * cut.rows_hi + r) * (HD + 2);
    float m = -INFINITY, l = 0.0f, o[HD / 64] = {};
    auto fold = [](float& m, float& l, float* o, float m1, float l1, const float* o1) {
        const float mn = fmaxf(m, m1), base = mn == -INFINITY ? 0.0f : mn;
        const float f = __builtin_amdgcn_exp2f(m - base);
        const float f1 = m1 == -INFINITY && l1 == 0.0f ? 0.0f
                         : __builtin_amdgcn_exp2f((m1 == -INFINITY ? 0.0f : m1) - base);
        m = mn;
        l = l * f + l1 * f1;
        for (int c = 0; c < HD / 64; c++) o[c] = o[c] * f + o1[c] * f1;
    };
    for (int i = wave; i < parts; i += 4) {
        const float* p = w + (size_t)i * stride;
        float o1[HD / 64];
        for (int c = 0; c < HD / 64; c++) o1[c] = p[64 * c + lane];
        fold(m, l, o, p[HD], p[HD + 1], o1);
    }
    for (int c = 0; c < HD / 64; c++) s_o[wave][64 * c + lane] = o[c];
    if (lane == 0) s_m[wave] = m, s_l[wave] = l;
    __syncthreads();
    if (wave) return;
    for (int k = 1; k < 4; k++) {
        float o1[HD / 64];
        for (int c = 0; c < HD / 64; c++) o1[c] = s_o[k][64 * c + lane];
        fold(m, l, o, s_m[k], s_l[k], o1);
    }
    float* out = a.out + ((size_t)s.row0 + r / G) * a.out_stride + (size_t)(head * G + r % G) * HD;
    for (int c = 0; c < HD / 64; c++) out[64 * c + lane] = o[c] / l;
}

// Sequences of few rows: wavefronts over pages, tiles of 16 rows; of more: wavefronts over
// rows, tiles of 128.
constexpr int kFewRows = 64, kTileFew = 16, kTileMany = 128;
constexpr int kTarget = 1024;  // workgroups that a launch is cut into

struct Launch {
    Cut cut;
    size_t floats;
    bool any;
};
Launch plan_launch(const std::vector<KvSeq>& seqs, const KvView& kv, const PagedArgs& a, bool many) {
    const int G = a.heads / kv.kv_heads, tile = many ? kTileMany : kTileFew;
    Launch r{};
    r.cut.rows_lo = many ? kFewRows + 1 : 1;
    long long work = 0, groups = 0, pages = 0;
    int longest = 0;
    for (const KvSeq& s : seqs) {
        const int rows = s.n_new * G;
        pages = s.table0 + (s.past + s.n_new + kPage - 1) / kPage;
        if (rows < 1 || (rows > kFewRows) != many) continue;
        r.any = true;
        const int tiles = (rows + tile - 1) / tile;
        r.cut.rows_hi = std::max(r.cut.rows_hi, rows);
        r.cut.tiles = std::max(r.cut.tiles, tiles);
        groups += tiles;
        for (int t = 0; t < tiles; t++) {
            const Span sp = tile_span(s.past + t * tile / G, s.past + (std::min(rows, (t + 1) * tile) - 1) / G, a.window, a.sinks);
            work += sp.count;
            longest = std::max(longest, sp.count);
        }
    }
    work *= kv.kv_heads;
    groups *= kv.kv_heads;
    // pages of a part: as many workgroups as the card takes at a time, unless
    // the tiles alone are
    const int least = many ? 1 : 4;
    long long chunk = groups >= kTarget ? longest : std::max<long long>(least, (work + kTarget - 1) / kTarget);
    for (;; chunk *= 2) {
        r.cut.chunk = (int)std::min<long long>(chunk, std::max(longest, 1));
        r.cut.splits = (longest + r.cut.chunk - 1) / std::max(r.cut.chunk, 1);
        r.floats = r.cut.splits < 2 ? 0
                                    : (size_t)(pages / r.cut.chunk + seqs.size() + 1) * kv.kv_heads * r.cut.rows_hi *
                                          (kv.head_dim + 2);
        if (r.floats <= ((size_t)64 << 20)) break;  // 256 MB
    }
    return r;
}

template <int HD, int R, bool PAGES>
int launch_one(hipStream_t s, const Launch& l, const KvView& kv, const KvPlanView& p, const PagedArgs& a) {
    const float scale = 1.4426950408889634f / sqrtf((float)HD);  // scores in units of log 2
    const size_t grid = (size_t)p.n_seqs * l.cut.tiles * l.cut.splits * kv.kv_heads;
    const size_t merge = (size_t)l.cut.rows_hi * kv.kv_heads;
    if (grid > (size_t)INT32_MAX || merge > (size_t)INT32_MAX)
        return set_error(SQ_ERR_SHAPE, "sdpa_paged: ShapeMismatch (too many rows)");
    hipLaunchKernelGGL((sdpa_paged_kernel<HD, R, PAGES>), dim3((unsigned)grid), dim3(256), 0, s, kv, p, a, l.cut, scale);
    if (l.cut.splits > 1)
        hipLaunchKernelGGL((sdpa_merge_kernel<HD>), dim3((unsigned)merge, p.n_seqs), dim3(256), 0, s, kv, p, a, l.cut,
                           PAGES ? kTileFew : kTileMany);
    return check_launch("sdpa_paged");
}

}  // namespace

size_t sdpa_paged_floats(const std::vector<KvSeq>& seqs, const KvView& kv, const PagedArgs& a) {
    return std::max(plan_launch(seqs, kv, a, false).floats, plan_launch(seqs, kv, a, true).floats);
}

int launch_sdpa_paged(hipStream_t s, const std::vector<KvSeq>& seqs, const KvView& kv, const KvPlanView& p,
                      const PagedArgs& a, float* ws) {
    for (bool many : {false, true}) {
        Launch l = plan_launch(seqs, kv, a, many);
        if (!l.any) continue;
        l.cut.ws = ws;
        int st;
        if (kv.head_dim == 64)
            st = many ? launch_one<64, 2, false>(s, l, kv, p, a) : launch_one<64, 1, true>(s, l, kv, p, a);
        else
            st = many ? launch_one<128, 2, false>(s, l, kv, p, a) : launch_one<128, 1, true>(s, l, kv, p, a);
        if (st) return st;
    }
    return 0;
}

}  // namespace sq
