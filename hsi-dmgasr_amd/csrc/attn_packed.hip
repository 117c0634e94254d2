// Attention over packed sequences: the C entry points, the choice of tile and split, and the small kernels around the main ones
// (attn_packed.h): joining split key ranges, the backward pass's row sums, adding split partial gradients.
#include "attn_packed.h"
#include <cmath>

namespace hsidm {

// Joins the shares of a split forward pass: part [S][T][Hq][D] fp32 normalised outputs, plse [S][Hq][T]; a row's weight of share s is
// exp(lse_s - lse).  Four elements a thread.
template <typename T>
__global__ __launch_bounds__(256) void attn_join_kernel(const float* __restrict__ part, const float* __restrict__ plse, int S, int64_t T_, int Hq, int D,
                                                        T* __restrict__ out, T* __restrict__ lo, float* __restrict__ lse) {
    const int per_row = D / 4;
    const int64_t n = T_ * Hq * per_row, rows = T_ * Hq;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / per_row;
        const int d = (int)(i - row * per_row) * 4, head = (int)(row % Hq);
        const int64_t at = head * T_ + row / Hq;
        float m = -INFINITY;
        for (int s = 0; s < S; ++s) m = fmaxf(m, plse[s * rows + at]);
        const float mm = m == -INFINITY ? 0.f : m;
        float l = 0.f;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < S; ++s) {
            const float w = __expf(plse[s * rows + at] - mm);
            const f32x4 x = *reinterpret_cast<const f32x4*>(part + (s * rows + row) * D + d);
            l += w;
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] += w * x[k];
        }
        typedef T vec __attribute__((ext_vector_type(4)));
        vec r, e;
        const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
        for (int k = 0; k < 4; ++k) { v[k] *= inv; r[k] = (T)v[k]; e[k] = (T)(v[k] - (float)r[k]); }
        *reinterpret_cast<vec*>(out + row * D + d) = r;
        if (lo) *reinterpret_cast<vec*>(lo + row * D + d) = e;
        if (lse && d == 0) lse[at] = mm + logf(l);
    }
}

// out[t][h][d] = sum over the shares of part[s * share + (t * H + h) * D + d], in order; up to three such sums (dK, dV, dQ) in one launch
struct AttnSum { const float* part; int64_t share; AttnTensor out; int S, H; };
struct AttnSums { AttnSum s[3]; };

template <typename T>
__global__ __launch_bounds__(256) void attn_add_kernel(AttnSums sums, int64_t T_, int D) {
    const AttnSum a = sums.s[blockIdx.y];
    const int per_row = D / 4;
    const int64_t n = T_ * a.H * per_row;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / per_row, token = row / a.H;
        const int d = (int)(i - row * per_row) * 4, head = (int)(row - token * a.H);
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < a.S; ++s) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(a.part + s * a.share + row * D + d);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] += x[k];
        }
        typedef T vec __attribute__((ext_vector_type(4)));
        vec r;
#pragma unroll
        for (int k = 0; k < 4; ++k) r[k] = (T)v[k];
        *reinterpret_cast<vec*>(reinterpret_cast<T*>(const_cast<char*>(a.out.p) + token * a.out.ts + head * a.out.hs) + d) = r;
    }
}

// delta[h][t] = sum_d dO O per row, O with its rounding residual where the forward pass kept it (without it, delta's error is as large as
// that of rounding dS and adds to it in dQ and dK: 1.55 ... 1.7 instead of 1.4 times the output's own rounding).  `group` lanes, a power of two
// that covers a row's 16-byte pieces, share a row.
struct DeltaRows {
    AttnTensor dout, o;
    const char* lo;
    int pieces, group;
};
__device__ __forceinline__ float group_sum(float x, int group) {
    for (int s = group >> 1; s > 0; s >>= 1) x += __shfl_xor(x, s, 64);
    return x;
}
// one row's dO . O, and this lane's share of |dO|^2
template <typename T>
__device__ __forceinline__ float delta_row(const DeltaRows& a, int64_t token, int head, int sub, bool live, float& sq) {
    constexpr int E = 16 / (int)sizeof(T);
    typedef T vec __attribute__((ext_vector_type(E)));
    float dot = 0.f;
    sq = 0.f;
    if (live && sub < a.pieces) {
        const vec x = *reinterpret_cast<const vec*>(a.dout.p + token * a.dout.ts + head * a.dout.hs + sub * 16);
        const vec y = *reinterpret_cast<const vec*>(a.o.p + token * a.o.ts + head * a.o.hs + sub * 16);
#pragma unroll
        for (int k = 0; k < E; ++k) { dot += (float)x[k] * (float)y[k]; sq += (float)x[k] * (float)x[k]; }
        if (sizeof(T) == 2 && a.lo) {
            const vec z = *reinterpret_cast<const vec*>(a.lo + token * a.o.ts + head * a.o.hs + sub * 16);
#pragma unroll
            for (int k = 0; k < E; ++k) dot += (float)x[k] * (float)z[k];
        }
    }
    return group_sum(dot, a.group);
}

constexpr int kDeltaBlocks = 512;

template <typename T>
__global__ __launch_bounds__(256) void attn_delta_kernel(DeltaRows a, int64_t T_, int Hq, float* __restrict__ delta) {
    const int sub = threadIdx.x & (a.group - 1), per = 256 / a.group;
    for (int64_t r0 = (int64_t)blockIdx.x * per; r0 < T_ * Hq; r0 += (int64_t)gridDim.x * per) {
        const int64_t r = r0 + threadIdx.x / a.group, token = r / Hq;
        const int head = (int)(r - token * Hq);
        float sq;
        const float dot = delta_row<T>(a, token, head, sub, r < T_ * Hq, sq);
        if (r < T_ * Hq && sub == 0) delta[head * T_ + token] = dot;
    }
}

// fp16: a workgroup per (64-row tile, key head), which also leaves the largest |dO|^2 and |V|^2 of the tile's finite rows (GradScale) at the
// tile's first token.
template <typename T>
__global__ __launch_bounds__(256) void attn_delta_tiles_kernel(DeltaRows a, AttnTensor v, const AttnTile* __restrict__ tiles, int64_t T_, int g, float* __restrict__ delta,
                                                               float* __restrict__ top_do, float* __restrict__ top_v) {
    constexpr int E = 16 / (int)sizeof(T);
    typedef T vec __attribute__((ext_vector_type(E)));
    __shared__ float red[2][4];
    const AttnTile tile = tiles[blockIdx.x];
    const int kvh = blockIdx.y, sub = threadIdx.x & (a.group - 1), per = 256 / a.group, rows = min(64, tile.len - tile.row0);
    const int64_t first = (int64_t)tile.start + tile.row0;
    float ma = 0.f, mb = 0.f;
    for (int r0 = 0; r0 < rows * g; r0 += per) {                     // (a token's heads one behind the other)
        const int r = r0 + threadIdx.x / a.group, row = r / g, head = kvh * g + (r - row * g);
        const bool live = row < rows;
        float sq;
        const float dot = delta_row<T>(a, first + row, head, sub, live, sq);
        ma = fmaxf(ma, finite_or_zero(group_sum(sq, a.group)));
        if (live && sub == 0) delta[head * T_ + first + row] = dot;
    }
    for (int r0 = 0; r0 < rows; r0 += per) {
        const int row = r0 + threadIdx.x / a.group;
        float sq = 0.f;
        if (row < rows && sub < a.pieces) {
            const vec x = *reinterpret_cast<const vec*>(v.p + (first + row) * v.ts + kvh * v.hs + sub * 16);
#pragma unroll
            for (int k = 0; k < E; ++k) sq += (float)x[k] * (float)x[k];
        }
        mb = fmaxf(mb, finite_or_zero(group_sum(sq, a.group)));
    }
    ma = wave_max(ma); mb = wave_max(mb);
    if ((threadIdx.x & 63) == 0) { red[0][threadIdx.x >> 6] = ma; red[1][threadIdx.x >> 6] = mb; }
    __syncthreads();
    if (threadIdx.x == 0) {
        top_do[kvh * T_ + first] = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
        top_v[kvh * T_ + first] = fmaxf(fmaxf(red[1][0], red[1][1]), fmaxf(red[1][2], red[1][3]));
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------
struct Cut { int waves, ntiles, splits; };
static int row_bytes(int D, int es) { return (D <= 32 ? 32 : D <= 64 ? 64 : D <= 128 ? 128 : 256) * es; }
static int tile_rows(int D, int es) { return row_bytes(D, es) <= 256 ? 64 : 32; }

// Tile height and split of the walked axis.  128-row tiles (4 waves) where they fill half the chip or the walk is long enough to split,
// else 64-row ones.  The walk is split where that pays by a coarse estimate of the time, in seconds, per number of shares:
//   tiles of equal work: rounds of resident workgroups times a share's steps;
//   unequal ones (causal, ragged; heaviest first): all work at the full rate, and 0.45 of the longest share at the end, alone;
//   plus the shares' partial sums, written in fp32 and read again.
// The rates and `resident` are constants of the estimate, fitted to the shares that measured best on a handful of cases when the forward
// kernel took 165 registers at D = 64; they decide the number of shares and nothing else.  They are not what the kernels have today: registers
// allow four forward workgroups of four waves at rows of 128 bytes (three are counted) and three at 256 in the 16-bit types (two), and the
// query-gradient walk runs beside the key walk, two at most (three are counted at 128 bytes).  Shares stay at four steps or more.
struct Walk { int resident, products; bool kv; };            // workgroups of four waves per CU, matrix products per tile pair
// waves: 0 to choose, 2 or 4 to go with another kernel's tiles
static Cut cut_work(const hsidm_attn_desc* d, int es, const Walk& k, int waves) {
    const int heads = k.kv ? d->Hk : d->Hq, walks = k.kv ? d->Hq / d->Hk : 1, rows = tile_rows(d->D, es), width = row_bytes(d->D, es) / es;
    const int64_t steps = (d->longest + rows - 1) / rows * walks;
    const double cus = device_cus(), rate = es == 4 ? 105e12 : width <= 32 ? 250e12 : width <= 64 ? 600e12 : 750e12;
    Cut c;
    c.waves = waves ? waves : (double)d->n128 * heads >= 0.5 * cus || steps >= 16 ? 4 : 2;
    c.ntiles = c.waves == 4 ? d->n128 : d->n64;
    const int tile = 32 * c.waves;
    const double slots = cus * k.resident * (4 / c.waves), n = (double)c.ntiles * heads;
    const double step = 2.0 * rows * tile * width * k.products;                            // flops
    const double total = d->pairs * heads * walks / ((double)tile * rows) * step;
    const double bytes = 2.0 * 4.0 * d->T * heads * d->D * (k.kv ? 2 : 1);                 // of one share's sums, there and back
    const bool equal = total > 0.9 * n * steps * step;
    double best = 1e300;
    c.splits = 1;
    for (int s = 1; s <= 16 && (s == 1 || steps / s >= 4); ++s) {
        const double share = (double)((steps + s - 1) / s) * step;
        double t = equal ? std::ceil(n * s / slots) * share * slots / rate : total / rate + 0.45 * share * cus / rate;
        if (s > 1) t += s * bytes / 4.5e12 + 5e-6;
        if (t < 0.97 * best) { best = t; c.splits = s; }
    }
    return c;
}
static Cut cut_queries(const hsidm_attn_desc* d, int es, int products, int waves = 0) {
    const int rb = row_bytes(d->D, es);
    return cut_work(d, es, {rb <= 128 ? 3 : rb <= (products == 2 ? 512 : 256) ? 2 : 1, products, false}, waves);
}
static Cut cut_keys(const hsidm_attn_desc* d, int es) {
    const int rb = row_bytes(d->D, es);
    return cut_work(d, es, {rb <= 256 ? 2 : 1, d->D > 128 ? 6 : 4, true}, 0);
}

// (token strides: the kernels hold 64 rows' offsets in 32 bits)
static bool rows_ok(const void* p, int64_t ts, int64_t hs, int es) {
    return p && (uintptr_t)p % 16 == 0 && ts >= 0 && hs >= 0 && ts <= (1 << 24) / es && ts * es % 16 == 0 && hs * es % 16 == 0;
}
static int check_attn(const hsidm_attn_desc* d, int& es) {
    if (!d || (d->prec != HSIDM_BF16 && d->prec != HSIDM_F16 && d->prec != HSIDM_F32X3)) return HSIDM_E_BADARG;
    es = d->prec == HSIDM_F32X3 ? 4 : 2;
    if (d->T <= 0 || d->T > 0x7fffff00 || d->Hk <= 0 || d->Hq <= 0 || d->Hq % d->Hk || d->Hq > 65535) return HSIDM_E_BADARG;
    if (d->D < 16 / es || d->D > 256 || d->D * es % 16) return HSIDM_E_BADARG;
    if (!(d->scale > 0.f) || !(d->scale < 1e30f)) return HSIDM_E_BADARG;
    if (!rows_ok(d->q, d->q_ts, d->q_hs, es) || !rows_ok(d->k, d->k_ts, d->k_hs, es) || !rows_ok(d->v, d->v_ts, d->v_hs, es)) return HSIDM_E_BADARG;
    if (!d->qtiles64 || !d->qtiles128 || !d->ktiles64 || !d->ktiles128 || d->n64 <= 0 || d->n128 <= 0 || d->longest <= 0 || !(d->pairs > 0)) return HSIDM_E_BADARG;
    return 0;
}
static AttnTensor tensor(const void* p, int64_t ts, int64_t hs, int es) { return {(const char*)p, ts * es, hs * es}; }
static int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }
static int launch(int prec, int kind, const void* args, const Cut& c, hipStream_t s) {
    if (prec == HSIDM_BF16) return attn_launch<bf16>(kind, args, c.waves, c.ntiles, s);
    if (prec == HSIDM_F16) return attn_launch<f16>(kind, args, c.waves, c.ntiles, s);
    return attn_launch<float>(kind, args, c.waves, c.ntiles, s);
}
static unsigned blocks_for(int64_t n) { const int64_t b = (n + 255) / 256; return (unsigned)(b < 65536 ? b : 65536); }

struct BwdPlan { Cut q, kv; int64_t delta, top_do, top_v, part_kv, part_q, bytes; };
static BwdPlan bwd_plan(const hsidm_attn_desc* d, int es) {
    BwdPlan p;
    p.kv = cut_keys(d, es);
    p.q = cut_queries(d, es, 3, p.kv.waves);                          // (one launch: one tile height)
    const int64_t top = es == 2 ? up16(d->T * d->Hk * 4) : 0;         // (one layout for the 16-bit types; fp16 uses it)
    p.delta = 0;
    p.top_do = up16(d->T * d->Hq * 4);
    p.top_v = p.top_do + top;
    p.part_kv = p.top_v + top;
    p.part_q = p.part_kv + (p.kv.splits > 1 ? (int64_t)p.kv.splits * 2 * d->T * d->Hk * d->D * 4 : 0);
    p.bytes = p.part_q + (p.q.splits > 1 ? (int64_t)p.q.splits * d->T * d->Hq * d->D * 4 : 0);
    return p;
}

template <typename T>
static void launch_delta(const DeltaRows& a, const hsidm_attn_desc* d, float* delta, hipStream_t s) {
    const int64_t blocks = (d->T * d->Hq * a.group + 255) / 256;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attn_delta_kernel<T>), dim3((unsigned)(blocks < kDeltaBlocks ? blocks : kDeltaBlocks)), dim3(256), 0, s, a, d->T, d->Hq, delta);
}
// (at most 2^32 threads along an axis: more tiles go in several launches)
static void launch_delta_f16(const DeltaRows& a, const AttnTensor& v, const hsidm_attn_desc* d, float* delta, float* top_do, float* top_v, hipStream_t s) {
    const AttnTile* tiles = (const AttnTile*)d->qtiles64;
    for (int64_t left = d->n64, most = 0xffffffffLL / 256; left > 0; left -= most, tiles += most)
        hipLaunchKernelGGL(HIP_KERNEL_NAME(attn_delta_tiles_kernel<f16>), dim3((unsigned)(left < most ? left : most), d->Hk), dim3(256), 0, s, a, v, tiles, d->T, d->Hq / d->Hk,
                           delta, top_do, top_v);
}
template <typename T>
static void launch_add(const AttnSums& sums, int n, int heads, int64_t T_, int D, hipStream_t s) {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attn_add_kernel<T>), dim3(blocks_for(T_ * heads * D / 4), n), dim3(256), 0, s, sums, T_, D);
}

}  // namespace hsidm

using namespace hsidm;

extern "C" int64_t hsidm_attention_packed_workspace_bytes(const hsidm_attn_desc* d) {
    int es;
    if (int rc = check_attn(d, es)) return rc;
    const Cut c = cut_queries(d, es, 2);
    return c.splits > 1 ? (int64_t)c.splits * d->T * d->Hq * (d->D + 1) * 4 : 0;
}

extern "C" int hsidm_attention_packed(const hsidm_attn_desc* d, void* out, void* out_lo, float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
    int es;
    if (int rc = check_attn(d, es)) return rc;
    if (!rows_ok(out, 0, 0, es) || (uintptr_t)out_lo % 16) return HSIDM_E_BADARG;
    const Cut c = cut_queries(d, es, 2);
    const int64_t rows = d->T * d->Hq;
    if (c.splits > 1 && (!rows_ok(workspace, 0, 0, 4) || workspace_bytes < c.splits * rows * (d->D + 1) * 4)) return HSIDM_E_BADARG;
    AttnFwdArgs a;
    a.q = tensor(d->q, d->q_ts, d->q_hs, es); a.k = tensor(d->k, d->k_ts, d->k_hs, es); a.v = tensor(d->v, d->v_ts, d->v_hs, es);
    float* part = (float*)workspace;
    a.out = c.splits > 1 ? (void*)part : out;
    a.lo = c.splits > 1 ? nullptr : out_lo;
    a.lse = c.splits > 1 ? part + c.splits * rows * d->D : lse;
    a.tiles = (const AttnTile*)(c.waves == 4 ? d->qtiles128 : d->qtiles64);
    a.T = d->T; a.Hq = d->Hq; a.Hk = d->Hk; a.D = d->D; a.causal = d->causal; a.splits = c.splits; a.scale = d->scale;
    hipStream_t s = (hipStream_t)stream;
    if (int rc = launch(d->prec, ATTN_FWD, &a, c, s)) return rc;
    if (c.splits > 1) {
        const dim3 grid(blocks_for(rows * d->D / 4));
        const float* pl = part + c.splits * rows * d->D;
#define JOIN(OUT) hipLaunchKernelGGL(HIP_KERNEL_NAME(attn_join_kernel<OUT>), grid, dim3(256), 0, s, (const float*)part, pl, c.splits, d->T, d->Hq, d->D, (OUT*)out, (OUT*)out_lo, lse)
        if (d->prec == HSIDM_BF16) JOIN(bf16);
        else if (d->prec == HSIDM_F16) JOIN(f16);
        else JOIN(float);
#undef JOIN
    }
    return (int)hipGetLastError();
}

extern "C" int64_t hsidm_attention_packed_bwd_workspace_bytes(const hsidm_attn_desc* d) {
    int es;
    if (int rc = check_attn(d, es)) return rc;
    return bwd_plan(d, es).bytes;
}

extern "C" int hsidm_attention_packed_bwd(const hsidm_attn_desc* d, const void* out, const void* out_lo, const float* lse, const void* dout, int64_t do_ts, int64_t do_hs,
                                          void* dq, int64_t dq_ts, int64_t dq_hs, void* dk, int64_t dk_ts, int64_t dk_hs, void* dv, int64_t dv_ts,
                                          int64_t dv_hs, void* workspace, int64_t workspace_bytes, void* stream) {
    int es;
    if (int rc = check_attn(d, es)) return rc;
    if (!lse || !rows_ok(out, 0, 0, es) || (uintptr_t)out_lo % 16 || !rows_ok(dout, do_ts, do_hs, es) || !rows_ok(dq, dq_ts, dq_hs, es) || !rows_ok(dk, dk_ts, dk_hs, es) ||
        !rows_ok(dv, dv_ts, dv_hs, es))
        return HSIDM_E_BADARG;
    const BwdPlan p = bwd_plan(d, es);
    if (!rows_ok(workspace, 0, 0, 4) || workspace_bytes < p.bytes) return HSIDM_E_BADARG;
    char* ws = (char*)workspace;
    float *delta = (float*)(ws + p.delta), *top_do = (float*)(ws + p.top_do), *top_v = (float*)(ws + p.top_v);
    hipStream_t s = (hipStream_t)stream;
    AttnBwdArgs a;
    a.q = tensor(d->q, d->q_ts, d->q_hs, es); a.k = tensor(d->k, d->k_ts, d->k_hs, es); a.v = tensor(d->v, d->v_ts, d->v_hs, es);
    a.dout = tensor(dout, do_ts, do_hs, es);
    a.dq = tensor(dq, dq_ts, dq_hs, es); a.dk = tensor(dk, dk_ts, dk_hs, es); a.dv = tensor(dv, dv_ts, dv_hs, es);
    a.lse = lse; a.delta = delta; a.top_do = top_do; a.top_v = top_v;
    a.T = d->T; a.Hq = d->Hq; a.Hk = d->Hk; a.D = d->D; a.causal = d->causal; a.scale = d->scale;
    DeltaRows rows = {a.dout, tensor(out, (int64_t)d->Hq * d->D, d->D, es), (const char*)out_lo, d->D * es / 16, 1};
    while (rows.group < rows.pieces) rows.group *= 2;
    if (d->prec == HSIDM_BF16) launch_delta<bf16>(rows, d, delta, s);
    else if (d->prec == HSIDM_F16) launch_delta_f16(rows, a.v, d, delta, top_do, top_v, s);
    else launch_delta<float>(rows, d, delta, s);
    const bool tall = p.kv.waves == 4;
    AttnBwdPair pair = {a, a};
    pair.kv.splits = p.kv.splits; pair.kv.part = (float*)(ws + p.part_kv);
    pair.kv.tiles = (const AttnTile*)(tall ? d->ktiles128 : d->ktiles64);
    pair.q.splits = p.q.splits; pair.q.part = (float*)(ws + p.part_q);
    pair.q.tiles = (const AttnTile*)(tall ? d->qtiles128 : d->qtiles64);
    if (int rc = launch(d->prec, ATTN_BWD, &pair, p.kv, s)) return rc;
    AttnSums sums;
    int n = 0, heads = 0;
    if (p.kv.splits > 1) {
        const int64_t one = d->T * d->Hk * d->D;
        sums.s[n++] = {pair.kv.part, 2 * one, a.dk, p.kv.splits, d->Hk};
        sums.s[n++] = {pair.kv.part + one, 2 * one, a.dv, p.kv.splits, d->Hk};
        heads = d->Hk;
    }
    if (p.q.splits > 1) {
        sums.s[n++] = {pair.q.part, d->T * d->Hq * d->D, a.dq, p.q.splits, d->Hq};
        heads = d->Hq;
    }
    if (n) {
        if (d->prec == HSIDM_BF16) launch_add<bf16>(sums, n, heads, d->T, d->D, s);
        else if (d->prec == HSIDM_F16) launch_add<f16>(sums, n, heads, d->T, d->D, s);
        else launch_add<float>(sums, n, heads, d->T, d->D, s);
    }
    return (int)hipGetLastError();
}
