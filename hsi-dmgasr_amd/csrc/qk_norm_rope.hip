// RMS norm of queries and keys per head, and the rotation by positions with several axes, in one pass - forward and backward.
//   n = x * r * w, r = rsqrt(mean_d x^2 + eps);   y = R n: pair p = (n[p], n[p + D/2]) turned by angle(p) = pos[token][axis(p)] * f(p)
//   backward (R is orthogonal): dn = R^T dy, g = dn * w, xhat = x * r:  dx = r * (g - xhat * mean_d(g * xhat)),  dw = sum dn * xhat
// Bound by HBM: x is read once and y written once (backward: x and dy read, dx written; r is recomputed, nothing is saved).
// A lane holds 8 elements of the first half of a head and the 8 they pair with, so the rotation needs no exchange; D/16 lanes (rounded up
// to a power of two) share a head, and walk the token's heads with ONE set of sines and cosines: those are the costly part - the angle is
// formed in 64 bits, as turns, and only its fraction is rounded, so that far positions (10^5 and more radians) keep their angle.
// 5 x 128 x 128 tokens, 8 + 2 heads of 64, bf16: 50 us, 4.2 TB/s (a large copy reaches 4.9); 19215 tokens, 4 + 4 heads of 128, fp16: forward 17
// us, backward 37 + 4 us.  Tried and not kept: stores past the caches (backward 9 % faster, forward 11 % slower, and the next kernel reads the
// result), more than one workgroup per token block once every CU has two.
#include "common.h"
#include "../../include/hsidm.h"

namespace hsidm {

struct RopeShape {
    int64_t T;
    int Hq, Hk, D, P, axes, group, heads_per;      // P rotated pairs; group lanes per head; heads_per heads per workgroup (of q | k in a row)
    int bound[HSIDM_ROPE_AXES];                    // first pair behind each axis's section
    float eps;
};
struct RopeSide { const void* x; int64_t ts, hs; const float* w; };

// cosines and sines of a lane's 8 pairs (p0 .. p0+7); pairs beyond P are not turned
__device__ __forceinline__ void rope_angles(const RopeShape& s, const int32_t* __restrict__ pos, const double* __restrict__ freq, int64_t token,
                                            int p0, bool live, float (&c)[8], float (&sn)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int p = p0 + j;
        c[j] = 1.f; sn[j] = 0.f;
        if (live && p < s.P) {
            int ax = 0;
#pragma unroll
            for (int a = 0; a + 1 < HSIDM_ROPE_AXES; ++a) ax += p >= s.bound[a] ? 1 : 0;
            const double turns = (double)pos[token * s.axes + ax] * freq[p];
            sincospif(2.0f * (float)(turns - rint(turns)), &sn[j], &c[j]);
        }
    }
}

__device__ __forceinline__ float group_sum(float v, int group) {
    for (int o = group >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

template <typename T>
__device__ __forceinline__ void load16(const T* p, int half, bool live, float (&a)[8], float (&b)[8]) {
    if (live) { Vec8<T>::load(p, a); Vec8<T>::load(p + half, b); }
    else {
#pragma unroll
        for (int j = 0; j < 8; ++j) { a[j] = 0.f; b[j] = 0.f; }
    }
}
// (conversions round to nearest even and keep infinities and NaN: fp16 does not saturate here)
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&v)[8]) { Vec8<T>::store(p, v); }
template <> __device__ __forceinline__ void store8<f16>(f16* p, const float (&v)[8]) {
    f16x8 r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = (f16)v[j];
    *reinterpret_cast<f16x8*>(p) = r;
}

template <typename T>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(RopeShape s, RopeSide q, RopeSide k, const int32_t* __restrict__ pos,
                                                           const double* __restrict__ freq, T* __restrict__ oq, T* __restrict__ ok) {
    const int sub = threadIdx.x & (s.group - 1), half = s.D >> 1;
    const int64_t token = (int64_t)blockIdx.x * (256 / s.group) + threadIdx.x / s.group;
    const bool live = token < s.T && sub * 8 < half;
    const int h0 = blockIdx.y * s.heads_per, h1 = min(h0 + s.heads_per, s.Hq + s.Hk);
    float c[8], sn[8];
    rope_angles(s, pos, freq, token, sub * 8, live, c, sn);
    auto side = [&](const RopeSide& in, T* out, int heads, int lo, int hi) __attribute__((always_inline)) {
        if (lo >= hi) return;
        float wa[8], wb[8];
        load16<float>(in.w + sub * 8, half, live, wa, wb);
        const T* src = reinterpret_cast<const T*>(in.x) + token * in.ts + sub * 8;
        T* dst = out + token * heads * s.D + sub * 8;
        for (int h = lo; h < hi; ++h) {
            float a[8], b[8];
            load16<T>(src + h * in.hs, half, live, a, b);
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) ss += a[j] * a[j] + b[j] * b[j];
            const float r = rsqrtf(group_sum(ss, s.group) / (float)s.D + s.eps);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float na = a[j] * r * wa[j], nb = b[j] * r * wb[j];
                a[j] = na * c[j] - nb * sn[j];
                b[j] = na * sn[j] + nb * c[j];
            }
            if (live) { store8<T>(dst + (int64_t)h * s.D, a); store8<T>(dst + (int64_t)h * s.D + half, b); }
        }
    };
    side(q, oq, s.Hq, h0, min(h1, s.Hq));
    side(k, ok, s.Hk, max(h0 - s.Hq, 0), h1 - s.Hq);
}

struct RopeGradSide { const void* dy; void* dx; int64_t ts, hs; };       // dy contiguous; dx's strides

template <typename T>
__global__ __launch_bounds__(256) void qk_norm_rope_bwd_kernel(RopeShape s, RopeSide q, RopeSide k, RopeGradSide gq, RopeGradSide gk,
                                                               const int32_t* __restrict__ pos, const double* __restrict__ freq,
                                                               float* __restrict__ part) {
    __shared__ float red[256 * 16];
    const int sub = threadIdx.x & (s.group - 1), half = s.D >> 1, groups = 256 / s.group, grp = threadIdx.x / s.group;
    const int h0 = blockIdx.y * s.heads_per, h1 = min(h0 + s.heads_per, s.Hq + s.Hk);
    float dwq[16], dwk[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) { dwq[j] = 0.f; dwk[j] = 0.f; }
    for (int64_t t0 = (int64_t)blockIdx.x * groups; t0 < s.T; t0 += (int64_t)gridDim.x * groups) {
        const int64_t token = t0 + grp;
        const bool live = token < s.T && sub * 8 < half;
        float c[8], sn[8];
        rope_angles(s, pos, freq, token, sub * 8, live, c, sn);
        auto side = [&](const RopeSide& in, const RopeGradSide& g, int heads, int lo, int hi, float (&dw)[16]) __attribute__((always_inline)) {
            if (lo >= hi) return;
            float wa[8], wb[8];
            load16<float>(in.w + sub * 8, half, live, wa, wb);
            const T* src = reinterpret_cast<const T*>(in.x) + token * in.ts + sub * 8;
            const T* dyp = reinterpret_cast<const T*>(g.dy) + token * heads * s.D + sub * 8;
            T* dst = reinterpret_cast<T*>(g.dx) + token * g.ts + sub * 8;
            for (int h = lo; h < hi; ++h) {
                float a[8], b[8], da[8], db[8];
                load16<T>(src + h * in.hs, half, live, a, b);
                load16<T>(dyp + (int64_t)h * s.D, half, live, da, db);
                float ss = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) ss += a[j] * a[j] + b[j] * b[j];
                float r = rsqrtf(group_sum(ss, s.group) / (float)s.D + s.eps);
                r = token < s.T ? r : 0.f;               // (behind the last token the row is zeros: with eps = 0, 0 * infinity)
                float dot = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float na = da[j] * c[j] + db[j] * sn[j], nb = db[j] * c[j] - da[j] * sn[j];       // dn
                    a[j] *= r; b[j] *= r;                                                                   // xhat
                    dw[j] += na * a[j]; dw[8 + j] += nb * b[j];
                    da[j] = na * wa[j]; db[j] = nb * wb[j];                                                 // g
                    dot += da[j] * a[j] + db[j] * b[j];
                }
                const float m = group_sum(dot, s.group) / (float)s.D;
#pragma unroll
                for (int j = 0; j < 8; ++j) { da[j] = r * (da[j] - a[j] * m); db[j] = r * (db[j] - b[j] * m); }
                if (live) { store8<T>(dst + h * g.hs, da); store8<T>(dst + h * g.hs + half, db); }
            }
        };
        side(q, gq, s.Hq, h0, min(h1, s.Hq), dwq);
        side(k, gk, s.Hk, max(h0 - s.Hq, 0), h1 - s.Hq, dwk);
    }
    // the workgroup's sums over its tokens and heads: part[workgroup][q | k][D]
    float* out = part + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 * s.D;
    auto reduce = [&](const float (&dw)[16], float* to) __attribute__((always_inline)) {
        __syncthreads();
        if (sub * 8 < half) {
#pragma unroll
            for (int j = 0; j < 8; ++j) { red[grp * s.D + sub * 8 + j] = dw[j]; red[grp * s.D + half + sub * 8 + j] = dw[8 + j]; }
        }
        __syncthreads();
        for (int d = threadIdx.x; d < s.D; d += 256) {
            float v = 0.f;
            for (int g = 0; g < groups; ++g) v += red[g * s.D + d];
            to[d] = v;
        }
    };
    reduce(dwq, out);
    reduce(dwk, out + s.D);
}

// dw[c] = sum over the workgroups' rows, in a fixed order, 64-bit sums; column c of part's 2 D.  32 columns and 32 threads down the rows
// per workgroup, four loads in flight each: the sums are latency, and with 4 threads down the rows this launch was a
// third of a training pass (19215 tokens, 4 + 4 heads of 128: 101 -> 67 us).
__global__ __launch_bounds__(1024) void rope_dw_kernel(const float* __restrict__ part, int rows, int D, float* __restrict__ dwq, float* __restrict__ dwk) {
    __shared__ double red[32][33];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5, c = blockIdx.x * 32 + x;
    double v = 0.0;
    const float* col = part + c;                                     // (2 D is a multiple of 32)
    int r = y;
    for (; r + 96 < rows; r += 128) {
        const float a0 = col[(int64_t)r * 2 * D], a1 = col[(int64_t)(r + 32) * 2 * D], a2 = col[(int64_t)(r + 64) * 2 * D], a3 = col[(int64_t)(r + 96) * 2 * D];
        v += (double)a0; v += (double)a1; v += (double)a2; v += (double)a3;
    }
    for (; r < rows; r += 32) v += (double)col[(int64_t)r * 2 * D];
    red[y][x] = v;
    __syncthreads();
    if (y == 0) {
        for (int k = 1; k < 32; ++k) v += red[k][x];
        if (c < D) dwq[c] = (float)v; else dwk[c - D] = (float)v;
    }
}

static bool aligned(const void* p, int64_t ts, int64_t hs, int es) {
    return p && (uintptr_t)p % 16 == 0 && (ts * es) % 16 == 0 && (hs * es) % 16 == 0;
}

static int rope_shape(const hsidm_rope_desc* d, RopeShape& s, int& es) {
    if (!d) return HSIDM_E_BADARG;
    if (d->prec != HSIDM_BF16 && d->prec != HSIDM_F16 && d->prec != HSIDM_F32X3) return HSIDM_E_BADARG;
    es = d->prec == HSIDM_F32X3 ? 4 : 2;
    if (d->T <= 0 || d->T > 0x7fffffff || d->Hq <= 0 || d->Hk <= 0 || d->Hq > 65535 || d->Hk > 65535 || d->D < 16 || d->D > 256 || d->D % 16) return HSIDM_E_BADARG;
    if (d->axes < 1 || d->axes > HSIDM_ROPE_AXES || !d->pos || !d->freq || !(d->eps >= 0.f)) return HSIDM_E_BADARG;
    if (!aligned(d->q, d->q_ts, d->q_hs, es) || !aligned(d->k, d->k_ts, d->k_hs, es) || !aligned(d->wq, 0, 0, 4) || !aligned(d->wk, 0, 0, 4)) return HSIDM_E_BADARG;
    s.T = d->T; s.Hq = d->Hq; s.Hk = d->Hk; s.D = d->D; s.axes = d->axes; s.eps = d->eps;
    s.P = 0;
    for (int a = 0; a < HSIDM_ROPE_AXES; ++a) {
        if (a < d->axes) {
            if (d->sections[a] < 0 || d->sections[a] > d->D / 2) return HSIDM_E_BADARG;
            s.P += d->sections[a];
        }
        s.bound[a] = a + 1 < d->axes ? s.P : 0x7fffffff;
    }
    if (s.P > s.D / 2) return HSIDM_E_BADARG;
    s.group = 1;
    while (s.group < s.D / 16) s.group *= 2;
    s.heads_per = s.Hq + s.Hk;
    return 0;
}

// With few tokens a token's heads go to several workgroups, which compute its angles again: until there are about two workgroups per CU.
static void split_heads(RopeShape& s, int64_t token_blocks) {
    const int heads = s.Hq + s.Hk;
    int64_t parts = 512 / (token_blocks > 0 ? token_blocks : 1);
    if (parts > heads) parts = heads;
    if (parts > 1) s.heads_per = (int)((heads + parts - 1) / parts);
}

constexpr int kBwdBlocks = 512;              // two workgroups per CU, each with one row of dw sums (1024: 67 instead of 64 us a training pass)

static void bwd_grid(RopeShape& s, int& gx, int& gy) {
    const int64_t tb = (s.T * s.group + 255) / 256;
    split_heads(s, tb);
    gy = (s.Hq + s.Hk + s.heads_per - 1) / s.heads_per;
    int64_t x = kBwdBlocks / gy > 0 ? kBwdBlocks / gy : 1;
    gx = (int)(tb < x ? tb : x);
}

}  // namespace hsidm

using namespace hsidm;

extern "C" int hsidm_qk_norm_rope(const hsidm_rope_desc* d, void* out_q, void* out_k, void* stream) {
    RopeShape s;
    int es;
    if (int rc = rope_shape(d, s, es)) return rc;
    if (!aligned(out_q, 0, 0, es) || !aligned(out_k, 0, 0, es)) return HSIDM_E_BADARG;
    const int64_t tb = (s.T * s.group + 255) / 256;
    split_heads(s, tb);
    const dim3 grid((unsigned)tb, (unsigned)((s.Hq + s.Hk + s.heads_per - 1) / s.heads_per));
    const RopeSide q = {d->q, d->q_ts, d->q_hs, d->wq}, k = {d->k, d->k_ts, d->k_hs, d->wk};
    hipStream_t st = (hipStream_t)stream;
#define ROPE_FWD(T) hipLaunchKernelGGL(HIP_KERNEL_NAME(qk_norm_rope_kernel<T>), grid, dim3(256), 0, st, s, q, k, d->pos, d->freq, (T*)out_q, (T*)out_k)
    if (d->prec == HSIDM_BF16) ROPE_FWD(bf16);
    else if (d->prec == HSIDM_F16) ROPE_FWD(f16);
    else ROPE_FWD(float);
#undef ROPE_FWD
    return (int)hipGetLastError();
}

extern "C" int64_t hsidm_qk_norm_rope_bwd_workspace_bytes(const hsidm_rope_desc* d) {
    RopeShape s;
    int es, gx, gy;
    if (int rc = rope_shape(d, s, es)) return rc;
    bwd_grid(s, gx, gy);
    return (int64_t)gx * gy * 2 * s.D * (int64_t)sizeof(float);
}

extern "C" int hsidm_qk_norm_rope_bwd(const hsidm_rope_desc* d, const void* d_out_q, const void* d_out_k, void* dq, int64_t dq_ts, int64_t dq_hs,
                                      void* dk, int64_t dk_ts, int64_t dk_hs, float* dwq, float* dwk, void* workspace, int64_t workspace_bytes,
                                      void* stream) {
    RopeShape s;
    int es, gx, gy;
    if (int rc = rope_shape(d, s, es)) return rc;
    if (!aligned(d_out_q, 0, 0, es) || !aligned(d_out_k, 0, 0, es) || !aligned(dq, dq_ts, dq_hs, es) || !aligned(dk, dk_ts, dk_hs, es)) return HSIDM_E_BADARG;
    if (!dwq || !dwk || !workspace) return HSIDM_E_BADARG;
    bwd_grid(s, gx, gy);
    if (workspace_bytes < (int64_t)gx * gy * 2 * s.D * (int64_t)sizeof(float)) return HSIDM_E_BADARG;
    const RopeSide q = {d->q, d->q_ts, d->q_hs, d->wq}, k = {d->k, d->k_ts, d->k_hs, d->wk};
    const RopeGradSide gq = {d_out_q, dq, dq_ts, dq_hs}, gk = {d_out_k, dk, dk_ts, dk_hs};
    hipStream_t st = (hipStream_t)stream;
#define ROPE_BWD(T) hipLaunchKernelGGL(HIP_KERNEL_NAME(qk_norm_rope_bwd_kernel<T>), dim3(gx, gy), dim3(256), 0, st, s, q, k, gq, gk, d->pos, d->freq, (float*)workspace)
    if (d->prec == HSIDM_BF16) ROPE_BWD(bf16);
    else if (d->prec == HSIDM_F16) ROPE_BWD(f16);
    else ROPE_BWD(float);
#undef ROPE_BWD
    hipLaunchKernelGGL(rope_dw_kernel, dim3(2 * s.D / 32), dim3(1024), 0, st, (const float*)workspace, gx * gy, s.D, dwq, dwk);
    return (int)hipGetLastError();
}
