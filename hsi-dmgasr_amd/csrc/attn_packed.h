// Attention over packed sequences: what the forward and backward kernels share.
//
// Every product runs on 32x32 matrix instructions with the SAME operand roles, for the 16-bit types and for fp32:
//   row operand     lane (r = lane % 32, h = lane / 32) holds row r of a tile, 16 bytes at a time: step t of a contraction over D takes
//                   its 16-byte piece 2t + h - one v_mfma_f32_32x32x16 (8 elements a lane) or four v_mfma_f32_32x32x2_f32 (4 elements);
//   score tile      lands with column = lane % 32 and rows 8*(j/4) + 4h + j%4 in register j;
//   column operand  (a tile's transpose, contracted over its 32 rows): the score tile's registers ARE the other operand if slot s of
//                   half h stands for row 8*(s/4) + 4h + s%4, so no probability is ever moved between lanes; the 16-bit types fetch
//                   the column operand with the transposing LDS read, fp32 reads it element by element (one register a row).
// Tiles live in LDS row by row (DP elements, D padded up), the 16-byte pieces of a row exchanged by an XOR with the row number, so that
// row reads (8 rows at one piece), transposing reads (4 rows x 32 bytes) and the fp32 column reads all spread over the banks; they are
// filled by loads that go to LDS directly.  Rows past a sequence's end re-read its last row and pieces past D the last one: what they
// hold is finite wherever the inputs are, and never counts (scores are masked, the register operand is zero there).
#pragma once
#include "common.h"
#include "../../include/hsidm.h"

namespace hsidm {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef s16x4 __attribute__((address_space(3))) * lds_s16x4_p;

// one sequence tile: rows [row0, row0 + tile) of the sequence of `len` tokens that begins at token `start`
struct AttnTile { int32_t start, len, row0, reserved; };

struct AttnTensor { const char* p; int64_t ts, hs; };      // base, token and head stride in BYTES

constexpr float kLog2e = 1.4426950408889634f;

// ---- 16 bytes of one operand row against 16 bytes of another: acc += A B over the elements they hold -------------------------
template <typename T> __device__ __forceinline__ void mma16(f32x16& acc, u32x4 a, u32x4 b) {
    typedef typename Elem<T>::x8 x8;
    acc = Elem<T>::mfma(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), acc);
}
template <> __device__ __forceinline__ void mma16<float>(f32x16& acc, u32x4 a, u32x4 b) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x[i], y[i], acc, 0, 0, 0);
}

// ---- LDS tiles ---------------------------------------------------------------------------------------------------------------
template <typename T, int DP> struct Row {
    static constexpr int BYTES = DP * (int)sizeof(T), PIECES = BYTES / 16, STEPS = PIECES / 2;
    static __device__ __forceinline__ int swz(int r) {
        if constexpr (PIECES >= 8) return ((r & 3) << 1) | ((r >> 2) & 1);
        else return (((r >> 1) & 1) << 1) | ((r >> 2) & 1);
    }
    // byte offset of a piece of a row
    static __device__ __forceinline__ int at(int row, int piece) { return row * BYTES + ((piece ^ swz(row)) << 4); }
};

// Requests rows [row0, row0 + ROWS) of a sequence (clamped to its last) into an LDS tile: every wave of the workgroup takes its share of
// 1 KB instructions.  base: the sequence's first row, this head.  Complete after wait_loads() and a barrier.  A lane's place among the
// rows is a 32-bit offset made once; what moves from tile to tile and from instruction to instruction is a scalar base, so that a whole
// tile costs the vector unit nothing (with 64-bit addresses per lane it was a quarter of its work at D = 64).
template <typename T, int DP, int ROWS, int NW> struct Stage {
    typedef Row<T, DP> R;
    static constexpr int PER_WAVE = ROWS * R::PIECES / 64 / NW, STEP = NW * 64 / R::PIECES;      // STEP: rows from one instruction to the next
    static constexpr int PAT = STEP % 8 == 0 ? 1 : 8 / STEP;         // instructions until the exchange of pieces repeats
    static_assert(ROWS * R::PIECES % (64 * NW) == 0 && (STEP % 8 == 0 || 8 % STEP == 0), "a tile is whole instructions of every wave");
    uint32_t off[PAT], ts;
    int r0;
    __device__ __forceinline__ Stage(int64_t token_stride, int pieces, int wave, int lane) : ts((uint32_t)token_stride) {
        const int idx = wave * 64 + lane;
        r0 = idx / R::PIECES;
#pragma unroll
        for (int x = 0; x < PAT; ++x) off[x] = (uint32_t)r0 * ts + (uint32_t)min((idx % R::PIECES) ^ R::swz(r0 + x * STEP), pieces - 1) * 16u;
    }
    __device__ __forceinline__ void operator()(const char* base, int row0, int len, char* tile, int wave) const {
        if (row0 + ROWS <= len) {
#pragma unroll
            for (int i = 0; i < PER_WAVE; ++i) load(base + (int64_t)(row0 + i * STEP) * ts, off[i % PAT], tile, wave, i);
        } else {
#pragma unroll
            for (int i = 0; i < PER_WAVE; ++i) {
                const int g = min(row0 + r0 + i * STEP, len - 1) - row0;             // (row0 < len: the tile has a row)
                load(base + (int64_t)row0 * ts, off[i % PAT] + (uint32_t)(g - r0) * ts, tile, wave, i);
            }
        }
    }
    static __device__ __forceinline__ void load(const char* base, uint32_t offset, char* tile, int wave, int i) {
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(base + offset),
                                         (__attribute__((address_space(3))) void*)(tile + (i * NW + wave) * 1024), 16, 0, 0);
    }
};
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// a row of a sequence in registers, as the row operand of every step: zero beyond D
template <typename T, int DP>
__device__ __forceinline__ void load_row(const char* row, int pieces, int h, u32x4 (&f)[Row<T, DP>::STEPS]) {
#pragma unroll
    for (int t = 0; t < Row<T, DP>::STEPS; ++t) {
        const int c = 2 * t + h;
        u32x4 v = {0u, 0u, 0u, 0u};
        if (c < pieces) v = *reinterpret_cast<const u32x4*>(row + c * 16);
        f[t] = v;
    }
}

// This lane's places in a tile.  The exchange by XOR reaches the low three bits of a piece's number, and neither 32 rows nor 8 pieces
// further on change it: a handful of offsets per lane serve every step, the rest is the instructions' immediate offset.
template <typename T, int DP> struct Places {
    typedef Row<T, DP> R;
    static constexpr int NR = R::STEPS < 4 ? R::STEPS : 4, NC = sizeof(T) == 2 ? (DP > 32 ? 2 : 1) : 4;
    int row[NR], col[NC];
    __device__ __forceinline__ Places(int lane) {
        const int lr = lane & 31, h = lane >> 5;
#pragma unroll
        for (int x = 0; x < NR; ++x) row[x] = R::at(lr, 2 * x + h);
        if constexpr (sizeof(T) == 2) {
            const int gi = lane & 15;
#pragma unroll
            for (int x = 0; x < NC; ++x) col[x] = R::at(4 * h + (gi >> 2), 4 * x + 2 * ((lane >> 4) & 1) + ((gi & 3) >> 1)) + 8 * (gi & 1);
        } else {
#pragma unroll
            for (int x = 0; x < NC; ++x) col[x] = R::at(4 * h + x, lr >> 2) + 4 * (lr & 3);
        }
    }
};

// scores of 32 tile rows (from rb on) against the row in registers: acc[row][lane's column] = sum_d tile[row][d] * f[d]
template <typename T, int DP>
__device__ __forceinline__ void row_product(f32x16& acc, const char* tile, int rb, const Places<T, DP>& at, const u32x4 (&f)[Row<T, DP>::STEPS]) {
    typedef Row<T, DP> R;
#pragma unroll
    for (int t = 0; t < R::STEPS; ++t) mma16<T>(acc, *reinterpret_cast<const u32x4*>(tile + at.row[t & 3] + (rb * R::BYTES + (t >> 2) * 128)), f[t]);
}

// a score tile as the operand that is contracted over its rows
template <typename T> struct ColFrag {
    typedef typename Elem<T>::x8 x8;
    x8 v[2];
    __device__ __forceinline__ void set(const f32x16& s) {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const auto p = cvt_pair_hw<T>(s[8 * kk + 2 * i], s[8 * kk + 2 * i + 1]);
                v[kk][2 * i] = p[0]; v[kk][2 * i + 1] = p[1];
            }
    }
};
template <> struct ColFrag<float> {
    f32x16 v;
    __device__ __forceinline__ void set(const f32x16& s) { v = s; }
};

// acc[d = 32 dt + row][lane's column] += sum over the 32 tile rows from rb on of tile[row][d] * p[row]
template <typename T, int DP>
__device__ __forceinline__ void col_product(f32x16& acc, const char* tile, int rb, int dt, const Places<T, DP>& at, const ColFrag<T>& p) {
    typedef Row<T, DP> R;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const char* q = tile + at.col[dt & 1] + ((rb + 16 * kk) * R::BYTES + (dt >> 1) * 128);
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_p)(q));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_p)(q + 8 * R::BYTES));
            const s16x8 a = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            acc = Elem<T>::mfma(__builtin_bit_cast(typename Elem<T>::x8, a), p.v[kk], acc);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const float a = *reinterpret_cast<const float*>(tile + at.col[j & 3] + ((rb + 8 * (j >> 2)) * R::BYTES + dt * 128));
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a, p.v[j], acc, 0, 0, 0);
        }
    }
}

__device__ __forceinline__ void zero16(f32x16& a) {
#pragma unroll
    for (int j = 0; j < 16; ++j) a[j] = 0.f;
}
// the larger of the two halves' values, in both (lane l and l + 32 hold the same column)
__device__ __forceinline__ float both_halves_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float both_halves_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Writes acc * f, rows d of one 32-wide tile of D, to out + d (this lane's row): four elements at a time, those beyond D left out
template <typename T>
__device__ __forceinline__ void store_column(T* out, const f32x16& acc, float f, int d0, int h, int D) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int d = d0 + 8 * g + 4 * h;
        if (d < D) {                                       // D is a multiple of 8 (16-bit) or 4 (fp32)
            typedef T vec __attribute__((ext_vector_type(4)));
            vec v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = (T)(acc[4 * g + i] * f);
            *reinterpret_cast<vec*>(out + d) = v;
        }
    }
}

// what rounding acc * f to the type left behind, rounded to the type itself
template <typename T>
__device__ __forceinline__ void store_residual(T* out, const f32x16& acc, float f, int d0, int h, int D) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int d = d0 + 8 * g + 4 * h;
        if (d < D) {
            typedef T vec __attribute__((ext_vector_type(4)));
            vec v;
#pragma unroll
            for (int i = 0; i < 4; ++i) { const float x = acc[4 * g + i] * f; v[i] = (T)(x - (float)(T)x); }
            *reinterpret_cast<vec*>(out + d) = v;
        }
    }
}

// Workgroup -> (tile, head): all heads of a tile follow each other (the tiles come heaviest first, and a late heavy one would leave
// the chip waiting), heads that share keys on one XCD (workgroups go to the eight XCDs in turn, each with an L2 of its own).
__device__ __forceinline__ void which_tile(int block, int heads, int& tile, int& head) {
    tile = block / heads;
    const int j = block - tile * heads;
    head = (heads & 7) == 0 ? (j & 7) * (heads >> 3) + (j >> 3) : j;
}

// ---- forward -------------------------------------------------------------------------------------------------------------------
struct AttnFwdArgs {
    AttnTensor q, k, v;
    void* out;                       // [T][Hq][D] of the type, or fp32 [splits][T][Hq][D]
    void* lo;                        // the rounding residual of out, like out; may be null (and is with splits: the join writes it)
    float* lse;                      // [Hq][T], or [splits][Hq][T]; may be null without splits
    const AttnTile* tiles;
    int64_t T;
    int Hq, Hk, D, causal, splits;
    float scale;
};

// How a probability is held ahead of its product with V: times 2^shift, the row's largest between 2^shift and 2^(shift + lazy).  bf16 and
// fp32 have the exponents for any row.  fp16 rounds what is below 2^-14 to steps of 2^-24: at scale one, keys at 2^-26 of the largest would
// vanish from the sum (a thousandth of a row of 65536 of them) and stay in the softmax's denominator.  Held between 2^11 and 2^15 (65504 is
// the largest fp16) half a step is 2^-36 of the largest: 2^25 keys lose less than the output's rounding.
template <typename T> struct ProbScale { static constexpr float shift = 0.f, lazy = 8.f, back = 1.f; };
template <> struct ProbScale<f16> { static constexpr float shift = 11.f, lazy = 4.f, back = 1.f / 2048.f; };

// O^T = V^T P^T with the softmax's running maximum and sum per column (= query = lane).  The maximum that scales the accumulators
// follows the true one lazily: only when some query's grew by more than 2^lazy (ProbScale) are they rescaled; sums are fp32 in any case.  NW waves of 32 queries each walk the key tiles together; two LDS buffers: a tile arrives while the one
// before it is multiplied.
// What it spends its time on: matrix products and the softmax between them, one after the other.  At D = 64 a tile has 680 cycles of vector
// work and 512 of the matrix pipe's; counted, the vector unit is active 58 % of the time and the matrix pipe 34 %, with 2.2 waves on a SIMD - the
// two hardly overlap, neither is full, and of the 182 us a pass takes, 127 would be those two in strict turn at 2.4 GHz (73 if they overlapped).
// fp16, 2 x 16384 tokens, one head of 64: 187 us, 735 TFLOP/s; bf16 causal, 20115 tokens in six sequences, 16 / 4 heads of 128: 502 ... 530 us,
// 880 ... 930 TFLOP/s of the pairs that count; fp32 (exact products, peak 157), 2 x 4096 tokens of 128: 154 us, 112 TFLOP/s.  D = 256, 8 x 2048
// tokens, 8 heads: bf16 297 us, fp16 311 (925 and 883 TFLOP/s); fp32, 2 x 4096, one head: 312, 110.  Head sizes between the widths of 32, 64, 128 and 256 do
// the products of the next one: 8 x 2048 tokens, 16 heads, bf16: D = 80 313 us, 96 322, 128 334 ... 350.
template <typename T, int DP, int NW>
__global__ __launch_bounds__(64 * NW, (Row<T, DP>::BYTES <= 512 ? 2 : 1)) void attn_fwd_kernel(AttnFwdArgs a) {
    typedef Row<T, DP> R;
    constexpr int BN = R::BYTES <= 256 ? 64 : 32, ND = DP / 32, TILE = BN * R::BYTES;
    // Where the accumulators reach into the second half of the register file (fp32, D > 128), a jump around work on them costs a move of every
    // one of them on either way: that kernel does masked tiles too and rescales every time.
    constexpr bool SKIP = R::BYTES <= 512;
    extern __shared__ __attribute__((aligned(16))) char lds[];       // [2][K tile, V tile]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 31, h = lane >> 5;
    int ti, head;
    which_tile(blockIdx.x, a.Hq, ti, head);
    const AttnTile tile = a.tiles[ti];
    const int len = tile.len, q0 = tile.row0 + wave * 32, kvh = head / (a.Hq / a.Hk), pieces = a.D * (int)sizeof(T) / 16;
    const char* kb = a.k.p + (int64_t)tile.start * a.k.ts + kvh * a.k.hs;
    const char* vb = a.v.p + (int64_t)tile.start * a.v.ts + kvh * a.v.hs;
    // this workgroup's key tiles
    const int kend = a.causal ? min(len, tile.row0 + 32 * NW) : len;
    const int nkt = (kend + BN - 1) / BN, per = (nkt + a.splits - 1) / a.splits;
    const int t0 = blockIdx.y * per, t1 = min(nkt, t0 + per);
    const int row = q0 + lr, rowc = min(row, len - 1);
    u32x4 qf[R::STEPS];
    load_row<T, DP>(a.q.p + (int64_t)(tile.start + rowc) * a.q.ts + head * a.q.hs, pieces, h, qf);
    f32x16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) zero16(o[d]);
    const Places<T, DP> at(lane);
    const float c = a.scale * kLog2e;
    float m = -INFINITY, l = 0.f;                                    // m: the scaling maximum in score units; l: this half's share of the sum
    const Stage<T, DP, BN, NW> kst(a.k.ts, pieces, wave, lane), vst(a.v.ts, pieces, wave, lane);
    auto stage = [&](int t, int buf) __attribute__((always_inline)) {
        kst(kb, t * BN, len, lds + buf * 2 * TILE, wave);
        vst(vb, t * BN, len, lds + buf * 2 * TILE + TILE, wave);
    };
    if (t0 < t1) stage(t0, 0);
    wait_loads();
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        const int buf = (t - t0) & 1, k0 = t * BN;
        if (t + 1 < t1) stage(t + 1, buf ^ 1);
        if (!SKIP || (q0 < len && (!a.causal || k0 <= q0 + 31))) {   // (uniform over the wave)
            const char* kt = lds + buf * 2 * TILE;
            const char* vt = kt + TILE;
            f32x16 s[BN / 32];
#pragma unroll
            for (int b = 0; b < BN / 32; ++b) { zero16(s[b]); row_product<T, DP>(s[b], kt, 32 * b, at, qf); }
            if (k0 + BN > len || (a.causal && k0 + BN - 1 > q0)) {
                const int last = a.causal ? min(len - 1, row) : len - 1;
#pragma unroll
                for (int b = 0; b < BN / 32; ++b)
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (k0 + 32 * b + 8 * (j >> 2) + 4 * h + (j & 3) > last) s[b][j] = -INFINITY;
            }
            float mt = s[0][0];
#pragma unroll
            for (int b = 0; b < BN / 32; ++b)
#pragma unroll
                for (int j = 0; j < 16; ++j) mt = fmaxf(mt, s[b][j]);
            mt = both_halves_max(mt);
            if (!SKIP || __any(!((mt - m) * c <= ProbScale<T>::lazy) && mt != -INFINITY)) {
                const float mn = fmaxf(m, mt), f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * c);
                m = mn;
                l *= f;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int j = 0; j < 16; ++j) o[d][j] *= f;
            }
            const float mc = (m == -INFINITY ? 0.f : m * c) - ProbScale<T>::shift;
            ColFrag<T> p[BN / 32];
#pragma unroll
            for (int b = 0; b < BN / 32; ++b) {
#pragma unroll
                for (int j = 0; j < 16; ++j) { s[b][j] = __builtin_amdgcn_exp2f(fmaf(s[b][j], c, -mc)); l += s[b][j]; }
                p[b].set(s[b]);
            }
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int b = 0; b < BN / 32; ++b) col_product<T, DP>(o[d], vt, 32 * b, d, at, p[b]);
        }
        wait_loads();
        __syncthreads();
    }
    if (row >= len) return;
    l = both_halves_sum(l);
    const float inv = l == 0.f ? 0.f : 1.0f / l;                     // (no key in this split's share)
    const int64_t token = (int64_t)tile.start + row;
    if (a.splits > 1) {
        float* out = reinterpret_cast<float*>(a.out) + ((blockIdx.y * a.T + token) * a.Hq + head) * a.D;
#pragma unroll
        for (int d = 0; d < ND; ++d) store_column<float>(out, o[d], inv, 32 * d, h, a.D);
    } else {
        T* out = reinterpret_cast<T*>(a.out) + (token * a.Hq + head) * a.D;
#pragma unroll
        for (int d = 0; d < ND; ++d) store_column<T>(out, o[d], inv, 32 * d, h, a.D);
        if (sizeof(T) == 2 && a.lo) {
            T* lo = reinterpret_cast<T*>(a.lo) + (token * a.Hq + head) * a.D;
#pragma unroll
            for (int d = 0; d < ND; ++d) store_residual<T>(lo, o[d], inv, 32 * d, h, a.D);
        }
    }
    if (a.lse && h == 0) a.lse[((int64_t)blockIdx.y * a.Hq + head) * a.T + token] = l == 0.f ? -INFINITY : m * a.scale + logf(l * ProbScale<T>::back);
}

// ---- backward ------------------------------------------------------------------------------------------------------------------
//   P = exp(S - lse), dP = dO V^T, delta = rowsum(dO o O), dS = P o (dP - delta):  dQ = scale dS K, dK = scale dS^T Q, dV = P^T dO
// Two kinds of workgroups recompute S and dP: one owns key tiles and walks the queries of every head that shares them (dK, dV: the sum over a group's
// heads stays in registers), one owns query tiles and walks the keys (dQ).  Nothing is added atomically: results do not depend on order.
// fp16: P and dS are stored to 11 bits with exponents down to 2^-14 only, and both shrink with the number of keys and the gradient's
// size.  P is kept times 2^10 and dS times a power of two chosen from |dO| and |V| (|dP - delta| <= 2 |dO| |V|): neither overflows, and
// underflow starts 2^10 and more lower.  dQ takes the power from its row's own |dO|; dK, a sum over rows, from the largest of the rows that see
// the tile's keys; |V| is the sequence's largest.  (One power for a whole call lost a long sequence beside a short one whose gradients are 2^18
// times as large.)  Only finite rows count: one with an infinity or a NaN has no finite gradient to scale.  bf16 has fp32's exponents and needs
// none of it.
struct AttnBwdArgs {
    AttnTensor q, k, v, dout, dq, dk, dv;
    const float *lse, *delta;        // [Hq][T]
    const float *top_do, *top_v;     // fp16, [Hk][T]: at a 64-row tile's first token, the largest |dO|^2 (over the group's heads) and |V|^2 of its rows
    float* part;                     // partial sums of split work: dQ [splits][T][Hq][D], or (dK | dV) [splits][2][T][Hk][D]
    const AttnTile* tiles;
    int64_t T;
    int Hq, Hk, D, causal, splits;
    float scale;
};

template <typename T> struct GradScale {
    static constexpr bool on = false;
    static constexpr float p_shift = 0.f, p_back = 1.f;          // P is kept times 2^p_shift
};
template <> struct GradScale<f16> {
    static constexpr bool on = true;
    static constexpr float p_shift = 10.f, p_back = 1.f / 1024.f;
};
__device__ __forceinline__ float finite_or_zero(float x) { return x < INFINITY ? x : 0.f; }      // (of a sum of squares: NaN compares false)

// the largest of a sequence's 64-row tiles from row `from` (a tile's first) on; the same in every lane
__device__ __forceinline__ float top_of_tiles(const float* top, int from, int len, int lane) {
    float m = 0.f;
    for (int64_t r = from + 64 * lane; r < len; r += 64 * 64) m = fmaxf(m, top[r]);
    return wave_max(m);
}
// The power of two that dS = P' (dP - delta), P' = 2^10 P, is multiplied by, from |dO|^2 and |V|^2.  Those are of finite fp16 rows, at most
// 256 * 65504^2 each, so that `top` is finite; it is zero only where dO or V is, and dS then is too.
__device__ __forceinline__ float grad_factor(float do2, float v2) {
    const float top = 2048.f * sqrtf(do2) * sqrtf(v2);           // |P' (dP - delta)|
    if (!(top > 0.f)) return 1.f;
    int e;
    frexpf(32768.f / top, &e);
    e = max(min(e - 1, 60), -60);
    return ldexpf(1.f, e);
}

template <typename T> __device__ __forceinline__ void store_grad(const AttnTensor& out, int64_t token, int head, const f32x16& acc, float f, int d0, int h, int D) {
    store_column<T>(reinterpret_cast<T*>(const_cast<char*>(out.p) + token * out.ts + head * out.hs), acc, f, d0, h, D);
}

// dK and dV of 32 keys per wave.  ND: 32-wide tiles of D that a workgroup accumulates (D > 128: half of them, the scores are computed
// once more by the workgroup of the other half - four full rows do not fit the registers)
template <typename T, int DP> struct KvTiles { static constexpr int ND = DP > 128 ? DP / 64 : DP / 32, PARTS = DP / 32 / ND; };

template <typename T, int DP, int NW>
__device__ __forceinline__ void attn_bwd_kv(const AttnBwdArgs& a, char* lds, int block, int share, int part) {
    typedef Row<T, DP> R;
    constexpr int BQ = R::BYTES <= 256 ? 64 : 32, ND = KvTiles<T, DP>::ND, TILE = BQ * R::BYTES, BUF = 2 * TILE + 512;
    // lds: [2][Q tile, dO tile, lse[64], delta[64]]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 31, h = lane >> 5;
    int ti, kvh;
    which_tile(block, a.Hk, ti, kvh);
    const AttnTile tile = a.tiles[ti];
    const int len = tile.len, k0 = tile.row0 + wave * 32, group = a.Hq / a.Hk, pieces = a.D * (int)sizeof(T) / 16;
    // this workgroup's work: the query tiles that see its keys, for every head of the group, one head behind the other
    const int tq0 = a.causal ? tile.row0 / BQ : 0, ntq = (len + BQ - 1) / BQ - tq0, work = ntq * group;
    const int per = (work + a.splits - 1) / a.splits, w0 = share * per, w1 = min(work, w0 + per);
    const int key = k0 + lr, keyc = min(key, len - 1);
    u32x4 kf[R::STEPS], vf[R::STEPS];
    load_row<T, DP>(a.k.p + (int64_t)(tile.start + keyc) * a.k.ts + kvh * a.k.hs, pieces, h, kf);
    load_row<T, DP>(a.v.p + (int64_t)(tile.start + keyc) * a.v.ts + kvh * a.v.hs, pieces, h, vf);
    const Places<T, DP> at(lane);
    const int dbytes = part * ND * 32 * (int)sizeof(T);        // this workgroup's part of D
    f32x16 dk[ND], dv[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) { zero16(dk[d]); zero16(dv[d]); }
    const float c = a.scale * kLog2e;
    float f = 1.f;
    if constexpr (GradScale<T>::on) {
        const int64_t first = kvh * a.T + tile.start;
        f = grad_factor(top_of_tiles(a.top_do + first, a.causal ? tile.row0 : 0, len, lane), top_of_tiles(a.top_v + first, 0, len, lane));
    }
    const Stage<T, DP, BQ, NW> qst(a.q.ts, pieces, wave, lane), gst(a.dout.ts, pieces, wave, lane);
    auto stage = [&](int w, int buf) __attribute__((always_inline)) {
        const int g = w / ntq, t = tq0 + w - g * ntq, head = kvh * group + g;
        char* b = lds + buf * BUF;
        qst(a.q.p + (int64_t)tile.start * a.q.ts + head * a.q.hs, t * BQ, len, b, wave);
        gst(a.dout.p + (int64_t)tile.start * a.dout.ts + head * a.dout.hs, t * BQ, len, b + TILE, wave);
        if (wave < 2) {                                              // 64 floats each; rows past the tile are not read back
            const float* src = (wave == 0 ? a.lse : a.delta) + head * a.T + tile.start + min(t * BQ + lane, len - 1);
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                             (__attribute__((address_space(3))) void*)(b + 2 * TILE + wave * 256), 4, 0, 0);
        }
    };
    if (w0 < w1) stage(w0, 0);
    wait_loads();
    __syncthreads();
    for (int w = w0; w < w1; ++w) {
        const int buf = (w - w0) & 1, q0 = (tq0 + w % ntq) * BQ;
        if (w + 1 < w1) stage(w + 1, buf ^ 1);
        const char* qt = lds + buf * BUF;
        const char* gt = qt + TILE;
        const float* rows = reinterpret_cast<const float*>(qt + 2 * TILE);
        // (no wave skips a tile: a jump around the products would have the accumulators change registers on either way)
#pragma unroll
        for (int b = 0; b < BQ / 32; ++b) {
            const char *qb = qt + b * 32 * R::BYTES, *gb = gt + b * 32 * R::BYTES;
            const float* rb = rows + 32 * b + 4 * h;
            f32x16 s, dp;
            zero16(s); zero16(dp);
            row_product<T, DP>(s, qb, 0, at, kf);
            row_product<T, DP>(dp, gb, 0, at, vf);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 l4 = *reinterpret_cast<const f32x4*>(rb + 8 * g);
                const f32x4 d4 = *reinterpret_cast<const f32x4*>(rb + 64 + 8 * g);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = 4 * g + i;
                    const float p = __builtin_amdgcn_exp2f(fmaf(s[j], c, GradScale<T>::p_shift - l4[i] * kLog2e));
                    float x = p * (dp[j] - d4[i]);
                    if constexpr (GradScale<T>::on) x *= f;
                    s[j] = p; dp[j] = x;
                }
            }
            const int qr = q0 + 32 * b;
            if (qr + 32 > len || (a.causal && qr < k0 + 31)) {       // (a pass of its own: selects, no branch per element)
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const int q = qr + 8 * (j >> 2) + 4 * h + (j & 3);
                    const bool gone = q >= len || (a.causal && q < key);
                    s[j] = gone ? 0.f : s[j];
                    dp[j] = gone ? 0.f : dp[j];
                }
            }
            ColFrag<T> pf, sf;
            pf.set(s); sf.set(dp);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                col_product<T, DP>(dv[d], gb + dbytes, 0, d, at, pf);
                col_product<T, DP>(dk[d], qb + dbytes, 0, d, at, sf);
            }
        }
        wait_loads();
        __syncthreads();
    }
    if (key >= len) return;
    const int64_t token = (int64_t)tile.start + key;
    const float fk = a.scale * GradScale<T>::p_back / f, fv = GradScale<T>::p_back;
    if (a.splits > 1) {
        float* out = a.part + (((int64_t)share * 2 * a.T + token) * a.Hk + kvh) * a.D;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            const int d0 = 32 * (part * ND + d);
            store_column<float>(out, dk[d], fk, d0, h, a.D);
            store_column<float>(out + a.T * a.Hk * a.D, dv[d], fv, d0, h, a.D);
        }
    } else {
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            const int d0 = 32 * (part * ND + d);
            store_grad<T>(a.dk, token, kvh, dk[d], fk, d0, h, a.D);
            store_grad<T>(a.dv, token, kvh, dv[d], fv, d0, h, a.D);
        }
    }
}

// dQ of 32 queries per wave
template <typename T, int DP, int NW>
__device__ __forceinline__ void attn_bwd_q(const AttnBwdArgs& a, char* lds, int block, int share) {
    typedef Row<T, DP> R;
    constexpr int BN = R::BYTES <= 256 ? 64 : 32, ND = DP / 32, TILE = BN * R::BYTES;
    constexpr bool SKIP = R::BYTES <= 256;                           // (as in the forward kernel)
    // lds: [2][K tile, V tile]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 31, h = lane >> 5;
    int ti, head;
    which_tile(block, a.Hq, ti, head);
    const AttnTile tile = a.tiles[ti];
    const int len = tile.len, q0 = tile.row0 + wave * 32, kvh = head / (a.Hq / a.Hk), pieces = a.D * (int)sizeof(T) / 16;
    const char* kb = a.k.p + (int64_t)tile.start * a.k.ts + kvh * a.k.hs;
    const char* vb = a.v.p + (int64_t)tile.start * a.v.ts + kvh * a.v.hs;
    const int kend = a.causal ? min(len, tile.row0 + 32 * NW) : len;
    const int nkt = (kend + BN - 1) / BN, per = (nkt + a.splits - 1) / a.splits;
    const int t0 = share * per, t1 = min(nkt, t0 + per);
    const int row = q0 + lr, rowc = min(row, len - 1);
    const int64_t rtok = (int64_t)tile.start + rowc;
    u32x4 qf[R::STEPS], gf[R::STEPS];
    load_row<T, DP>(a.q.p + rtok * a.q.ts + head * a.q.hs, pieces, h, qf);
    load_row<T, DP>(a.dout.p + rtok * a.dout.ts + head * a.dout.hs, pieces, h, gf);
    const float lse2 = a.lse[head * a.T + rtok] * kLog2e - GradScale<T>::p_shift, delta = a.delta[head * a.T + rtok];
    const Places<T, DP> at(lane);
    f32x16 dq[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) zero16(dq[d]);
    const float c = a.scale * kLog2e;
    float f = 1.f;
    if constexpr (GradScale<T>::on) {                                // (this lane's row)
        float sq = 0.f;
#pragma unroll
        for (int t = 0; t < R::STEPS; ++t) {
            const auto x = __builtin_bit_cast(typename Elem<T>::x8, gf[t]);
#pragma unroll
            for (int i = 0; i < 8; ++i) sq += (float)x[i] * (float)x[i];
        }
        f = grad_factor(finite_or_zero(both_halves_sum(sq)), top_of_tiles(a.top_v + kvh * a.T + tile.start, 0, len, lane));
    }
    const Stage<T, DP, BN, NW> kst(a.k.ts, pieces, wave, lane), vst(a.v.ts, pieces, wave, lane);
    auto stage = [&](int t, int buf) __attribute__((always_inline)) {
        kst(kb, t * BN, len, lds + buf * 2 * TILE, wave);
        vst(vb, t * BN, len, lds + buf * 2 * TILE + TILE, wave);
    };
    if (t0 < t1) stage(t0, 0);
    wait_loads();
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        const int buf = (t - t0) & 1, k0 = t * BN;
        if (t + 1 < t1) stage(t + 1, buf ^ 1);
        const char* kt = lds + buf * 2 * TILE;
        const char* vt = kt + TILE;
        if (!SKIP || q0 < len) {
            const int last = a.causal ? min(len - 1, row) : len - 1;
#pragma unroll
            for (int b = 0; b < BN / 32; ++b) {
                if (SKIP && (k0 + 32 * b >= len || (a.causal && k0 + 32 * b > q0 + 31))) continue;       // (uniform over the wave)
                f32x16 s, dp;
                zero16(s); zero16(dp);
                row_product<T, DP>(s, kt, 32 * b, at, qf);
                row_product<T, DP>(dp, vt, 32 * b, at, gf);
                const bool edge = k0 + 32 * b + 32 > len || (a.causal && k0 + 32 * b + 31 > q0);
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    float x = __builtin_amdgcn_exp2f(fmaf(s[j], c, -lse2)) * (dp[j] - delta);
                    if constexpr (GradScale<T>::on) x *= f;
                    s[j] = x;
                }
                if (edge) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) s[j] = k0 + 32 * b + 8 * (j >> 2) + 4 * h + (j & 3) > last ? 0.f : s[j];
                }
                ColFrag<T> sf;
                sf.set(s);
#pragma unroll
                for (int d = 0; d < ND; ++d) col_product<T, DP>(dq[d], kt, 32 * b, d, at, sf);
            }
        }
        wait_loads();
        __syncthreads();
    }
    if (row >= len) return;
    const float fq = a.scale * GradScale<T>::p_back / f;
    if (a.splits > 1) {
        float* out = a.part + (((int64_t)share * a.T + rtok) * a.Hq + head) * a.D;
#pragma unroll
        for (int d = 0; d < ND; ++d) store_column<float>(out, dq[d], fq, 32 * d, h, a.D);
    } else {
#pragma unroll
        for (int d = 0; d < ND; ++d) store_grad<T>(a.dq, rtok, head, dq[d], fq, 32 * d, h, a.D);
    }
}

// Both in one launch, the key tiles' workgroups first: neither depends on the other, and the query tiles fill what the key tiles leave
// free - a launch of its own would begin when the last of them ends (fp16 4 x 256 tokens, 8 heads of 64: 13 us instead of 25; bf16 causal,
// 10739 tokens in five sequences, 8 / 2 heads of 128: 304 us instead of 412).
// Bound by the matrix pipe together with the vector work and the LDS reads between its instructions (four products per pair of tiles read
// 32 KB a wave at D = 128, as long as they multiply).  8 x 2048 tokens, 16 heads, bf16: D = 128 1086 ... 1114 us, D = 64 529 ... 575 us - 875 and 870
// TFLOP/s of the seven products that run (two of them recompute S and dP); fp32, 2 x 4096 tokens of 128: 528 ... 540 us, 114 TFLOP/s.
// Registers: D = 128 in the 16-bit types spills 10 ... 20 of them (28 ... 52 bytes of scratch a lane), fp32 D = 64 two or three, fp32 D = 256 65 ... 106 (168
// ... 244 bytes); what that costs was not measured.  D = 256 recomputes the scores for either half of D and has one wave on a SIMD: 8 x 2048 tokens, 8
// heads, bf16 1703 us, fp16 1763 (at D = 128 and 16 heads, as many products: 1086 and 1179); fp32, 2 x 4096, one head: 1347, 2.5 times D = 128.
template <typename T, int DP, int NW>
__global__ __launch_bounds__(64 * NW, (Row<T, DP>::BYTES <= 256 ? 2 : 1)) void attn_bwd_kernel(AttnBwdArgs kv, AttnBwdArgs q, int kv_blocks, int q_blocks) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    int b = blockIdx.x;
    const int kv_all = kv_blocks * kv.splits * KvTiles<T, DP>::PARTS;
    if (b < kv_all) {
        const int rest = b / kv_blocks;
        attn_bwd_kv<T, DP, NW>(kv, lds, b - rest * kv_blocks, rest % kv.splits, rest / kv.splits);
    } else {
        b -= kv_all;
        attn_bwd_q<T, DP, NW>(q, lds, b % q_blocks, b / q_blocks);
    }
}

// ---- launches: one translation unit per element type (attn_packed_<type>.hip) ---------------------------------------------------
// kind: which kernel; waves: 2 or 4 per workgroup (a tile is 32 rows per wave)
enum { ATTN_FWD = 0, ATTN_BWD = 1 };
struct AttnBwdPair { AttnBwdArgs kv, q; };
template <typename T> int attn_launch(int kind, const void* args, int waves, int ntiles, hipStream_t s);
extern template int attn_launch<bf16>(int, const void*, int, int, hipStream_t);
extern template int attn_launch<f16>(int, const void*, int, int, hipStream_t);
extern template int attn_launch<float>(int, const void*, int, int, hipStream_t);

}  // namespace hsidm
