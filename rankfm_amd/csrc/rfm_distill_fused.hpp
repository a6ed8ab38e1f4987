// rfm_distill_fused.hpp -- the distillation loss and its gradients without the score matrix (included by rfm_distill.hip).
//
// fp32 products on the fp16 matrix cores.  Every fp32 factor is the sum of two fp16 parts, x = h + m: 11 bits of the significand each, rounded to
// nearest at each cut, so that 2^-24 of x is left over -- half a step of fp32.  Of the four products of two such sums m m' is left out, 2^-24 of
// |x x'| at most and 2^-27 in the mean: an fp32 product rounds away as much.  Three v_mfma_f32_32x32x16_f16 take 3 / 16 of the time of the
// fp32 matrix instructions (six with bf16 parts, which hold 8 bits: measured, 1.16 -> 0.66 ms for the k = 64 step of 8192 rows x 50 k items).
// fp16 has little range, so every tile of 32 rows is scaled by a power of two, its largest finite value to 2^14 .. 2^15: what is 2^-16 of that
// or more keeps its 22 bits, what is less an absolute error of 2^-40 of it.  The scales are taken back exactly where the sums are used.
//
// Fragments.  A 32 x 16 operand of that instruction is, for both sides, 8 consecutive k of row (lane & 31), k block (lane >> 5).  The tables are
// laid out once per call in exactly that order, [tile of 32 rows][k / 16][part][lane][8], so that a wavefront's operand is a contiguous
// kilobyte in memory and in LDS.  A second copy is transposed, for the products that sum over the rows: [tile][factor / 32][row / 16][part][lane][8],
// lane holding factor (lane & 31).  The accumulator of a 32 x 32 product holds, in lane l, column l & 31 and rows (r & 3) + 8 (r >> 2) + 4 (l >> 5)
// of register r: taken as the other operand of the second product its registers 8 t .. 8 t + 7 are k = 16 t + (j & 3) + 8 (j >> 2) + 4 (l >> 5).
// The sum over k does not care in which order the k's come as long as both sides agree, so the transposed copy is written in that order, and the
// weights go from one product to the next without leaving their lane.
//
//   forward_kernel   columns: 32 users per wavefront, fixed; streams item tiles through LDS.  z^T = items . users^T; a column's maximum and sum are
//                    in-lane; weighted sums O^T += items^T . exp2(z^T - max).
//   items_kernel     columns: 32 items per wavefront, fixed; streams user tiles.  z = users . items^T, dz from the row's lse, O^T += users^T . dz.
#pragma once

namespace rfm {
namespace distill {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kItemData = 64;                    // floats that travel with an item tile: 32 biases (log2 units), 2^-e, e, 2^e, for its scale 2^e
constexpr int kUserData = 64;                    // ... with each copy of a user tile: 32 lse (log2 units) and 2^-e; 32 coefficients, e and 2^e
constexpr int kFusedTeacher = 256;               // teacher entries of the fused path: a tile's 32 x n entries are sorted in LDS
constexpr float kLowest = -3.402823466e38f;
constexpr float kUnit = 7.0f;                    // a column's largest weight is 2^7 when its maximum is set, and at most 2^15 (fp16 ends at 2^16)
constexpr float kLimit = 15.0f;

template <int KP> struct Frag {
    static constexpr int steps = KP / 16, cols = KP / 32;
    static constexpr int bytes = KP * 128;       // one copy of a tile: KP / 16 x 2 parts x 1 KB; the transposed copy has as many
};

struct FusedArgs {
    rfm_distill_args a;
    int user_tiles, item_tiles, item_blocks;     // tiles of 32 rows; blocks of items_kernel's workgroups
    int splits, chunk;                           // of the streamed tiles
    char *user_frag, *user_frag_t, *item_frag, *item_frag_t;
    float *item_data, *user_data, *user_data_t;  // [item_tiles, kItemData], [user_tiles, kUserData] twice
    int32_t *mask_row;                           // [user_tiles * 32] mask of each row, -1 = none
    float *part_m, *part_l, *part_o;             // forward: [splits, user_tiles * 32 (, KP)]
    uint2 *entry;                                // [user_tiles, 32 n]: (item << 5 | row, p), ascending
    int32_t *entry_at;                           // [user_tiles, item_blocks + 1] where a block's entries begin
    float *part_items, *part_bias;               // items: [splits, item_tiles * 32 (, KP)]
};

__device__ __forceinline__ void split2(float x, _Float16 &h, _Float16 &m) {
    h = (_Float16)x;
    m = (_Float16)(x - (float)h);
}

// the exponent that brings a tile's largest value to 2^14 .. 2^15.  A tile of zeros or nearly so is scaled as if it held 2^-26: its weights then
// stay out of the way of the others' (the running maximum below is that of weight / scale).
__device__ __forceinline__ int tile_exponent(float largest) {
    const int e = 14 - (largest > 0.0f ? ilogbf(largest) : -1000);
    return min(max(e, -100), 40);
}
// largest of a value per thread; every thread gets it
__device__ __forceinline__ float block_max(float x, float *s_max) {
    x = wave_max(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = x;
    __syncthreads();
    return fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
}

// One workgroup per tile of 32 rows of a table: its fragments.  One copy holds row * `by`, the transposed one row * weight[row] (1 without), each with
// a scale of its own.  Rows without a usable teacher entry (live) count as zeros: they may be padding.
template <int KP>
__device__ void write_frags(const float *__restrict__ x, long long stride, int tile, long long rows, int factors, float by, const float *__restrict__ live,
                            const float *__restrict__ weight, float all_weight, char *frag, char *frag_t, float *lds, float *s_max, int *e_out, int *e_t_out) {
    constexpr int ld = KP + 1;
    float big = 0.0f, big_t = 0.0f;
    for (int e = threadIdx.x; e < 32 * KP; e += 256) {
        const int row = e / KP, k = e % KP;
        const long long r = (long long)tile * 32 + row;
        float v = 0.0f;
        if (r < rows && k < factors && (!live || live[r] > 0.0f)) {
            v = x[r * stride + k];
            const float a = fabsf(v * by), b = fabsf(v * (weight ? weight[r] * all_weight : all_weight));
            if (a < INFINITY) big = fmaxf(big, a);
            if (b < INFINITY) big_t = fmaxf(big_t, b);
        }
        lds[row * ld + k] = v;
    }
    const int ex = tile_exponent(block_max(big, s_max)), ex_t = tile_exponent(block_max(big_t, s_max));
    *e_out = ex;
    *e_t_out = ex_t;
    for (int e = threadIdx.x; e < KP * 4; e += 256) {            // 8 factors of a row each
        const int s = e >> 6, lane = e & 63;
        f16x8 h, m;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            _Float16 a, b;
            split2(ldexpf(lds[(lane & 31) * ld + 16 * s + 8 * (lane >> 5) + j] * by, ex), a, b);
            h[j] = a; m[j] = b;
        }
        f16x8 *out = reinterpret_cast<f16x8 *>(frag + (size_t)tile * Frag<KP>::bytes) + s * 128 + lane;
        out[0] = h; out[64] = m;
    }
    if (!frag_t) return;
    for (int e = threadIdx.x; e < KP * 4; e += 256) {            // 8 rows of a factor each
        const int ct = e >> 6, lane = e & 63, half = lane >> 5;
        f16x8 h, m;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int row = 16 * (ct & 1) + (j & 3) + 8 * (j >> 2) + 4 * half;
            const long long r = (long long)tile * 32 + row;
            const float v = lds[row * ld + 32 * (ct >> 1) + (lane & 31)], g = weight && r < rows ? weight[r] * all_weight : all_weight;
            _Float16 a, b;
            split2(v == 0.0f ? 0.0f : ldexpf(v * g, ex_t), a, b);
            h[j] = a; m[j] = b;
        }
        f16x8 *out = reinterpret_cast<f16x8 *>(frag_t + (size_t)tile * Frag<KP>::bytes) + ct * 128 + lane;
        out[0] = h; out[64] = m;
    }
}

template <int KP>
__global__ void __launch_bounds__(256) frags_kernel(const FusedArgs f, float c, const float *__restrict__ mass) {
    __shared__ float lds[32 * (KP + 1)], s_max[4];
    const rfm_distill_args &a = f.a;
    const bool grad = a.d_users != nullptr;
    const int b = blockIdx.x;
    int e, e_t;
    if (b < f.user_tiles) {
        write_frags<KP>(a.users, a.user_stride, b, a.n_rows, a.n_factors, c, mass, grad ? a.row_weight : nullptr, a.temperature, f.user_frag, grad ? f.user_frag_t : nullptr, lds, s_max, &e, &e_t);
        if (threadIdx.x == 0) {
            f.user_data[(size_t)b * kUserData + 32] = ldexpf(1.0f, -e);
            f.user_data_t[(size_t)b * kUserData + 32] = (float)e_t;
            f.user_data_t[(size_t)b * kUserData + 33] = ldexpf(1.0f, e_t);
        }
        if (threadIdx.x < 32 && a.allowed) {
            const long long r = (long long)b * 32 + threadIdx.x;
            long long m = -1;
            if (r < a.n_rows) m = a.allowed_rows ? (long long)a.allowed_rows[r] : (a.n_allowed == 1 ? 0 : r);
            f.mask_row[r] = m >= 0 && m < a.n_allowed ? (int32_t)m : -1;
        }
    } else {
        const int t = b - f.user_tiles;
        write_frags<KP>(a.items, a.item_stride, t, a.n_items, a.n_factors, 1.0f, nullptr, nullptr, 1.0f, f.item_frag, grad ? f.item_frag_t : nullptr, lds, s_max, &e, &e_t);
        float *data = f.item_data + (size_t)t * kItemData;
        if (threadIdx.x < 32) {
            const long long i = (long long)t * 32 + threadIdx.x;
            data[threadIdx.x] = i < a.n_items ? (a.bias ? a.bias[i] * c : 0.0f) : -INFINITY;
        }
        if (threadIdx.x == 32) { data[32] = ldexpf(1.0f, -e); data[33] = (float)e_t; data[34] = ldexpf(1.0f, e_t); }
    }
}

// ---- LDS staging: a kilobyte per instruction straight from memory (global_load_lds, 16 bytes per lane) --------------------------------------------
__device__ __forceinline__ void stage16(const char *from, char *to) {            // `to` is the wavefront's own kilobyte, `from` the lane's 16 bytes
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from, (__attribute__((address_space(3))) void *)to, 16, 0, 0);
}
__device__ __forceinline__ void stage4(const char *from, char *to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from, (__attribute__((address_space(3))) void *)to, 4, 0, 0);
}
// one copy of a tile, and the floats that go with it
template <int KP, int WAVES>
__device__ __forceinline__ void stage_copy(const char *frag, int tile, char *buf, int wave, int lane) {
    constexpr int bytes = Frag<KP>::bytes, kb = bytes / 1024;
    const char *src = frag + (size_t)tile * bytes + lane * 16;
#pragma unroll
    for (int q = 0; q < (kb + WAVES - 1) / WAVES; ++q) {
        const int k = q * WAVES + wave;
        if (kb % WAVES == 0 || k < kb) stage16(src + k * 1024, buf + k * 1024);
    }
}
__device__ __forceinline__ void stage_data(const float *data, char *buf, int wave, int lane) {
    if (wave == 0) stage4(reinterpret_cast<const char *>(data + lane), buf);
}
__device__ __forceinline__ void staged() {       // this wavefront's staging is in LDS
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

__device__ __forceinline__ f32x16 mfma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
// c + (ah + am) (bh + bm), the small products first
__device__ __forceinline__ f32x16 mfma3(const f16x8 *a, const f16x8 *b, f32x16 c) {
    c = mfma(a[1], b[0], c);
    c = mfma(a[0], b[1], c);
    return mfma(a[0], b[0], c);
}
// the two parts of the 16 weights.  x - h in one instruction (v_fma_mix_f32 takes a half of a packed pair as a factor); the compiler makes three
__device__ __forceinline__ void split_weights(const f32x16 &w, f16x8 (*p)[2]) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        u32x4 h, m;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float a = w[8 * t + 2 * j], b = w[8 * t + 2 * j + 1];
            const f16x2 pair = {(_Float16)a, (_Float16)b};
            h[j] = __builtin_bit_cast(unsigned, pair);
            float ra, rb;
            asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(ra) : "v"(h[j]), "v"(a));
            asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(rb) : "v"(h[j]), "v"(b));
            const f16x2 rest = {(_Float16)ra, (_Float16)rb};
            m[j] = __builtin_bit_cast(unsigned, rest);
        }
        p[t][0] = __builtin_bit_cast(f16x8, h);
        p[t][1] = __builtin_bit_cast(f16x8, m);
    }
}
// o[c] = o[c] * by + rows of the transposed tile . weights.  A tile's 32 terms are summed by themselves first: the running sum sees one
// operation per tile
template <int KP>
__device__ __forceinline__ void weighted_sum(const char *tile_t, int lane, const f16x8 (*p)[2], float by, f32x16 *o) {
#pragma unroll
    for (int c = 0; c < Frag<KP>::cols; ++c) {
        f32x16 sum = {0};
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const f16x8 *at = reinterpret_cast<const f16x8 *>(tile_t) + (c * 2 + t) * 128 + lane;
            const f16x8 a[2] = {at[0], at[64]};
            sum = mfma3(a, p[t], sum);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) o[c][r] = fmaf(o[c][r], by, sum[r]);
    }
}
template <int KP>
__device__ __forceinline__ f32x16 tile_scores(const char *tile, int lane, const f16x8 (*x)[2]) {
    f32x16 s = {0};
#pragma unroll
    for (int k = 0; k < Frag<KP>::steps; ++k) {
        const f16x8 *at = reinterpret_cast<const f16x8 *>(tile) + k * 128 + lane;
        const f16x8 a[2] = {at[0], at[64]};
        s = mfma3(a, x[k], s);
    }
    return s;
}
template <int KP>
__device__ __forceinline__ void load_columns(const char *frag, int tile, int lane, f16x8 (*x)[2]) {
    const f16x8 *src = reinterpret_cast<const f16x8 *>(frag + (size_t)tile * Frag<KP>::bytes) + lane;
#pragma unroll
    for (int k = 0; k < Frag<KP>::steps; ++k)
#pragma unroll
        for (int p = 0; p < 2; ++p) x[k][p] = src[k * 128 + p * 64];
}
__device__ __forceinline__ float largest16(const f32x16 &s) {
    float high = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) high = fmaxf(high, s[r]);
    return high;
}
__device__ __forceinline__ float sum16(const f32x16 &s) {
    float sum[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) sum[q] = (s[4 * q] + s[4 * q + 1]) + (s[4 * q + 2] + s[4 * q + 3]);
    return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// Both kernels keep a column's sums in units of 2^(top - 7): a weight 2^x of a tile of scale 2^e enters as 2^(x - e - top + 7), against the tile's
// values times 2^e.  `top` is moved only when that passes 2^15; it is the same in both halves of the wavefront, and a whole number, so that every scale
// is an exact power of two (a fractional one rounds differently where it is put in and where it is taken out: up to 7e-7 of a column).
//
// Block b: split b % splits of the items, columns block b / splits: with a multiple of 8 splits the workgroups of one XCD stream the same items.
// The loop is one tile deep in flight: while the vector unit turns tile t's scores into weights, the matrix cores make tile t + 1's.
template <int KP, bool GRAD, bool MASK, int WAVES>
__global__ void __launch_bounds__(WAVES * 64, 2) forward_kernel(const FusedArgs f) {
    constexpr int kBytes = Frag<KP>::bytes, kBuf = kBytes + kItemData * 4;
    __shared__ __attribute__((aligned(16))) char buf[2][kBuf], buf_t[GRAD ? 2 : 1][GRAD ? kBytes : 16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), half = lane >> 5;
    const int split = (int)blockIdx.x % f.splits, tile = (int)blockIdx.x / f.splits * WAVES + wave;
    const int mine = tile < f.user_tiles ? tile : f.user_tiles - 1;              // (a wavefront without users works on the last ones and writes nothing)
    const int t0 = split * f.chunk, t1 = min(t0 + f.chunk, f.item_tiles);
    f16x8 x[Frag<KP>::steps][2];
    load_columns<KP>(f.user_frag, mine, lane, x);
    const float unscale = f.user_data[(size_t)mine * kUserData + 32];
    const uint32_t *mask = nullptr;
    if constexpr (MASK) {
        const int m = f.mask_row[mine * 32 + (lane & 31)];
        if (m >= 0) mask = f.a.allowed + (size_t)m * (size_t)f.item_tiles;
    }
    float top = kLowest, total = 0.0f;
    f32x16 o[GRAD ? Frag<KP>::cols : 1];
    if constexpr (GRAD)
        for (int c = 0; c < Frag<KP>::cols; ++c) o[c] = f32x16{0};
    auto stage_scores = [&](int t) {
        stage_copy<KP, WAVES>(f.item_frag, t, buf[t & 1], wave, lane);
        stage_data(f.item_data + (size_t)t * kItemData, buf[t & 1] + kBytes, wave, lane);
    };
    unsigned word = 0xffffffffu, next_word = 0xffffffffu;
    auto finish = [&](int t, f32x16 &s, float &high, float &e, float &scale) {       // z of tile t (log2 units) out of its products, and the tile's scale
        const f32x4 *data = reinterpret_cast<const f32x4 *>(buf[t & 1] + kBytes);
        const f32x4 last = data[8];
        const float by = last[0] * unscale;
        e = last[1];
        scale = last[2];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x4 b = data[half + 2 * q];
#pragma unroll
            for (int k = 0; k < 4; ++k) s[4 * q + k] = fmaf(s[4 * q + k], by, b[k]);
        }
        if constexpr (MASK) {
            const unsigned w = word >> (4 * half);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = (w >> ((r & 3) + 8 * (r >> 2))) & 1u ? s[r] : -INFINITY;
        }
        high = largest16(s) - e;
    };
    if constexpr (MASK)
        if (mask) { word = mask[t0]; next_word = mask[min(t0 + 1, t1 - 1)]; }
    stage_scores(t0);
    if constexpr (GRAD) stage_copy<KP, WAVES>(f.item_frag_t, t0, buf_t[t0 & 1], wave, lane);
    staged();
    if (t0 + 1 < t1) stage_scores(t0 + 1);
    // one tile: its z is in `s`; that of the next one is left in `next`
    auto step = [&](int t, f32x16 &s, float high, float e, float scale, f32x16 &next, float &next_high, float &next_e, float &next_scale) {
        staged();                                                // tile t + 1's scores copy and tile t's other copy are in LDS; the buffers of before are free
        if (t + 1 < t1) {
            word = next_word;
            if constexpr (MASK)
                if (mask && t + 2 < t1) next_word = mask[t + 2];
            if (t + 2 < t1) stage_scores(t + 2);
            if constexpr (GRAD) stage_copy<KP, WAVES>(f.item_frag_t, t + 1, buf_t[(t + 1) & 1], wave, lane);
        }
        float by = 1.0f;
        if (__any(high > top + (kLimit - kUnit))) {
            const float to = fmaxf(top, ceilf(fmaxf(high, __shfl_xor(high, 32))));
            by = __builtin_amdgcn_exp2f(top - to);
            top = to;
        }
        const float off = top + (e - kUnit);
        next = tile_scores<KP>(buf[(t + 1) & 1], lane, x);       // (behind the last tile: of what is left in LDS, and not used)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(s[r] - off);
        total = fmaf(sum16(s), scale, total * by);
        if constexpr (GRAD) {
            f16x8 p[2][2];
            split_weights(s, p);
            weighted_sum<KP>(buf_t[t & 1], lane, p, by, o);
        }
        finish(t + 1, next, next_high, next_e, next_scale);
    };
    f32x16 s0 = tile_scores<KP>(buf[t0 & 1], lane, x), s1;
    float h0, h1, e0, e1, c0, c1;
    finish(t0, s0, h0, e0, c0);
    for (int t = t0; t < t1; t += 2) {
        step(t, s0, h0, e0, c0, s1, h1, e1, c1);
        if (t + 1 >= t1) break;
        step(t + 1, s1, h1, e1, c1, s0, h0, e0, c0);
    }
    if (tile >= f.user_tiles) return;
    total += __shfl_xor(total, 32);
    const size_t at = (size_t)split * f.user_tiles * 32 + (size_t)tile * 32 + (lane & 31);
    if (half == 0) { f.part_m[at] = top; f.part_l[at] = total; }
    if constexpr (GRAD) {
#pragma unroll
        for (int c = 0; c < Frag<KP>::cols; ++c)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 v = {o[c][4 * q], o[c][4 * q + 1], o[c][4 * q + 2], o[c][4 * q + 3]};
                *reinterpret_cast<f32x4 *>(f.part_o + at * KP + 32 * c + 8 * q + 4 * half) = v;
            }
    }
}

// One wavefront per row: the splits joined; loss, the users' gradient, and what items_kernel needs of the row.
template <int KP>
__global__ void __launch_bounds__(256) join_rows_kernel(const FusedArgs f, const float *__restrict__ part, const float *__restrict__ mass, const float *__restrict__ acc) {
    const int lane = threadIdx.x & 63;
    const long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6), padded = (long long)f.user_tiles * 32;
    if (r >= padded) return;
    const bool grad = f.a.d_users != nullptr;
    const size_t at = (size_t)(r >> 5) * kUserData + (r & 31);
    const float has = r < f.a.n_rows ? mass[r] : 0.0f;
    if (!(has > 0.0f)) {                                         // no row, nothing to learn from, or a mask that does not exist
        if (r < f.a.n_rows) {
            if (lane == 0) f.a.loss[r] = has;                    // (0 or NaN)
            if (grad)
                for (int k = lane; k < f.a.n_factors; k += 64) f.a.d_users[(size_t)r * f.a.n_factors + k] = 0.0f;
        }
        if (grad && lane == 0) { f.user_data[at] = INFINITY; f.user_data_t[at] = 0.0f; }
        return;
    }
    float top = kLowest;
    for (int s = lane; s < f.splits; s += 64) top = fmaxf(top, f.part_m[(size_t)s * padded + r]);
    top = wave_max(top);
    float total = 0.0f;
    for (int s = lane; s < f.splits; s += 64) total += f.part_l[(size_t)s * padded + r] * __builtin_amdgcn_exp2f(f.part_m[(size_t)s * padded + r] - top);
    total = wave_sum(total);
    const float lse2 = top - kUnit + log2f(total);
    if (lane == 0) f.a.loss[r] = f.a.temperature * f.a.temperature * (part[r] + lse2 * 0.693147180559945309f);
    if (!grad) return;
    const float coef = f.a.temperature * (f.a.row_weight ? f.a.row_weight[r] : 1.0f);
    if (lane == 0) { f.user_data[at] = lse2; f.user_data_t[at] = coef; }
    for (int k = lane; k < f.a.n_factors; k += 64) {
        float o = 0.0f;
        for (int s = 0; s < f.splits; ++s) o += f.part_o[((size_t)s * padded + r) * KP + k] * __builtin_amdgcn_exp2f(f.part_m[(size_t)s * padded + r] - top);
        f.a.d_users[(size_t)r * f.a.n_factors + k] = coef * (o / total - acc[(size_t)r * KP + k]);
    }
}

// One workgroup per tile of 32 rows: the tile's usable teacher entries by item (and row), an item that stands in a row's list more than once as one
// entry, and where each block of items_kernel begins in them.
__global__ void __launch_bounds__(256) sort_entries_kernel(long long rows, int n, int block_items, int blocks, int p2, const int32_t *__restrict__ item,
                                                           const float *__restrict__ p, uint2 *__restrict__ entry, int32_t *__restrict__ entry_at) {
    extern __shared__ unsigned long long s_key[];
    const long long r0 = (long long)blockIdx.x * 32;
    const int count = (int)min(32ll, rows - r0) * n;
    for (int e = threadIdx.x; e < p2; e += 256) {
        const int i = e < count ? item[r0 * n + e] : -1;
        s_key[e] = i >= 0 ? ((unsigned long long)(unsigned)i << 13) | (unsigned)(e / n) << 8 | (unsigned)(e % n) : ~0ull;
    }
    __syncthreads();
    for (int k = 2; k <= p2; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int t = threadIdx.x; t < p2 / 2; t += 256) {
                const int i = ((t & ~(j - 1)) << 1) | (t & (j - 1)), l = i + j;
                const unsigned long long a = s_key[i], b = s_key[l];
                if ((a > b) == ((i & k) == 0)) { s_key[i] = b; s_key[l] = a; }
            }
            __syncthreads();
        }
    uint2 *out = entry + (size_t)blockIdx.x * 32 * n;
    for (int e = threadIdx.x; e < 32 * n; e += 256) {
        const unsigned long long key = s_key[e];
        if (key == ~0ull) { out[e] = make_uint2(0xffffffffu, 0); continue; }
        auto value = [&](unsigned long long k) { return p[(r0 + ((k >> 8) & 31)) * n + (k & 255)]; };
        float v = 0.0f;
        if (e == 0 || (s_key[e - 1] >> 8) != (key >> 8)) {       // the first of its item and row takes the others
            v = value(key);
            for (int q = e + 1; q < 32 * n && (s_key[q] >> 8) == (key >> 8); ++q) v += value(s_key[q]);
            out[e] = make_uint2((unsigned)(key >> 8), __float_as_uint(v));
        } else out[e] = make_uint2(0xffffffffu, 0);
    }
    int32_t *at = entry_at + (size_t)blockIdx.x * (blocks + 1);
    for (int b = threadIdx.x; b <= blocks; b += 256) {
        const unsigned long long first = (unsigned long long)b * block_items << 13;
        int lo = 0, hi = 32 * n;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (s_key[mid] < first) lo = mid + 1; else hi = mid;
        }
        at[b] = lo;
    }
}

// The items' gradient.  p of the teacher enters through a 32 x 32 patch of LDS per wavefront: the few entries that fall into the tile are written
// there, read back as the lanes hold dz, and cleared; a wavefront's LDS operations run in order, so no barrier is needed.
constexpr int kPatch = 36;                       // floats per item of the patch: 32 rows, and 16-byte reads without bank conflicts
template <int KP, bool MASK, int WAVES>
__global__ void __launch_bounds__(WAVES * 64, 2) items_kernel(const FusedArgs f) {
    constexpr int kBytes = Frag<KP>::bytes, kBuf = kBytes + kUserData * 4;
    __shared__ __attribute__((aligned(16))) char buf[2][kBuf], buf_t[2][kBuf];
    __shared__ __attribute__((aligned(16))) float patches[WAVES][32 * kPatch];
    __shared__ __attribute__((aligned(16))) unsigned words[MASK ? WAVES : 1][32];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), half = lane >> 5, col = lane & 31;
    const int split = (int)blockIdx.x % f.splits, block = (int)blockIdx.x / f.splits, tile = block * WAVES + wave;
    const int mine = tile < f.item_tiles ? tile : f.item_tiles - 1;
    const int t0 = split * f.chunk, t1 = min(t0 + f.chunk, f.user_tiles), n32 = 32 * f.a.n_teacher;
    float *patch = patches[wave];
    for (int k = lane; k < 32 * kPatch; k += 64) patch[k] = 0.0f;
    f16x8 x[Frag<KP>::steps][2];
    load_columns<KP>(f.item_frag, mine, lane, x);
    const float bias = f.item_data[(size_t)mine * kItemData + col], unscale = f.item_data[(size_t)mine * kItemData + 32];
    const unsigned base = (unsigned)tile * 32u;
    f32x16 o[Frag<KP>::cols];
    for (int c = 0; c < Frag<KP>::cols; ++c) o[c] = f32x16{0};
    float top = kLowest, d_bias = 0.0f;
    auto mask_word = [&](int t) {                                // of row `col` of the tile, the bits of this wavefront's items
        const int m = f.mask_row[t * 32 + col];
        return m < 0 ? 0xffffffffu : f.a.allowed[(size_t)m * (size_t)f.item_tiles + mine];
    };
    auto stage_scores = [&](int t) {
        stage_copy<KP, WAVES>(f.user_frag, t, buf[t & 1], wave, lane);
        stage_data(f.user_data + (size_t)t * kUserData, buf[t & 1] + kBytes, wave, lane);
    };
    auto stage_rest = [&](int t) {
        stage_copy<KP, WAVES>(f.user_frag_t, t, buf_t[t & 1], wave, lane);
        stage_data(f.user_data_t + (size_t)t * kUserData, buf_t[t & 1] + kBytes, wave, lane);
    };
    unsigned word = 0, next_word = 0;
    auto finish = [&](int t, f32x16 &s, float &high) {           // log2 of q of tile t out of its products
        const f32x4 *data = reinterpret_cast<const f32x4 *>(buf[t & 1] + kBytes);
        const float by = data[8][0] * unscale;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x4 lse = data[half + 2 * q];
#pragma unroll
            for (int k = 0; k < 4; ++k) s[4 * q + k] = fmaf(s[4 * q + k], by, bias) - lse[k];
        }
        if constexpr (MASK) {
            if (half == 0) words[wave][col] = word;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const u32x4 w = reinterpret_cast<const u32x4 *>(words[wave])[2 * q + half];
#pragma unroll
                for (int k = 0; k < 4; ++k) s[4 * q + k] = (w[k] >> col) & 1u ? s[4 * q + k] : -INFINITY;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        high = largest16(s);
    };
    if constexpr (MASK) { word = mask_word(t0); next_word = mask_word(min(t0 + 1, t1 - 1)); }
    int begin = f.entry_at[(size_t)t0 * (f.item_blocks + 1) + block], end = f.entry_at[(size_t)t0 * (f.item_blocks + 1) + block + 1];
    stage_scores(t0);
    stage_rest(t0);
    staged();
    if (t0 + 1 < t1) stage_scores(t0 + 1);
    auto step = [&](int t, f32x16 &s, float high, f32x16 &next, float &next_high) {
        staged();
        const int from = begin, to = end;
        uint2 entry = make_uint2(0xffffffffu, 0);
        if (from + lane < to) entry = f.entry[(size_t)t * n32 + from + lane];
        if (t + 1 < t1) {
            begin = f.entry_at[(size_t)(t + 1) * (f.item_blocks + 1) + block];
            end = f.entry_at[(size_t)(t + 1) * (f.item_blocks + 1) + block + 1];
            if constexpr (MASK) {
                word = next_word;
                if (t + 2 < t1) next_word = mask_word(t + 2);
            }
            if (t + 2 < t1) stage_scores(t + 2);
            stage_rest(t + 1);
        }
        const f32x4 *data = reinterpret_cast<const f32x4 *>(buf_t[t & 1] + kBytes);
        const float e = data[8][0], scale = data[8][1];
        float by = 1.0f;
        high -= e;
        if (__any(high > top + (kLimit - kUnit))) {
            const float now = fmaxf(top, ceilf(fmaxf(high, __shfl_xor(high, 32))));
            by = __builtin_amdgcn_exp2f(top - now);
            top = now;
        }
        next = tile_scores<KP>(buf[(t + 1) & 1], lane, x);       // (behind the last tile: of what is left in LDS, and not used)
        {
            const float off = top + (e - kUnit);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(s[r] - off);
        }
        // the teacher's share
        bool any = false;
        for (int k = from; k < to; k += 64) {
            if (k > from) entry = k + lane < to ? f.entry[(size_t)t * n32 + k + lane] : make_uint2(0xffffffffu, 0);
            const unsigned at = (entry.x >> 5) - base;
            const bool hit = entry.x != 0xffffffffu && at < 32u;
            if (hit) patch[at * kPatch + (entry.x & 31)] = __uint_as_float(entry.y);
            any |= __any(hit);
        }
        if (any) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            f32x4 *cell = reinterpret_cast<f32x4 *>(patch + col * kPatch + 4 * half);
            f32x4 p[4];
            float most = 0.0f;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                p[q] = cell[2 * q];
                cell[2 * q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                most = fmaxf(fmaxf(most, fmaxf(p[q][0], p[q][1])), fmaxf(p[q][2], p[q][3]));
            }
            const float log_p = log2f(most) - e;                 // (-inf where there is none)
            if (__any(log_p > top + (kLimit - kUnit))) {
                const float now = fmaxf(top, ceilf(fmaxf(log_p, __shfl_xor(log_p, 32))));
                const float by_p = __builtin_amdgcn_exp2f(top - now);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] *= by_p;
                by *= by_p;
                top = now;
            }
            const float unit = __builtin_amdgcn_exp2f(kUnit - e - top);
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int k = 0; k < 4; ++k) s[4 * q + k] -= p[q][k] == 0.0f ? 0.0f : p[q][k] * unit;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x4 coef = data[half + 2 * q];
#pragma unroll
            for (int k = 0; k < 4; ++k) sum[k] = fmaf(s[4 * q + k], coef[k], sum[k]);
        }
        d_bias = fmaf((sum[0] + sum[1]) + (sum[2] + sum[3]), scale, d_bias * by);
        f16x8 p[2][2];
        split_weights(s, p);
        weighted_sum<KP>(buf_t[t & 1], lane, p, by, o);
        finish(t + 1, next, next_high);
    };
    f32x16 s0 = tile_scores<KP>(buf[t0 & 1], lane, x), s1;
    float h0, h1;
    finish(t0, s0, h0);
    for (int t = t0; t < t1; t += 2) {
        step(t, s0, h0, s1, h1);
        if (t + 1 >= t1) break;
        step(t + 1, s1, h1, s0, h0);
    }
    if (tile >= f.item_tiles) return;
    d_bias += __shfl_xor(d_bias, 32);
    const float unit = __builtin_amdgcn_exp2f(top - kUnit);
    const size_t at = (size_t)split * f.item_tiles * 32 + (size_t)tile * 32 + col;
    if (half == 0) f.part_bias[at] = d_bias * unit;
#pragma unroll
    for (int c = 0; c < Frag<KP>::cols; ++c)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x4 v = {o[c][4 * q], o[c][4 * q + 1], o[c][4 * q + 2], o[c][4 * q + 3]};
            *reinterpret_cast<f32x4 *>(f.part_items + at * KP + 32 * c + 8 * q + 4 * half) = v * unit;
        }
}

template <int KP>
__global__ void __launch_bounds__(256) join_items_kernel(const FusedArgs f) {
    const long long padded = (long long)f.item_tiles * 32, n = (long long)f.a.n_items * f.a.n_factors;
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < n; e += (long long)gridDim.x * 256) {
        const long long i = e / f.a.n_factors;
        const int k = (int)(e - i * f.a.n_factors);
        float s = 0.0f;
        for (int q = 0; q < f.splits; ++q) s += f.part_items[((size_t)q * padded + i) * KP + k];
        f.a.d_items[e] = s;
        if (k == 0 && f.a.d_bias) {
            float b = 0.0f;
            for (int q = 0; q < f.splits; ++q) b += f.part_bias[(size_t)q * padded + i];
            f.a.d_bias[i] = b;
        }
    }
}

__global__ void __launch_bounds__(256) zero_kernel(float *x, long long n) {
    for (long long k = (long long)blockIdx.x * 256 + threadIdx.x; k < n; k += (long long)gridDim.x * 256) x[k] = 0.0f;
}

}  // namespace distill
}  // namespace rfm
