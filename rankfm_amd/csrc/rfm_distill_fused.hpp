// rfm_distill_fused.hpp -- the distillation loss and its gradients without the score matrix (included by rfm_distill.hip).
//
// fp32 products on the fp16 matrix cores.  Every fp32 factor is the sum of two fp16 parts, x = h + m: 11 bits of the significand each, rounded to
// nearest at each cut.  The last of fp32's 24 bits is lost where m is large and the bit is set: 2^-23 of x at most, in a quarter of all values.  Of the
// four products of two such sums m m' is left out, 2^-22 of |x x'| at most and 2^-25 in the mean.  So a product is off by up to 2^-21 (2^-24.2 in the
// mean), where an fp32 product rounds away 2^-24 (2^-25.5): 8 times as much at worst, 2.4 times in the mean, and in a score as much as the additions of 8 terms
// may round away.  With the fourth product it would be 2^-22 still, and 2^-24.6 in the mean (loss of 8192 rows x 50 k items at k = 64: 179 -> 198 us, gradients
// 708 -> 823; 2048 x 200 k, k = 128: 1255 -> 1496).  Three v_mfma_f32_32x32x16_f16 take 3 / 16 of the time of the fp32 matrix instructions (six with
// bf16 parts, which hold 8 bits: gradients at k = 64 took 1164 us with those, 794 with these).
// fp16 has little range, so every tile of 32 rows is scaled by a power of two, its largest finite value to 2^14 .. 2^15: what is 2^-16 of that
// or more keeps its 22 bits, what is less an absolute error of 2^-40 of it (the scale is 2^40 at most: 2^-65 then).  The scales are taken back
// exactly where the sums are used.
//
// Fragments.  A 32 x 16 operand of that instruction is, for both sides, 8 consecutive k of row (lane & 31), k block (lane >> 5).  The tables are
// laid out once per call in exactly that order, [tile of 32 rows][k / 16][part][lane][8], so that a wavefront's operand is a contiguous
// kilobyte in memory and in LDS.  A second copy is transposed, for the products that sum over the rows: [tile][factor / 32][row / 16][part][lane][8],
// lane holding factor (lane & 31).  The accumulator of a 32 x 32 product holds, in lane l, column l & 31 and rows (r & 3) + 8 (r >> 2) + 4 (l >> 5)
// of register r: taken as the other operand of the second product its registers 8 t .. 8 t + 7 are k = 16 t + (j & 3) + 8 (j >> 2) + 4 (l >> 5).
// The sum over k does not care in which order the k's come as long as both sides agree, so the transposed copy is written in that order, and the
// weights go from one product to the next without leaving their lane.
//
//   forward_kernel   columns: 32 or 64 users per wavefront, fixed; streams item tiles through LDS.  z^T = items . users^T; a column's maximum and sum are
//                    in-lane; weighted sums O^T += 2^(high - top) items^T . exp2(z^T - high), `high` the tile's and `top` the column's.
//   thin_forward_kernel   the same for one or two tiles of users over a large table, which it takes as it is: no copies of the items.
//   items_kernel     columns: 32 or 64 items per wavefront, fixed; streams user tiles.  z = users . items^T, dz from the row's lse, O^T += users^T . dz.
//
// What bounds them: 8192 rows x 50 k items at k = 64, lists of 32, gradients: 0.71 ms in all, of which forward_kernel 323 us, items_kernel 420, prepare 24, the joins 14 and
// 11 (under a profiler, which adds a few percent).  2 x 6 x 8192 x 50 k x 64 x 2 operations are 0.63 TFLOP: 393 us at
// the 1.6 PFLOP/s that a loop of nothing but these instructions holds (its power sets its clock).  The matrix cores are busy in 53 % of the
// cycles of forward_kernel and 39 % of items_kernel; vector instructions issue in 53 % of both.  In copies: no LDS reads of the streamed tiles -18 .. -27 %,
// no teacher's entries -5 %, no test for a larger maximum -2 .. -4 %, no exponentials or a higher wave priority next to nothing.  The loss alone:
// 165 us.  2048 rows x 200 k items at k = 128: 1.27 ms, of which 549 + 706; 63 % and 46 %.
#pragma once

namespace rfm {
namespace distill {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kItemData = 64;                    // floats that travel with an item tile: 32 biases (log2 units), 2^-e, e, 2^e, for its scale 2^e
constexpr int kUserData = 64;                    // ... with a user tile: 32 lse (log2 units, whole), 2^-e of one copy, e and 2^e of the other; 32 row weights, 32 rests of the lse
constexpr int kBuckets = 1024;                   // of a tile's teacher entries, by block of items
constexpr float kLowest = -3.402823466e38f;
constexpr float kUnit = 15.0f;                   // a column's largest weight in a tile is 2^14 .. 2^15 (fp16 ends at 2^16)
constexpr float kSlack = 8.0f;                   // how far a tile may be above a column's running unit before that is moved
constexpr float kHead = 24.0f;                   // ... and how far above the tile it is moved

template <int KP> struct Frag {
    static constexpr int steps = KP / 16, cols = KP / 32;
    static constexpr int bytes = KP * 128;       // one copy of a tile: KP / 16 x 2 parts x 1 KB; the transposed copy has as many
    static constexpr int waves = KP <= 64 ? 4 : 8;               // wavefronts of a workgroup
};
// Wavefronts per SIMD that the registers are kept to.  Up to 64 factors a wavefront may have two tiles of 32 columns, NC = 2: what it reads of a streamed
// tile from LDS then serves both, at two wavefronts per SIMD instead of three and half as many workgroups (8192 rows x 50 k items at k = 64: 728 -> 689 us;
// at k = 128, where it would leave one wavefront per SIMD, 12 % slower).
template <int KP, int NC> constexpr int kPerSimd = KP <= 64 && NC == 1 ? 3 : 2;

struct FusedArgs {
    rfm_distill_args a;
    int user_tiles, item_tiles, item_blocks;     // tiles of 32 rows; blocks of items_kernel's workgroups
    int splits, chunk, lanes;                    // forward: how the item tiles are split; workgroups that a block of users is given (`splits`, or a few more)
    int units;                                   // items: (block, user tile) pairs per workgroup
    int few;                                     // user tiles, rounded up to a power of two, where they are few (thin_forward_kernel); else 0
    float c;                                     // log2 e / temperature
    char *user_frag, *user_frag_t, *item_frag, *item_frag_t;
    float *item_data, *user_data, *user_data_t;  // [item_tiles, kItemData], [user_tiles, kUserData] twice
    int32_t *mask_row;                           // [user_tiles * 32] mask of each row, -1 = none, -2 = a row that counts nowhere
    float *part_m, *part_l, *part_o;             // forward: [splits, user_tiles * 32 (, KP)]
    uint2 *entry;                                // [user_tiles, 32 n]: (item << 5 | row, p), by bucket
    int32_t *entry_at;                           // [user_tiles, kBuckets + 1] where a bucket's entries begin
    float *part_items, *part_bias;               // items: [workgroups + item_blocks, rows of a block (, KP)]
};

__device__ __forceinline__ void split2(float x, _Float16 &h, _Float16 &m) {
    h = (_Float16)x;
    m = (_Float16)(x - (float)h);
}

// the scales of two tiles taken back.  Where their largest values multiply beyond float32's range a score of them does, too, and one of 0 stays 0
__device__ __forceinline__ float unscaled(float a, float b) { return fminf(a * b, -kLowest); }

// the exponent that brings a tile's largest value to 2^14 .. 2^15.  A tile of zeros or nearly so is scaled as if it held 2^-26: its weights then
// stay out of the way of the others' (the running maximum below is that of weight / scale).
__device__ __forceinline__ int tile_exponent(float largest) {
    const int e = 14 - (largest > 0.0f ? ilogbf(largest) : -1000);
    return min(max(e, -113), 40);                                // (-113: float32 ends there)
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
// a scale of its own -- the transposed one that of the largest product, so a row of little weight is cut as one of small factors is.  Rows without a usable teacher entry (live [32]) count as zeros: they may be padding.  In the transposed copy, which the weights
// multiply, so does a factor that is not finite: where it counts the score and with it the row's sum is NaN already, where a mask has taken it out its
// weight is 0.
template <int KP>
__device__ void write_frags(const float *__restrict__ x, long long stride, int tile, long long rows, int factors, float by, const float *live,
                            const float *__restrict__ weight, char *frag, char *frag_t, float *lds, float *s_weight, float *s_max, int *e_out, int *e_t_out) {
    constexpr int ld = KP + 1;
    float big = 0.0f, big_t = 0.0f;
    if (threadIdx.x < 32) {
        const long long r = (long long)tile * 32 + threadIdx.x;
        s_weight[threadIdx.x] = weight && r < rows ? weight[r] : 1.0f;
    }
    Four v[KP / 32];                                             // all of a thread's loads first
#pragma unroll
    for (int q = 0; q < KP / 32; ++q) {
        const int e = q * 256 + (int)threadIdx.x, row = e / (KP / 4), k = e % (KP / 4) * 4;
        const long long r = (long long)tile * 32 + row;
        v[q] = Four{{0.0f, 0.0f, 0.0f, 0.0f}};
        if (r < rows && k < factors && (!live || live[row] > 0.0f)) v[q] = load_four(x + r * stride, k, factors);
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < KP / 32; ++q) {
        const int e = q * 256 + (int)threadIdx.x, row = e / (KP / 4), k = e % (KP / 4) * 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float a = fabsf(v[q].v[j] * by), b = fabsf(v[q].v[j] * s_weight[row]);
            if (a < INFINITY) big = fmaxf(big, a);
            if (b < INFINITY) big_t = fmaxf(big_t, b);
            lds[row * ld + k + j] = v[q].v[j];
        }
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
            const float v = lds[row * ld + 32 * (ct >> 1) + (lane & 31)], g = s_weight[row];
            _Float16 a, b;
            split2(v == 0.0f || !(fabsf(v) < INFINITY) ? 0.0f : ldexpf(v * g, ex_t), a, b);
            h[j] = a; m[j] = b;
        }
        f16x8 *out = reinterpret_cast<f16x8 *>(frag_t + (size_t)tile * Frag<KP>::bytes) + ct * 128 + lane;
        out[0] = h; out[64] = m;
    }
}

// One launch: the teacher's rows, four per workgroup (first: a row is a chain of loads, the tiles are bandwidth), the users' tiles and the items' tiles.
template <int KP, bool GRAD>
__global__ void __launch_bounds__(256) prepare_kernel(const FusedArgs f, float c, float *__restrict__ part, float *__restrict__ mass, int32_t *__restrict__ ids,
                                                      float *__restrict__ ps, float *__restrict__ acc) {
    extern __shared__ int s_dyn[];
    __shared__ float lds[32 * (KP + 1)], s_max[4], live[32], s_weight[32];
    const rfm_distill_args &a = f.a;
    const int teachers = (int)((a.n_rows + 3) / 4), b = (int)blockIdx.x - teachers;
    int e, e_t;
    if (b < 0) {
        teacher_row<GRAD, (KP + 63) / 64>(a, (long long)blockIdx.x * 4 + (threadIdx.x >> 6), KP, s_dyn, part, mass, ids, ps, acc);
    } else if (b < f.user_tiles) {
        // a row is live when its list has a usable entry (and its mask exists): 8 threads look through each
        {
            const int row = threadIdx.x >> 3, sub = threadIdx.x & 7;
            const long long r = (long long)b * 32 + row;
            bool some = false, bad = false;
            if (r < a.n_rows) {
                const uint32_t *mask = row_mask(a, r, &bad);
                for (int j = sub; j < a.n_teacher; j += 8) some |= usable(a, mask, a.teacher_items[(size_t)r * a.n_teacher + j], a.teacher_scores[(size_t)r * a.n_teacher + j]);
            }
            const unsigned long long any = __ballot(some && !bad);
            if (sub == 0) live[row] = (any >> ((threadIdx.x & 63) & ~7)) & 0xff ? 1.0f : 0.0f;
        }
        __syncthreads();
        write_frags<KP>(a.users, a.user_stride, b, a.n_rows, a.n_factors, c, live, GRAD ? a.row_weight : nullptr, f.user_frag, GRAD ? f.user_frag_t : nullptr, lds, s_weight, s_max, &e, &e_t);
        if (threadIdx.x == 0) {
            f.user_data[(size_t)b * kUserData + 32] = ldexpf(1.0f, -e);
            f.user_data[(size_t)b * kUserData + 33] = (float)e_t;
            f.user_data[(size_t)b * kUserData + 34] = ldexpf(1.0f, e_t);
        }
        if (threadIdx.x < 32 && a.allowed) {
            const long long r = (long long)b * 32 + threadIdx.x;
            long long m = -2;
            if (live[threadIdx.x] > 0.0f) m = max(a.allowed_rows ? (long long)a.allowed_rows[r] : (a.n_allowed == 1 ? 0 : r), -1ll);
            f.mask_row[r] = (int32_t)m;                          // (below n_allowed: the row would not be live)
        }
    } else {
        const int t = b - f.user_tiles;
        write_frags<KP>(a.items, a.item_stride, t, a.n_items, a.n_factors, 1.0f, nullptr, nullptr, f.item_frag, GRAD ? f.item_frag_t : nullptr, lds, s_weight, s_max, &e, &e_t);
        float *data = f.item_data + (size_t)t * kItemData;
        if (threadIdx.x < 32) {
            const long long i = (long long)t * 32 + threadIdx.x;
            data[threadIdx.x] = i < a.n_items ? (a.bias ? a.bias[i] * c : 0.0f) : -INFINITY;
        }
        if (threadIdx.x == 32) { data[32] = ldexpf(1.0f, -e); data[33] = (float)e_t; data[34] = ldexpf(1.0f, e_t); }
    }
}

// ---- LDS staging: a kilobyte per instruction straight from memory (global_load_lds, 16 bytes per lane).  Written out rather than by the builtin:
// the compiler holds every later LDS read of the step back until such loads have arrived (s_waitcnt vmcnt(0): it cannot tell the buffers apart), which
// is the latency they are meant to hide (the step of 2048 rows x 200 k items at k = 128: 1338 -> 1292 us).  Nothing but LDS is written by them; what
// waits for them is staged() below.  `to`: the wavefront's own place in LDS, `from`: the lane's own bytes.
__device__ __forceinline__ unsigned lds_offset(const void *p) { return (unsigned)(size_t)(const __attribute__((address_space(3))) char *)p; }
__device__ __forceinline__ void stage16(const char *from, char *to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(__builtin_amdgcn_readfirstlane(lds_offset(to))), "v"(from) : "memory", "m0");
}
__device__ __forceinline__ void stage4(const char *from, char *to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(__builtin_amdgcn_readfirstlane(lds_offset(to))), "v"(from) : "memory", "m0");
}
// One copy of a tile, and the floats that go with it.  Every wavefront issues the same number of instructions (some fetch what another fetches too):
// that number is what a wavefront may leave in flight when it waits for the group before.
template <int KP, int WAVES> constexpr int kCopyLoads = (Frag<KP>::bytes / 1024 + WAVES - 1) / WAVES;
template <int KP, int WAVES>
__device__ __forceinline__ void stage_copy(const char *frag, int tile, char *buf, int wave, int lane) {
    constexpr int bytes = Frag<KP>::bytes, kb = bytes / 1024;
    const char *src = frag + (size_t)tile * bytes + lane * 16;
#pragma unroll
    for (int q = 0; q < kCopyLoads<KP, WAVES>; ++q) {
        const int k = kb % WAVES == 0 ? q * WAVES + wave : min(q * WAVES + wave, kb - 1);
        stage16(src + k * 1024, buf + k * 1024);
    }
}
__device__ __forceinline__ void stage_data(const float *data, char *buf, int lane) { stage4(reinterpret_cast<const char *>(data + lane), buf); }
// all but the last LEFT loads of this wavefront have arrived, and everyone else's too
template <int LEFT>
__device__ __forceinline__ void staged() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LEFT) : "memory");       // (its reads of the buffer that is fetched into next are over, too)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

__device__ __forceinline__ f32x16 mfma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
// c + (ah + am) (bh + bm), the small products first; SWAP: those in the other order
template <bool SWAP = false>
__device__ __forceinline__ f32x16 mfma3(const f16x8 *a, const f16x8 *b, f32x16 c) {
    c = SWAP ? mfma(a[0], b[1], c) : mfma(a[1], b[0], c);
    c = SWAP ? mfma(a[1], b[0], c) : mfma(a[0], b[1], c);
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
// o[n][c] += unit[n] * rows of the transposed tile . weights of column tile n.  A tile's 32 terms are summed by themselves first: the running sum
// sees one operation per tile
template <int KP, int NC>
__device__ __forceinline__ void weighted_sum(const char *tile_t, int lane, const f16x8 (*p)[2][2], const float *unit, f32x16 (*o)[Frag<KP>::cols]) {
#pragma unroll
    for (int c = 0; c < Frag<KP>::cols; ++c) {
        f32x16 sum[NC];
#pragma unroll
        for (int n = 0; n < NC; ++n) sum[n] = f32x16{0};
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const f16x8 *at = reinterpret_cast<const f16x8 *>(tile_t) + (c * 2 + t) * 128 + lane;
            const f16x8 a[2] = {at[0], at[64]};
#pragma unroll
            for (int n = 0; n < NC; ++n) sum[n] = mfma3(a, p[n][t], sum[n]);
        }
#pragma unroll
        for (int n = 0; n < NC; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[n][c][r] = fmaf(sum[n][r], unit[n], o[n][c][r]);
    }
}
// SWAP: the columns are the items (the same sums in the same order as where they are the rows: a score has the same bits in both kernels, so that the largest
// share of a row is as exact as the row's sum, however large the scores are)
template <int KP, int NC, bool SWAP = false>
__device__ __forceinline__ void tile_scores(const char *tile, int lane, const f16x8 (*x)[Frag<KP>::steps][2], f32x16 *s) {
#pragma unroll
    for (int n = 0; n < NC; ++n) s[n] = f32x16{0};
#pragma unroll
    for (int k = 0; k < Frag<KP>::steps; ++k) {
        const f16x8 *at = reinterpret_cast<const f16x8 *>(tile) + k * 128 + lane;
        const f16x8 a[2] = {at[0], at[64]};
#pragma unroll
        for (int n = 0; n < NC; ++n) s[n] = mfma3<SWAP>(a, x[n][k], s[n]);
    }
}
template <int KP>
__device__ __forceinline__ void load_columns(const char *frag, int tile, int lane, f16x8 (*x)[2]) {
    const f16x8 *src = reinterpret_cast<const f16x8 *>(frag + (size_t)tile * Frag<KP>::bytes) + lane;
#pragma unroll
    for (int k = 0; k < Frag<KP>::steps; ++k)
#pragma unroll
        for (int p = 0; p < 2; ++p) x[k][p] = src[k * 128 + p * 64];
}
// s where bit (r & 3) + 8 (r >> 2) of w is set for register r, else -inf
__device__ __forceinline__ void mask16(f32x16 &s, unsigned w) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const unsigned keep = (unsigned)((int)(w << (31 - ((r & 3) + 8 * (r >> 2)))) >> 31);
        s[r] = __uint_as_float((keep & __float_as_uint(s[r])) | (~keep & 0xff800000u));
    }
}
// ... and where the mask of register r's row holds the bit of this lane's column: lane i holds the word of row i.  Two rows' words, one for each
// half of the wavefront, are a mask of lanes as they stand
__device__ __forceinline__ void mask16_rows(f32x16 &s, unsigned word) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int row = (r & 3) + 8 * (r >> 2);
        const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)word, row), hi = (unsigned)__builtin_amdgcn_readlane((int)word, row + 4);
        s[r] = __builtin_amdgcn_inverse_ballot_w64((unsigned long long)hi << 32 | lo) ? s[r] : -INFINITY;
    }
}
__device__ __forceinline__ float largest16(const f32x16 &s) {
    float high = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) high = fmaxf(high, s[r]);
    return high;
}
// the larger of a column's two halves, for both (v_permlane32_swap_b32 exchanges one's upper with the other's lower lanes)
__device__ __forceinline__ float both_halves(float x) {
    const auto pair = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(pair[0]), __uint_as_float(pair[1]));
}
__device__ __forceinline__ float sum16(const f32x16 &s) {
    float sum[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) sum[q] = (s[4 * q] + s[4 * q + 1]) + (s[4 * q + 2] + s[4 * q + 3]);
    return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// A weight 2^x is cut into its two parts as 2^(x - off), off = high - 15, `high` being the least whole number that none of its column's in the tile is above: the parts
// end at 2^-25, 2^-40 of the column's largest weight in the TILE.  (With one unit for all tiles, the column's largest so far, they ended at 2^-32 of that:
// of 200 k items 16 nats below the first the users' gradient lost 1.4e-3, at 20 nats a tenth, and an item on a teacher's list the shares of all other users
// below 2^-9 of its own.)  The running sums are in units of 2^top, top >= off - e - 8 for a tile whose values are scaled by 2^e: what a tile
// gives is multiplied by 2^(off - e - top) where it is added, and `top` moved only when that would pass 2^8 -- by 24 more than it has to be, so that a
// column is moved once and not at every larger tile (an item's first entry of a teacher's list is some 2^13 above its shares: gradients of 8192 rows x
// 50 k items at k = 64, 702 us without, 691 with).  All of these are the same in both halves of the wavefront, and whole numbers, so that every scale is
// an exact power of two (a fractional one rounds differently where it is put in and where it is taken out: up to 7e-7 of a column).
__device__ __forceinline__ float below(float high) {
    const float off = high - kUnit;
    return high - off > kUnit ? high - 7.0f : off;               // (beyond 2^24 a step of float32 is 2 and more: 2^16 would be infinite in fp16)
}
template <int COLS>
__device__ __forceinline__ float tile_unit(float off, float e, float &top, float &total, f32x16 (&o)[COLS]) {
    const float over = (off - top) - e;
    if (__any(over > kSlack)) {                                  // (top is kLowest at first)
        const float to = over > kSlack ? (off - e) + kHead : top, by = __builtin_amdgcn_exp2f(top - to);
        top = to;
        total *= by;
#pragma unroll
        for (int c = 0; c < COLS; ++c)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[c][r] *= by;
    }
    return __builtin_amdgcn_exp2f((off - top) - e);
}
// the weights of exponents s, and their sum
__device__ __forceinline__ float weigh(f32x16 &s, float off) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(s[r] - off);
    return sum16(s);
}
// Where nothing but their sum is wanted they are not cut, and the unit is the column's largest so far (50 k items, k = 64, 8192 rows: 174 us; 185 with a unit
// per tile)
__device__ __forceinline__ void add_weights(f32x16 &s, float &top, float &total) {
    const float high = largest16(s);
    if (__any(high > top + kSlack)) {
        const float to = fmaxf(top, ceilf(both_halves(high)));
        total *= __builtin_amdgcn_exp2f(top - to);
        top = to;
    }
    total += weigh(s, top);
}

// Workgroup b: split b % lanes of the items, columns block b / lanes.  Workgroups go round the XCDs: where `lanes` is a multiple of 8, those of one XCD stream
// the same items, out of its L2 (512 rows x 50 k items, k = 20, gradients: 75.1 us without, 72.8 with; 1503 x 35 k, 61 splits: 141.3 with 61 lanes, 139.3 with 64).
template <int KP, int NC, bool GRAD, bool MASK>
__global__ void __launch_bounds__(Frag<KP>::waves * 64, (GRAD ? kPerSimd<KP, NC> : NC == 1 ? 4 : 2)) forward_kernel(const FusedArgs f) {
    constexpr int WAVES = Frag<KP>::waves;
    constexpr int kBytes = Frag<KP>::bytes, kBuf = kBytes * (GRAD ? 2 : 1) + kItemData * 4, kGroup = kCopyLoads<KP, WAVES> * (GRAD ? 2 : 1) + 1;
    __shared__ __attribute__((aligned(16))) char buf[3][kBuf];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), half = lane >> 5, col = lane & 31;
    const int split = (int)blockIdx.x % f.lanes, tile = ((int)blockIdx.x / f.lanes * WAVES + wave) * NC;
    if (split >= f.splits) return;
    const int t0 = split * f.chunk, t1 = min(t0 + f.chunk, f.item_tiles);
    f16x8 x[NC][Frag<KP>::steps][2];
    float unscale[NC], top[NC], total[NC];
    const uint32_t *mask[NC];
    unsigned next_word[NC];
    f32x16 o[NC][GRAD ? Frag<KP>::cols : 1];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        const int mine = min(tile + n, f.user_tiles - 1);        // (where there are no users left, the last ones are worked on and nothing is written)
        load_columns<KP>(f.user_frag, mine, lane, x[n]);
        unscale[n] = f.user_data[(size_t)mine * kUserData + 32];
        top[n] = kLowest;
        total[n] = 0.0f;
        mask[n] = nullptr;
        next_word[n] = 0xffffffffu;
        if constexpr (MASK) {
            const int m = f.mask_row[mine * 32 + col];
            if (m >= 0) { mask[n] = f.a.allowed + (size_t)m * (size_t)f.item_tiles; next_word[n] = mask[n][t0]; }
        }
        if constexpr (GRAD)
            for (int c = 0; c < Frag<KP>::cols; ++c) o[n][c] = f32x16{0};
    }
    // Three buffers: what a step needs was asked for two steps before.  Behind the last tile the last one is fetched again, so that a group always has
    // the same number of loads.
    auto stage = [&](int t, int at) {
        const int from = min(t, t1 - 1);
        stage_copy<KP, WAVES>(f.item_frag, from, buf[at], wave, lane);
        if constexpr (GRAD) stage_copy<KP, WAVES>(f.item_frag_t, from, buf[at] + kBytes, wave, lane);
        stage_data(f.item_data + (size_t)from * kItemData, buf[at] + kBuf - kItemData * 4, lane);
    };
    stage(t0, 0);
    stage(t0 + 1, 1);
    for (int t = t0, i = 0; t < t1; ++t, i = i == 2 ? 0 : i + 1) {
        staged<kGroup>();                                        // tile t is in LDS, and nobody reads tile t - 1 any more
        unsigned word[NC];
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            word[n] = next_word[n];
            if constexpr (MASK) {
                asm volatile("" : "+v"(word[n]));                // (no instruction: it is here, and is taken before anything else is asked for)
                if (mask[n]) next_word[n] = mask[n][min(t + 1, t1 - 1)];
            }
        }
        stage(t + 2, i == 0 ? 2 : i - 1);
        if (tile >= f.user_tiles) continue;                      // (a wavefront without users only fetches)
        f32x16 s[NC];
        tile_scores<KP, NC>(buf[i], lane, x, s);
        const f32x4 *data = reinterpret_cast<const f32x4 *>(buf[i] + kBuf - kItemData * 4);
        const f32x4 last = data[8];
        const float e = last[1], scale = last[2];
        float by[NC];                                            // (the gradients' alone, as the two above)
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const float unit = unscaled(last[0], unscale[n]);
#pragma unroll
            for (int q = 0; q < 4; ++q) {                        // z in log2 units
                const f32x4 b = data[half + 2 * q];
#pragma unroll
                for (int k = 0; k < 4; ++k) s[n][4 * q + k] = fmaf(s[n][4 * q + k], unit, b[k]);
            }
            if constexpr (MASK) mask16(s[n], word[n] >> (4 * half));
            if constexpr (GRAD) {
                const float high = fmaxf(ceilf(both_halves(largest16(s[n]))), kLowest);      // (kLowest: nothing is allowed, all weights are 0)
                const float off = below(high);
                by[n] = tile_unit(off, e, top[n], total[n], o[n]);
                total[n] = fmaf(weigh(s[n], off), by[n] * scale, total[n]);
            } else add_weights(s[n], top[n], total[n]);
        }
        if constexpr (GRAD) {
            f16x8 p[NC][2][2];
#pragma unroll
            for (int n = 0; n < NC; ++n) split_weights(s[n], p[n]);
            weighted_sum<KP, NC>(buf[i] + kBytes, lane, p, by, o);
        }
    }
    staged<0>();                                                 // nothing is on its way into this workgroup's LDS when it ends
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        if (tile + n >= f.user_tiles) return;
        const float sum = total[n] + __shfl_xor(total[n], 32);
        const size_t at = (size_t)split * f.user_tiles * 32 + (size_t)(tile + n) * 32 + col;
        if (half == 0) { f.part_m[at] = top[n]; f.part_l[at] = sum; }
        if constexpr (GRAD) {
#pragma unroll
            for (int c = 0; c < Frag<KP>::cols; ++c)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f32x4 v = {o[n][c][4 * q], o[n][c][4 * q + 1], o[n][c][4 * q + 2], o[n][c][4 * q + 3]};
                    *reinterpret_cast<f32x4 *>(f.part_o + at * KP + 32 * c + 8 * q + 4 * half) = v;
                }
        }
    }
}

// ---- Few users -----------------------------------------------------------------------------------------------------------------------------
// With one or two tiles of users the items' two copies cost more than what is done with them: 4 x the table's bytes written and read again.  Here they
// are not made (29 rows x 150 k items at k = 60: preparation 21 -> 12 us, this pass 38 -> 19; 1.9 TB/s of the table: its rows are read 16 bytes a lane).  A wavefront takes a tile of 32 items from the table itself -- its rows are the lanes, 8 factors each per step, as the operand wants
// them -- cuts it into parts in its registers, and passes the parts through LDS (a word per factor: both parts) for the second product, where the lanes
// are the factors.  Nothing is shared and nobody waits; the wavefronts of a workgroup that have the same users join their sums at the end.
//
// A tile of a table, the lane's factors of its row in operand order; the exponent of its scale is returned.  odd: something in it is not finite.
template <int KP>
__device__ __forceinline__ int raw_tile(const float *__restrict__ table, long long stride, int tile, int rows, int factors, int lane, Four (*raw)[2], bool &odd) {
    const int half = lane >> 5, row = tile * 32 + (lane & 31);
    const float *from = table + (size_t)min(row, rows - 1) * stride;
#pragma unroll
    for (int s = 0; s < Frag<KP>::steps; ++s)
#pragma unroll
        for (int q = 0; q < 2; ++q) raw[s][q] = load_four(from, 16 * s + 8 * half + 4 * q, factors);
    if (tile * 32 + 32 > rows) {                                 // (the same for all)
#pragma unroll
        for (int s = 0; s < Frag<KP>::steps; ++s)
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int j = 0; j < 4; ++j) raw[s][q].v[j] = row < rows ? raw[s][q].v[j] : 0.0f;
    }
    unsigned most = 0;                                           // |x| orders like its bits; what is not finite lies above all that is
#pragma unroll
    for (int s = 0; s < Frag<KP>::steps; ++s)
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int j = 0; j < 4; ++j) most = max(most, __float_as_uint(raw[s][q].v[j]) & 0x7fffffffu);
    odd = __any(most >= 0x7f800000u);
    if (odd) {
        most = 0;
#pragma unroll
        for (int s = 0; s < Frag<KP>::steps; ++s)
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const unsigned b = __float_as_uint(raw[s][q].v[j]) & 0x7fffffffu;
                    most = b < 0x7f800000u ? max(most, b) : most;
                }
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) most = max(most, (unsigned)__shfl_xor((int)most, d));
    return tile_exponent(__uint_as_float(most));
}
// ... and one step of it as an operand, by = 2^e
__device__ __forceinline__ void raw_step(const Four *raw, float by, f16x8 *x) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        _Float16 h, m;
        split2(raw[j >> 2].v[j & 3] * by, h, m);
        x[0][j] = h; x[1][j] = m;
    }
}

constexpr int kThinWaves = 8;
template <int KP, bool GRAD> constexpr int kThinPerSimd = KP <= (GRAD ? 32 : 64) ? 4 : 2;
// Workgroup b: its wavefronts are f.few tiles of users times 8 / f.few tiles of items, which go round all workgroups.
template <int KP, bool GRAD, bool MASK>
__global__ void __launch_bounds__(kThinWaves * 64, (kThinPerSimd<KP, GRAD>)) thin_forward_kernel(const FusedArgs f) {
    constexpr int ld = KP + 4;
    __shared__ __attribute__((aligned(16))) unsigned words[GRAD ? kThinWaves : 1][GRAD ? 32 * ld : 4];
    __shared__ __attribute__((aligned(16))) float row_bias[kThinWaves][32];
    __shared__ float tops[kThinWaves][32], totals[kThinWaves][32];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), half = lane >> 5, col = lane & 31;
    const int user = wave & (f.few - 1), group = wave / f.few, groups = kThinWaves / f.few, mine = min(user, f.user_tiles - 1);
    f16x8 x[Frag<KP>::steps][2];
    load_columns<KP>(f.user_frag, mine, lane, x);
    const float unscale = f.user_data[(size_t)mine * kUserData + 32];
    const uint32_t *mask = nullptr;
    if constexpr (MASK) {
        const int m = f.mask_row[mine * 32 + col];
        if (m >= 0) mask = f.a.allowed + (size_t)m * (size_t)f.item_tiles;
    }
    float top = kLowest, total = 0.0f;
    f32x16 o[GRAD ? Frag<KP>::cols : 1];
    for (int c = 0; c < (GRAD ? Frag<KP>::cols : 1); ++c) o[c] = f32x16{0};
    const int last_tile = user < f.user_tiles ? f.item_tiles : 0;
    for (int tile = (int)blockIdx.x * groups + group; tile < last_tile; tile += (int)gridDim.x * groups) {
        const int item = tile * 32 + col;
        const float b_of = item < f.a.n_items ? (f.a.bias ? f.a.bias[item] * f.c : 0.0f) : -INFINITY;
        unsigned word = 0xffffffffu;
        if constexpr (MASK)
            if (mask) word = mask[tile];
        Four raw[Frag<KP>::steps][2];
        bool odd;
        const int e_tile = raw_tile<KP>(f.a.items, f.a.item_stride, tile, f.a.n_items, f.a.n_factors, lane, raw, odd);
        const float e = (float)e_tile, unit = unscaled(unscale, ldexpf(1.0f, -e_tile)), scale = ldexpf(1.0f, e_tile);
        if (half == 0) row_bias[wave][col] = b_of;
        f32x16 s = f32x16{0};
#pragma unroll
        for (int k = 0; k < Frag<KP>::steps; ++k) {
            f16x8 a[2];
            raw_step(raw[k], scale, a);
            s = mfma3(a, x[k], s);
            if constexpr (GRAD) {
                const u32x4 h = __builtin_bit_cast(u32x4, a[0]), m = __builtin_bit_cast(u32x4, a[1]);
                u32x4 w[2];
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j >> 2][j & 3] = __builtin_amdgcn_perm(m[j >> 1], h[j >> 1], j & 1 ? 0x07060302u : 0x05040100u);
                if (odd) {                                       // (a part h that is not finite is one whose factor is not)
#pragma unroll
                    for (int j = 0; j < 8; ++j) w[j >> 2][j & 3] = (w[j >> 2][j & 3] & 0x7c00u) == 0x7c00u ? 0u : w[j >> 2][j & 3];
                }
                u32x4 *to = reinterpret_cast<u32x4 *>(words[wave] + col * ld + 16 * k + 8 * half);
                to[0] = w[0];
                to[1] = w[1];
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const f32x4 *data = reinterpret_cast<const f32x4 *>(row_bias[wave]);
#pragma unroll
        for (int q = 0; q < 4; ++q) {                            // z in log2 units
            const f32x4 b = data[half + 2 * q];
#pragma unroll
            for (int k = 0; k < 4; ++k) s[4 * q + k] = fmaf(s[4 * q + k], unit, b[k]);
        }
        if constexpr (MASK) mask16(s, word >> (4 * half));
        float by = 1.0f;
        if constexpr (GRAD) {
            const float off = below(fmaxf(ceilf(both_halves(largest16(s))), kLowest));
            by = tile_unit(off, e, top, total, o);
            total = fmaf(weigh(s, off), by * scale, total);
        } else add_weights(s, top, total);
        if constexpr (GRAD) {
            f16x8 p[2][2];
            split_weights(s, p);
#pragma unroll
            for (int c = 0; c < Frag<KP>::cols; ++c) {
                f32x16 sum = f32x16{0};
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    u32x4 h, m;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {                // rows 2 j and 2 j + 1 of this lane's eight
                        const int r = 16 * t + ((2 * j) & 3) + 8 * (j >> 1) + 4 * half;
                        const unsigned w0 = words[wave][r * ld + 32 * c + col], w1 = words[wave][(r + 1) * ld + 32 * c + col];
                        h[j] = __builtin_amdgcn_perm(w1, w0, 0x05040100u);
                        m[j] = __builtin_amdgcn_perm(w1, w0, 0x07060302u);
                    }
                    const f16x8 parts[2] = {__builtin_bit_cast(f16x8, h), __builtin_bit_cast(f16x8, m)};
                    sum = mfma3(parts, p[t], sum);
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) o[c][r] = fmaf(sum[r], by, o[c][r]);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    // the wavefronts of the same users, in their order
    const float sum = total + __shfl_xor(total, 32);
    if (half == 0) { tops[wave][col] = top; totals[wave][col] = sum; }
    __syncthreads();
    float highest = kLowest;
    for (int g = 0; g < groups; ++g) highest = fmaxf(highest, tops[g * f.few + user][col]);
    const float part = __builtin_amdgcn_exp2f(top - highest);
    const size_t at = (size_t)blockIdx.x * f.user_tiles * 32 + (size_t)user * 32 + col;
    if (group == 0 && half == 0 && user < f.user_tiles) {
        float all = 0.0f;
        for (int g = 0; g < groups; ++g) all = fmaf(totals[g * f.few + user][col], __builtin_amdgcn_exp2f(tops[g * f.few + user][col] - highest), all);
        f.part_m[at] = highest;
        f.part_l[at] = all;
    }
    if constexpr (GRAD) {
        float *joined = reinterpret_cast<float *>(words[user]);  // (nobody needs the words any more)
        for (int g = 0; g < groups; ++g) {
            if (g == group && user < f.user_tiles) {
#pragma unroll
                for (int c = 0; c < Frag<KP>::cols; ++c)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        f32x4 *cell = reinterpret_cast<f32x4 *>(joined + col * ld + 32 * c + 8 * q + 4 * half);
                        f32x4 v = f32x4{o[c][4 * q], o[c][4 * q + 1], o[c][4 * q + 2], o[c][4 * q + 3]} * part;
                        if (g > 0) v += *cell;
                        if (g < groups - 1) *cell = v;
                        else *reinterpret_cast<f32x4 *>(f.part_o + at * KP + 32 * c + 8 * q + 4 * half) = v;
                    }
            }
            __syncthreads();
        }
    }
}

// The splits of a row joined: loss, the users' gradient, and what items_kernel needs of the row.  W: wavefronts per row, this one the `share`-th (more than
// one where rows are few and splits are many: 29 rows, 256 splits, k = 96: 16.9 us by one, 8.5 by eight).  weight: 64 floats of LDS, sums: W x (KP + 1)
template <int KP, int W>
__device__ void join_row(const FusedArgs &f, long long r, int share, const float *__restrict__ part, const float *__restrict__ mass, const float *__restrict__ acc, float *weight,
                         float *sums) {
    const int lane = threadIdx.x & 63;
    const long long padded = (long long)f.user_tiles * 32;
    const bool grad = f.a.d_users != nullptr;
    const size_t at = (size_t)(r >> 5) * kUserData + (r & 31);
    const float has = r < f.a.n_rows ? mass[r] : 0.0f;
    if (!(has > 0.0f)) {                                         // no row, nothing to learn from, or a mask that does not exist (the same for the W)
        if (share > 0) return;
        if (r < f.a.n_rows) {
            if (lane == 0) f.a.loss[r] = has;                    // (0 or NaN)
            if (grad)
                for (int k = lane; k < f.a.n_factors; k += 64) f.a.d_users[(size_t)r * f.a.n_factors + k] = 0.0f;
        }
        if (grad && lane == 0) { f.user_data[at] = INFINITY; f.user_data_t[at] = 0.0f; f.user_data_t[at + 32] = 0.0f; }
        return;
    }
    float top = kLowest;
    for (int s = lane; s < f.splits; s += 64) top = fmaxf(top, f.part_m[(size_t)s * padded + r]);
    top = wave_max(top);
    // KP / 4 lanes take four factors each of one split, the lanes behind them of the next ones
    constexpr int at_once = 64 / (KP / 4);
    const int mine = lane / (KP / 4), k4 = lane % (KP / 4) * 4;
    float total = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = share * 64; s0 < f.splits; s0 += 64 * W) {
        const int s = s0 + lane;
        const float w = s < f.splits ? __builtin_amdgcn_exp2f(f.part_m[(size_t)s * padded + r] - top) : 0.0f;
        if (s < f.splits) total += f.part_l[(size_t)s * padded + r] * w;
        if (!grad) continue;
        weight[lane] = w;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const int count = min(64, f.splits - s0);
        const float *from = f.part_o + ((size_t)s0 * padded + r) * KP + k4;
        if (mine < at_once) {
            constexpr int ahead = 8;                             // loads in flight: they are far apart
            for (int q0 = mine; q0 < count; q0 += ahead * at_once) {
                f32x4 x[ahead];
#pragma unroll
                for (int h = 0; h < ahead; ++h) x[h] = *reinterpret_cast<const f32x4 *>(from + (size_t)min(q0 + h * at_once, count - 1) * padded * KP);
#pragma unroll
                for (int h = 0; h < ahead; ++h) {
                    const int q = q0 + h * at_once;
                    const float by = q < count ? weight[q] : 0.0f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[j] = q < count ? fmaf(x[h][j], by, o[j]) : o[j];
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    total = wave_sum(total);
    if (grad) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float sum = o[j];
            for (int d = 1; d < at_once; ++d) sum += __shfl(o[j], lane + d * (KP / 4));
            o[j] = sum;                                          // (of the first KP / 4 lanes)
        }
    }
    if constexpr (W > 1) {
        float *own = sums + share * (KP + 1);
        if (grad && mine == 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j) own[k4 + j] = o[j];
        }
        if (lane == 0) own[KP] = total;
        __syncthreads();                                         // (all W are here: a row is theirs alone)
        if (share > 0) return;
        for (int v = 1; v < W; ++v) {
            const float *other = sums + v * (KP + 1);
            total += other[KP];
            if (grad && mine == 0) {
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] += other[k4 + j];
            }
        }
    }
    // lse (log2 units) as a whole number and a rest, neither of which loses what the other is rounded to
    const int power = total > 0.0f && total < INFINITY ? ilogbf(total) : 0;
    const float lse2 = top + (float)power, rest = log2f(ldexpf(total, -power)) + ((top - lse2) + (float)power);
    if (lane == 0) f.a.loss[r] = f.a.temperature * (f.a.temperature * (part[r] + (lse2 + rest) * 0.693147180559945309f));
    if (!grad) return;
    const float weight_of = f.a.row_weight ? f.a.row_weight[r] : 1.0f, coef = f.a.temperature * weight_of;
    if (lane == 0) { f.user_data[at] = lse2; f.user_data_t[at] = weight_of; f.user_data_t[at + 32] = rest; }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int k = k4 + j;
        if (mine == 0 && k < f.a.n_factors) f.a.d_users[(size_t)r * f.a.n_factors + k] = coef * (o[j] / total - acc[(size_t)r * KP + k]);
    }
}

// One workgroup per tile of 32 rows: the tile's teacher entries by the block of items_kernel that they fall into, modulo kBuckets (a block skips what
// is not its own).  Their order inside a bucket is whatever it comes to: no two of them are the same item of the same row, and all that is done
// with them is to be written to that place.  count: kBuckets + 8 ints of LDS.
__device__ void bucket_entries(const FusedArgs &f, int tile, int block_items, const int32_t *__restrict__ item, const float *__restrict__ p, int *count) {
    const int n = f.a.n_teacher, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long r0 = (long long)tile * 32;
    const int entries = (int)min(32ll, f.a.n_rows - r0) * n;
    static_assert(kBuckets == 1024, "two counters per thread of 512");
    count[threadIdx.x] = 0;
    count[threadIdx.x + 512] = 0;
    __syncthreads();
    for (int e = threadIdx.x; e < entries; e += 512) {
        const int i = item[r0 * n + e];
        if (i >= 0) atomicAdd(count + (i / block_items) % kBuckets, 1);
    }
    __syncthreads();
    const int c0 = count[2 * threadIdx.x], c1 = count[2 * threadIdx.x + 1];
    int before = c0 + c1;                                        // inclusive prefix over the wavefront, then over the wavefronts
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(before, d);
        if (lane >= d) before += o;
    }
    if (lane == 63) count[kBuckets + wave] = before;
    __syncthreads();
    int add = 0;
    for (int w = 0; w < wave; ++w) add += count[kBuckets + w];
    const int at1 = add + before - c1, at0 = at1 - c0;
    count[2 * threadIdx.x] = at0;
    count[2 * threadIdx.x + 1] = at1;
    int32_t *at = f.entry_at + (size_t)tile * (kBuckets + 1);
    at[2 * threadIdx.x] = at0;
    at[2 * threadIdx.x + 1] = at1;
    if (threadIdx.x == 511) at[kBuckets] = at1 + c1;
    __syncthreads();
    uint2 *out = f.entry + (size_t)tile * 32 * n;
    for (int e = threadIdx.x; e < entries; e += 512) {
        const int i = item[r0 * n + e];
        if (i >= 0) out[atomicAdd(count + (i / block_items) % kBuckets, 1)] = make_uint2((unsigned)i << 5 | (unsigned)(e / n), __float_as_uint(p[r0 * n + e]));
    }
}

// Two things that wait for different kernels and for nothing of each other, in one launch: the rows joined (8 / W per workgroup), and the tiles' entries
// (workgroups behind the rows').
template <int KP, int W>
__global__ void __launch_bounds__(512) join_rows_kernel(const FusedArgs f, int row_blocks, int block_items, const float *__restrict__ part, const float *__restrict__ mass,
                                                        const float *__restrict__ acc, const int32_t *__restrict__ item, const float *__restrict__ p) {
    __shared__ int lds[kBuckets + 8];
    if ((int)blockIdx.x >= row_blocks) {
        bucket_entries(f, (int)blockIdx.x - row_blocks, block_items, item, p, lds);
        return;
    }
    __shared__ float sums[W > 1 ? W * (KP + 1) : 1];
    const int wave = threadIdx.x >> 6;
    static_assert(W == 1 || W == 8, "a barrier for the W wavefronts of a row is one for the workgroup");
    join_row<KP, W>(f, (long long)blockIdx.x * (8 / W) + wave / W, wave % W, part, mass, acc, reinterpret_cast<float *>(lds) + wave * 64, sums);
}

// The items' gradient.  p of the teacher enters through a 32 x 32 patch of LDS per wavefront: the few entries that fall into the tile are written
// there, read back as the lanes hold dz, and cleared; a wavefront's LDS operations run in order, so no barrier is needed.
constexpr int kPatch = 36;                       // floats per item of the patch: 32 rows, and 16-byte reads without bank conflicts
// The work is cut into equal ranges of (block of items, user tile) pairs, one per workgroup that fits on the chip: no workgroup waits for a last
// round.  A block that lies inside one range is written out as it is; the others' parts go to slot workgroup + block -- workgroups and blocks
// both ascend along the ranges, so no two parts share one -- and are joined in that order.
// RAW: the items' own operands are made from the table (few users: no copies)
template <int KP, int NC, bool MASK, bool RAW = false>
__global__ void __launch_bounds__(Frag<KP>::waves * 64, (kPerSimd<KP, NC>)) items_kernel(const FusedArgs f) {
    constexpr int WAVES = Frag<KP>::waves;
    constexpr int kBytes = Frag<KP>::bytes, kBuf = 2 * kBytes + 2 * kUserData * 4;
    __shared__ __attribute__((aligned(16))) char buf[2][kBuf];
    __shared__ __attribute__((aligned(16))) float patches[WAVES][NC * 32 * kPatch];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), half = lane >> 5, col = lane & 31;
    const int n32 = 32 * f.a.n_teacher;
    float *patch = patches[wave];
    for (int k = lane; k < NC * 32 * kPatch; k += 64) patch[k] = 0.0f;
    const long long last_unit = min((long long)(blockIdx.x + 1) * f.units, (long long)f.item_blocks * f.user_tiles);
    for (long long unit = (long long)blockIdx.x * f.units; unit < last_unit;) {
        const int block = (int)(unit / f.user_tiles), t0 = (int)(unit - (long long)block * f.user_tiles);
        const int t1 = (int)min((long long)f.user_tiles, t0 + (last_unit - unit));
        unit += t1 - t0;
        const int tile = (block * WAVES + wave) * NC;
        const unsigned base = (unsigned)tile * 32u;
        f16x8 x[NC][Frag<KP>::steps][2];
        float bias[NC], unscale[NC], top[NC], d_bias[NC];
        unsigned next_word[NC];
        f32x16 o[NC][Frag<KP>::cols];
        auto mask_word = [&](int t, int n) {                     // of row `col` of the tile, the bits of this wavefront's items
            const int m = f.mask_row[min(t, t1 - 1) * 32 + col];
            const unsigned word = f.a.allowed[(size_t)max(m, 0) * (size_t)f.item_tiles + min(tile + n, f.item_tiles - 1)];
            return m >= 0 ? word : (unsigned)(-2 - m);           // (-1: all of them, -2: none)
        };
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const int mine = min(tile + n, f.item_tiles - 1);
            if constexpr (RAW) {
                bool odd;
                const int item = mine * 32 + col;
                Four raw[Frag<KP>::steps][2];
                const int e_raw = raw_tile<KP>(f.a.items, f.a.item_stride, mine, f.a.n_items, f.a.n_factors, lane, raw, odd);
                unscale[n] = ldexpf(1.0f, -e_raw);
#pragma unroll
                for (int k = 0; k < Frag<KP>::steps; ++k) raw_step(raw[k], ldexpf(1.0f, e_raw), x[n][k]);
                bias[n] = item < f.a.n_items ? (f.a.bias ? f.a.bias[item] * f.c : 0.0f) : -INFINITY;
            } else {
                load_columns<KP>(f.item_frag, mine, lane, x[n]);
                bias[n] = f.item_data[(size_t)mine * kItemData + col];
                unscale[n] = f.item_data[(size_t)mine * kItemData + 32];
            }
            top[n] = kLowest;
            d_bias[n] = 0.0f;
            next_word[n] = 0;
            if constexpr (MASK) next_word[n] = mask_word(t0, n);
            for (int c = 0; c < Frag<KP>::cols; ++c) o[n][c] = f32x16{0};
        }
        auto stage = [&](int t) {
            stage_copy<KP, WAVES>(f.user_frag, t, buf[t & 1], wave, lane);
            stage_copy<KP, WAVES>(f.user_frag_t, t, buf[t & 1] + kBytes, wave, lane);
            stage_data(f.user_data + (size_t)t * kUserData, buf[t & 1] + 2 * kBytes, lane);
            stage_data(f.user_data_t + (size_t)t * kUserData, buf[t & 1] + 2 * kBytes + kUserData * 4, lane);
        };
        // the tile's teacher entries: where they are is known two steps ahead (scalar loads), the first 64 are asked for one step ahead
        const int bucket = block % kBuckets;
        typedef const __attribute__((address_space(4))) int32_t *scalar_ptr;
        auto bounds = [&](int t, int &begin, int &end, int &all) {
            const scalar_ptr at = (scalar_ptr)(f.entry_at + (size_t)min(t, t1 - 1) * (kBuckets + 1));
            begin = at[bucket];
            end = at[bucket + 1];
            all = at[kBuckets];                                  // of all buckets: 0 where the tile has no live row
        };
        auto entry_of = [&](int t, int begin) { return f.entry[(size_t)min(t, t1 - 1) * n32 + min(begin + lane, n32 - 1)]; };
        int begin, end, all, begin1, end1, all1;
        bounds(t0, begin, end, all);
        bounds(t0 + 1, begin1, end1, all1);
        uint2 next_entry = entry_of(t0, begin);
        stage(t0);
        for (int t = t0; t < t1; ++t) {
            staged<0>();
            const char *now = buf[t & 1];
            const int from = begin, to = end, entries = all;
            uint2 entry = next_entry;
            unsigned word[NC];
            // (no instructions: what was asked for a step ago is here, and is taken before anything else is asked for)
            asm volatile("" : "+v"(entry.x), "+v"(entry.y));
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                word[n] = next_word[n];
                if constexpr (MASK) {
                    asm volatile("" : "+v"(word[n]));
                    next_word[n] = mask_word(t + 1, n);
                }
            }
            begin = begin1;
            end = end1;
            all = all1;
            bounds(t + 2, begin1, end1, all1);
            next_entry = entry_of(t + 1, begin);
            if (t + 1 < t1) stage(t + 1);
            f32x16 s[NC];
            tile_scores<KP, NC, true>(now, lane, x, s);
            const f32x4 *data = reinterpret_cast<const f32x4 *>(now + 2 * kBytes);
            const f32x4 last = data[8];
            const float e = last[1], scale = last[2];
            // a tile without a live row gives nothing, whatever the items hold.  (Beside a live one no row is without all items: where those are not finite
            // the live row's own share is not, either)
            if (!entries) continue;
            float high[NC], off[NC];
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                const float unit = unscaled(last[0], unscale[n]);
#pragma unroll
                for (int q = 0; q < 4; ++q) {                    // log2 of the shares: z as forward_kernel has it, less the row's lse
                    const f32x4 lse = data[half + 2 * q], rest = data[kUserData / 4 + 8 + half + 2 * q];
#pragma unroll
                    for (int k = 0; k < 4; ++k) s[n][4 * q + k] = (fmaf(s[n][4 * q + k], unit, bias[n]) - lse[k]) - rest[k];
                }
                if constexpr (MASK) mask16_rows(s[n], word[n]);
                high[n] = fmaxf(ceilf(both_halves(largest16(s[n]))), kLowest);
                off[n] = below(high[n]);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[n][r] = __builtin_amdgcn_exp2f(s[n][r] - off[n]);
            }
            // the teacher's share
            unsigned any = 0;                                    // a bit per column tile that is hit
            for (int k = from; k < to; k += 64) {
                if (k > from) entry = entry_of(t, k);
                const unsigned at = (entry.x >> 5) - base;
                const bool hit = k + lane < to && at < 32u * NC;
                if (hit) patch[at * kPatch + (entry.x & 31)] = __uint_as_float(entry.y);
#pragma unroll
                for (int n = 0; n < NC; ++n) any |= __any(hit && (at >> 5) == (unsigned)n) ? 1u << n : 0u;
            }
            if (any) {
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int n = 0; n < NC; ++n) {
                    if (!((any >> n) & 1u)) continue;
                    f32x4 *cell = reinterpret_cast<f32x4 *>(patch + (n * 32 + col) * kPatch + 4 * half);
                    f32x4 p[4];
                    unsigned most = 0;                           // (p is never negative: its bits order like its value)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        p[q] = cell[2 * q];
                        cell[2 * q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int k = 0; k < 4; ++k) most = max(most, __float_as_uint(p[q][k]));
                    }
                    const float log_p = both_halves(__builtin_amdgcn_logf(__uint_as_float(most)));       // (-inf where there is none)
                    if (__any(log_p > high[n])) {
                        const float to = below(fmaxf(high[n], ceilf(log_p))), by_p = __builtin_amdgcn_exp2f(off[n] - to);
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[n][r] *= by_p;
                        off[n] = to;
                    }
                    const float unit = fminf(__builtin_amdgcn_exp2f(-off[n]), -kLowest);      // (finite where a column has no weight: 0 stays 0)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
#pragma unroll
                        for (int k = 0; k < 4; ++k) s[n][4 * q + k] = fmaf(p[q][k], -unit, s[n][4 * q + k]);
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
            f16x8 p[NC][2][2];
            float by[NC];
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                by[n] = tile_unit(off[n], e, top[n], d_bias[n], o[n]);
                float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f32x4 coef = data[kUserData / 4 + half + 2 * q];
#pragma unroll
                    for (int k = 0; k < 4; ++k) sum[k] = fmaf(s[n][4 * q + k], coef[k], sum[k]);
                }
                d_bias[n] = fmaf((sum[0] + sum[1]) + (sum[2] + sum[3]), by[n] * scale, d_bias[n]);
                split_weights(s[n], p[n]);
            }
            weighted_sum<KP, NC>(now + kBytes, lane, p, by, o);
        }
        __syncthreads();                                         // the buffers are free for the next block
        const bool whole = t0 == 0 && t1 == f.user_tiles;
        const int K = f.a.n_factors;
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const float sum = d_bias[n] + __shfl_xor(d_bias[n], 32);
            // out of their unit 2^top, which may be below float32's smallest where its sums are not: by the exponent, not by a factor
            const int unit = (int)fminf(fmaxf(top[n], -1000.0f), 1000.0f);
            const float tau = f.a.temperature;
            auto out_of_unit = [&](int c, int q) {
                const f32x4 v = f32x4{o[n][c][4 * q], o[n][c][4 * q + 1], o[n][c][4 * q + 2], o[n][c][4 * q + 3]} * tau;
                return f32x4{ldexpf(v[0], unit), ldexpf(v[1], unit), ldexpf(v[2], unit), ldexpf(v[3], unit)};
            };
            const int item = (tile + n) * 32 + col;
            if (whole && item < f.a.n_items) {
                float *out = f.a.d_items + (size_t)item * K;
                if (half == 0 && f.a.d_bias) f.a.d_bias[item] = ldexpf(sum * tau, unit);
#pragma unroll
                for (int c = 0; c < Frag<KP>::cols; ++c)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int k = 32 * c + 8 * q + 4 * half;
                        const f32x4 v = out_of_unit(c, q);
                        store_four(out, k, K, v[0], v[1], v[2], v[3]);
                    }
            } else if (!whole) {
                const size_t at = ((size_t)(blockIdx.x + block) * WAVES * NC + wave * NC + n) * 32 + col;
                if (half == 0) f.part_bias[at] = ldexpf(sum * tau, unit);
#pragma unroll
                for (int c = 0; c < Frag<KP>::cols; ++c)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        *reinterpret_cast<f32x4 *>(f.part_items + at * KP + 32 * c + 8 * q + 4 * half) = out_of_unit(c, q);
            }
        }
    }
}

// One workgroup per tile of items: the parts of a block that was cut, in the order of its user tiles.
template <int KP>
__global__ void __launch_bounds__(256) join_items_kernel(const FusedArgs f, int tiles) {
    const int block = (int)blockIdx.x / tiles, in_block = (int)blockIdx.x % tiles * 32, K = f.a.n_factors;
    const int first = (int)((long long)block * f.user_tiles / f.units), last = (int)(((long long)(block + 1) * f.user_tiles - 1) / f.units);
    if (first == last) return;
    const int i0 = block * tiles * 32 + in_block;
    for (int e = threadIdx.x; e < 32 * KP / 4; e += 256) {
        const int row = e / (KP / 4), k = e % (KP / 4) * 4;
        if (i0 + row >= f.a.n_items || k >= K) continue;
        f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
        const float *from = f.part_items + ((size_t)block * tiles * 32 + in_block + row) * KP + k;
        int g = first;
        for (; g + 3 <= last; g += 4) {                          // (four loads in flight)
            f32x4 x[4];
#pragma unroll
            for (int h = 0; h < 4; ++h) x[h] = *reinterpret_cast<const f32x4 *>(from + (size_t)(g + h) * tiles * 32 * KP);
#pragma unroll
            for (int h = 0; h < 4; ++h) s += x[h];
        }
        for (; g <= last; ++g) s += *reinterpret_cast<const f32x4 *>(from + (size_t)g * tiles * 32 * KP);
        store_four(f.a.d_items + (size_t)(i0 + row) * K, k, K, s[0], s[1], s[2], s[3]);
    }
    if (!f.a.d_bias || threadIdx.x >= 32 || i0 + (int)threadIdx.x >= f.a.n_items) return;
    float s = 0.0f;
#pragma unroll 8
    for (int g = first; g <= last; ++g) s += f.part_bias[(size_t)(g + block) * tiles * 32 + in_block + threadIdx.x];
    f.a.d_bias[i0 + threadIdx.x] = s;
}

__global__ void __launch_bounds__(256) zero_kernel(float *x, long long n) {
    for (long long k = (long long)blockIdx.x * 256 + threadIdx.x; k < n; k += (long long)gridDim.x * 256) x[k] = 0.0f;
}

}  // namespace distill
}  // namespace rfm
