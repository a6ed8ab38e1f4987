// rfm_distill_fused.hpp -- the distillation loss and its gradients without the score matrix (included by rfm_distill.hip).
//
// fp32 products on the bf16 matrix cores.  Every fp32 factor is the sum of three bf16 parts, x = h + m + l (8 + 8 + 8 bits of the 24-bit
// significand, rounded to nearest at each cut); of the nine products of two such sums the six of order 2^-16 and above are computed,
// l h', h l', m m', m h', h m', h h', and the three left out are below 2^-24 of |x x'|: half a step of fp32, the size of the rounding that an
// fp32 product makes itself.  Six v_mfma_f32_32x32x16_bf16 take 6 / 16 of the time of the fp32 matrix instructions for the same product.
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

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kRowData = 64;                     // floats that travel with a tile: 32 biases (+ 32 unused), or 32 lse and 32 coefficients
constexpr int kFusedTeacher = 256;               // teacher entries of the fused path: a tile's 32 x n entries are sorted in LDS
constexpr float kLowest = -3.402823466e38f;

template <int KP> struct Frag {
    static constexpr int steps = KP / 16, cols = KP / 32;
    static constexpr int bytes = KP * 192;       // one copy of a tile: KP / 16 x 3 parts x 1 KB; the transposed copy has as many
};

struct FusedArgs {
    rfm_distill_args a;
    int user_tiles, item_tiles, item_blocks;     // tiles of 32 rows; blocks of items_kernel's workgroups
    int splits, chunk;                           // of the streamed tiles
    const char *user_frag, *user_frag_t, *item_frag, *item_frag_t;
    const float *bias2;                          // [(item_tiles + 2) * 32] bias * log2(e) / temperature, -inf behind the last item
    const int32_t *mask_row;                     // [user_tiles * 32] mask of each row, -1 = none
    float *part_m, *part_l, *part_o;             // forward: [splits, user_tiles * 32 (, KP)]
    const float *row_data;                       // [user_tiles, 64] lse (log2 units) and coefficient of each row
    const uint2 *entry;                          // [user_tiles, 32 n]: (item << 5 | row, p), ascending
    const int32_t *entry_at;                     // [user_tiles, item_blocks + 1] where a block's entries begin
    float *part_items, *part_bias;               // items: [splits, item_tiles * 32 (, KP)]
};

__device__ __forceinline__ void split3(float x, __bf16 &h, __bf16 &m, __bf16 &l) {
    h = (__bf16)x;
    const float r = x - (float)h;
    m = (__bf16)r;
    l = (__bf16)(r - (float)m);
}

// One workgroup per tile of 32 rows of a table: its fragments.  Rows without a usable teacher entry (live) count as zeros: they may be padding.
template <int KP>
__device__ void write_frags(const float *__restrict__ x, long long stride, int tile, long long rows, int factors, float scale, const float *__restrict__ live, char *frag,
                            char *frag_t, float *lds) {
    constexpr int ld = KP + 1;
    for (int e = threadIdx.x; e < 32 * KP; e += 256) {
        const int row = e / KP, k = e % KP;
        const long long r = (long long)tile * 32 + row;
        lds[row * ld + k] = r < rows && k < factors && (!live || live[r] > 0.0f) ? x[r * stride + k] : 0.0f;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < KP * 4; e += 256) {            // 8 factors of a row each
        const int s = e >> 6, lane = e & 63;
        bf16x8 h, m, l;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            __bf16 a, b, c;
            split3(lds[(lane & 31) * ld + 16 * s + 8 * (lane >> 5) + j] * scale, a, b, c);
            h[j] = a; m[j] = b; l[j] = c;
        }
        bf16x8 *out = reinterpret_cast<bf16x8 *>(frag + (size_t)tile * Frag<KP>::bytes) + s * 192 + lane;
        out[0] = h; out[64] = m; out[128] = l;
    }
    if (!frag_t) return;
    for (int e = threadIdx.x; e < KP * 4; e += 256) {            // 8 rows of a factor each
        const int ct = e >> 6, lane = e & 63, half = lane >> 5;
        bf16x8 h, m, l;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            __bf16 a, b, c;
            split3(lds[(16 * (ct & 1) + (j & 3) + 8 * (j >> 2) + 4 * half) * ld + 32 * (ct >> 1) + (lane & 31)], a, b, c);
            h[j] = a; m[j] = b; l[j] = c;
        }
        bf16x8 *out = reinterpret_cast<bf16x8 *>(frag_t + (size_t)tile * Frag<KP>::bytes) + ct * 192 + lane;
        out[0] = h; out[64] = m; out[128] = l;
    }
}

template <int KP>
__global__ void __launch_bounds__(256) frags_kernel(const rfm_distill_args a, int user_tiles, int item_tiles, float c, const float *__restrict__ mass, char *user_frag,
                                                    char *user_frag_t, char *item_frag, char *item_frag_t, float *bias2, int32_t *mask_row) {
    __shared__ float lds[32 * (KP + 1)];
    const int b = blockIdx.x;
    if (b < user_tiles) {
        write_frags<KP>(a.users, a.user_stride, b, a.n_rows, a.n_factors, c, mass, user_frag, user_frag_t, lds);
        if (threadIdx.x < 32 && a.allowed) {
            const long long r = (long long)b * 32 + threadIdx.x;
            long long m = -1;
            if (r < a.n_rows) m = a.allowed_rows ? (long long)a.allowed_rows[r] : (a.n_allowed == 1 ? 0 : r);
            mask_row[r] = m >= 0 && m < a.n_allowed ? (int32_t)m : -1;
        }
    } else {
        const int t = b - user_tiles;
        write_frags<KP>(a.items, a.item_stride, t, a.n_items, a.n_factors, 1.0f, nullptr, item_frag, item_frag_t, lds);
        if (threadIdx.x < 32) {
            const long long i = (long long)t * 32 + threadIdx.x;
            bias2[i] = i < a.n_items ? (a.bias ? a.bias[i] * c : 0.0f) : -INFINITY;
        }
        if (t == item_tiles - 1 && threadIdx.x < 64) bias2[(size_t)item_tiles * 32 + threadIdx.x] = -INFINITY;
    }
}

// ---- LDS staging: a kilobyte per instruction straight from memory (global_load_lds, 16 bytes per lane) --------------------------------------------
__device__ __forceinline__ void stage16(const char *from, char *to) {            // `to` is the wavefront's own kilobyte, `from` the lane's 16 bytes
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from, (__attribute__((address_space(3))) void *)to, 16, 0, 0);
}
__device__ __forceinline__ void stage4(const char *from, char *to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from, (__attribute__((address_space(3))) void *)to, 4, 0, 0);
}
template <int KP, bool T, int WAVES>
__device__ __forceinline__ void stage_tile(const char *frag, const char *frag_t, const float *data, int tile, char *buf, int wave, int lane) {
    constexpr int bytes = Frag<KP>::bytes, kb = bytes / 1024;
    const char *src = frag + (size_t)tile * bytes + lane * 16;
#pragma unroll
    for (int q = 0; q < (kb + WAVES - 1) / WAVES; ++q) {
        const int k = q * WAVES + wave;
        if (kb % WAVES == 0 || k < kb) stage16(src + k * 1024, buf + k * 1024);
    }
    if constexpr (T) {
        const char *src_t = frag_t + (size_t)tile * bytes + lane * 16;
#pragma unroll
        for (int q = 0; q < (kb + WAVES - 1) / WAVES; ++q) {
            const int k = q * WAVES + wave;
            if (kb % WAVES == 0 || k < kb) stage16(src_t + k * 1024, buf + bytes + k * 1024);
        }
    }
    if (wave == 0) stage4(reinterpret_cast<const char *>(data) + lane * 4, buf + (T ? 2 : 1) * bytes);
}
__device__ __forceinline__ void staged() {       // this wavefront's staging is in LDS
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
// c + (ah + am + al) (bh + bm + bl), the small products first
__device__ __forceinline__ f32x16 mfma6(const bf16x8 *a, const bf16x8 *b, f32x16 c) {
    c = mfma(a[2], b[0], c); c = mfma(a[0], b[2], c); c = mfma(a[1], b[1], c);
    c = mfma(a[1], b[0], c); c = mfma(a[0], b[1], c);
    return mfma(a[0], b[0], c);
}
__device__ __forceinline__ void split_weights(const f32x16 &w, bf16x8 (*p)[3]) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            __bf16 h, m, l;
            split3(w[8 * t + j], h, m, l);
            p[t][0][j] = h; p[t][1][j] = m; p[t][2][j] = l;
        }
}
// o[c] += rows of the transposed tile . weights.  A tile's 32 terms are summed by themselves first: the running sum sees one addition per tile
template <int KP>
__device__ __forceinline__ void weighted_sum(const char *tile_t, int lane, const bf16x8 (*p)[3], f32x16 *o) {
#pragma unroll
    for (int c = 0; c < Frag<KP>::cols; ++c) {
        f32x16 sum = {0};
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const bf16x8 *at = reinterpret_cast<const bf16x8 *>(tile_t) + (c * 2 + t) * 192 + lane;
            const bf16x8 a[3] = {at[0], at[64], at[128]};
            sum = mfma6(a, p[t], sum);
        }
        o[c] += sum;
    }
}
template <int KP>
__device__ __forceinline__ f32x16 tile_scores(const char *tile, int lane, const bf16x8 (*x)[3], f32x16 s) {
#pragma unroll
    for (int k = 0; k < Frag<KP>::steps; ++k) {
        const bf16x8 *at = reinterpret_cast<const bf16x8 *>(tile) + k * 192 + lane;
        const bf16x8 a[3] = {at[0], at[64], at[128]};
        s = mfma6(a, x[k], s);
    }
    return s;
}
template <int KP>
__device__ __forceinline__ void load_columns(const char *frag, int tile, int lane, bf16x8 (*x)[3]) {
    const bf16x8 *src = reinterpret_cast<const bf16x8 *>(frag + (size_t)tile * Frag<KP>::bytes) + lane;
#pragma unroll
    for (int k = 0; k < Frag<KP>::steps; ++k)
#pragma unroll
        for (int p = 0; p < 3; ++p) x[k][p] = src[k * 192 + p * 64];
}

// Block b: split b % splits of the items, columns block b / splits: with a multiple of 8 splits the workgroups of one XCD stream the same items.
template <int KP, bool GRAD, bool MASK, int WAVES>
__global__ void __launch_bounds__(WAVES * 64, 2) forward_kernel(const FusedArgs f) {
    constexpr int kBytes = (GRAD ? 2 : 1) * Frag<KP>::bytes + kRowData * 4;
    __shared__ __attribute__((aligned(16))) char buf[2][kBytes];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), half = lane >> 5;
    const int split = (int)blockIdx.x % f.splits, tile = (int)blockIdx.x / f.splits * WAVES + wave;
    const int mine = tile < f.user_tiles ? tile : f.user_tiles - 1;              // (a wavefront without users works on the last ones and writes nothing)
    const int t0 = split * f.chunk, t1 = min(t0 + f.chunk, f.item_tiles);
    bf16x8 x[Frag<KP>::steps][3];
    load_columns<KP>(f.user_frag, mine, lane, x);
    const uint32_t *mask = nullptr;
    if constexpr (MASK) {
        const int m = f.mask_row[mine * 32 + (lane & 31)];
        if (m >= 0) mask = f.a.allowed + (size_t)m * (size_t)f.item_tiles;
    }
    float top = kLowest, total = 0.0f;
    f32x16 o[GRAD ? Frag<KP>::cols : 1];
    if constexpr (GRAD)
        for (int c = 0; c < Frag<KP>::cols; ++c) o[c] = f32x16{0};
    stage_tile<KP, GRAD, WAVES>(f.item_frag, f.item_frag_t, f.bias2 + (size_t)t0 * 32, t0, buf[0], wave, lane);
    unsigned word = 0xffffffffu, next_word = 0xffffffffu;
    if constexpr (MASK)
        if (mask) next_word = mask[t0];
    for (int t = t0; t < t1; ++t) {
        const char *now = buf[(t - t0) & 1];
        staged();
        if constexpr (MASK) word = next_word;
        if (t + 1 < t1) {
            if constexpr (MASK)
                if (mask) next_word = mask[t + 1];
            stage_tile<KP, GRAD, WAVES>(f.item_frag, f.item_frag_t, f.bias2 + (size_t)(t + 1) * 32, t + 1, buf[(t - t0 + 1) & 1], wave, lane);
        }
        f32x16 s;
        const f32x4 *bias = reinterpret_cast<const f32x4 *>(now + (GRAD ? 2 : 1) * Frag<KP>::bytes) + half;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x4 b = bias[2 * q];
#pragma unroll
            for (int k = 0; k < 4; ++k) s[4 * q + k] = b[k];
        }
        s = tile_scores<KP>(now, lane, x, s);
        if constexpr (MASK) {
            const unsigned w = word >> (4 * half);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = (w >> ((r & 3) + 8 * (r >> 2))) & 1u ? s[r] : -INFINITY;
        }
        float high = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) high = fmaxf(high, s[r]);
        // the maximum is moved only when a score passes it by 2^8: the weights stay below 256 and the sums are rarely scaled
        if (__any(high > top + 8.0f)) {
            const float to = fmaxf(top, fmaxf(high, __shfl_xor(high, 32)));
            const float by = __builtin_amdgcn_exp2f(top - to);
            total *= by;
            if constexpr (GRAD)
                for (int c = 0; c < Frag<KP>::cols; ++c) o[c] *= by;
            top = to;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(s[r] - top);
        float sum[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) sum[q] = (s[4 * q] + s[4 * q + 1]) + (s[4 * q + 2] + s[4 * q + 3]);
        total += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        if constexpr (GRAD) {
            bf16x8 p[2][3];
            split_weights(s, p);
            weighted_sum<KP>(now + Frag<KP>::bytes, lane, p, o);
        }
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
__global__ void __launch_bounds__(256) join_rows_kernel(const FusedArgs f, const float *__restrict__ part, const float *__restrict__ mass, const float *__restrict__ acc,
                                                        float *__restrict__ row_data) {
    const int lane = threadIdx.x & 63;
    const long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6), padded = (long long)f.user_tiles * 32;
    if (r >= padded) return;
    const bool grad = f.a.d_users != nullptr;
    float *data = row_data + (r >> 5) * kRowData + (r & 31);
    const float has = r < f.a.n_rows ? mass[r] : 0.0f;
    if (!(has > 0.0f)) {                                         // no row, nothing to learn from, or a mask that does not exist
        if (r < f.a.n_rows) {
            if (lane == 0) f.a.loss[r] = has;                    // (0 or NaN)
            if (grad)
                for (int k = lane; k < f.a.n_factors; k += 64) f.a.d_users[(size_t)r * f.a.n_factors + k] = 0.0f;
        }
        if (grad && lane == 0) { data[0] = INFINITY; data[32] = 0.0f; }
        return;
    }
    float top = kLowest;
    for (int s = lane; s < f.splits; s += 64) top = fmaxf(top, f.part_m[(size_t)s * padded + r]);
    top = wave_max(top);
    float total = 0.0f;
    for (int s = lane; s < f.splits; s += 64) total += f.part_l[(size_t)s * padded + r] * __builtin_amdgcn_exp2f(f.part_m[(size_t)s * padded + r] - top);
    total = wave_sum(total);
    const float lse2 = top + log2f(total);
    if (lane == 0) f.a.loss[r] = f.a.temperature * f.a.temperature * (part[r] + lse2 * 0.693147180559945309f);
    if (!grad) return;
    const float coef = f.a.temperature * (f.a.row_weight ? f.a.row_weight[r] : 1.0f);
    if (lane == 0) { data[0] = lse2; data[32] = coef; }
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
    constexpr int kBytes = 2 * Frag<KP>::bytes + kRowData * 4;
    __shared__ __attribute__((aligned(16))) char buf[2][kBytes];
    __shared__ __attribute__((aligned(16))) float patches[WAVES][32 * kPatch];
    __shared__ __attribute__((aligned(16))) unsigned words[MASK ? WAVES : 1][32];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), half = lane >> 5, col = lane & 31;
    const int split = (int)blockIdx.x % f.splits, block = (int)blockIdx.x / f.splits, tile = block * WAVES + wave;
    const int mine = tile < f.item_tiles ? tile : f.item_tiles - 1;
    const int t0 = split * f.chunk, t1 = min(t0 + f.chunk, f.user_tiles), n32 = 32 * f.a.n_teacher;
    float *patch = patches[wave];
    for (int k = lane; k < 32 * kPatch; k += 64) patch[k] = 0.0f;
    bf16x8 x[Frag<KP>::steps][3];
    load_columns<KP>(f.item_frag, mine, lane, x);
    const float bias = f.bias2[mine * 32 + col];
    const unsigned base = (unsigned)tile * 32u;
    f32x16 o[Frag<KP>::cols];
    for (int c = 0; c < Frag<KP>::cols; ++c) o[c] = f32x16{0};
    float d_bias = 0.0f;
    auto mask_word = [&](int t) {                                // of row `col` of the tile, the bits of this wavefront's items
        const int m = f.mask_row[t * 32 + col];
        return m < 0 ? 0xffffffffu : f.a.allowed[(size_t)m * (size_t)f.item_tiles + mine];
    };
    stage_tile<KP, true, WAVES>(f.user_frag, f.user_frag_t, f.row_data + (size_t)t0 * kRowData, t0, buf[0], wave, lane);
    unsigned next_word = 0;
    if constexpr (MASK) next_word = mask_word(t0);
    int begin = f.entry_at[(size_t)t0 * (f.item_blocks + 1) + block], end = f.entry_at[(size_t)t0 * (f.item_blocks + 1) + block + 1];
    for (int t = t0; t < t1; ++t) {
        const char *now = buf[(t - t0) & 1];
        staged();
        const int from = begin, to = end;
        uint2 e = make_uint2(0xffffffffu, 0);
        if (from + lane < to) e = f.entry[(size_t)t * n32 + from + lane];
        unsigned word = 0;
        if constexpr (MASK) word = next_word;
        if (t + 1 < t1) {
            begin = f.entry_at[(size_t)(t + 1) * (f.item_blocks + 1) + block];
            end = f.entry_at[(size_t)(t + 1) * (f.item_blocks + 1) + block + 1];
            if constexpr (MASK) next_word = mask_word(t + 1);
            stage_tile<KP, true, WAVES>(f.user_frag, f.user_frag_t, f.row_data + (size_t)(t + 1) * kRowData, t + 1, buf[(t - t0 + 1) & 1], wave, lane);
        }
        f32x16 s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = bias;
        s = tile_scores<KP>(now, lane, x, s);
        const f32x4 *data = reinterpret_cast<const f32x4 *>(now + 2 * Frag<KP>::bytes) + half;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x4 lse = data[2 * q];
#pragma unroll
            for (int k = 0; k < 4; ++k) s[4 * q + k] = __builtin_amdgcn_exp2f(s[4 * q + k] - lse[k]);
        }
        if constexpr (MASK) {
            if (half == 0) words[wave][col] = word;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const u32x4 w = reinterpret_cast<const u32x4 *>(words[wave])[2 * q + half];
#pragma unroll
                for (int k = 0; k < 4; ++k) s[4 * q + k] = (w[k] >> col) & 1u ? s[4 * q + k] : 0.0f;
            }
        }
        // the teacher's share
        bool any = false;
        for (int k = from; k < to; k += 64) {
            if (k > from) e = k + lane < to ? f.entry[(size_t)t * n32 + k + lane] : make_uint2(0xffffffffu, 0);
            const unsigned at = (e.x >> 5) - base;
            const bool hit = e.x != 0xffffffffu && at < 32u;
            if (hit) patch[at * kPatch + (e.x & 31)] = __uint_as_float(e.y);
            any |= __any(hit);
        }
        if (any) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                f32x4 *cell = reinterpret_cast<f32x4 *>(patch + col * kPatch + 8 * q + 4 * half);
                const f32x4 p = *cell;
#pragma unroll
                for (int k = 0; k < 4; ++k) s[4 * q + k] -= p[k];
                *cell = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x4 coef = data[8 + 2 * q];
#pragma unroll
            for (int k = 0; k < 4; ++k) s[4 * q + k] *= coef[k];
        }
        float sum[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) sum[q] = (s[4 * q] + s[4 * q + 1]) + (s[4 * q + 2] + s[4 * q + 3]);
        d_bias += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        bf16x8 p[2][3];
        split_weights(s, p);
        weighted_sum<KP>(now + Frag<KP>::bytes, lane, p, o);
    }
    if (tile >= f.item_tiles) return;
    d_bias += __shfl_xor(d_bias, 32);
    const size_t at = (size_t)split * f.item_tiles * 32 + (size_t)tile * 32 + col;
    if (half == 0) f.part_bias[at] = d_bias;
#pragma unroll
    for (int c = 0; c < Frag<KP>::cols; ++c)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x4 v = {o[c][4 * q], o[c][4 * q + 1], o[c][4 * q + 2], o[c][4 * q + 3]};
            *reinterpret_cast<f32x4 *>(f.part_items + at * KP + 32 * c + 8 * q + 4 * half) = v;
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
