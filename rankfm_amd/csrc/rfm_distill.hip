// rfm_distill.hip -- learning from another model's top scores: the loss of a student's catalogue distribution against a teacher's lists, and
// its gradients (include/rankfm_hip.h rfm_distill_device).
//
//   z[r, i] = < users[r], items[i] > + bias[i],  q = softmax(z / tau) over the allowed items,  p = softmax(teacher / tau) over usable entries
//   loss[r] = tau^2 sum_j p_j (log p_j - z[r, t_j] / tau + lse_r),   lse_r = log sum_i exp(z[r, i] / tau)
//   dz = tau * weight[r] * (q - p);   d_users = dz . items;   d_items = dz^T . users;   d_bias = column sums of dz
//
// Two paths.  Up to 128 factors the scores never leave the registers: one pass over the items per block of rows keeps a
// running maximum and sum (and, for the gradients, the weighted sum of item rows), a second one over the rows per block of items gives the
// items' gradient (rfm_distill_fused.hpp).  Beyond, the matrix path: the scores of a block of rows are written out, turned into dz in place
// and multiplied.  Every sum has a fixed order on both.
#include <hip/hip_runtime.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "../../include/rankfm_hip.h"

namespace rfm {
namespace distill {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kMaxTeacher = 1024;                // entries of a teacher's list (their ids sit in LDS)

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) x += __shfl_xor(x, m);
    return x;
}
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) x = fmaxf(x, __shfl_xor(x, m));
    return x;
}

// the row's mask of allowed items (nullptr: everything is); `bad`: it names one behind the last
__device__ __forceinline__ const uint32_t *row_mask(const rfm_distill_args &a, long long r, bool *bad) {
    if (!a.allowed) return nullptr;
    const long long m = a.allowed_rows ? (long long)a.allowed_rows[r] : (a.n_allowed == 1 ? 0 : r);
    if (m >= a.n_allowed) { *bad = true; return nullptr; }
    return m < 0 ? nullptr : a.allowed + (size_t)m * (size_t)((a.n_items + 31) / 32);
}

// whether a teacher's entry counts
__device__ __forceinline__ bool usable(const rfm_distill_args &a, const uint32_t *mask, int item, float score) {
    return item >= 0 && item < a.n_items && !(score == -INFINITY) && (!mask || ((mask[item >> 5] >> (item & 31)) & 1u));
}

struct __attribute__((packed, aligned(4))) Four { float v[4]; };
// factors 4 f .. 4 f + 3 of a row, zeros behind its end; rows start anywhere, the hardware takes 16 bytes at any address
__device__ __forceinline__ Four load_four(const float *row, int k, int factors) {
    Four x;
    if (k + 4 <= factors) __builtin_memcpy(&x, reinterpret_cast<const Four *>(row + k), sizeof(x));
    else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x.v[j] = k + j < factors ? row[k + j] : 0.0f;
    }
    return x;
}

// ... and written
__device__ __forceinline__ void store_four(float *row, int k, int factors, float a, float b, float c, float d) {
    if (k + 4 <= factors) {
        const Four x = {{a, b, c, d}};
        __builtin_memcpy(reinterpret_cast<Four *>(row + k), &x, sizeof(x));
    } else {
        const float x[4] = {a, b, c, d};
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (k + j < factors) row[k + j] = x[j];
    }
}

// One wavefront per row: the teacher's distribution over the usable entries, and its part of the loss.
//   part[r] = sum_j p_j (log p_j - z[r, t_j] / tau)     mass[r] = 1, 0 without a usable entry, NaN where the row's mask does not exist
// For the gradients the list is left with the usable entries' p (-1, 0 elsewhere).  MERGE: merged too -- an item's first entry holds the sum of
// its entries' p, the others are off, so that no two entries of a row meet in one element of dz.  ACC > 0: 64 ACC factors at most, in registers;
// acc [rows, kp] = sum_j p_j items[t_j] where it is asked for.  s_dyn: per wavefront ids [n] and p [n].  No barrier: a wavefront works by itself.
template <bool MERGE, int ACC>
__device__ void teacher_row(const rfm_distill_args &a, long long r, int kp, int *s_dyn, float *__restrict__ part, float *__restrict__ mass, int32_t *__restrict__ merged_item,
                            float *__restrict__ merged_p, float *__restrict__ acc_out) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = a.n_teacher;
    if (r >= a.n_rows) return;
    int *id = s_dyn + wave * 2 * n;
    float *pr = reinterpret_cast<float *>(id + n);
    bool bad = false;
    const uint32_t *mask = row_mask(a, r, &bad);
    const int32_t *ti = a.teacher_items + (size_t)r * n;
    const float *ts = a.teacher_scores + (size_t)r * n;
    const float inv_tau = 1.0f / a.temperature;
    float top = -INFINITY;
    bool nan = false;
    int some = 0;
    for (int j = lane; j < n; j += 64) {
        const int i = ti[j];
        const float t = ts[j];
        const bool use = usable(a, mask, i, t);
        id[j] = use ? i : -1;
        if (use) { some = 1; nan |= isnan(t); top = fmaxf(top, t); }
    }
    some = __any(some);
    top = wave_max(top);
    if (__any(nan)) top = __uint_as_float(0x7fc00000u);
    float sum = 0.0f;
    for (int j = lane; j < n; j += 64) {
        const float e = id[j] >= 0 ? expf((ts[j] - top) * inv_tau) : 0.0f;
        pr[j] = e;
        sum += e;
    }
    sum = wave_sum(sum);
    const float log_sum = logf(sum), inv = 1.0f / sum;
    // sum_j p_j (log p_j - bias / tau) here, the products of factors below: sum_j p_j < u, v_j > = < u, sum_j p_j v_j >
    float acc = 0.0f;
    for (int j = lane; j < n; j += 64) {
        const float e = pr[j];
        const int i = id[j];
        if (!(e == 0.0f)) acc += e * inv * ((ts[j] - top) * inv_tau - log_sum - (a.bias ? a.bias[i] * inv_tau : 0.0f));
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    // 16 lanes per entry, the loads of several entries of each group of lanes in flight
    const float *u = a.users + (size_t)r * a.user_stride;
    const int sub = lane & 15, grp = lane >> 4;
    float dot = 0.0f;
    if constexpr (ACC > 0) {
        constexpr int AHEAD = ACC == 1 ? 8 : 5;
        Four mine[ACC], wsum[ACC];
#pragma unroll
        for (int q = 0; q < ACC; ++q) {
            mine[q] = load_four(u, 64 * q + 4 * sub, a.n_factors);
            wsum[q] = Four{{0.0f, 0.0f, 0.0f, 0.0f}};
        }
        for (int j0 = 0; j0 < n; j0 += 4 * AHEAD) {
            Four x[AHEAD][ACC];
            float e[AHEAD];
#pragma unroll
            for (int h = 0; h < AHEAD; ++h) {
                const int j = j0 + 4 * h + grp, item = j < n ? id[j] : -1;
                e[h] = item >= 0 ? pr[j] : 0.0f;
#pragma unroll
                for (int q = 0; q < ACC; ++q) {
                    x[h][q] = Four{{0.0f, 0.0f, 0.0f, 0.0f}};
                    if (item >= 0) x[h][q] = load_four(a.items + (size_t)item * a.item_stride, 64 * q + 4 * sub, a.n_factors);
                }
            }
#pragma unroll
            for (int h = 0; h < AHEAD; ++h)
#pragma unroll
                for (int q = 0; q < ACC; ++q)
#pragma unroll
                    for (int k = 0; k < 4; ++k) wsum[q].v[k] = fmaf(e[h], x[h][q].v[k], wsum[q].v[k]);
        }
#pragma unroll
        for (int q = 0; q < ACC; ++q)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                dot = fmaf(mine[q].v[k], wsum[q].v[k], dot);
                float x = wsum[q].v[k];
                x += __shfl_xor(x, 16);
                x += __shfl_xor(x, 32);
                const int at = 64 * q + 4 * sub + k;
                if (acc_out && grp == 0 && at < kp) acc_out[(size_t)r * kp + at] = some ? x * inv : 0.0f;
            }
    } else {
        for (int j = grp; j < n; j += 4) {
            const int item = id[j];
            if (item < 0) continue;
            float d = 0.0f;
            for (int f = 4 * sub; f < a.n_factors; f += 64) {
                const Four x = load_four(a.items + (size_t)item * a.item_stride, f, a.n_factors), y = load_four(u, f, a.n_factors);
#pragma unroll
                for (int k = 0; k < 4; ++k) d = fmaf(y.v[k], x.v[k], d);
            }
            dot = fmaf(pr[j], d, dot);
        }
    }
    acc = wave_sum(acc) - wave_sum(dot) * inv * inv_tau;
    if (lane == 0) {
        part[r] = some ? acc : 0.0f;
        mass[r] = bad ? __uint_as_float(0x7fc00000u) : some ? 1.0f : 0.0f;
    }
    if (!merged_item) return;
    auto merge = [&](int j0, auto slots) {                       // some entries per lane against all of them
        constexpr int S = decltype(slots)::value;
        int i[S];
        float p[S];
        bool first[S];
#pragma unroll
        for (int q = 0; q < S; ++q) {
            const int j = j0 + 64 * q + lane;
            i[q] = j < n ? id[j] : -1;
            p[q] = MERGE || i[q] < 0 ? 0.0f : pr[j];
            first[q] = true;
        }
        if constexpr (MERGE) {
#pragma unroll 4
            for (int k = 0; k < n; ++k) {
                const int at = id[k];
                const float more = pr[k];
#pragma unroll
                for (int q = 0; q < S; ++q) {
                    const bool twin = at == i[q];
                    first[q] &= !twin || k >= j0 + 64 * q + lane;
                    p[q] += twin ? more : 0.0f;
                }
            }
        }
#pragma unroll
        for (int q = 0; q < S; ++q) {
            const int j = j0 + 64 * q + lane;
            const bool on = i[q] >= 0 && first[q] && !bad;
            if (j < n) {
                merged_item[(size_t)r * n + j] = on ? i[q] : -1;
                merged_p[(size_t)r * n + j] = on ? p[q] * inv : 0.0f;
            }
        }
    };
    int j0 = 0;
    for (; n - j0 > 128; j0 += 256) merge(j0, std::integral_constant<int, 4>());
    if (n - j0 > 64) merge(j0, std::integral_constant<int, 2>());
    else if (n > j0) merge(j0, std::integral_constant<int, 1>());
}
__global__ void __launch_bounds__(256) teacher_kernel(const rfm_distill_args a, float *__restrict__ part, float *__restrict__ mass, int32_t *__restrict__ merged_item,
                                                      float *__restrict__ merged_p) {
    extern __shared__ int s_dyn[];
    teacher_row<true, 0>(a, (long long)blockIdx.x * 4 + (threadIdx.x >> 6), 0, s_dyn, part, mass, merged_item, merged_p, nullptr);
}

// C[m, n] (+)= sum_k A[m, k] B[k, n] (+ bias[n]), any strides; slices of k (blockIdx.y) go to slices of C.  live: rows k of B whose entry is 0
// or NaN count as zeros, whatever they hold (rows without a usable teacher entry may be padding).  finite: so do elements of B that are not
// finite -- in the products with dz: where they count that row of dz is NaN already, where a mask has taken them out dz is 0.  64 x 64 tile per
// workgroup, four wavefronts of one 32 x 32 accumulator each (v_mfma_f32_32x32x2_f32, exact fp32), k in LDS stages of 32.
constexpr int kKT = 32, kLd = kKT + 1;
__global__ void __launch_bounds__(256) gemm_kernel(const float *__restrict__ A, long long am, long long ak, const float *__restrict__ B, long long bk, long long bn,
                                                   const float *__restrict__ bias, float *__restrict__ C, long long cm, long long slice_stride, long long M, int N, int K,
                                                   int k_slice, int n_tiles, int accumulate, const float *__restrict__ live, int finite) {
    __shared__ float sA[64 * kLd], sB[64 * kLd];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wr = wave >> 1, wc = wave & 1;
    const long long m0 = (long long)(blockIdx.x / n_tiles) * 64;
    const int n0 = (int)(blockIdx.x % n_tiles) * 64;
    const int kb = (int)blockIdx.y * k_slice, ke = min(K - kb, k_slice) + kb;
    C += (size_t)blockIdx.y * slice_stride;
    f32x16 acc = {0};
    for (int k0 = kb; k0 < ke; k0 += kKT) {
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const int e = tid + 256 * q;
            const int ra = ak == 1 ? e >> 5 : e & 63, ca = ak == 1 ? e & 31 : e >> 6;      // (consecutive threads along the contiguous side)
            const int rb = bk == 1 ? e >> 5 : e & 63, cb = bk == 1 ? e & 31 : e >> 6;
            sA[ra * kLd + ca] = m0 + ra < M && k0 + ca < ke ? A[(m0 + ra) * am + (long long)(k0 + ca) * ak] : 0.0f;
            const float b = n0 + rb < N && k0 + cb < ke && (!live || live[k0 + cb] > 0.0f) ? B[(long long)(k0 + cb) * bk + (long long)(n0 + rb) * bn] : 0.0f;
            sB[rb * kLd + cb] = finite && !(fabsf(b) < INFINITY) ? 0.0f : b;
        }
        __syncthreads();
        const float *pa = sA + (wr * 32 + (lane & 31)) * kLd + (lane >> 5), *pb = sB + (wc * 32 + (lane & 31)) * kLd + (lane >> 5);
#pragma unroll
        for (int k = 0; k < kKT; k += 2) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(pa[k], pb[k], acc, 0, 0, 0);
        __syncthreads();
    }
    const int col = n0 + wc * 32 + (lane & 31);
    if (col >= N) return;
    const float b = bias ? bias[col] : 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const long long row = m0 + wr * 32 + (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5);
        if (row < M) {
            float *c = C + row * cm + col;
            *c = accumulate ? *c + acc[r] : acc[r] + b;
        }
    }
}

// One workgroup per row of a block: lse and loss; for the gradients the row of scores becomes the row of dz.
__global__ void __launch_bounds__(256) softmax_rows_kernel(const rfm_distill_args a, long long row0, float *__restrict__ z, const float *__restrict__ part,
                                                           const float *__restrict__ mass, const int32_t *__restrict__ merged_item,
                                                           const float *__restrict__ merged_p) {
    __shared__ float sm[4], sl[4];
    const long long r = row0 + blockIdx.x;
    float *row = z + (size_t)blockIdx.x * a.n_items;
    const float c = 1.0f / a.temperature;
    bool bad = false;
    const uint32_t *mask = row_mask(a, r, &bad);
    float m = -INFINITY, l = 0.0f;
    bool nan = false;
    for (int i = threadIdx.x; i < a.n_items; i += 256) {
        const bool ok = !mask || ((mask[i >> 5] >> (i & 31)) & 1u);
        const float x = ok ? row[i] * c : -INFINITY;
        nan |= isnan(x);
        if (x > m) { l = l * expf(m - x) + 1.0f; m = x; }
        else if (x > -INFINITY) l += expf(x - m);
    }
    const float wm = wave_max(m);
    l = wave_sum(m > -INFINITY ? l * expf(m - wm) : 0.0f);
    if (__any(nan)) l = __uint_as_float(0x7fc00000u);
    if ((threadIdx.x & 63) == 0) { sm[threadIdx.x >> 6] = wm; sl[threadIdx.x >> 6] = l; }
    __syncthreads();
    m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    l = 0.0f;
    for (int w = 0; w < 4; ++w) l += sm[w] > -INFINITY || isnan(sl[w]) ? sl[w] * expf(sm[w] - m) : 0.0f;
    const float log_l = logf(l), has = mass[r];                  // (m and log l apart: their sum would lose what m is rounded to)
    if (threadIdx.x == 0) a.loss[r] = has == 0.0f ? 0.0f : a.temperature * (a.temperature * (part[r] + has * (m + log_l)));
    if (!a.d_users) return;
    const float coef = a.temperature * (a.row_weight ? a.row_weight[r] : 1.0f);
    for (int i = threadIdx.x; i < a.n_items; i += 256) {
        const bool ok = !mask || ((mask[i >> 5] >> (i & 31)) & 1u);
        row[i] = has == 0.0f || bad || !ok ? 0.0f : coef * expf((row[i] * c - m) - log_l);
    }
    __syncthreads();
    for (int j = threadIdx.x; j < a.n_teacher; j += 256) {
        const int i = merged_item[(size_t)r * a.n_teacher + j];
        if (i >= 0) row[i] -= coef * merged_p[(size_t)r * a.n_teacher + j];
    }
}

__global__ void __launch_bounds__(256) column_sum_kernel(const float *__restrict__ dz, long long rows, int n_items, float *__restrict__ out, int accumulate) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= n_items) return;
    float s = accumulate ? out[i] : 0.0f;
    for (long long r = 0; r < rows; ++r) s += dz[(size_t)r * n_items + i];
    out[i] = s;
}

__global__ void __launch_bounds__(256) sum_slices_kernel(const float *__restrict__ part, long long n, int slices, float *__restrict__ out) {
    for (long long k = (long long)blockIdx.x * 256 + threadIdx.x; k < n; k += (long long)gridDim.x * 256) {
        float s = part[k];
        for (int q = 1; q < slices; ++q) s += part[(size_t)q * n + k];
        out[k] = s;
    }
}

}  // namespace distill
}  // namespace rfm

#include "rfm_distill_fused.hpp"

namespace rfm {
namespace distill {

static int check(const rfm_distill_args *a) {
    if (!a || a->n_rows < 0 || a->n_items < 1 || a->n_factors < 1 || a->n_teacher < 1) return RFM_ERR_BAD_ARG;
    if (!(a->temperature >= 0x1p-126f && a->temperature < INFINITY)) return RFM_ERR_BAD_ARG;      // (below, its inverse is infinite)
    if (a->user_stride < a->n_factors || a->item_stride < a->n_factors) return RFM_ERR_BAD_ARG;
    if (a->allowed && (a->n_allowed < 1 || (!a->allowed_rows && a->n_allowed != 1 && a->n_allowed < a->n_rows))) return RFM_ERR_BAD_ARG;
    if (!a->d_users != !a->d_items || (a->d_bias && !a->d_items)) return RFM_ERR_BAD_ARG;
    if (a->n_factors > 1024 || a->n_teacher > kMaxTeacher || a->n_items > (1 << 25) || a->n_rows > (1 << 24)) return RFM_ERR_UNSUPPORTED;      // (launches stay below 2^32 threads)
    return RFM_OK;
}

static size_t up(size_t bytes) { return (bytes + 255) & ~(size_t)255; }

// The fused path holds a wavefront's factors and sums in registers.
static bool fused(const rfm_distill_args *a) { return a->n_factors <= 128; }

struct MatrixLayout {
    long long block;                             // rows whose scores are kept at once
    int slices;                                  // of the items, for the users' gradient
    size_t part, mass, merged_item, merged_p, z, d_part, bytes;
};
static MatrixLayout matrix_layout(const rfm_distill_args *a) {
    MatrixLayout w;
    const size_t R = (size_t)a->n_rows, I = (size_t)a->n_items, n = (size_t)a->n_teacher;
    w.block = std::max<long long>(64, std::min<long long>(4096, ((long long)1 << 28) / a->n_items));
    w.block = std::min<long long>(w.block, std::max<long long>(1, a->n_rows));
    w.slices = (int)std::max<size_t>(1, std::min<size_t>(16, I / 2048));
    size_t off = 0;
    auto take = [&](size_t bytes) { const size_t at = off; off += up(bytes ? bytes : 1); return at; };
    const bool grad = a->d_users != nullptr;
    w.part = take(4 * R); w.mass = take(4 * R);
    w.merged_item = take(grad ? 4 * R * n : 0); w.merged_p = take(grad ? 4 * R * n : 0);
    w.z = take(4 * (size_t)w.block * I);
    w.d_part = take(grad ? 4 * (size_t)w.slices * (size_t)w.block * (size_t)a->n_factors : 0);
    w.bytes = off;
    return w;
}

static int run_matrix(const rfm_distill_args *a, char *base, hipStream_t stream) {
    const MatrixLayout w = matrix_layout(a);
    const bool grad = a->d_users != nullptr;
    float *part = (float *)(base + w.part), *mass = (float *)(base + w.mass), *z = (float *)(base + w.z), *d_part = (float *)(base + w.d_part);
    int32_t *mi = grad ? (int32_t *)(base + w.merged_item) : nullptr;
    float *mp = grad ? (float *)(base + w.merged_p) : nullptr;
    const int I = a->n_items, K = a->n_factors;
    teacher_kernel<<<dim3((unsigned)((a->n_rows + 3) / 4)), dim3(256), (size_t)a->n_teacher * 2 * 4 * 4, stream>>>(*a, part, mass, mi, mp);
    const int it = (I + 63) / 64, kt = (K + 63) / 64;
    const int slice = ((I + w.slices - 1) / w.slices + 31) / 32 * 32;
    const int slices = (I + slice - 1) / slice;
    for (long long r0 = 0; r0 < a->n_rows; r0 += w.block) {
        const long long nr = std::min<long long>(w.block, a->n_rows - r0);
        const float *u = a->users + (size_t)r0 * a->user_stride;
        const unsigned rt = (unsigned)((nr + 63) / 64);
        const int more = r0 > 0;
        gemm_kernel<<<dim3(rt * (unsigned)it), dim3(256), 0, stream>>>(u, a->user_stride, 1, a->items, 1, a->item_stride, a->bias, z, I, 0, nr, I, K, K, it, 0, nullptr, 0);
        softmax_rows_kernel<<<dim3((unsigned)nr), dim3(256), 0, stream>>>(*a, r0, z, part, mass, mi, mp);
        if (!grad) continue;
        gemm_kernel<<<dim3(rt * (unsigned)kt, (unsigned)slices), dim3(256), 0, stream>>>(z, I, 1, a->items, a->item_stride, 1, nullptr, d_part, K, nr * K, nr, K, I, slice, kt, 0, nullptr, 1);
        sum_slices_kernel<<<dim3(1024), dim3(256), 0, stream>>>(d_part, nr * K, slices, a->d_users + (size_t)r0 * K);
        gemm_kernel<<<dim3((unsigned)it * (unsigned)kt), dim3(256), 0, stream>>>(z, 1, I, u, a->user_stride, 1, nullptr, a->d_items, K, 0, I, K, (int)nr, 1 << 20, kt, more, mass + r0, 1);
        if (a->d_bias) column_sum_kernel<<<dim3((unsigned)((I + 255) / 256)), dim3(256), 0, stream>>>(z, nr, I, a->d_bias, more);
    }
    return RFM_OK;
}

// How often the streamed tiles are split: workgroups run `slots` at a time, a workgroup costs its tiles and about four more to start and end,
// a split costs its partial sums.  The cheapest count wins; the sums of a count are always joined in the same order.
constexpr int kCus = 256;
static int pick_splits(int blocks, int tiles, int slots) {
    int best = 1;
    double least = 1e30;
    for (int s = 1; s <= 256 && s <= std::max(1, tiles / 2); ++s) {
        const int chunk = (tiles + s - 1) / s, used = (tiles + chunk - 1) / chunk;
        if (used != s) continue;
        const double rounds = (double)(((long long)blocks * s + slots - 1) / slots);
        const double cost = rounds * (chunk + 4) + 0.25 * s;
        if (cost < least) { least = cost; best = s; }
    }
    return best;
}

struct FusedLayout {
    int kp, few, columns, block_tiles, user_tiles, item_tiles, user_blocks, item_blocks, splits_f, lanes_f, groups_i, units_i;
    size_t part, mass, ids, ps, acc, user_frag, user_frag_t, item_frag, item_frag_t, item_data, user_data, user_data_t, mask_row, part_m, part_l, part_o, entry, entry_at, part_items, part_bias, bytes;
};
static FusedLayout fused_layout(const rfm_distill_args *a) {
    FusedLayout w;
    const bool grad = a->d_users != nullptr;
    w.kp = (a->n_factors + 31) / 32 * 32;
    const size_t R = (size_t)a->n_rows, n = (size_t)a->n_teacher, kp = (size_t)w.kp;
    w.user_tiles = (int)((a->n_rows + 31) / 32);
    w.item_tiles = (a->n_items + 31) / 32;
    // Few users: no copies of the items' table are made (thin_forward_kernel).  Measured with copies / without, us, gradients of 29 rows: k = 20, 6 k items
    // 25.7 / 26.4, 190 k 73 / 43; k = 64, 6 k 28.8 / 31.6, 10 k 35.7 / 33.6, 150 k 88 / 60; k = 128, 6 k 42.0 / 50.4, 20 k 59.5 / 57.7, 150 k 151 / 109; the loss
    // alone, k = 64: 2 k 14.3 / 14.7, 3.7 k 14.8 / 14.8, 150 k 46 / 25.  With three or four tiles of users they come out even, at any size.
    const bool thin = w.user_tiles <= 2 && w.item_tiles >= (grad ? 5 * w.kp : w.kp + 64);
    w.few = thin ? w.user_tiles : 0;
    // Column tiles per wavefront: two read LDS half as often, one leaves more workgroups to spread.  Measured with two against one, k = 64, gradients / loss
    // alone: 512 rows x 50 k items 1.10 / 1.13, 2048 x 50 k 1.01 / 0.96, 4096 x 20 k 1.00 / 0.95, 4096 x 50 k 0.95 / 0.93, 2048 x 200 k 0.96 / 0.93; k = 20
    // crosses at the same place; with masks one is the faster throughout (2048 x 50 k 1.06).
    w.columns = !thin && w.kp <= 64 && !a->allowed && (long long)w.user_tiles * w.item_tiles >= (1 << 17) ? 2 : 1;
    w.block_tiles = (w.kp <= 64 ? 4 : 8) * w.columns;
    w.user_blocks = (w.user_tiles + w.block_tiles - 1) / w.block_tiles;
    w.item_blocks = (w.item_tiles + w.block_tiles - 1) / w.block_tiles;
    // workgroups that fit on the chip at once, by registers and LDS (the loss alone needs fewer of both)
    const int slots = kCus * (w.kp > 64 ? 1 : w.columns == 2 ? 2 : 3), slots_loss = kCus * (w.kp <= 64 && w.columns == 1 ? 4 : 2);
    const int slots_f = grad ? slots : slots_loss;
    w.splits_f = pick_splits(w.user_blocks, w.item_tiles, slots_f);
    // a multiple of the 8 XCDs, where that takes no more rounds
    const int even = (w.splits_f + 7) / 8 * 8;
    auto rounds = [&](int each) { return ((long long)w.user_blocks * each + slots_f - 1) / slots_f; };
    w.lanes_f = rounds(even) == rounds(w.splits_f) ? even : w.splits_f;
    if (w.few) {                                 // workgroups, each with 8 / few tiles of items at a time
        const int at_once = kThinWaves / w.few;
        w.splits_f = w.lanes_f = std::min(kCus, (w.item_tiles + at_once - 1) / at_once);
    }
    // items_kernel: equal ranges for the workgroups that fit on the chip at once, no shorter than 4 tiles (or a block, if that is less)
    const long long units = (long long)w.item_blocks * w.user_tiles;
    w.units_i = (int)std::max<long long>((units + slots - 1) / slots, std::min(w.user_tiles, 4));
    w.groups_i = (int)((units + w.units_i - 1) / w.units_i);
    const size_t ur = (size_t)w.user_tiles * 32, ir = (size_t)w.item_tiles * 32;
    size_t off = 0;
    auto take = [&](size_t bytes) { const size_t at = off; off += up(bytes ? bytes : 1); return at; };
    w.part = take(4 * R); w.mass = take(4 * R);
    w.ids = take(grad ? 4 * R * n : 0); w.ps = take(grad ? 4 * R * n : 0); w.acc = take(grad ? 4 * R * kp : 0);
    w.user_frag = take(4 * ur * kp); w.item_frag = take(w.few ? 0 : 4 * ir * kp);
    w.user_frag_t = take(grad ? 4 * ur * kp : 0); w.item_frag_t = take(grad && !w.few ? 4 * ir * kp : 0);
    w.item_data = take((size_t)w.item_tiles * kItemData * 4); w.user_data = take((size_t)w.user_tiles * kUserData * 4); w.user_data_t = take((size_t)w.user_tiles * kUserData * 4);
    w.mask_row = take(a->allowed ? 4 * ur : 0);
    w.part_m = take(4 * w.splits_f * ur); w.part_l = take(4 * w.splits_f * ur); w.part_o = take(grad ? 4 * w.splits_f * ur * kp : 0);
    w.entry = take(grad ? ur * n * 8 : 0); w.entry_at = take(grad ? 4 * (size_t)w.user_tiles * (kBuckets + 1) : 0);
    const size_t parts = (size_t)(w.groups_i + w.item_blocks) * w.block_tiles * 32;
    w.part_items = take(grad ? 4 * parts * kp : 0); w.part_bias = take(grad ? 4 * parts : 0);
    w.bytes = off;
    return w;
}

template <int KP, int NC>
static int run_fused(const rfm_distill_args *a, const FusedLayout &w, char *base, hipStream_t stream) {
    const bool grad = a->d_users != nullptr;
    auto at = [&](size_t off) { return base + off; };
    float *part = (float *)at(w.part), *mass = (float *)at(w.mass), *acc = (float *)at(w.acc), *ps = (float *)at(w.ps);
    int32_t *ids = (int32_t *)at(w.ids);
    FusedArgs f = {};
    f.a = *a;
    f.user_tiles = w.user_tiles; f.item_tiles = w.item_tiles; f.item_blocks = w.item_blocks;
    f.user_frag = at(w.user_frag); f.user_frag_t = at(w.user_frag_t); f.item_frag = at(w.item_frag); f.item_frag_t = at(w.item_frag_t);
    f.item_data = (float *)at(w.item_data); f.user_data = (float *)at(w.user_data); f.user_data_t = (float *)at(w.user_data_t); f.mask_row = (int32_t *)at(w.mask_row);
    f.part_m = (float *)at(w.part_m); f.part_l = (float *)at(w.part_l); f.part_o = (float *)at(w.part_o);
    f.entry = (uint2 *)at(w.entry); f.entry_at = (int32_t *)at(w.entry_at);
    f.part_items = (float *)at(w.part_items); f.part_bias = (float *)at(w.part_bias);
    const float c = 1.4426950408889634f / a->temperature;
    f.c = c;
    f.few = w.few;
    const size_t lds = (size_t)a->n_teacher * 2 * 4 * 4;
    const dim3 grid_p((unsigned)(w.user_tiles + (w.few ? 0 : w.item_tiles) + (a->n_rows + 3) / 4));
    if (grad) prepare_kernel<KP, true><<<grid_p, dim3(256), lds, stream>>>(f, c, part, mass, ids, ps, acc);
    else prepare_kernel<KP, false><<<grid_p, dim3(256), lds, stream>>>(f, c, part, mass, nullptr, nullptr, nullptr);
    f.splits = w.splits_f;
    f.chunk = (w.item_tiles + w.splits_f - 1) / w.splits_f;
    f.lanes = w.lanes_f;
    const dim3 grid_f((unsigned)(w.user_blocks * w.lanes_f)), threads(Frag<KP>::waves * 64);
    if (w.few) {
        if constexpr (NC == 1) {
            const dim3 grid_t((unsigned)w.splits_f), threads_t(kThinWaves * 64);
            if (grad && a->allowed) thin_forward_kernel<KP, true, true><<<grid_t, threads_t, 0, stream>>>(f);
            if (!grad && a->allowed) thin_forward_kernel<KP, false, true><<<grid_t, threads_t, 0, stream>>>(f);
            if (grad && !a->allowed) thin_forward_kernel<KP, true, false><<<grid_t, threads_t, 0, stream>>>(f);
            if (!grad && !a->allowed) thin_forward_kernel<KP, false, false><<<grid_t, threads_t, 0, stream>>>(f);
        }
    } else {
        if constexpr (NC == 1) {
            if (grad && a->allowed) forward_kernel<KP, NC, true, true><<<grid_f, threads, 0, stream>>>(f);
            if (!grad && a->allowed) forward_kernel<KP, NC, false, true><<<grid_f, threads, 0, stream>>>(f);
        }
        if (grad && !a->allowed) forward_kernel<KP, NC, true, false><<<grid_f, threads, 0, stream>>>(f);
        if (!grad && !a->allowed) forward_kernel<KP, NC, false, false><<<grid_f, threads, 0, stream>>>(f);
    }
    const bool wide = w.user_tiles <= 8 && w.splits_f > 64;      // (few rows, many splits)
    const int row_blocks = w.user_tiles * (wide ? 32 : 4);
    const dim3 grid_j((unsigned)(row_blocks + (grad ? w.user_tiles : 0)));
    if (wide) join_rows_kernel<KP, 8><<<grid_j, dim3(512), 0, stream>>>(f, row_blocks, w.block_tiles * 32, part, mass, acc, ids, ps);
    else join_rows_kernel<KP, 1><<<grid_j, dim3(512), 0, stream>>>(f, row_blocks, w.block_tiles * 32, part, mass, acc, ids, ps);
    if (!grad) return RFM_OK;
    f.units = w.units_i;
    const dim3 grid_i((unsigned)w.groups_i);
    if constexpr (NC == 1) {
        if (w.few && a->allowed) items_kernel<KP, NC, true, true><<<grid_i, threads, 0, stream>>>(f);
        if (w.few && !a->allowed) items_kernel<KP, NC, false, true><<<grid_i, threads, 0, stream>>>(f);
        if (!w.few && a->allowed) items_kernel<KP, NC, true><<<grid_i, threads, 0, stream>>>(f);
    }
    if (!w.few && !a->allowed) items_kernel<KP, NC, false><<<grid_i, threads, 0, stream>>>(f);
    // (a block is cut where a range ends inside it)
    if (w.groups_i > 1 && w.units_i % w.user_tiles != 0) join_items_kernel<KP><<<dim3((unsigned)(w.item_blocks * w.block_tiles)), dim3(256), 0, stream>>>(f, w.block_tiles);
    return RFM_OK;
}

}  // namespace distill
}  // namespace rfm

using namespace rfm;

extern "C" {

size_t rfm_distill_workspace_bytes(const rfm_distill_args *a) {
    if (distill::check(a) != RFM_OK) return 0;
    return distill::fused(a) ? distill::fused_layout(a).bytes : distill::matrix_layout(a).bytes;
}

int rfm_distill_device(const rfm_distill_args *a, void *workspace, size_t workspace_bytes, void *hip_stream) {
    int rc = distill::check(a);
    if (rc != RFM_OK) return rc;
    hipStream_t stream = (hipStream_t)hip_stream;
    if (!a->items || (a->n_rows > 0 && (!a->users || !a->teacher_items || !a->teacher_scores || !a->loss))) return RFM_ERR_BAD_ARG;
    if (!workspace || workspace_bytes < rfm_distill_workspace_bytes(a)) return RFM_ERR_WORKSPACE;
    if (a->n_rows == 0) {                        // nothing to learn from: the items' gradients are zero
        if (a->d_items) distill::zero_kernel<<<dim3(1024), dim3(256), 0, stream>>>(a->d_items, (long long)a->n_items * a->n_factors);
        if (a->d_bias) distill::zero_kernel<<<dim3(1024), dim3(256), 0, stream>>>(a->d_bias, a->n_items);
    } else if (!distill::fused(a)) {
        rc = distill::run_matrix(a, (char *)workspace, stream);
    } else {
        const distill::FusedLayout w = distill::fused_layout(a);
        char *base = (char *)workspace;
        if (w.kp == 32) rc = w.columns == 2 ? distill::run_fused<32, 2>(a, w, base, stream) : distill::run_fused<32, 1>(a, w, base, stream);
        else if (w.kp == 64) rc = w.columns == 2 ? distill::run_fused<64, 2>(a, w, base, stream) : distill::run_fused<64, 1>(a, w, base, stream);
        else if (w.kp == 96) rc = distill::run_fused<96, 1>(a, w, base, stream);
        else rc = distill::run_fused<128, 1>(a, w, base, stream);
    }
    if (rc != RFM_OK) return rc;
    return hipGetLastError() == hipSuccess ? RFM_OK : RFM_ERR_HIP;
}

}  // extern "C"
