// rfm_distill.hip -- learning from another model's top scores: the loss of a student's catalogue distribution against a teacher's lists, and
// its gradients (include/rankfm_hip.h rfm_distill_device).
//
//   z[r, i] = < users[r], items[i] > + bias[i],  q = softmax(z / tau) over the allowed items,  p = softmax(teacher / tau) over usable entries
//   loss[r] = tau^2 sum_j p_j (log p_j - z[r, t_j] / tau + lse_r),   lse_r = log sum_i exp(z[r, i] / tau)
//   dz = tau * weight[r] * (q - p);   d_users = dz . items;   d_items = dz^T . users;   d_bias = column sums of dz
//
// The matrix path: the scores of a block of rows are written out, turned into dz in place and multiplied; every sum has a fixed order.
#include <hip/hip_runtime.h>
#include <math.h>

#include <algorithm>

#include "../../include/rankfm_hip.h"

namespace rfm {
namespace distill {

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

// One wavefront per row: the teacher's distribution over the usable entries, and its part of the loss.
//   part[r] = sum_j p_j (log p_j - z[r, t_j] / tau)     mass[r] = 1, 0 without a usable entry, NaN where the row's mask does not exist
// For the gradients the list is left merged: an item's first entry holds the sum of its entries' p, the others are off (-1, 0), so that no
// two entries of a row meet in one element of dz.
__global__ void __launch_bounds__(256) teacher_kernel(const rfm_distill_args a, float *__restrict__ part, float *__restrict__ mass, int32_t *__restrict__ merged_item,
                                                      float *__restrict__ merged_p) {
    extern __shared__ int s_dyn[];               // per wavefront: ids [n], p [n]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = a.n_teacher;
    const long long r = (long long)blockIdx.x * 4 + wave;
    if (r >= a.n_rows) return;                   // (no barrier below: a wavefront works by itself)
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
        const bool use = i >= 0 && i < a.n_items && !(t == -INFINITY) && (!mask || ((mask[i >> 5] >> (i & 31)) & 1u));
        id[j] = use ? i : -1;
        if (use) { some = 1; nan |= isnan(t); top = fmaxf(top, t); }
    }
    some = __any(some);
    if (__any(nan)) top = __uint_as_float(0x7fc00000u);
    top = wave_max(top);
    if (__any(isnan(top))) top = __uint_as_float(0x7fc00000u);
    float sum = 0.0f;
    for (int j = lane; j < n; j += 64) {
        const float e = id[j] >= 0 ? expf((ts[j] - top) * inv_tau) : 0.0f;
        pr[j] = e;
        sum += e;
    }
    sum = wave_sum(sum);
    const float log_sum = logf(sum), inv = 1.0f / sum;
    // the student's scores of the entries: one dot product per entry, 16 lanes each
    const float *u = a.users + (size_t)r * a.user_stride;
    const int sub = lane & 15, grp = lane >> 4;
    float acc = 0.0f;
    for (int j0 = 0; j0 < n; j0 += 4) {
        const int j = j0 + grp;
        const int i = j < n ? id[j] : -1;
        float d = 0.0f;
        if (i >= 0) {
            const float *v = a.items + (size_t)i * a.item_stride;
            for (int f = sub; f < a.n_factors; f += 16) d = fmaf(u[f], v[f], d);
        }
#pragma unroll
        for (int m = 8; m > 0; m >>= 1) d += __shfl_xor(d, m);
        if (i >= 0 && sub == 0) {
            const float e = pr[j], z = d + (a.bias ? a.bias[i] : 0.0f);
            if (!(e == 0.0f)) acc += e * inv * ((ts[j] - top) * inv_tau - log_sum - z * inv_tau);
        }
    }
    acc = wave_sum(acc);
    if (lane == 0) {
        part[r] = some ? acc : 0.0f;
        mass[r] = bad ? __uint_as_float(0x7fc00000u) : some ? 1.0f : 0.0f;
    }
    if (!merged_item) return;
    for (int j = lane; j < n; j += 64) {
        int i = id[j];
        float p = i >= 0 ? pr[j] * inv : 0.0f;
        if (i >= 0) {
            bool first = true;
            for (int k = 0; k < j; ++k) first &= id[k] != i;
            if (first) {
                for (int k = j + 1; k < n; ++k)
                    if (id[k] == i) p += pr[k] * inv;
            } else { i = -1; p = 0.0f; }
        }
        merged_item[(size_t)r * n + j] = bad ? -1 : i;
        merged_p[(size_t)r * n + j] = p;
    }
}

// C[m, n] (+)= sum_k A[m, k] B[k, n] (+ bias[n]), any strides; slices of k (blockIdx.y) go to slices of C.  64 x 64 tile per workgroup, four
// wavefronts of one 32 x 32 accumulator each (v_mfma_f32_32x32x2_f32, exact fp32), k in LDS stages of 32.
typedef float f32x16 __attribute__((ext_vector_type(16)));
constexpr int kKT = 32, kLd = kKT + 1;
__global__ void __launch_bounds__(256) gemm_kernel(const float *__restrict__ A, long long am, long long ak, const float *__restrict__ B, long long bk, long long bn,
                                                   const float *__restrict__ bias, float *__restrict__ C, long long cm, long long slice_stride, long long M, int N, int K,
                                                   int k_slice, int n_tiles, int accumulate) {
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
            sB[rb * kLd + cb] = n0 + rb < N && k0 + cb < ke ? B[(long long)(k0 + cb) * bk + (long long)(n0 + rb) * bn] : 0.0f;
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
    const float lse = m + logf(l), has = mass[r];
    if (threadIdx.x == 0) a.loss[r] = has == 0.0f ? 0.0f : a.temperature * a.temperature * (part[r] + has * lse);
    if (!a.d_users) return;
    const float coef = a.temperature * (a.row_weight ? a.row_weight[r] : 1.0f);
    for (int i = threadIdx.x; i < a.n_items; i += 256) {
        const bool ok = !mask || ((mask[i >> 5] >> (i & 31)) & 1u);
        row[i] = has == 0.0f || bad || !ok ? 0.0f : coef * expf(row[i] * c - lse);
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

static int check(const rfm_distill_args *a) {
    if (!a || a->n_rows < 0 || a->n_items < 1 || a->n_factors < 1 || a->n_teacher < 1) return RFM_ERR_BAD_ARG;
    if (!(a->temperature > 0.0f && a->temperature < INFINITY)) return RFM_ERR_BAD_ARG;
    if (a->user_stride < a->n_factors || a->item_stride < a->n_factors) return RFM_ERR_BAD_ARG;
    if (a->allowed && (a->n_allowed < 1 || (!a->allowed_rows && a->n_allowed != 1 && a->n_allowed < a->n_rows))) return RFM_ERR_BAD_ARG;
    if (!a->d_users != !a->d_items || (a->d_bias && !a->d_items)) return RFM_ERR_BAD_ARG;
    if (a->n_factors > 1024 || a->n_teacher > kMaxTeacher || a->n_items > 0x7fffff00 || a->n_rows > 0x7fffff00) return RFM_ERR_UNSUPPORTED;
    return RFM_OK;
}

static size_t up(size_t bytes) { return (bytes + 255) & ~(size_t)255; }

struct Layout {
    long long block;                             // rows whose scores are kept at once
    int slices;                                  // of the items, for the users' gradient
    size_t part, mass, merged_item, merged_p, z, d_part, bytes;
};
static Layout layout(const rfm_distill_args *a) {
    Layout w;
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

}  // namespace distill
}  // namespace rfm

using namespace rfm;

extern "C" {

size_t rfm_distill_workspace_bytes(const rfm_distill_args *a) { return distill::check(a) == RFM_OK ? distill::layout(a).bytes : 0; }

int rfm_distill_device(const rfm_distill_args *a, void *workspace, size_t workspace_bytes, void *hip_stream) {
    const int rc = distill::check(a);
    if (rc != RFM_OK) return rc;
    hipStream_t stream = (hipStream_t)hip_stream;
    const bool grad = a->d_users != nullptr;
    if (!a->items || (a->n_rows > 0 && (!a->users || !a->teacher_items || !a->teacher_scores || !a->loss))) return RFM_ERR_BAD_ARG;
    const distill::Layout w = distill::layout(a);
    if (!workspace || workspace_bytes < w.bytes) return RFM_ERR_WORKSPACE;
    char *base = (char *)workspace;
    float *part = (float *)(base + w.part), *mass = (float *)(base + w.mass), *z = (float *)(base + w.z), *d_part = (float *)(base + w.d_part);
    int32_t *mi = grad ? (int32_t *)(base + w.merged_item) : nullptr;
    float *mp = grad ? (float *)(base + w.merged_p) : nullptr;
    const int I = a->n_items, K = a->n_factors;
    if (a->n_rows > 0)
        distill::teacher_kernel<<<dim3((unsigned)((a->n_rows + 3) / 4)), dim3(256), (size_t)a->n_teacher * 2 * 4 * 4, stream>>>(*a, part, mass, mi, mp);
    const int it = (I + 63) / 64, kt = (K + 63) / 64;
    const int slice = ((I + w.slices - 1) / w.slices + 31) / 32 * 32;
    const int slices = (I + slice - 1) / slice;
    for (long long r0 = 0; r0 < std::max<int64_t>(a->n_rows, grad ? 1 : 0); r0 += w.block) {      // (no rows at all: the items' gradients are still set, to zero)
        const long long nr = std::min<long long>(w.block, a->n_rows - r0);
        const float *u = a->users + (size_t)r0 * a->user_stride;
        if (nr > 0) {
            const unsigned rt = (unsigned)((nr + 63) / 64);
            distill::gemm_kernel<<<dim3(rt * (unsigned)it), dim3(256), 0, stream>>>(u, a->user_stride, 1, a->items, 1, a->item_stride, a->bias, z, I, 0, nr, I, K, K, it, 0);
            distill::softmax_rows_kernel<<<dim3((unsigned)nr), dim3(256), 0, stream>>>(*a, r0, z, part, mass, mi, mp);
            if (!grad) continue;
            distill::gemm_kernel<<<dim3(rt * (unsigned)kt, (unsigned)slices), dim3(256), 0, stream>>>(z, I, 1, a->items, a->item_stride, 1, nullptr, d_part, K, (long long)nr * K, nr, K,
                                                                                                       I, slice, kt, 0);
            distill::sum_slices_kernel<<<dim3(1024), dim3(256), 0, stream>>>(d_part, nr * K, slices, a->d_users + (size_t)r0 * K);
        }
        const int more = r0 > 0;
        distill::gemm_kernel<<<dim3((unsigned)it * (unsigned)kt), dim3(256), 0, stream>>>(z, 1, I, u, a->user_stride, 1, nullptr, a->d_items, K, 0, I, K, (int)std::max<long long>(nr, 0), 1 << 20, kt,
                                                                                           more);
        if (a->d_bias) distill::column_sum_kernel<<<dim3((unsigned)((I + 255) / 256)), dim3(256), 0, stream>>>(z, std::max<long long>(nr, 0), I, a->d_bias, more);
    }
    return hipGetLastError() == hipSuccess ? RFM_OK : RFM_ERR_HIP;
}

}  // extern "C"
