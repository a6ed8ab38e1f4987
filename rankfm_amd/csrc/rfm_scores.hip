// rfm_scores.hip -- rows of catalogue scores: rules applied to them, and their top entries.
//
//   rfm_adjust_scores_device   s' = rules(s): penalties for items of the row's history, biases, masks of allowed items
//   rfm_top_scores_device      the n best (item, score) of every row, rules applied on the way: the adjusted rows are never written
//
// The rules, for row r and item i with c = the number of times i stands in the row's history (all arithmetic in fp32, each operation
// rounded once and in this order, so that a caller's own elementary operations give the same bits):
//   c > 0:            s = s > 0 ? s / repetition[r] : s * repetition[r];   s = s - frequency[r] * c;   s = s - presence[r]
//   item_bias:        s = s + item_bias[i]
//   row_bias lists i: s = s + the value of the LAST entry of the row's list that names i
//   not allowed:      s = -inf, whatever it was (NaN and +inf included)
#include <hip/hip_runtime.h>
#include <math.h>

#include <algorithm>

#include "../../include/rankfm_hip.h"

namespace rfm {

constexpr int kThreads = 256;
constexpr int kTile = 2048;                      // scores a workgroup holds in registers at a time: 8 per thread
constexpr int kPer = kTile / kThreads;

// one row's share of the rules; every index is checked against the array it points into, so no list can lead a read astray
struct RowRules {
    const int32_t *hist = nullptr;               // the row's history
    long long hist_n = 0;
    const int32_t *bias_item = nullptr;          // the row's own biases
    const float *bias_value = nullptr;
    long long bias_n = 0;
    const uint32_t *mask = nullptr;              // the row's allowed items, one bit each
    float rho = 1.0f, phi = 0.0f, pi = 0.0f;
    bool bad = false;                            // the row names a history or a mask that does not exist: it comes out NaN
};

__device__ __forceinline__ RowRules row_rules(const rfm_score_rules &u, long long r, int n_items) {
    RowRules w;
    if (u.history_offsets) {
        const long long h = u.history_rows ? (long long)u.history_rows[r] : r;
        if (h >= u.n_history) w.bad = true;
        else if (h >= 0) {
            const long long a = max((long long)u.history_offsets[h], 0ll), b = min((long long)u.history_offsets[h + 1], (long long)u.n_history_items);
            w.hist = u.history_items + a;
            w.hist_n = b > a ? b - a : 0;
        }
        w.rho = u.repetition ? u.repetition[r] : u.repetition_all;
        w.phi = u.frequency ? u.frequency[r] : u.frequency_all;
        w.pi = u.presence ? u.presence[r] : u.presence_all;
    }
    if (u.bias_offsets) {
        const long long a = max((long long)u.bias_offsets[r], 0ll), b = min((long long)u.bias_offsets[r + 1], (long long)u.n_bias_items);
        w.bias_item = u.bias_items + a;
        w.bias_value = u.bias_values + a;
        w.bias_n = b > a ? b - a : 0;
    }
    if (u.allowed) {
        const long long m = u.allowed_rows ? (long long)u.allowed_rows[r] : (u.n_allowed == 1 ? 0 : r);
        if (m >= u.n_allowed) w.bad = true;
        else if (m >= 0) w.mask = u.allowed + (size_t)m * (size_t)((n_items + 31) / 32);
    }
    return w;
}

// ---- 16 bytes of a row at a time.  Rows of an odd item count start anywhere: the loads are written for the type's own alignment (the
// ---- hardware takes them at any address; a wavefront's kilobyte then touches nine lines instead of eight).
template <typename T> struct Vec { static constexpr int n = 16 / (int)sizeof(T); };
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Chunk { T v[16 / sizeof(T)]; };

template <typename T>
__device__ __forceinline__ void load_vec(const T *p, float *out) {
    Chunk<T> c;
    __builtin_memcpy(&c, reinterpret_cast<const Chunk<T> *>(p), sizeof(c));
#pragma unroll
    for (int k = 0; k < Vec<T>::n; ++k) out[k] = (float)c.v[k];
}
template <typename T>
__device__ __forceinline__ void store_vec(T *p, const float *in) {
    Chunk<T> c;
#pragma unroll
    for (int k = 0; k < Vec<T>::n; ++k) c.v[k] = (T)in[k];        // the one rounding of an adjusted score
    __builtin_memcpy(reinterpret_cast<Chunk<T> *>(p), &c, sizeof(c));
}

// the eight scores of this thread out of items [first, first + kTile): vector j of the tile belongs to thread j % 256
template <typename T>
__device__ __forceinline__ int element(int slot) {               // position inside the tile of this thread's slot-th score
    constexpr int ve = Vec<T>::n;
    return ((slot / ve) * kThreads + (int)threadIdx.x) * ve + slot % ve;
}
template <typename T>
__device__ __forceinline__ void load_tile(const T *row, int first, int n_items, float *s) {
    constexpr int ve = Vec<T>::n;
#pragma unroll
    for (int j = 0; j < kPer / ve; ++j) {
        const int i = first + (j * kThreads + (int)threadIdx.x) * ve;
        if (i + ve <= n_items) load_vec(row + i, s + j * ve);
        else {
#pragma unroll
            for (int k = 0; k < ve; ++k) s[j * ve + k] = i + k < n_items ? (float)row[i + k] : -INFINITY;
        }
    }
}

// where the row's lists name an item of the tile: count[item] of the history, and 1 + the position of the last bias entry
__device__ __forceinline__ void scan_lists(const RowRules &w, int first, int *count, int *last) {
    for (int k = threadIdx.x; k < kTile; k += kThreads) { count[k] = 0; last[k] = 0; }
    __syncthreads();
    for (long long k = threadIdx.x; k < w.hist_n; k += kThreads) {
        const unsigned at = (unsigned)(w.hist[k] - first);
        if (at < (unsigned)kTile) atomicAdd(count + at, 1);
    }
    for (long long k = threadIdx.x; k < w.bias_n; k += kThreads) {
        const unsigned at = (unsigned)(w.bias_item[k] - first);
        if (at < (unsigned)kTile) atomicMax(last + at, (int)k + 1);
    }
    __syncthreads();
}

template <typename T, bool LISTS>
__device__ __forceinline__ void apply_rules(const rfm_score_rules &u, const RowRules &w, int first, int n_items, const int *count, const int *last, float *s) {
    constexpr int ve = Vec<T>::n;
#pragma unroll
    for (int j = 0; j < kPer / ve; ++j) {
        const int at = (j * kThreads + (int)threadIdx.x) * ve, i = first + at;
        if (i >= n_items) continue;
        unsigned bits = 0xffffffffu;
        if (w.mask) {                                            // the ve items may lie in two words
            const int word = i >> 5, words = (n_items + 31) >> 5;
            const unsigned long long both = ((unsigned long long)w.mask[word + 1 < words ? word + 1 : word] << 32) | w.mask[word];
            bits = (unsigned)(both >> (i & 31));
        }
#pragma unroll
        for (int k = 0; k < ve; ++k) {
            float x = s[j * ve + k];
            if constexpr (LISTS) {
                const int c = count[at + k];
                if (c > 0) {
                    x = x > 0.0f ? x / w.rho : x * w.rho;
                    x = x - w.phi * (float)c;
                    x = x - w.pi;
                }
            }
            if (u.item_bias && i + k < n_items) x = x + u.item_bias[i + k];
            if constexpr (LISTS) {
                const int l = last[at + k];
                if (l > 0) x = x + w.bias_value[l - 1];
            }
            s[j * ve + k] = (bits >> k) & 1u ? x : -INFINITY;
        }
    }
}

// One workgroup per (row, tile of 2048 items): the row is read and written once, which is the floor.  The lists cost a scan per tile.
template <typename T>
__global__ void __launch_bounds__(kThreads) adjust_scores_kernel(const rfm_score_rules u, long long row0, int tiles, int n_items, const T *__restrict__ scores,
                                                                 long long stride, T *out, long long out_stride) {
    __shared__ int count[kTile], last[kTile];
    const long long r = row0 + blockIdx.x / tiles;
    const int first = (int)(blockIdx.x % tiles) * kTile;
    const RowRules w = row_rules(u, r, n_items);
    float s[kPer];
    load_tile(scores + r * stride, first, n_items, s);
    if (w.bad) {
#pragma unroll
        for (int k = 0; k < kPer; ++k) s[k] = __uint_as_float(0x7fc00000u);
    } else if (w.hist_n > 0 || w.bias_n > 0) {
        scan_lists(w, first, count, last);
        apply_rules<T, true>(u, w, first, n_items, count, last, s);
    } else {
        apply_rules<T, false>(u, w, first, n_items, count, last, s);
    }
    constexpr int ve = Vec<T>::n;
    T *o = out + r * out_stride;
#pragma unroll
    for (int j = 0; j < kPer / ve; ++j) {
        const int i = first + (j * kThreads + (int)threadIdx.x) * ve;
        if (i + ve <= n_items) store_vec(o + i, s + j * ve);
        else {
#pragma unroll
            for (int k = 0; k < ve; ++k)
                if (i + k < n_items) o[i + k] = (T)s[j * ve + k];
        }
    }
}

// ---- top scores ---------------------------------------------------------------------------------------------------------------------------
// A score and its item become one 64-bit key that orders like (score descending, item ascending): the score's bits made monotone in the
// upper half (-0 counted as 0), the item's complement in the lower.  0 is no key: NaN and -inf have none and never rank.
typedef unsigned long long u64;
__device__ __forceinline__ unsigned score_key(float x) {
    const unsigned b = __float_as_uint(x + 0.0f);
    return x > -INFINITY ? (b & 0x80000000u ? ~b : b | 0x80000000u) : 0u;      // (false for NaN)
}
__device__ __forceinline__ float key_score(u64 key) {
    const unsigned b = (unsigned)(key >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ int key_item(u64 key) { return (int)~(unsigned)key; }

constexpr int kBuf = 2 * kTile;                  // candidates a workgroup holds: a tile's worth on top of what is kept
constexpr int kRound = 1024;                     // most entries kept at a time; a longer list is taken in rounds of this many
constexpr int kSuper = 4;                        // tiles whose scores are in registers at once

// descending bitonic sort of buf[0 .. p2), p2 a power of two
__device__ __forceinline__ void sort_keys(u64 *buf, int p2) {
    for (int k = 2; k <= p2; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int t = threadIdx.x; t < p2 / 2; t += kThreads) {
                const int i = (t / j) * 2 * j + t % j, l = i + j;
                const u64 a = buf[i], b = buf[l];
                if ((a < b) == ((i & k) == 0)) { buf[i] = b; buf[l] = a; }
            }
            __syncthreads();
        }
}

// keeps the best `keep` of the m candidates, sorted; returns how many there are now.  m <= kBuf.
__device__ __forceinline__ int compact(u64 *buf, int m, int keep) {
    int p2 = 2;
    while (p2 < m) p2 <<= 1;
    for (int k = m + threadIdx.x; k < p2; k += kThreads) buf[k] = 0;
    __syncthreads();
    sort_keys(buf, p2);
    return m < keep ? m : keep;
}

// One workgroup per (row, segment of the row): ONE pass over the scores.  Candidates above the running threshold go to LDS; when they no
// longer fit, they are sorted and the threshold becomes the n-th best.  The first threshold comes from the first 8192 scores: each of the
// 1024 groups of eight holds its maximum in a register, a wavefront finds by bisection over ballots the value that ceil(n / 4) of its group
// maxima reach, and the least of the four wavefronts' values is reached by at least n scores.  So the sort sees a few times n keys, not the
// row.  FROM_KEYS: the "scores" are the sorted keys that the segments of a row left behind.
template <typename T, bool RULED, bool FROM_KEYS>
__global__ void __launch_bounds__(kThreads) top_scores_kernel(const rfm_score_rules u, long long row0, int segments, int segment, int n_items,
                                                              const T *__restrict__ scores, long long stride, const u64 *__restrict__ keys_in, int n_keys,
                                                              int n, u64 *__restrict__ keys_out, int32_t *__restrict__ items, float *__restrict__ values) {
    __shared__ u64 buf[kBuf];
    __shared__ int count[RULED ? kTile : 1], last[RULED ? kTile : 1];
    __shared__ int appended[3];
    __shared__ unsigned wave_t[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long r = row0 + blockIdx.x / segments;
    const int seg = (int)(blockIdx.x % segments);
    const int begin = FROM_KEYS ? 0 : seg * segment, end = FROM_KEYS ? n_keys : min(n_items - begin, segment) + begin;
    RowRules w;
    if constexpr (RULED) w = row_rules(u, r, n_items);
    const bool lists = RULED && (w.hist_n > 0 || w.bias_n > 0);
    const T *row = FROM_KEYS ? nullptr : scores + r * stride;
    const u64 *krow = FROM_KEYS ? keys_in + (size_t)(r - row0) * n_keys : nullptr;
    u64 ceiling = ~0ull;                                         // keys of earlier rounds are at or above it
    for (int base = 0; base < n; base += kRound) {
        const int want = min(n - base, kRound);
        u64 thr = 0;                                             // a key passes when it is above
        int m = 0, step = 0;
        if (threadIdx.x < 3) appended[threadIdx.x] = 0;
        __syncthreads();
        for (int t0 = begin; t0 < end && !(RULED && w.bad); t0 += kSuper * kTile) {
            u64 key[kSuper * kPer];
#pragma unroll
            for (int q = 0; q < kSuper; ++q) {
                const int first = t0 + q * kTile;
                if constexpr (FROM_KEYS) {
#pragma unroll
                    for (int k = 0; k < kPer; ++k) {
                        const int e = first + k * kThreads + (int)threadIdx.x;
                        const u64 x = e < end ? krow[e] : 0;
                        key[q * kPer + k] = x < ceiling ? x : 0;
                    }
                } else {
                    float s[kPer];
#pragma unroll
                    for (int k = 0; k < kPer; ++k) s[k] = -INFINITY;
                    if (first < end) {
                        load_tile(row, first, end, s);
                        if constexpr (RULED) {
                            if (lists) {
                                scan_lists(w, first, count, last);
                                apply_rules<T, true>(u, w, first, n_items, count, last, s);
                                __syncthreads();                 // (the next tile's scan clears the counts)
                            } else apply_rules<T, false>(u, w, first, n_items, count, last, s);
                        }
                    }
#pragma unroll
                    for (int k = 0; k < kPer; ++k) {
                        const int i = first + element<T>(k);
                        const unsigned v = i < end ? score_key(s[k]) : 0u;
                        const u64 x = v ? ((u64)v << 32) | (unsigned)~i : 0;
                        key[q * kPer + k] = x < ceiling ? x : 0;
                    }
                }
            }
            if (t0 == begin) {                                   // the first threshold
                unsigned g[kSuper];
#pragma unroll
                for (int q = 0; q < kSuper; ++q) {
                    g[q] = 0;
#pragma unroll
                    for (int k = 0; k < kPer; ++k) g[q] = max(g[q], (unsigned)(key[q * kPer + k] >> 32));
                }
                const int need = (want + 3) / 4;
                if (need <= 32) { g[0] = max(max(g[0], g[1]), max(g[2], g[3])); g[1] = g[2] = g[3] = 0; }
                unsigned t = 0;
                for (int bit = 31; bit >= 0; --bit) {
                    const unsigned c = t | (1u << bit);
                    int reach = 0;
#pragma unroll
                    for (int q = 0; q < kSuper; ++q) reach += __popcll(__ballot(g[q] >= c));
                    if (reach >= need) t = c;
                }
                if (lane == 0) wave_t[wave] = t;
                __syncthreads();
                t = min(min(wave_t[0], wave_t[1]), min(wave_t[2], wave_t[3]));
                thr = t ? ((u64)t << 32) - 1 : 0;
            }
#pragma unroll
            for (int q = 0; q < kSuper; ++q) {                   // at most kTile of them pass, and there is room for that many
                if (t0 + q * kTile >= end) break;                // (the same for all)
                const int slot = step % 3;
                if (threadIdx.x == 0) appended[(step + 1) % 3] = 0;
                int mine = 0;
#pragma unroll
                for (int k = 0; k < kPer; ++k) mine += key[q * kPer + k] > thr;
                int before = mine;                               // inclusive prefix over the wavefront
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) {
                    const int o = __shfl_up(before, d);
                    if (lane >= d) before += o;
                }
                const int total = __shfl(before, 63);
                if (total > 0) {
                    int at = 0;
                    if (lane == 63) at = atomicAdd(appended + slot, total);
                    at = m + __shfl(at, 63) + before - mine;
#pragma unroll
                    for (int k = 0; k < kPer; ++k)
                        if (key[q * kPer + k] > thr) buf[at++] = key[q * kPer + k];
                }
                __syncthreads();
                m += appended[slot];
                ++step;
                if (m > kBuf - kTile) {
                    m = compact(buf, m, want);
                    if (m == want) thr = buf[want - 1];
                    __syncthreads();
                }
            }
        }
        __syncthreads();
        m = compact(buf, m, want);
        const size_t row_out = FROM_KEYS || segments == 1 ? (size_t)r * n : ((size_t)(r - row0) * segments + seg) * n;
        for (int k = threadIdx.x; k < want; k += kThreads) {
            const u64 x = k < m ? buf[k] : 0;
            if (!FROM_KEYS && segments > 1) keys_out[row_out + base + k] = x;
            else {
                items[row_out + base + k] = x ? key_item(x) : -1;
                values[row_out + base + k] = x ? key_score(x) : -INFINITY;
            }
        }
        ceiling = m == want ? buf[want - 1] : 0;                 // 0: nothing is left for further rounds
        __syncthreads();
    }
}

// how many segments a row is cut into: with few rows, enough to give every CU work, of at least one 8192-score block each.  A list longer
// than one round is not cut.
static int top_segments(long long n_rows, int n_items, int n) {
    constexpr int block = kSuper * kTile;
    if (n > kRound || n_rows >= 512) return 1;
    const long long blocks = ((long long)n_items + block - 1) / block;
    return (int)std::max<long long>(1, std::min<long long>(blocks, (512 + n_rows - 1) / n_rows));
}
static int top_segment(int n_items, int segments) {
    constexpr int block = kSuper * kTile;
    const long long blocks = ((long long)n_items + block - 1) / block;
    return (int)std::min<long long>(n_items, (blocks + segments - 1) / segments * block);
}

// a launch holds fewer than 2^32 threads per dimension
constexpr long long kMaxBlocks = 1ll << 23;

static int check_rules(const rfm_score_rules *u, int64_t n_rows) {
    if (!u) return RFM_ERR_BAD_ARG;
    if (u->history_offsets) {
        if (u->n_history < 0 || u->n_history_items < 0 || (u->n_history_items > 0 && !u->history_items)) return RFM_ERR_BAD_ARG;
        if (!u->history_rows && u->n_history < n_rows) return RFM_ERR_BAD_ARG;
        if (!u->repetition && !(u->repetition_all > 0.0f && u->repetition_all < INFINITY)) return RFM_ERR_BAD_ARG;
        if (!u->frequency && !isfinite(u->frequency_all)) return RFM_ERR_BAD_ARG;
        if (!u->presence && !isfinite(u->presence_all)) return RFM_ERR_BAD_ARG;
    }
    if (u->bias_offsets && (u->n_bias_items < 0 || u->n_bias_items > 0x7ffffffe || (u->n_bias_items > 0 && (!u->bias_items || !u->bias_values)))) return RFM_ERR_BAD_ARG;
    if (u->allowed && (u->n_allowed < 1 || (!u->allowed_rows && u->n_allowed != 1 && u->n_allowed < n_rows))) return RFM_ERR_BAD_ARG;
    return RFM_OK;
}

template <typename T>
static void launch_adjust(const rfm_score_rules &u, long long n_rows, int n_items, const void *in, long long in_stride, void *out, long long out_stride, hipStream_t stream) {
    const int tiles = (n_items + kTile - 1) / kTile;
    const long long step = std::max<long long>(1, kMaxBlocks / tiles);
    for (long long r = 0; r < n_rows; r += step)
        adjust_scores_kernel<T><<<dim3((unsigned)(std::min(step, n_rows - r) * tiles)), dim3(kThreads), 0, stream>>>(u, r, tiles, n_items, (const T *)in, in_stride,
                                                                                                                      (T *)out, out_stride);
}

template <typename T, bool RULED>
static void launch_top(const rfm_score_rules &u, long long n_rows, int n_items, const void *in, long long stride, int n, int32_t *items, float *values, u64 *keys,
                       hipStream_t stream) {
    int segments = top_segments(n_rows, n_items, n);
    const int segment = top_segment(n_items, segments);
    segments = (n_items + segment - 1) / segment;
    const long long step = std::max<long long>(1, kMaxBlocks / segments);
    for (long long r = 0; r < n_rows; r += step) {               // (more than one only without segments: top_segments)
        const long long rows = std::min(step, n_rows - r);
        top_scores_kernel<T, RULED, false><<<dim3((unsigned)(rows * segments)), dim3(kThreads), 0, stream>>>(u, r, segments, segment, n_items, (const T *)in, stride,
                                                                                                              nullptr, 0, n, keys, items, values);
        if (segments > 1)
            top_scores_kernel<T, false, true><<<dim3((unsigned)rows), dim3(kThreads), 0, stream>>>(u, r, 1, n_items, n_items, (const T *)nullptr, 0, keys, segments * n, n,
                                                                                                    nullptr, items, values);
    }
}

}  // namespace rfm

using namespace rfm;

extern "C" {

int rfm_adjust_scores_device(const rfm_score_rules *rules, int32_t dtype, int64_t n_rows, int32_t n_items, const void *scores, int64_t stride, void *out,
                             int64_t out_stride, void *hip_stream) {
    if (n_rows < 0 || n_items < 1 || dtype < RFM_F32 || dtype > RFM_BF16 || stride < n_items || out_stride < n_items) return RFM_ERR_BAD_ARG;
    const int rc = check_rules(rules, n_rows);
    if (rc != RFM_OK) return rc;
    if (n_rows == 0) return RFM_OK;
    if (!scores || !out || n_items > 0x7fffffff - 4 * kTile) return RFM_ERR_BAD_ARG;
    hipStream_t stream = (hipStream_t)hip_stream;
    if (dtype == RFM_F32) launch_adjust<float>(*rules, n_rows, n_items, scores, stride, out, out_stride, stream);
    else if (dtype == RFM_F16) launch_adjust<_Float16>(*rules, n_rows, n_items, scores, stride, out, out_stride, stream);
    else launch_adjust<__bf16>(*rules, n_rows, n_items, scores, stride, out, out_stride, stream);
    return hipGetLastError() == hipSuccess ? RFM_OK : RFM_ERR_HIP;
}

size_t rfm_top_scores_workspace_bytes(int64_t n_rows, int32_t n_items, int32_t n) {
    if (n_rows < 0 || n_items < 1 || n < 1 || n > n_items) return 0;
    const int segments = top_segments(n_rows, n_items, n);
    return segments > 1 ? sizeof(u64) * (size_t)n_rows * (size_t)segments * (size_t)n : 8;
}

int rfm_top_scores_device(const rfm_score_rules *rules, int32_t dtype, int64_t n_rows, int32_t n_items, const void *scores, int64_t stride, int32_t n,
                          int32_t *items, float *values, void *workspace, size_t workspace_bytes, void *hip_stream) {
    if (n_rows < 0 || n_items < 1 || n < 1 || n > n_items || dtype < RFM_F32 || dtype > RFM_BF16 || stride < n_items) return RFM_ERR_BAD_ARG;
    if (rules) {
        const int rc = check_rules(rules, n_rows);
        if (rc != RFM_OK) return rc;
    }
    if (n_rows == 0) return RFM_OK;
    if (!scores || !items || !values || n_items > 0x7fffffff - 8 * kTile) return RFM_ERR_BAD_ARG;
    if (workspace_bytes < rfm_top_scores_workspace_bytes(n_rows, n_items, n) || !workspace) return RFM_ERR_WORKSPACE;
    hipStream_t stream = (hipStream_t)hip_stream;
    u64 *keys = (u64 *)workspace;
    const rfm_score_rules none = {};
    const rfm_score_rules &u = rules ? *rules : none;
    auto go = [&](auto type) {
        using T = decltype(type);
        if (rules) launch_top<T, true>(u, n_rows, n_items, scores, stride, n, items, values, keys, stream);
        else launch_top<T, false>(u, n_rows, n_items, scores, stride, n, items, values, keys, stream);
    };
    if (dtype == RFM_F32) go(float(0));
    else if (dtype == RFM_F16) go(_Float16(0));
    else go(__bf16(0));
    return hipGetLastError() == hipSuccess ? RFM_OK : RFM_ERR_HIP;
}

}  // extern "C"
