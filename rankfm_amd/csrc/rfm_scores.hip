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
#include <type_traits>

#include "../../include/rankfm_hip.h"

namespace rfm {

constexpr int kThreads = 256;

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

// The P scores of this thread out of items [first, first + 256 P): vector j of the tile belongs to thread j % 256.
template <typename T>
__device__ __forceinline__ int element(int slot) {               // position inside the tile of this thread's slot-th score
    constexpr int ve = Vec<T>::n;
    return ((slot / ve) * kThreads + (int)threadIdx.x) * ve + slot % ve;
}
template <typename T, int P>
__device__ __forceinline__ void load_tile(const T *row, int first, int n_items, float *s) {
    constexpr int ve = Vec<T>::n;
    if (first + P * kThreads <= n_items) {                       // (the same for all: no branch between the loads)
#pragma unroll
        for (int j = 0; j < P / ve; ++j) load_vec(row + first + (j * kThreads + (int)threadIdx.x) * ve, s + j * ve);
        return;
    }
#pragma unroll
    for (int j = 0; j < P / ve; ++j) {
        const int i = first + (j * kThreads + (int)threadIdx.x) * ve;
        if (i + ve <= n_items) load_vec(row + i, s + j * ve);
        else {
#pragma unroll
            for (int k = 0; k < ve; ++k) s[j * ve + k] = i + k < n_items ? (float)row[i + k] : -INFINITY;
        }
    }
}

// x[k] of a lane's own k
template <int N>
__device__ __forceinline__ float pick(const float (&x)[N], int k) {
    if constexpr (N == 1) return x[0];
    else {
        const unsigned upper = 0u - (unsigned)((k / (N / 2)) & 1);             // (bits, not an index: an indexed array would live in memory)
        float half[N / 2];
#pragma unroll
        for (int j = 0; j < N / 2; ++j) half[j] = __uint_as_float((__float_as_uint(x[j + N / 2]) & upper) | (__float_as_uint(x[j]) & ~upper));
        return pick<N / 2>(half, k);
    }
}

// what the row's lists name of a tile: count[item] of the history, and 1 + the position of the last bias entry
template <int P>
__device__ __forceinline__ void scan_lists(const RowRules &w, int first, int *count, int *last) {
    constexpr int tile = P * kThreads;
    for (int k = threadIdx.x; k < tile; k += kThreads) { count[k] = 0; last[k] = 0; }
    __syncthreads();
    for (long long k = threadIdx.x; k < w.hist_n; k += kThreads) {
        const unsigned at = (unsigned)w.hist[k] - (unsigned)first;               // (an id may be any 32 bits)
        if (at < (unsigned)tile) atomicAdd(count + at, 1);
    }
    for (long long k = threadIdx.x; k < w.bias_n; k += kThreads) {
        const unsigned at = (unsigned)w.bias_item[k] - (unsigned)first;
        if (at < (unsigned)tile) atomicMax(last + at, (int)k + 1);
    }
    __syncthreads();
}

// the rules of an item that the row's lists name (an allowed one)
__device__ __forceinline__ float listed_score(const rfm_score_rules &u, const RowRules &w, int item, int count, int last, float x) {
    if (count > 0) {
        x = x > 0.0f ? x / w.rho : x * w.rho;
        x = x - w.phi * (float)count;
        x = x - w.pi;
    }
    if (u.item_bias) x = x + u.item_bias[item];
    if (last > 0) x = x + w.bias_value[last - 1];
    return x;
}

// What the rules say of every item, for the scores of a tile: biases, and a bit per score that is allowed.  Asked for all at once, next to the scores:
// one after the other they are a chain of loads (1024 rows of 50 k items, the best ten under every rule: 82.6 us like that, 65.8 like this).  A tile
// starts at a multiple of 32 items, so a vector's bits lie in one word.
template <int P> struct Everyones { float bias[P]; unsigned allowed; };
template <typename T, int P>
__device__ __forceinline__ void load_everyones(const rfm_score_rules &u, const RowRules &w, int first, int n_items, Everyones<P> &e) {
    constexpr int ve = Vec<T>::n;
    const bool whole = first + P * kThreads <= n_items;          // (the same for all)
    unsigned word[P / ve];
    if (w.mask) {
#pragma unroll
        for (int j = 0; j < P / ve; ++j) word[j] = w.mask[min(first + (j * kThreads + (int)threadIdx.x) * ve, n_items - 1) >> 5];
    }
    if (u.item_bias) {
        if (whole) {
#pragma unroll
            for (int j = 0; j < P / ve; ++j)
#pragma unroll
                for (int k = 0; k < ve; k += 4) load_vec(u.item_bias + first + (j * kThreads + (int)threadIdx.x) * ve + k, e.bias + j * ve + k);
        } else {
#pragma unroll
            for (int k = 0; k < P; ++k) e.bias[k] = u.item_bias[min(first + element<T>(k), n_items - 1)];
        }
    }
    e.allowed = 0xffffffffu;
    if (w.mask) {
        e.allowed = 0;
#pragma unroll
        for (int j = 0; j < P / ve; ++j) e.allowed |= ((word[j] >> ((first + (j * kThreads + (int)threadIdx.x) * ve) & 31)) & ((1u << ve) - 1)) << (j * ve);
    }
}
template <int P>
__device__ __forceinline__ void apply_everyones(const rfm_score_rules &u, const Everyones<P> &e, float *s) {
    if (u.item_bias) {
#pragma unroll
        for (int k = 0; k < P; ++k) s[k] = s[k] + e.bias[k];
    }
    if (__any(e.allowed != 0xffffffffu)) {
#pragma unroll
        for (int k = 0; k < P; ++k) s[k] = (e.allowed >> k) & 1u ? s[k] : -INFINITY;
    }
}

// ... and with a row's lists: what they count for a tile
template <typename T, int P>
__device__ __forceinline__ void apply_counts(const rfm_score_rules &u, const RowRules &w, int first, int n_items, const int *count, const int *last, float *s) {
    constexpr int ve = Vec<T>::n;
#pragma unroll
    for (int j = 0; j < P / ve; ++j) {
        const int at = (j * kThreads + (int)threadIdx.x) * ve, i = first + at;
        if (i >= n_items) continue;
        const unsigned bits = w.mask ? w.mask[i >> 5] >> (i & 31) : 0xffffffffu;
#pragma unroll
        for (int k = 0; k < ve; ++k) {
            float x = s[j * ve + k];
            if (i + k < n_items) x = listed_score(u, w, i + k, count[at + k], last[at + k], x);
            s[j * ve + k] = (bits >> k) & 1u ? x : -INFINITY;
        }
    }
}

constexpr int kHits = kThreads;                  // list entries of a tile that are looked at by a thread each
constexpr int kCounted = 2048;                   // items whose counts are in LDS at a time, where there are more
struct Hits {
    int n;
    int2 at[kHits];                              // item; 0 for an entry of the history, else 1 + the position of the bias
};
struct Counted {
    int count[kCounted], last[kCounted];
};

// One workgroup per (row, tile of 256 P items): the row is read and written once, which is the floor.  The scores are asked for before the lists:
// their way through three dependent loads passes meanwhile.  A tile's few list entries are gathered in LDS; a thread each counts those of its item, makes
// that item's score and writes it over what the row's pass left there (read before anything of the tile is written: `out` may be `scores`).  Where
// there are more than 256, counts per item are made, 2048 items at a time.
// Bound by memory: 512 rows of 200 k items in bf16, 74 us = 5.5 TB/s read and written (a 4 GiB copy reaches 4.7); 1000 rows of 35 k in fp32 under every
// rule, 61.6 us = 4.5 TB/s; one row of 3.7 k, 4.6 us of the device's and 16 of the host's time.  8 (fp32) or 16 scores per thread are 32 bytes of
// a row either way: eight workgroups per CU, no loop.
template <typename T, int P>
__global__ void __launch_bounds__(kThreads) adjust_scores_kernel(const rfm_score_rules u, long long row0, int tiles, int n_items, const T *scores,
                                                                 long long stride, T *out, long long out_stride) {
    __shared__ union { Hits hits; Counted counted; } lists;
    const long long r = row0 + blockIdx.x / tiles;
    const int first = (int)(blockIdx.x % tiles) * P * kThreads;
    if (threadIdx.x == 0) lists.hits.n = 0;
    float s[P], value = 0.0f;
    int hits = 0, mine = -1;                                     // the item that the lists name and this thread sees to, and what becomes of its score
    load_tile<T, P>(scores + r * stride, first, n_items, s);
    const RowRules w = row_rules(u, r, n_items);
    Everyones<P> all;
    load_everyones<T, P>(u, w, first, n_items, all);
    if (w.bad) {
#pragma unroll
        for (int k = 0; k < P; ++k) s[k] = __uint_as_float(0x7fc00000u);
    } else {
        bool many = false;
        if (w.hist_n > 0 || w.bias_n > 0) {
            __syncthreads();
            auto note = [&](int item, int entry) {
                if ((unsigned)item - (unsigned)first >= (unsigned)(P * kThreads) || item >= n_items) return;
                const int at = atomicAdd(&lists.hits.n, 1);
                if (at < kHits) lists.hits.at[at] = make_int2(item, entry);
            };
            for (long long k = threadIdx.x; k < w.hist_n; k += kThreads) note(w.hist[k], 0);
            for (long long k = threadIdx.x; k < w.bias_n; k += kThreads) note(w.bias_item[k], (int)k + 1);
            __syncthreads();
            hits = lists.hits.n;
            many = hits > kHits;
            if (!many && (int)threadIdx.x < hits) {
                const int item = lists.hits.at[threadIdx.x].x;
                int c = 0, l = 0;
                bool before = false;                             // an earlier entry names the item: that thread sees to it
#pragma unroll 4
                for (int k = 0; k < hits; ++k) {
                    const int2 e = lists.hits.at[k];
                    const bool same = e.x == item;
                    before |= same && k < (int)threadIdx.x;
                    c += same && e.y == 0;
                    l = same ? max(l, e.y) : l;
                }
                if (!before) {
                    mine = item;
                    value = (float)scores[r * stride + item];
                    value = !w.mask || ((w.mask[item >> 5] >> (item & 31)) & 1u) ? listed_score(u, w, item, c, l, value) : -INFINITY;
                }
            }
            asm volatile("" : "+v"(value));                      // (no instruction: it is read by now)
            __syncthreads();                                     // `out` may be `scores`: no store before these reads
        }
        if (!many) apply_everyones<P>(u, all, s);
        else {
            constexpr int per = kCounted / kThreads;             // (tiles of P scores per thread lie in tiles of `per`: vectors of a tile come in order)
#pragma unroll
            for (int q = 0; q < P / per; ++q) {
                __syncthreads();
                const int from = first + q * kCounted;
                scan_lists<per>(w, from, lists.counted.count, lists.counted.last);
                apply_counts<T, per>(u, w, from, n_items, lists.counted.count, lists.counted.last, s + q * per);
            }
        }
    }
    constexpr int ve = Vec<T>::n;
    T *o = out + r * out_stride;
#pragma unroll
    for (int j = 0; j < P / ve; ++j) {
        const int i = first + (j * kThreads + (int)threadIdx.x) * ve;
        if (i + ve <= n_items) store_vec(o + i, s + j * ve);
        else {
#pragma unroll
            for (int k = 0; k < ve; ++k)
                if (i + k < n_items) o[i + k] = (T)s[j * ve + k];
        }
    }
    if (hits > 0) {                                              // (the same for all; none with counts)
        __syncthreads();                                         // behind the row's own stores
        if (mine >= 0) o[mine] = (T)value;
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

constexpr int kWaves = kThreads / 64;
constexpr int kPer = 8, kTile = kPer * kThreads; // scores per thread of a tile
// Under rules, half as many tiles are in registers at once (their biases and masks are too) and half as many candidates in LDS (it holds what the
// lists name as well): four workgroups per CU either way.
template <bool RULED> struct Top {
    static constexpr int super = RULED ? 2 : 4;  // tiles whose scores are in registers at once
    static constexpr int buf = RULED ? 512 : 1024;               // candidates a wavefront holds
    static constexpr int round = buf / 4 * 3;    // most entries kept at a time; a longer list is taken in rounds of this many
};
constexpr int kSlots = 1024;                     // hash slots for the items that a row's lists name
constexpr int kFull = kSlots - kThreads;         // lists that name more are scanned once per tile instead
constexpr int kWindow = 65536;                   // items whose membership bits are in LDS at a time

// x of lane ^ J.  Inside a row of 16 lanes that is an operand's modifier (DPP), inside 32 a fixed pattern, beyond a shuffle
template <int J>
__device__ __forceinline__ unsigned from_lane_xor(unsigned x) {
    if constexpr (J == 1) return (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0xb1, 0xf, 0xf, true);            // quad_perm 1 0 3 2
    else if constexpr (J == 2) return (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0x4e, 0xf, 0xf, true);       // quad_perm 2 3 0 1
    else if constexpr (J == 8) return (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0x128, 0xf, 0xf, true);      // row_ror 8
    else if constexpr (J < 32) return (unsigned)__builtin_amdgcn_ds_swizzle((int)x, J << 10 | 0x1f);
    else return __shfl_xor(x, J);
}
// the step of distance J of the stage of 2 * k's merges (nothing where the stage has no such step)
template <int R, int J>
__device__ __forceinline__ void exchange(u64 (&x)[R], int k, int lane) {
    if (J >= k) return;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const u64 other = (u64)from_lane_xor<J>((unsigned)(x[r] >> 32)) << 32 | from_lane_xor<J>((unsigned)x[r]);
        const bool larger = (((r * 64 + lane) & k) == 0) == ((lane & J) == 0);
        x[r] = (other > x[r]) == larger ? other : x[r];
    }
}
// Descending bitonic sort of `m` keys by a wavefront, in its registers: key r * 64 + lane is the r-th of its lane, so distances of 64 and more stay inside
// a lane and shorter ones are a shuffle; nothing waits for another wavefront but the writing back: key k is key `first` + k of the four buffers one
// behind the other, whose ends are s[].
template <int R, int BUF>
__device__ __forceinline__ void sort_in_registers(u64 *all, const int (&s)[kWaves - 1], int first, int m, int wave, int lane) {
    u64 x[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int k = r * 64 + lane, g = first + k, at = g < s[0] ? g : g < s[1] ? BUF + g - s[0] : g < s[2] ? 2 * BUF + g - s[1] : 3 * BUF + g - s[2];
        x[r] = k < m ? all[at] : 0;
    }
#pragma unroll 1
    for (int k = 2; k <= 64 * R; k <<= 1) {
#pragma unroll
        for (int d = R / 2; d > 0; d >>= 1) {
            if (d * 128 > k) continue;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (r & d) continue;
                const u64 a = x[r], b = x[r | d];
                const bool swap = (a < b) == ((r * 64 & k) == 0);
                x[r] = swap ? b : a;
                x[r | d] = swap ? a : b;
            }
        }
        exchange<R, 32>(x, k, lane);
        exchange<R, 16>(x, k, lane);
        exchange<R, 8>(x, k, lane);
        exchange<R, 4>(x, k, lane);
        exchange<R, 2>(x, k, lane);
        exchange<R, 1>(x, k, lane);
    }
    __syncthreads();                                             // the keys of all wavefronts are in registers
#pragma unroll
    for (int r = 0; r < R; ++r) all[wave * BUF + r * 64 + lane] = x[r];
}
// The same in LDS, for any number that the buffer holds (padded to a power of two): twice the time, and no registers
__device__ __forceinline__ void sort_in_place(u64 *buf, int m, int lane) {
    int p2 = 2;
    while (p2 < m) p2 <<= 1;
    for (int k = m + lane; k < p2; k += 64) buf[k] = 0;
    for (int k = 2; k <= p2; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            for (int t = lane; t < p2 / 2; t += 64) {
                const int i = ((t & ~(j - 1)) << 1) | (t & (j - 1)), l = i + j;
                const u64 a = buf[i], b = buf[l];
                if ((a < b) == ((i & k) == 0)) { buf[i] = b; buf[l] = a; }
            }
        }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
// what a row's lists name of a segment, when that is not much: a hash table of the items with their counts and last bias entries, and a bit per item of a
// window
struct Listed {
    int used, id[kSlots], count[kSlots], last[kSlots];
    unsigned bits[kWindow / 32];
};
struct Tiled {
    int count[kTile], last[kTile];               // (one tile at a time)
};
union ListMemory {
    Listed listed;
    Tiled tiled;
};

// false: there are too many of them for the table
__device__ __forceinline__ bool hash_lists(const RowRules &w, int begin, int end, Listed &m) {
    for (int k = threadIdx.x; k < kSlots; k += kThreads) { m.id[k] = -1; m.count[k] = 0; m.last[k] = 0; }
    if (threadIdx.x == 0) m.used = 0;
    __syncthreads();
    // (the walk ends: a table of more than kFull items is given up, and the threads that had not seen that yet fit in)
    auto slot_of = [&](int item) {
        unsigned at = (unsigned)item * 2654435761u >> 22;
        while (__hip_atomic_load(&m.used, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) <= kFull) {
            const int was = atomicCAS(m.id + at, -1, item);
            if (was == -1) atomicAdd(&m.used, 1);
            if (was == -1 || was == item) return (int)at;
            at = (at + 1) & (kSlots - 1);
        }
        return -1;
    };
    for (long long k = threadIdx.x; k < w.hist_n; k += kThreads) {
        const int i = w.hist[k];
        if (i >= begin && i < end) {
            const int at = slot_of(i);
            if (at < 0) break;
            atomicAdd(m.count + at, 1);
        }
    }
    for (long long k = threadIdx.x; k < w.bias_n; k += kThreads) {
        const int i = w.bias_item[k];
        if (i >= begin && i < end) {
            const int at = slot_of(i);
            if (at < 0) break;
            atomicMax(m.last + at, (int)k + 1);
        }
    }
    __syncthreads();
    const bool fits = m.used <= kFull;
    __syncthreads();                                             // (where it does not, counts of tiles take the table's place at once)
    return fits;
}
__device__ __forceinline__ void window_bits(Listed &m, int first) {
    __syncthreads();                                             // (nobody reads the last window's any more)
    for (int k = threadIdx.x; k < kWindow / 32; k += kThreads) m.bits[k] = 0;
    __syncthreads();
    for (int k = threadIdx.x; k < kSlots; k += kThreads) {
        const int i = m.id[k];
        if (i >= first && i - first < kWindow) atomicOr(m.bits + ((i - first) >> 5), 1u << (i & 31));
    }
    __syncthreads();
}

// One workgroup per (row, segment of the row): ONE pass over the scores.  Scores at or above the running threshold become keys in the wavefront's
// own part of LDS -- no barrier in the loop; when it is full, it is sorted and the threshold becomes the n-th best.  The first threshold comes
// from the first 8192 scores (4096 under rules): each group of eight holds its maximum in a register, a wavefront finds by bisection over ballots the
// value that its share of n of its group maxima reach, and the least of the four wavefronts' values is reached by at least n scores.  So the final
// sort sees a few times n keys, not the row (1837 rows of 640 items, the best two: 60 us when the empty wavefronts leave it none, 16 with it).  Under
// rules, items that the row's lists name are left out of the pass (a bit per item in LDS) and looked at by themselves afterwards.  FROM_KEYS: the "scores"
// are the sorted keys that the segments of a row left behind.
// Bound by memory without rules: 4096 rows of 50 k items, the best 64, 160 us = 5.1 TB/s read (a plain sum of as much reaches 4.0 - 4.7); under every
// rule 1024 rows take 63 us = 3.3 TB/s: the biases are as many loads again (54 us with them alone, 46 with nothing), from the L2, and so are the masks.  One
// row of 200 k: 17.5 us, two launches of which neither has enough work for the chip.
template <typename T, bool RULED, bool FROM_KEYS>
__global__ void __launch_bounds__(kThreads, 4) top_scores_kernel(const rfm_score_rules u, long long row0, int segments, int segment, int n_items,
                                                              const T *__restrict__ scores, long long stride, const u64 *__restrict__ keys_in, int n_keys,
                                                              int n, u64 *__restrict__ keys_out, int32_t *__restrict__ items, float *__restrict__ values) {
    constexpr int kSuper = Top<RULED>::super, kBuf = Top<RULED>::buf, kRound = Top<RULED>::round;
    constexpr int kAll = kSuper * kPer, ve = FROM_KEYS ? 1 : Vec<T>::n;
    __shared__ u64 buf[kWaves * kBuf];
    __shared__ typename std::conditional<RULED, ListMemory, int>::type lists_memory;
    __shared__ unsigned wave_t[kWaves], wave_q[kWaves];
    __shared__ int wave_m[kWaves];
    __shared__ u64 last_key;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const long long r = row0 + blockIdx.x / segments;
    const int seg = (int)(blockIdx.x % segments);
    const int begin = FROM_KEYS ? 0 : seg * segment, end = FROM_KEYS ? n_keys : min(n_items - begin, segment) + begin;
    RowRules w;
    if constexpr (RULED) w = row_rules(u, r, n_items);
    const bool listed = RULED && (w.hist_n > 0 || w.bias_n > 0);
    bool hashed = false;
    const T *row = FROM_KEYS ? nullptr : scores + r * stride;
    const u64 *krow = FROM_KEYS ? keys_in + (size_t)(r - row0) * n_keys : nullptr;
    u64 *mine = buf + wave * kBuf;
    if constexpr (RULED)
        if (listed && end - begin > kSuper * kTile) hashed = hash_lists(w, begin, end, lists_memory.listed);
    u64 ceiling = ~0ull;                                         // keys of earlier rounds are at or above it
    for (int base = 0; base < n; base += kRound) {
        const int want = min(n - base, kRound);
        if (threadIdx.x < kWaves) wave_q[threadIdx.x] = 0;      // (a barrier comes before the first is looked at: the first threshold's)
        u64 thr = 0;                                             // a key passes when it is above; a score is looked at when it is `reach` or more
        float reach = -3.402823466e38f;
        int m = 0;
        // The wavefront's part of LDS is full: the value that its n-th best reaches and the least of the four values that a quarter of n of each wavefront's
        // reach (as far as they have come there) are thresholds for everyone; what is above stays.  Found by bisection over ballots, cut to 20 bits,
        // a sort only where too many are equal.  (Sorting, and each wavefront its own n-th best alone: 500 rows of 190 k, 500 wanted, 305 us; 179 so.)
        auto make_room = [&]() {
            unsigned v[kBuf / 64];
#pragma unroll
            for (int k = 0; k < kBuf / 64; ++k) v[k] = k * 64 + lane < m ? (unsigned)(mine[k * 64 + lane] >> 32) : 0u;
            unsigned whole = 0, quarter = 0;
            for (int bit = 31; bit >= 12; --bit) {
                const unsigned cw = whole | (1u << bit), cq = quarter | (1u << bit);
                int nw = 0, nq = 0;
#pragma unroll
                for (int k = 0; k < kBuf / 64; ++k) { nw += __popcll(__ballot(v[k] >= cw)); nq += __popcll(__ballot(v[k] >= cq)); }
                if (nw >= want) whole = cw;
                if (nq >= (want + kWaves - 1) / kWaves) quarter = cq;
            }
            if (lane == 0) __hip_atomic_store(wave_q + wave, quarter, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            unsigned least = quarter;                            // (0 as long as one of them has not been full)
#pragma unroll
            for (int w = 0; w < kWaves; ++w)
                if (w != wave) least = min(least, __hip_atomic_load(wave_q + w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP));
            const unsigned t = max(whole, least);
            thr = max(thr, ((u64)t << 32) - (t ? 1 : 0));
            int kept = 0;
#pragma unroll 1
            for (int k = 0; k < m; k += 64) {
                const u64 key = k + lane < m ? mine[k + lane] : 0;
                const bool stays = key > thr;
                const unsigned long long who = __ballot(stays);
                if (stays) mine[kept + __popcll(who & ((1ull << lane) - 1))] = key;
                kept += __popcll(who);
            }
            m = kept;
            if (m > kBuf / 4 * 3) {                              // many of the same value: the first ones stay
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
                sort_in_place(mine, m, lane);
                m = want;                                        // (three quarters of the buffer at most)
                thr = max(thr, mine[want - 1]);
            }
            reach = key_score(thr);
        };
        auto keep = [&](bool pass, u64 key) {                    // (by whole wavefronts)
            pass = pass && key > thr && key < ceiling;
            const unsigned long long who = __ballot(pass);
            if (!who) return;
            if (m > kBuf - 64) {
                make_room();
                pass = pass && key > thr;
            }
            const unsigned long long still = __ballot(pass);
            if (pass) mine[m + __popcll(still & ((1ull << lane) - 1))] = key;
            m += __popcll(still);
        };
        int window = -1;
        for (int t0 = begin; t0 < end && !(RULED && w.bad); t0 += kSuper * kTile) {
            float x[kAll];
            if constexpr (FROM_KEYS) {
#pragma unroll
                for (int k = 0; k < kAll; ++k) {
                    const int e = t0 + k * kThreads + (int)threadIdx.x;
                    const u64 key = e < end ? krow[e] : 0;
                    x[k] = key && key < ceiling ? key_score(key) : -INFINITY;
                }
            } else {
                load_tile<T, kAll>(row, t0, end, x);
                if constexpr (RULED) {
                    if (!listed || hashed) {
                        Everyones<kAll> all;
                        load_everyones<T, kAll>(u, w, t0, n_items, all);
                        apply_everyones<kAll>(u, all, x);
                        if (hashed) {
                            if (t0 / kWindow != window) { window = t0 / kWindow; window_bits(lists_memory.listed, window * kWindow); }
#pragma unroll
                            for (int j = 0; j < kAll / ve; ++j) {
                                const int at = t0 - window * kWindow + (j * kThreads + (int)threadIdx.x) * ve;       // (ve divides 32: one word)
                                const unsigned bits = lists_memory.listed.bits[at >> 5] >> (at & 31);
#pragma unroll
                                for (int k = 0; k < ve; ++k) x[j * ve + k] = (bits >> k) & 1u ? -INFINITY : x[j * ve + k];
                            }
                        }
                    } else {
#pragma unroll
                        for (int q = 0; q < kSuper; ++q) {
                            if (t0 + q * kTile >= end) break;    // (the same for all)
                            scan_lists<kPer>(w, t0 + q * kTile, lists_memory.tiled.count, lists_memory.tiled.last);
                            apply_counts<T, kPer>(u, w, t0 + q * kTile, n_items, lists_memory.tiled.count, lists_memory.tiled.last, x + q * kPer);
                            __syncthreads();                     // (the next tile's scan clears the counts)
                        }
                    }
                }
            }
            auto key_of = [&](int k, float value) {
                if constexpr (FROM_KEYS) {
                    const int e = t0 + k * kThreads + (int)threadIdx.x;
                    return e < end ? krow[e] : 0ull;
                } else {
                    const int i = t0 + (k / kPer) * kTile + element<T>(k % kPer);
                    const unsigned v = i < end ? score_key(value) : 0u;
                    return v ? ((u64)v << 32) | (unsigned)~i : 0ull;
                }
            };
            if (t0 == begin) {                                   // the first threshold (in later rounds, of the scores below what was taken)
                const float taken = base == 0 ? INFINITY : key_score(ceiling);
                unsigned g[kSuper];
#pragma unroll
                for (int q = 0; q < kSuper; ++q) {
                    float high = -INFINITY;
#pragma unroll
                    for (int k = 0; k < kPer; ++k) high = fmaxf(high, base == 0 || x[q * kPer + k] < taken ? x[q * kPer + k] : -INFINITY);
                    g[q] = score_key(high);
                }
                // Every wavefront's share of the wanted is that of the groups it holds scores of: the vectors of a short row do not reach them all.
                const int vectors = (min(end - t0, kSuper * kTile) + ve - 1) / ve;
                int groups = min(max(vectors - wave * 64, 0), 64), of = min(vectors, kThreads);
                if (2 * want <= of) {                            // few are wanted: one group per lane
#pragma unroll
                    for (int q = 1; q < kSuper; ++q) { g[0] = max(g[0], g[q]); g[q] = 0; }
                } else {
#pragma unroll
                    for (int q = 1; q < kSuper; ++q) {
                        const int left = vectors - q * (kPer / ve) * kThreads;
                        groups += min(max(left - wave * 64, 0), 64);
                        of += min(max(left, 0), kThreads);
                    }
                }
                // the largest value (cut to 20 bits: a little below the exact one) that this wavefront's share of the wanted reaches
                unsigned t = 0;
                auto bisect = [&](auto reaching) {
                    const int need = (want * groups + of - 1) / of;
                    for (int bit = 31; bit >= 12; --bit) {
                        const unsigned c = t | (1u << bit);
                        if (reaching(c) >= need) t = c;
                    }
                };
                bool each = false;
                if constexpr (!FROM_KEYS) {
                    // A short row has too few groups for a long list: its scores are counted one by one (few of a lane's places hold any).  3319 rows of
                    // 1222, 394 wanted: 142 -> 74 us; at 0.8 of the groups (2000 rows of 5000, 500 wanted) 69 -> 72
                    each = 8 * want > 7 * of;
                    if (each) {
                        groups = 0;
                        of = vectors;
                        int above = 0;                           // the scores of earlier rounds
                        auto count = [&](float cut) {
                            int found = 0;
#pragma unroll
                            for (int j = 0; j < kAll / ve; ++j) {
                                if (j * kThreads >= vectors) break;
#pragma unroll
                                for (int k = 0; k < ve; ++k) found += __popcll(__ballot(x[j * ve + k] >= cut));
                            }
                            return found;
                        };
                        for (int j = 0; j * kThreads < vectors; ++j) groups += min(max(vectors - j * kThreads - wave * 64, 0), 64);
                        if (base > 0) above = count(taken);
                        bisect([&](unsigned c) { return count(key_score((u64)c << 32)) - above; });
                    }
                }
                if (!each)
                    bisect([&](unsigned c) {
                        int found = 0;
#pragma unroll
                        for (int q = 0; q < kSuper; ++q) found += __popcll(__ballot(g[q] >= c));
                        return found;
                    });
                if (lane == 0) wave_t[wave] = t;
                __syncthreads();
                t = min(min(wave_t[0], wave_t[1]), min(wave_t[2], wave_t[3]));
                if (t) { thr = ((u64)t << 32) - 1; reach = key_score((u64)t << 32); }
            }
            // a bit per score that reaches the threshold (bit 31 - k for slot k); then one score of every lane at a time, picked out of the registers
            unsigned reached = 0;
#pragma unroll
            for (int k = 0; k < kAll; ++k) reached = reached + reached + (x[k] >= reach ? 1u : 0u);
            reached <<= 32 - kAll;
            while (__any(reached != 0)) {
                const int k = __clz((int)reached) & (kAll - 1);
                const bool pass = reached != 0;
                reached &= ~(0x80000000u >> k);
                keep(pass, key_of(k, pick(x, k)));
            }
        }
        if constexpr (RULED) {
            if (hashed && !w.bad) {                              // the items left out
                const Listed &l = lists_memory.listed;
#pragma unroll 1
                for (int k = 0; k < kSlots / kThreads; ++k) {
                    const int at = k * kThreads + (int)threadIdx.x, i = l.id[at];
                    const bool here = i >= begin && i < end;
                    float s = -INFINITY;
                    if (here && (!w.mask || ((w.mask[i >> 5] >> (i & 31)) & 1u))) {
                        s = (float)row[i];
                        s = listed_score(u, w, i, l.count[at], l.last[at], s);
                    }
                    const unsigned v = score_key(s);
                    keep(v != 0, ((u64)v << 32) | (unsigned)~i);
                }
            }
        }
        // The candidates in order.  Few are placed by counting: a key's place is the number of larger ones (keys are unique).  Otherwise every wavefront
        // sorts an equal share of them (the vectors of a short row go to the first wavefronts), and a key's place is its place there and the number of
        // larger keys of the other three, each found by bisection.  (Sorting all of them together takes a barrier for each of its steps: 4096 rows of
        // 50 k, 64 wanted, 194 -> 165 us.  The shares: 2377 rows of 1039, 390 wanted, 200 -> 152; 6 of 3204, 365 wanted, 31 -> 22.)  Counting is the
        // square of the work; 256 are few where rows are and one workgroup's way to the end is what counts.
        if (lane == 0) wave_m[wave] = m;
        if (threadIdx.x == 0) last_key = 0;
        __syncthreads();
        int in_wave[kWaves], total = 0;
#pragma unroll
        for (int v = 0; v < kWaves; ++v) {
            in_wave[v] = __builtin_amdgcn_readfirstlane(wave_m[v]);
            total += in_wave[v];
        }
        const int got = total < want ? total : want;
        const size_t row_out = FROM_KEYS || segments == 1 ? (size_t)r * n : ((size_t)(r - row0) * segments + seg) * n;
        auto put = [&](int place, u64 key) {
            if (place == want - 1) last_key = key;
            if (!FROM_KEYS && segments > 1) keys_out[row_out + base + place] = key;
            else {
                items[row_out + base + place] = key ? key_item(key) : -1;
                values[row_out + base + place] = key ? key_score(key) : -INFINITY;
            }
        };
        if (total <= (FROM_KEYS || segments > 1 ? 256 : 64)) {
            for (int k = lane; k < m; k += 64) {
                const u64 key = mine[k];
                int place = 0;
#pragma unroll
                for (int v = 0; v < kWaves; ++v)
#pragma unroll 4
                    for (int q = 0; q < in_wave[v]; ++q) place += buf[v * kBuf + q] > key;
                if (place < want) put(place, key);
            }
        } else {
            const int share = (total + kWaves - 1) / kWaves;
            if (share <= 512) {
                const int ends[kWaves - 1] = {in_wave[0], in_wave[0] + in_wave[1], in_wave[0] + in_wave[1] + in_wave[2]}, first = wave * share;
                m = min(max(total - first, 0), share);
                if (share <= 64) sort_in_registers<1, kBuf>(buf, ends, first, m, wave, lane);
                else if (share <= 128) sort_in_registers<2, kBuf>(buf, ends, first, m, wave, lane);
                else if (share <= 256) sort_in_registers<4, kBuf>(buf, ends, first, m, wave, lane);
                else sort_in_registers<8, kBuf>(buf, ends, first, m, wave, lane);
#pragma unroll
                for (int v = 0; v < kWaves; ++v) in_wave[v] = min(max(total - v * share, 0), share);
            } else sort_in_place(mine, m, lane);
            __syncthreads();
            int count[kWaves - 1], most = 0;                     // of the other wavefronts
            const u64 *other[kWaves - 1];
#pragma unroll
            for (int v = 0; v < kWaves - 1; ++v) {
                const int who = (wave + 1 + v) & (kWaves - 1);
                other[v] = buf + who * kBuf;
                count[v] = who == 0 ? in_wave[0] : who == 1 ? in_wave[1] : who == 2 ? in_wave[2] : in_wave[3];
                most = max(most, count[v]);
            }
            const int steps = most > 0 ? 1 << (31 - __clz(most)) : 0;
            auto place_keys = [&](auto keys) {                   // `keys` of a lane at a time: their reads follow each other, not their bisections
                constexpr int at_once = decltype(keys)::value;
                for (int k0 = 0; k0 < min(m, want); k0 += 64 * at_once) {
                    u64 key[at_once];
                    int above[at_once][kWaves - 1];
#pragma unroll
                    for (int h = 0; h < at_once; ++h) {
                        key[h] = k0 + h * 64 + lane < m ? mine[k0 + h * 64 + lane] : 0;
#pragma unroll
                        for (int v = 0; v < kWaves - 1; ++v) above[h][v] = 0;
                    }
                    for (int step = steps; step > 0; step >>= 1)
#pragma unroll
                        for (int h = 0; h < at_once; ++h)
#pragma unroll
                            for (int v = 0; v < kWaves - 1; ++v) {
                                const int next = above[h][v] + step;
                                above[h][v] = next <= count[v] && other[v][min(next, kBuf) - 1] > key[h] ? next : above[h][v];
                            }
#pragma unroll
                    for (int h = 0; h < at_once; ++h) {
                        int place = k0 + h * 64 + lane;
                        const bool on = place < m;
#pragma unroll
                        for (int v = 0; v < kWaves - 1; ++v) place += above[h][v];
                        if (on && place < want) put(place, key[h]);
                    }
                }
            };
            if (min(m, want) <= 64) place_keys(std::integral_constant<int, 1>());
            else place_keys(std::integral_constant<int, 2>());
        }
        for (int k = got + threadIdx.x; k < want; k += kThreads) put(k, 0);
        __syncthreads();
        ceiling = last_key;                                      // 0: nothing is left for further rounds
        __syncthreads();
    }
}

// How many segments a row is cut into: with few rows, enough to give every CU work, of at least one block of 8192 scores each.  Lists of more than 1024
// are not cut: every segment would hand that many on.  From 256 rows on joining costs more than the second workgroup per CU gives (400 rows of 17 k, n = 10 / 100 /
// 450, cut in two: 20.4 / 35.6 / 79.0 us, whole: 12.5 / 19.0 / 44.4; of 190 k: 71 / 129 / 191 and 61 / 129 / 157), but for long rows under rules
// (500 of 190 k, n = 10: 91 and 118).  Below 256 rows the rule knows the row's length by its blocks alone, and cuts short rows that would be faster
// whole (255 rows of 17 k, cut, with the call: 25 / 36 / 67 us; 256, whole: 21 / 27 / 50).  Uncut, a long list is walked by one workgroup: one row of
// 200 k, n = 1024 / 1025 / 5000: 310 / 240 / 979 us.
constexpr int kBlock = 8192;
static int top_segments(long long n_rows, int n_items, int n, bool ruled) {
    const long long blocks = ((long long)n_items + kBlock - 1) / kBlock;
    if (n > 1024 || n_rows >= 512 || (n_rows >= 256 && !(ruled && blocks > 12))) return 1;
    return (int)std::max<long long>(1, std::min<long long>(blocks, (512 + n_rows - 1) / n_rows));
}
static int top_segment(int n_items, int segments) {
    const long long blocks = ((long long)n_items + kBlock - 1) / kBlock;
    return (int)std::min<long long>(n_items, (blocks + segments - 1) / segments * kBlock);
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
    constexpr int per = sizeof(T) == 4 ? 8 : 16; // 32 bytes of a row per thread either way
    const int tiles = (n_items + per * kThreads - 1) / (per * kThreads);
    const long long step = std::max<long long>(1, kMaxBlocks / tiles);
    for (long long r = 0; r < n_rows; r += step)
        adjust_scores_kernel<T, per><<<dim3((unsigned)(std::min(step, n_rows - r) * tiles)), dim3(kThreads), 0, stream>>>(u, r, tiles, n_items, (const T *)in, in_stride,
                                                                                                                      (T *)out, out_stride);
}

template <typename T, bool RULED>
static void launch_top(const rfm_score_rules &u, long long n_rows, int n_items, const void *in, long long stride, int n, int32_t *items, float *values, u64 *keys,
                       hipStream_t stream) {
    int segments = top_segments(n_rows, n_items, n, RULED);
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
    const int segments = top_segments(n_rows, n_items, n, true);            // (with rules there are as many or more)
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
    const bool ruled = u.history_offsets || u.item_bias || u.bias_offsets || u.allowed;
    auto go = [&](auto type) {
        using T = decltype(type);
        if (ruled) launch_top<T, true>(u, n_rows, n_items, scores, stride, n, items, values, keys, stream);
        else launch_top<T, false>(u, n_rows, n_items, scores, stride, n, items, values, keys, stream);
    };
    if (dtype == RFM_F32) go(float(0));
    else if (dtype == RFM_F16) go(_Float16(0));
    else go(__bf16(0));
    return hipGetLastError() == hipSuccess ? RFM_OK : RFM_ERR_HIP;
}

}  // extern "C"
