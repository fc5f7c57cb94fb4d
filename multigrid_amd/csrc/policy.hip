// libmgrid_hip.so - what stands between the simulator and a policy network, for gfx950 (MI355X):
//   embedding of cells and tokens, and its gradient;
//   adjustment of logits (penalties, bias, mask), and its gradient;
//   draw of a token from logits;
//   log-probability and entropy of given tokens, and their gradient.
// The formulas stand in include/mgrid.h beside each entry point.
//
// Sums, maxima and probabilities are held in 32 bits (64 in the draw, where a token's borders decide); a value is
// rounded to its type once, when it is stored.
//
// On this card a copy of 1 GiB moves 5.1 TB/s (read and written together), a fill 6.9, torch's float32 sum reads 4.0; the smallest
// launch takes 3.6 us.  The times beside the kernels are theirs, without the host.  A pass that reads much takes longer behind one that
// has written much, while the caches still write that back: where two times are given, the first is of the pass by itself.

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "mgrid.h"
#include "mgrid_error.h"

namespace {

using bf16 = __bf16;
using f16 = _Float16;
using float4_t = __attribute__((__vector_size__(16))) float;
using ushort2_t = unsigned short __attribute__((ext_vector_type(2)));

constexpr int THREADS = 256;
constexpr float NEG_INF = -__builtin_inff();
constexpr float LEAST_TEMPERATURE = 0x1p-126f;  // its reciprocal is finite

// V elements at any element's alignment: global loads and stores of gfx950 take 16 bytes at any address
template <class T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Vec {
    T v[V];
};

// Words, not elements, go to memory: as elements a store and the one of a row's end beside it would be taken apart and merged.
template <class T, int V>
__device__ __forceinline__ void store(T *p, const float (&x)[V]) {
    constexpr int WORDS = V * sizeof(T) / 4;
    Vec<T, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = static_cast<T>(x[i]);
    uint32_t w[WORDS];
    __builtin_memcpy(w, &r, sizeof r);
    struct __attribute__((packed, aligned(sizeof(T)))) Words {
        uint32_t w[WORDS];
    } q;
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
        asm("" : "+v"(w[i]));
        q.w[i] = w[i];
    }
    *reinterpret_cast<Words *>(p) = q;
}

// elements in 16 bytes
template <class T>
constexpr int WIDE = 16 / static_cast<int>(sizeof(T));

// 16 bytes moved down by `bits` (1 .. 128), `fills` behind them
__device__ __forceinline__ void move_down(uint32_t (&w)[4], int bits, uint32_t fills) {
    const uint64_t all = static_cast<uint64_t>(fills) << 32 | fills, lo = static_cast<uint64_t>(w[1]) << 32 | w[0], hi = static_cast<uint64_t>(w[3]) << 32 | w[2];
    uint64_t to, top;
    if (bits < 64) {
        to = lo >> bits | hi << (64 - bits);
        top = hi >> bits | all << (64 - bits);
    } else {
        to = bits == 64 ? hi : (bits == 128 ? all : hi >> (bits - 64) | all << (128 - bits));
        top = all;
    }
    w[0] = static_cast<uint32_t>(to);
    w[1] = static_cast<uint32_t>(to >> 32);
    w[2] = static_cast<uint32_t>(top);
    w[3] = static_cast<uint32_t>(top >> 32);
}

// Words of W adjacent elements at p, which stay packed until they are used.  `left` elements are the row's, the others become
// `fill` (an element's bits).  A row of at least W elements is never read element by element (each would be waited for): the W
// elements that end where the row does are read and moved down.
template <class T, int W>
__device__ __forceinline__ void load_words(const T *p, int left, int length, uint32_t fill, uint32_t (&w)[(W * sizeof(T) + 3) / 4]) {
    constexpr int WORDS = (W * sizeof(T) + 3) / 4, BITS = 8 * sizeof(T);
    if constexpr (W * sizeof(T) < 4) {
        w[0] = left > 0 ? *reinterpret_cast<const uint16_t *>(p) : fill;
        return;
    } else {
        struct __attribute__((packed, aligned(sizeof(T)))) Words {
            uint32_t w[WORDS];
        };
        const uint32_t fills = BITS == 32 ? fill : fill * 0x10001u;
        if (left >= W) {
            const Words r = *reinterpret_cast<const Words *>(p);
#pragma unroll
            for (int i = 0; i < WORDS; ++i) w[i] = r.w[i];
        } else if (left > 0 && length >= W) {
            const Words r = *reinterpret_cast<const Words *>(p - (W - left));
            const int down = (W - left) * BITS;
            if constexpr (WORDS == 1) {
                w[0] = r.w[0] >> 16 | fills << 16;
            } else if constexpr (WORDS == 2) {
                const uint64_t to = (static_cast<uint64_t>(r.w[1]) << 32 | r.w[0]) >> down | (static_cast<uint64_t>(fills) << 32 | fills) << (64 - down);
                w[0] = static_cast<uint32_t>(to);
                w[1] = static_cast<uint32_t>(to >> 32);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = r.w[i];
                move_down(w, down, fills);
            }
        } else if constexpr (WORDS > 1) {  // a short row: its halves
            if (left > 0) {
                uint32_t half[WORDS / 2], rest[WORDS / 2];
                load_words<T, W / 2>(p, left, length, fill, half);
                load_words<T, W / 2>(p + W / 2, left - W / 2, length, fill, rest);
#pragma unroll
                for (int i = 0; i < WORDS / 2; ++i) {
                    w[i] = half[i];
                    w[WORDS / 2 + i] = rest[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < WORDS; ++i) w[i] = fills;
            }
        } else {  // one element of a word, or none
            w[0] = fills;
            if (left > 0) w[0] = BITS == 32 ? *reinterpret_cast<const uint32_t *>(p) : (fills & 0xFFFF0000u) | *reinterpret_cast<const uint16_t *>(p);
        }
    }
}

// 2, 4 or 8 bytes of elements of ALIGN bytes from an address that was a number: a pointer made of one is no pointer to global memory
// to the compiler, and its loads would be waited for together with everything else.
template <int BYTES, int ALIGN>
__device__ __forceinline__ void load_global(uint64_t at, uint32_t (&w)[(BYTES + 3) / 4]) {
    using one_t = uint32_t __attribute__((aligned(ALIGN)));
    using two_t = uint32_t __attribute__((ext_vector_type(2), aligned(ALIGN)));
#define GLOBAL_AT(type) *reinterpret_cast<const __attribute__((address_space(1))) type *>(at)
    if constexpr (BYTES == 2) {
        w[0] = GLOBAL_AT(uint16_t);
    } else if constexpr (BYTES == 4) {
        w[0] = GLOBAL_AT(one_t);
    } else {
        const two_t v = GLOBAL_AT(two_t);
        w[0] = v.x;
        w[1] = v.y;
    }
#undef GLOBAL_AT
}

// element i of words
template <class T>
__device__ __forceinline__ float element(const uint32_t *w, int i) {
    if constexpr (sizeof(T) == 4)
        return __builtin_bit_cast(float, w[i]);
    else
        return static_cast<float>(__builtin_bit_cast(T, static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1)))));
}

// N vectors of a row, number j at first + (j * lanes + lane) * V; behind the row's k elements `fill`.  All loads are under way
// before the first is looked at, so none stands behind a test (which would be waited for): a vector that passes the row's end is
// read where the row's last V elements lie, and moved down.  V elements or more lie before that end (the row has more than
// SHORT, and a piece of one begins behind others).
template <class T, int N>
__device__ __forceinline__ void load_vectors(const T *row, int k, int first, int lanes, int lane, uint32_t fill, uint32_t (&w)[N][4]) {
    constexpr int V = WIDE<T>;
    struct __attribute__((packed, aligned(sizeof(T)))) Words {
        uint32_t w[4];
    };
    const uint32_t fills = sizeof(T) == 4 ? fill : fill * 0x10001u;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const Words r = *reinterpret_cast<const Words *>(row + min(first + (j * lanes + lane) * V, k - V));
#pragma unroll
        for (int i = 0; i < 4; ++i) w[j][i] = r.w[i];
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int past = first + (j * lanes + lane) * V - (k - V);
        if (past > 0) move_down(w[j], min(past, V) * 8 * static_cast<int>(sizeof(T)), fills);
    }
}

template <class T, int V>
__device__ __forceinline__ void load(const T *p, float (&x)[V]) {
    uint32_t w[V * sizeof(T) / 4];
    load_words<T, V>(p, V, V, 0, w);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = element<T>(w, i);
}

template <class T>
constexpr uint32_t NEG_INF_BITS = sizeof(T) == 4 ? 0xFF800000u : (__is_same(T, f16) ? 0xFC00u : 0xFF80u);

template <class T, int V>
__device__ __forceinline__ void load_part(const T *p, int left, int length, float (&x)[V]) {
    uint32_t w[V * sizeof(T) / 4];
    load_words<T, V>(p, left, length, 0, w);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = element<T>(w, i);
}

// The first `left` of 16 bytes of elements: by halves, where they are not all of them.
template <class T>
__device__ __forceinline__ void store_words(T *p, int left, uint32_t (&w)[4]) {
    struct __attribute__((packed, aligned(sizeof(T)))) Four {
        uint32_t w[4];
    };
    struct __attribute__((packed, aligned(sizeof(T)))) Two {
        uint32_t w[2];
    };
    struct __attribute__((packed, aligned(sizeof(T)))) One {
        uint32_t w;
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("" : "+v"(w[i]));  // (else the elements that two ways have in common are stored by themselves)
    constexpr int V = WIDE<T>;
    char *to = reinterpret_cast<char *>(p);
    if (left >= V) {
        *reinterpret_cast<Four *>(to) = Four{{w[0], w[1], w[2], w[3]}};
    } else if (left > 0) {
        if (left & (V / 2)) {
            *reinterpret_cast<Two *>(to) = Two{{w[0], w[1]}};
            to += 8;
            w[0] = w[2];
            w[1] = w[3];
        }
        if (left & (V / 4)) {
            reinterpret_cast<One *>(to)->w = w[0];
            to += 4;
            w[0] = w[1];
        }
        if (V == 8 && (left & 1)) *reinterpret_cast<uint16_t *>(to) = static_cast<uint16_t>(w[0]);
    }
}

template <class T>
__device__ __forceinline__ void pack(const float (&x)[WIDE<T>], uint32_t (&w)[4]) {
    Vec<T, WIDE<T>> r;
#pragma unroll
    for (int i = 0; i < WIDE<T>; ++i) r.v[i] = static_cast<T>(x[i]);
    __builtin_memcpy(w, &r, sizeof r);
}

template <class T, int V>
__device__ __forceinline__ void store_part(T *p, int left, const float (&x)[V]) {
    static_assert(V % WIDE<T> == 0, "16 bytes, or several");
#pragma unroll
    for (int i = 0; i < V; i += WIDE<T>) {
        float y[WIDE<T>];
#pragma unroll
        for (int j = 0; j < WIDE<T>; ++j) y[j] = x[i + j];
        uint32_t w[4];
        pack<T>(y, w);
        store_words(p + i, left - i, w);
    }
}

// ---- embedding -----------------------------------------------------------------------------------------------------

struct EmbedArgs {
    int64_t n, ids_stride, field_stride, row_stride;
    int32_t fields, dim, rows;
    float scale;
    int32_t sizes[MG_MAX_FIELDS];
};

// One thread per 16 bytes of output; the threads of a token share its ids.  (Four tokens to a thread at once: no faster where
// there are many tokens, half as fast at 8190.)  Bound by the writes and by the rows that the cache does not hold: 16384 tokens x
// 2048 bfloat16 of 32000 rows 22 us (134 MB), 98 cells x 32 2.6 us.
template <class T, class I>
__global__ __launch_bounds__(THREADS) void embed_kernel(EmbedArgs a, const I *ids, const T *table, T *out, I *ids_copy) {
    constexpr int V = WIDE<T>;
    const int vecs = (a.dim + V - 1) / V;
    const int cols = min(vecs, THREADS), per_block = THREADS / cols;
    const int sub = threadIdx.x / cols, col = threadIdx.x - sub * cols;
    if (sub >= per_block) return;
    for (int64_t n = static_cast<int64_t>(blockIdx.x) * per_block + sub; n < a.n; n += static_cast<int64_t>(gridDim.x) * per_block) {
        const I *id_at = ids + n * a.ids_stride;
        T *to = out + n * a.dim;
        for (int c = col; c < vecs; c += cols) {
            const int d0 = c * V;
            // get(one row's elements) for every row that the token reads
            auto sum = [&](auto get) {
                float acc[V] = {};
                int64_t base = 0;
                for (int f = 0; f < a.fields; ++f) {
                    const int64_t id = static_cast<int64_t>(id_at[f * a.field_stride]);
                    if (id >= 0 && id < a.sizes[f]) {
                        float x[V];
                        get(table + (base + id) * a.row_stride + d0, x);
#pragma unroll
                        for (int i = 0; i < V; ++i) acc[i] += x[i];
                    }
                    base += a.sizes[f];
                }
#pragma unroll
                for (int i = 0; i < V; ++i) acc[i] *= a.scale;
                store_part<T, V>(to + d0, a.dim - d0, acc);
            };
            if (d0 + V <= a.dim)
                sum([](const T *from, float (&x)[V]) { load<T, V>(from, x); });
            else
                sum([&](const T *from, float (&x)[V]) { load_part<T, V>(from, a.dim - d0, a.dim, x); });
        }
        if (ids_copy && col == 0)
            for (int f = 0; f < a.fields; ++f) ids_copy[n * a.fields + f] = id_at[f * a.field_stride];
    }
}

// A table that LDS holds (cells: 24 rows): a block copies it there once, then takes `far` (up to FAR) tokens' ids at a time into LDS
// as row numbers, and writes those tokens' outputs 16 bytes a thread, four tokens to a thread at once.  Bound by the writes; with the
// table in memory or L1 each output waits for a chain of id, row and store.  401408 cells x 64 float32: 22.6 us (103 MB, 4.6 TB/s),
// 31.5 by embed_kernel.
constexpr int TABLE_BYTES = 32768, FAR = 512, TABLE_BLOCKS = 2048, UNITS = 256;

template <class T, class I>
__global__ __launch_bounds__(THREADS) void embed_table_kernel(EmbedArgs a, int far, const I *ids, const T *table, T *out, I *ids_copy) {
    constexpr int V = WIDE<T>, TOGETHER = 4;
    extern __shared__ __align__(16) char lds[];
    const int vecs = (a.dim + V - 1) / V, pitch = vecs * V;
    T *table_s = reinterpret_cast<T *>(lds);                                                  // [rows + 1][pitch], zeros in the last row
    uint16_t *rows_s = reinterpret_cast<uint16_t *>(lds + (a.rows + 1) * pitch * sizeof(T));  // [fields][FAR]
    for (int i = threadIdx.x; i < (a.rows + 1) * pitch; i += THREADS) {
        const int r = i / pitch, d = i - r * pitch;
        table_s[i] = r < a.rows && d < a.dim ? table[r * a.row_stride + d] : static_cast<T>(0.f);
    }
    const int cols = min(vecs, THREADS), per_block = THREADS / cols;
    const int sub = threadIdx.x / cols, col = threadIdx.x - sub * cols;
    for (int64_t n0 = static_cast<int64_t>(blockIdx.x) * far; n0 < a.n; n0 += static_cast<int64_t>(gridDim.x) * far) {
        const int tokens = static_cast<int>(min(static_cast<int64_t>(far), a.n - n0));
        __syncthreads();
        int base = 0;
        for (int f = 0; f < a.fields; ++f) {
            const I *from = ids + n0 * a.ids_stride + f * a.field_stride;
            I id[FAR / THREADS];
#pragma unroll
            for (int j = 0; j < FAR / THREADS; ++j) {
                const int t = j * THREADS + threadIdx.x;
                id[j] = t < tokens ? from[t * a.ids_stride] : static_cast<I>(0);
            }
#pragma unroll
            for (int j = 0; j < FAR / THREADS; ++j) {
                const int64_t v = static_cast<int64_t>(id[j]);
                rows_s[f * FAR + j * THREADS + threadIdx.x] = static_cast<uint16_t>(v >= 0 && v < a.sizes[f] ? base + v : a.rows);
                if (ids_copy && j * THREADS + static_cast<int>(threadIdx.x) < tokens) ids_copy[(n0 + j * THREADS + threadIdx.x) * a.fields + f] = id[j];
            }
            base += a.sizes[f];
        }
        __syncthreads();
        if (sub < per_block)
            for (int c = col; c < vecs; c += cols)
                for (int t0 = sub; t0 < tokens; t0 += per_block * TOGETHER) {
                    float acc[TOGETHER][V] = {};
                    for (int f = 0; f < a.fields; ++f)
#pragma unroll
                        for (int u = 0; u < TOGETHER; ++u) {
                            const int t = min(t0 + u * per_block, FAR - 1);
                            const uint4 q = *reinterpret_cast<const uint4 *>(table_s + rows_s[f * FAR + t] * pitch + c * V);
                            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                            for (int i = 0; i < V; ++i) acc[u][i] += element<T>(w, i);
                        }
#pragma unroll
                    for (int u = 0; u < TOGETHER; ++u) {
                        const int t = t0 + u * per_block;
                        if (t >= tokens) break;
#pragma unroll
                        for (int i = 0; i < V; ++i) acc[u][i] *= a.scale;
                        store_part<T, V>(out + (n0 + t) * a.dim + c * V, a.dim - c * V, acc[u]);
                    }
                }
    }
}

// the ids to a contiguous copy, by all blocks of a launch
template <class I>
__device__ __forceinline__ void copy_ids(const EmbedArgs &a, const I *ids, I *to) {
    constexpr int V = 16 / static_cast<int>(sizeof(I));
    const int64_t all = a.n * a.fields, step = static_cast<int64_t>(gridDim.x) * blockDim.x;
    int64_t e = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (a.ids_stride == a.fields && a.field_stride == 1) {
        for (int64_t i = e * V; i + V <= all; i += step * V) *reinterpret_cast<Vec<I, V> *>(to + i) = *reinterpret_cast<const Vec<I, V> *>(ids + i);
        e += all / V * V;
    }
    for (; e < all; e += step) {
        const int64_t n = e / a.fields;
        to[e] = ids[n * a.ids_stride + (e - n * a.fields) * a.field_stride];
    }
}

// The same where LDS holds the finished output of every combination of a token's ids, none included (cells: 12 x 7 x 8): worked
// out once a block, then each 16 bytes of output are one read of LDS and one store.  For rows of whole vectors (`dim` a multiple of V):
// storing other rows' ends element by element was slower than embed_table_kernel (4500000 cells x 31 bfloat16 174 us against 112).
// 6422528 cells x 32 bfloat16: 90 us (430 MB, 4.8 TB/s), 109 by embed_table_kernel, 185 by embed_kernel; x 16 float32 92, 93 and 151.
constexpr int COMBINED_BYTES = 53248, COMBINED_THREADS = 512, COMBINED_BLOCKS = 768;  // three blocks to a compute unit
static_assert(FAR == COMBINED_THREADS, "a token's ids to each thread");

template <class T, class I>
__global__ __launch_bounds__(COMBINED_THREADS) void embed_combined_kernel(EmbedArgs a, int combined, const I *ids, const T *table, T *out, I *ids_copy) {
    constexpr int V = WIDE<T>, TOGETHER = 4;
    extern __shared__ __align__(16) char lds[];
    const int vecs = a.dim / V, pitch = a.dim;
    T *done_s = reinterpret_cast<T *>(lds), *table_s = done_s + combined * pitch;  // [combined][pitch], [rows + 1][pitch]
    if (ids_copy) copy_ids(a, ids, ids_copy);  // (a stream of its own, before the others: 4 us; a launch of its own 10, beside each token's output 17)
    uint16_t *which_s = reinterpret_cast<uint16_t *>(table_s + (a.rows + 1) * pitch);
    for (int i = threadIdx.x; i < (a.rows + 1) * pitch; i += COMBINED_THREADS) {
        const int r = i / pitch, d = i - r * pitch;
        table_s[i] = r < a.rows ? table[r * a.row_stride + d] : static_cast<T>(0.f);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < combined * vecs; i += COMBINED_THREADS) {
        const int c = i / combined, at = i - c * combined;
        int row[MG_MAX_FIELDS], rest = at, base = a.rows;
#pragma unroll
        for (int f = MG_MAX_FIELDS - 1; f >= 0; --f)  // the last field varies first
            if (f < a.fields) {
                const int size = a.sizes[f], id = rest % (size + 1);
                rest /= size + 1;
                base -= size;
                row[f] = id < size ? base + id : a.rows;
            }
        float acc[V] = {};
#pragma unroll
        for (int f = 0; f < MG_MAX_FIELDS; ++f)  // in the order of the other two kernels: a token's bits do not depend on how many there are
            if (f < a.fields) {
                float x[V];
                load<T, V>(table_s + row[f] * pitch + c * V, x);
#pragma unroll
                for (int e = 0; e < V; ++e) acc[e] += x[e];
            }
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] *= a.scale;
        store<T, V>(done_s + at * pitch + c * V, acc);
    }
    const int cols = min(vecs, COMBINED_THREADS), per_block = COMBINED_THREADS / cols;
    const int sub = threadIdx.x / cols, col = threadIdx.x - sub * cols;
    I id[MG_MAX_FIELDS];
    auto fetch = [&](int64_t n0) {  // FAR is COMBINED_THREADS
        const I *from = ids + min(n0 + threadIdx.x, a.n - 1) * a.ids_stride;
#pragma unroll
        for (int f = 0; f < MG_MAX_FIELDS; ++f)
            if (f < a.fields) id[f] = from[f * a.field_stride];
    };
    const int64_t step = static_cast<int64_t>(gridDim.x) * FAR;
    int64_t n0 = static_cast<int64_t>(blockIdx.x) * FAR;
    if (n0 < a.n) fetch(n0);
    for (; n0 < a.n; n0 += step) {
        const int tokens = static_cast<int>(min(static_cast<int64_t>(FAR), a.n - n0));
        __syncthreads();
        {
            int which = 0;
#pragma unroll
            for (int f = 0; f < MG_MAX_FIELDS; ++f)
                if (f < a.fields) {
                    const int64_t v = static_cast<int64_t>(id[f]);
                    which = which * (a.sizes[f] + 1) + (v >= 0 && v < a.sizes[f] ? static_cast<int>(v) : a.sizes[f]);
                }
            which_s[threadIdx.x] = static_cast<uint16_t>(which);
        }
        if (n0 + step < a.n) fetch(n0 + step);  // on their way while this one's outputs are written
        __syncthreads();
        if (sub < per_block)
            for (int c = col; c < vecs; c += cols)
                for (int t0 = sub; t0 < tokens; t0 += per_block * TOGETHER) {
                    uint4 q[TOGETHER];
#pragma unroll
                    for (int u = 0; u < TOGETHER; ++u) q[u] = *reinterpret_cast<const uint4 *>(done_s + which_s[min(t0 + u * per_block, FAR - 1)] * pitch + c * V);
#pragma unroll
                    for (int u = 0; u < TOGETHER; ++u) {
                        const int t = t0 + u * per_block;
                        if (t >= tokens) break;
                        struct __attribute__((packed, aligned(sizeof(T)))) Words {
                            uint32_t w[4];
                        };
                        *reinterpret_cast<Words *>(out + (n0 + t) * a.dim + c * V) = Words{{q[u].x, q[u].y, q[u].z, q[u].w}};
                    }
                }
    }
}

// ---- gradient of the embedding -------------------------------------------------------------------------------------

// An id as it lies in memory (a negative one has a large upper or lower half), so that many can be under way before the first
// is looked at; f(load of the id at an element's index) runs under one test of the ids' type.
struct Id {
    uint32_t low, high;
};
template <class F>
__device__ __forceinline__ void with_ids(const void *ids, int type, F f) {
    if (type == MG_U8)
        f([=](int64_t at) { return Id{static_cast<const uint8_t *>(ids)[at], 0}; });
    else if (type == MG_I32)
        f([=](int64_t at) { return Id{static_cast<const uint32_t *>(ids)[at], 0}; });
    else
        f([=](int64_t at) {
            const uint2 v = static_cast<const uint2 *>(ids)[at];
            return Id{v.x, v.y};
        });
}
// as a row of the table, or `none`
__device__ __forceinline__ uint32_t row_of(Id id, uint32_t base, uint32_t size, uint32_t none) { return id.high == 0 && id.low < size ? base + id.low : none; }

// Few rows (up to FEW): the gradient is the product of the rows' indicator [rows][n] (1 where token n reads the row) and the
// incoming gradient [n][dim], which is what matrix instructions are for: 1 is exact in every type, so every product is, and
// the sums are held in float32.  16-bit gradients go in as they are, float32 ones as three bfloat16 parts of eight bits each (of 2^16
// times the number: bfloat16 ends at 2^-133, float32 at 2^-149).
//
// A wave takes 64 tokens at a time: lane n puts its token's rows into LDS, then two 16 x 16 x 32 products per 16 rows and 16
// columns.  The indicator's fragment (row l % 16, tokens 8 (l / 16) ...) is made from eight row numbers by three packed 16-bit
// instructions per pair; the gradient's fragment (column l % 16, the same tokens) comes straight from memory, W adjacent
// columns of a token to a lane, so that product i of W covers columns W * (0 .. 15) + i and pairs of tokens meet by one byte
// permutation each.  The order of the tokens within 32 is free: a load takes four adjacent tokens, whole lines of memory.
// Waves and blocks stride over the tokens, a block adds its four waves, embed_join_kernel the blocks, all in a fixed order.
//
// Bound by the reads: with the join, 6422528 cells x 32 bfloat16 81 us (430 MB with the ids, 5.3 TB/s), 128 behind the lookup that
// has written as much; 401408 x 64 float32 27 us (104 MB, 3.9 TB/s: four or five turns of a wave, and their beginning and end), 40
// behind the lookup.  By sorting the tokens these take 3250 and 172 us; with 64
// rows and 8190 tokens x 1024 the two are equal (28 and 26 us), with 2000 tokens x 64 it is 10 against 20.
//
// 0 times infinity or NaN is NaN: such a number would spoil a whole column.  A block whose sums are not all finite does its tokens
// again, one after the other, each added to its own rows only.
// Three blocks to a compute unit, two where a lane takes four columns and the registers allow no more.  Against 512, 1024 and 1536 in
// place of 768, over nine cases from 65536 x 64 float32 to 6422528 x 32 bfloat16: within 3 % for most; 512 gains 12 % with 401408 x 32
// bfloat16 and loses 12 % with 1500000 x 100 float16, 1024 and more lose up to 8 and 24 %.
constexpr int FEW = 64, FEW_BLOCKS = 768;
constexpr int64_t FAR_ROWS = 1 << 24;  // a stride up to which 64 tokens lie within 32-bit offsets

template <class T>
struct Operand {
    using type = __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16;
    static constexpr uint32_t ONE = 0x3F80;
    static __device__ __forceinline__ float4_t multiply(type a, type b, float4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Operand<f16> {
    using type = __attribute__((__vector_size__(8 * sizeof(_Float16)))) _Float16;
    static constexpr uint32_t ONE = 0x3C00;
    static __device__ __forceinline__ float4_t multiply(type a, type b, float4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

union Fragment {
    uint32_t w[4];
    Operand<float>::type b;
    Operand<f16>::type h;
    template <class T>
    __device__ __forceinline__ typename Operand<T>::type get() const {
        if constexpr (sizeof(typename Operand<T>::type) && __is_same(T, f16))
            return h;
        else
            return b;
    }
};

template <class T, int W, int TILES, int FIELDS>
__global__ __launch_bounds__(THREADS, TILES > 2 || W > 2 || FIELDS > 3 ? 2 : 3) void embed_grad_few_kernel(EmbedArgs a, const void *ids, int ids_type, const T *grad, T *out, float *parts) {
    constexpr int COLS = 16 * W, WORDS = (W * sizeof(T) + 3) / 4;
    // float32 numbers times this are three bfloat16 parts to the last bit, 2^-149 as well: bfloat16 ends at 2^-133.  All sums are whole
    // multiples of 2^-149 too, so dividing by it loses nothing; where it overflows, a sum is not finite (see above).
    constexpr float UP = 0x1p16f;
    __shared__ __align__(16) uint16_t rows_s[THREADS / 64][FIELDS][64];  // 0xFFFF: none
    __shared__ float sum_s[TILES * 16][COLS];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, l16 = lane % 16, quad = lane / 16;
    const int d0 = blockIdx.y * COLS, col = l16 * W;
    // the field that this lane's row of each tile belongs to, and the row twice in a word (a row that is none never matches)
    int field[TILES];
    uint32_t twice[TILES];
#pragma unroll
    for (int m = 0; m < TILES; ++m) {
        const int row = m * 16 + l16;
        int f = 0, base = 0;
        while (f + 1 < a.fields && row >= base + a.sizes[f]) base += a.sizes[f++];
        field[m] = f;
        twice[m] = row < a.rows ? static_cast<uint32_t>(row) * 0x10001u : 0xFFFEFFFEu;
    }
    float4_t acc[TILES][W];
#pragma unroll
    for (int m = 0; m < TILES; ++m)
#pragma unroll
        for (int i = 0; i < W; ++i) acc[m][i] = float4_t{0.f, 0.f, 0.f, 0.f};

    const int64_t step = static_cast<int64_t>(gridDim.x) * THREADS;
    // a lane at the row's end, or behind it, takes the last W columns and keeps of them those that are its own
    const int from_col = min(col, a.dim - d0 - W);
    const uint32_t stride = static_cast<uint32_t>(a.row_stride) * sizeof(T), own = quad * stride + (d0 + from_col) * sizeof(T);  // bytes, see FAR_ROWS
    // No load stands behind a branch: it would be waited for at the branch's end, and with it all that were on their way before.
    // So the last 64 tokens stand for a wave that passes the end (tokens of another wave's are given no row), the last field for
    // those that are not there, and of an id the aligned word that holds it (its other bytes, the tensor's or not, are in the same
    // page), or its lower half, is read, and an upper half, which only int64 has.
    const int id_shift = ids_type == MG_U8 ? 0 : (ids_type == MG_I32 ? 2 : 3);
    const uint32_t id_mask = ids_type == MG_U8 ? 0xFF : ~0u, high_mask = ids_type == MG_I64 ? ~0u : 0;
    auto id_at = [&](int64_t t0, int f) {
        return reinterpret_cast<uint64_t>(ids) + (((min(t0, a.n - 64) + lane) * a.ids_stride + min(f, a.fields - 1) * a.field_stride) << id_shift);
    };
    auto fetch_ids = [&](int64_t t0, Id (&id)[FIELDS]) {
#pragma unroll
        for (int f = 0; f < FIELDS; ++f) {
            const uint64_t at = id_at(t0, f) & ~3ull;
            uint32_t low[1], high[1];
            load_global<4, 4>(at, low);
            load_global<4, 4>(at + (high_mask & 4), high);
            id[f] = Id{low[0], high[0]};
        }
    };
    auto fetch = [&](int64_t t0, uint32_t (&x)[2][8][WORDS]) {
        // an address that is the same for the wave, and this lane's offset
        uint64_t from = reinterpret_cast<uint64_t>(grad + min(t0, a.n - 64) * a.row_stride);
        asm volatile("" : "+s"(from));
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) load_global<W * sizeof(T), sizeof(T)>(from + static_cast<uint64_t>(s * 32 + j * 4) * stride + own, x[s][j]);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto put_rows = [&](int64_t t0, const Id (&id)[FIELDS]) {
        __builtin_amdgcn_wave_barrier();  // the last tokens' rows are read
        const int place = (lane & 32) + (lane & 3) * 8 + (lane & 31) / 4;  // token j * 4 + quad is number j of the quad
        const bool live = min(t0, a.n - 64) + lane >= t0;
        uint32_t base = 0;
#pragma unroll
        for (int f = 0; f < FIELDS; ++f) {
            const uint32_t shift = ids_type == MG_U8 ? static_cast<uint32_t>(id_at(t0, f)) % 4 * 8 : 0, size = f < a.fields ? a.sizes[f] : 0;
            const Id own_id{(id[f].low >> shift) & id_mask, id[f].high & high_mask};
            rows_s[wave][f][place] = static_cast<uint16_t>(live ? row_of(own_id, base, size, 0xFFFF) : 0xFFFF);
            base += size;
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };
    auto add = [&](uint32_t (&x)[2][8][WORDS]) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int i = 0; i < WORDS; ++i) asm volatile("" : "+v"(x[s][j][i]));  // not before the next loads are on their way
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            Fragment hot[TILES];
#pragma unroll
            for (int m = 0; m < TILES; ++m) {
                const uint4 r = *reinterpret_cast<const uint4 *>(&rows_s[wave][field[m]][s * 32 + quad * 8]);
                const uint32_t rr[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
                for (int p = 0; p < 4; ++p) {  // ONE where the halves are equal: ONE - min(xor, 1) * ONE
                    ushort2_t d = __builtin_bit_cast(ushort2_t, rr[p] ^ twice[m]);
                    d = __builtin_elementwise_min(d, ushort2_t{1, 1});
                    constexpr uint16_t ONE = Operand<T>::ONE;
                    hot[m].w[p] = __builtin_bit_cast(uint32_t, static_cast<ushort2_t>(ushort2_t{ONE, ONE} - d * ushort2_t{ONE, ONE}));
                }
            }
#pragma unroll
            for (int i = 0; i < W; ++i) {
                Fragment g;
                if constexpr (sizeof(T) == 2) {
#pragma unroll
                    for (int p = 0; p < 4; ++p)
                        g.w[p] = __builtin_amdgcn_perm(x[s][2 * p + 1][i / 2], x[s][2 * p][i / 2], i & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
                    for (int m = 0; m < TILES; ++m) acc[m][i] = Operand<T>::multiply(hot[m].template get<T>(), g.template get<T>(), acc[m][i]);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[s][j][i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, x[s][j][i]) * UP);
#pragma unroll
                    for (int part = 0; part < 3; ++part) {
#pragma unroll
                        for (int p = 0; p < 4; ++p) {
                            g.w[p] = __builtin_amdgcn_perm(x[s][2 * p + 1][i], x[s][2 * p][i], 0x07060302u);
#pragma unroll
                            for (int o = 0; o < 2; ++o) {  // what the upper half leaves
                                uint32_t &v = x[s][2 * p + o][i];
                                v = __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, v) - __builtin_bit_cast(float, v & 0xFFFF0000u));
                            }
                        }
#pragma unroll
                        for (int m = 0; m < TILES; ++m) acc[m][i] = Operand<T>::multiply(hot[m].template get<T>(), g.template get<T>(), acc[m][i]);
                    }
                }
            }
        }
    };
    // two sets of registers in turn: while one is multiplied, the loads of the other are under way
    uint32_t x0[2][8][WORDS], x1[2][8][WORDS];
    Id id[FIELDS];
    int64_t t0 = (static_cast<int64_t>(blockIdx.x) * (THREADS / 64) + wave) * 64;
    auto turn = [&](uint32_t (&now)[2][8][WORDS], uint32_t (&next)[2][8][WORDS]) {
        if (t0 >= a.n) return false;
        put_rows(t0, id);
        fetch_ids(t0 + step, id);
        fetch(t0 + step, next);
        add(now);
        t0 += step;
        return true;
    };
    if (t0 < a.n) {
        fetch_ids(t0, id);
        fetch(t0, x0);
        while (turn(x0, x1) && turn(x1, x0)) {
        }
    }

    bool fine = true;
#pragma unroll
    for (int m = 0; m < TILES; ++m)
#pragma unroll
        for (int i = 0; i < W; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) fine &= fabsf(acc[m][i][q]) < -NEG_INF;
    if (__syncthreads_and(fine)) {
        for (int w = 0; w < THREADS / 64; ++w) {
            if (wave == w) {
#pragma unroll
                for (int m = 0; m < TILES; ++m)
#pragma unroll
                    for (int i = 0; i < W; ++i)
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            if (from_col + i >= col) {
                                float &s = sum_s[m * 16 + quad * 4 + q][from_col + i];
                                const float own_sum = sizeof(T) == 4 ? acc[m][i][q] * (1.f / UP) : acc[m][i][q];
                                s = w ? s + own_sum : own_sum;
                            }
            }
            __syncthreads();
        }
    } else {  // one thread for a column and every (THREADS / COLS)th row
        const int c = threadIdx.x % COLS, share = threadIdx.x / COLS;
        for (int r = share; r < TILES * 16; r += THREADS / COLS) sum_s[r][c] = 0.f;
        with_ids(ids, ids_type, [&](auto load_id) {
            for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * THREADS; t0 < a.n; t0 += step)
                for (int64_t t = t0; t < t0 + THREADS && t < a.n; ++t) {
                    uint32_t base = 0;
                    for (int f = 0; f < a.fields; ++f) {
                        const uint32_t r = row_of(load_id(t * a.ids_stride + f * a.field_stride), base, a.sizes[f], FEW);
                        if (r < FEW && r % (THREADS / COLS) == static_cast<uint32_t>(share) && d0 + c < a.dim) sum_s[r][c] += static_cast<float>(grad[t * a.row_stride + d0 + c]);
                        base += a.sizes[f];
                    }
                }
        });
        __syncthreads();
    }
    for (int i = threadIdx.x; i < a.rows * COLS; i += THREADS) {
        const int r = i / COLS, c = i % COLS;
        if (d0 + c >= a.dim) continue;
        if (parts)
            parts[(static_cast<int64_t>(blockIdx.x) * a.rows + r) * a.dim + d0 + c] = sum_s[r][c];
        else
            out[static_cast<int64_t>(r) * a.dim + d0 + c] = static_cast<T>(sum_s[r][c] * a.scale);
    }
}

// The blocks' sums of one table gradient added up: 16 adjacent elements and 64 shares of the blocks to a workgroup.
constexpr int JOIN_COLS = 16, JOIN_SHARES = 64;

template <class T>
__global__ __launch_bounds__(JOIN_COLS *JOIN_SHARES) void embed_join_kernel(const float *parts, int blocks, int64_t elements, float scale, T *out) {
    __shared__ float sum_s[JOIN_SHARES][JOIN_COLS];
    const int c = threadIdx.x % JOIN_COLS, share = threadIdx.x / JOIN_COLS;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * JOIN_COLS + c;
    float s = 0.f;
    if (at < elements)
#pragma unroll 8
        for (int b = share; b < blocks; b += JOIN_SHARES) s += parts[b * elements + at];
    sum_s[share][c] = s;
    __syncthreads();
    for (int half = JOIN_SHARES / 2; half > 0; half /= 2) {
        if (share < half) sum_s[share][c] += sum_s[share + half][c];
        __syncthreads();
    }
    if (share == 0 && at < elements) out[at] = static_cast<T>(sum_s[0][c] * scale);
}

// More rows: the entries (token n, field f) are sorted by row, order kept (a radix sort of up to 9 bits a pass), and the sorted
// list is cut into chunks of equal length whatever the rows' frequencies are.  A chunk adds up its runs of equal rows; a run
// that lies inside one chunk is finished there, one that passes a border leaves float32 parts for embed_span_kernel.
// 8190 tokens, 30011 rows x 1024 bfloat16: sort 19 us, runs 10, spans 7.4.
constexpr int MOST_BINS = 512, DIGIT = 9;

// The entries e0, e0 + step, ... (N of them, those below `end`): row (a.rows where the id reads none) and token.
template <int N>
__device__ __forceinline__ void load_entries(const EmbedArgs &a, const void *ids, int ids_type, int64_t e0, int64_t step, int64_t end, uint2 (&entry)[N]) {
    Id id[N];
    with_ids(ids, ids_type, [&](auto load_id) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int64_t e = min(e0 + j * step, end - 1), n = a.fields == 1 ? e : e / a.fields;
            id[j] = load_id(n * a.ids_stride + (e - n * a.fields) * a.field_stride);
        }
    });
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int64_t e = e0 + j * step, n = a.fields == 1 ? e : e / a.fields;
        uint32_t base = 0, size = a.sizes[0];
        for (int f = 1, at = static_cast<int>(e - n * a.fields); f <= at; ++f) {
            base += size;
            size = a.sizes[f];
        }
        entry[j] = make_uint2(row_of(id[j], base, size, a.rows), static_cast<uint32_t>(n));
    }
}

// Places among the wave's earlier entries of the same digit, counted in `count`: N digits of a lane, one after the other.  What
// waits (the counters) is under way for all of them at once.
template <int N>
__device__ __forceinline__ void places(uint32_t *count, const uint32_t (&digit)[N], const bool (&live)[N], int bits, uint32_t (&at)[N]) {
    uint32_t low[N], high[N];  // lanes with the same digit as this one
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const uint64_t all = __ballot(live[j]);
        low[j] = static_cast<uint32_t>(all);
        high[j] = static_cast<uint32_t>(all >> 32);
    }
    for (int b = 0; b < bits; ++b)
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t one = __builtin_amdgcn_sbfe(digit[j], b, 1);  // no bit, or all
            const uint64_t ones = __ballot(one != 0);
            low[j] &= ~(static_cast<uint32_t>(ones) ^ one);
            high[j] &= ~(static_cast<uint32_t>(ones >> 32) ^ one);
        }
    uint32_t before[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        at[j] = __builtin_amdgcn_mbcnt_hi(high[j], __builtin_amdgcn_mbcnt_lo(low[j], 0));
        before[j] = 0;
        // An earlier digit's count comes first, also if it is another lane's: one wave's accesses to LDS are done in the order of its
        // instructions, which the fence makes the compiler keep (it emits nothing).
        if (j > 0) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (live[j] && at[j] == 0) before[j] = atomicAdd(&count[digit[j]], static_cast<uint32_t>(__popc(low[j]) + __popc(high[j])));
    }
#pragma unroll
    for (int j = 0; j < N; ++j) at[j] += __shfl(before[j], low[j] ? __builtin_ctz(low[j]) : (high[j] ? 32 + __builtin_ctz(high[j]) : 0), 64);
}

// exclusive sums of v over the threads of a block
template <int N>
__device__ __forceinline__ uint32_t sum_before(uint32_t v, uint32_t *wave_sums, uint32_t *total) {
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    uint32_t s = v;
#pragma unroll
    for (int by = 1; by < 64; by *= 2) {
        const uint32_t o = __shfl_up(s, by, 64);
        if (lane >= by) s += o;
    }
    if (lane == 63) wave_sums[wave] = s;
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (int w = 0; w < N / 64; ++w) {
        if (w < wave) before += wave_sums[w];
        all += wave_sums[w];
    }
    if (total) *total = all;
    __syncthreads();
    return before + s - v;
}

// The gradient's bytes to 0, by the blocks beside those that sort: the rows that no token reads stay so, the others are written
// when their sums are known.
__device__ __forceinline__ void clear(char *out, int64_t bytes, int64_t block, int64_t blocks) {
    struct __attribute__((packed, aligned(1))) Words {
        uint32_t w[4];
    };
    for (int64_t i = (block * blockDim.x + threadIdx.x) * 16; i < bytes; i += blocks * blockDim.x * 16) {
        if (i + 16 <= bytes)
            *reinterpret_cast<Words *>(out + i) = Words{{0, 0, 0, 0}};
        else
            for (int64_t b = i; b < bytes; ++b) out[b] = 0;
    }
}

// Up to SORT_ONE entries and 2^18 - 1 rows: one workgroup sorts words of row << 14 | entry in LDS, while others clear the output.
// Bound by the one compute unit's instructions (the digits' comparison bit by bit); still the whole gradient of 8190 tokens x 64
// takes 30 us so and 45 with the three kernels below for each digit, of 16384 tokens 42 and 47.
constexpr int SORT_THREADS = 1024, SORT_ONE = 1 << 14, SORT_ROWS = (1 << 18) - 1;

__global__ __launch_bounds__(SORT_THREADS) void embed_sort_kernel(EmbedArgs a, const void *ids, int ids_type, int entries, int passes, int bits,
                                                                  uint32_t *rows_out, uint32_t *tokens_out, char *out, int64_t out_bytes) {
    constexpr int WAVES = SORT_THREADS / 64, ROUNDS = SORT_ONE / SORT_THREADS, TOGETHER = 4;
    if (blockIdx.x > 0) return clear(out, out_bytes, blockIdx.x - 1, gridDim.x - 1);
    __shared__ uint32_t word_s[SORT_ONE];
    __shared__ uint32_t count_s[WAVES][MOST_BINS], base_s[MOST_BINS];
    __shared__ uint32_t wave_sums[WAVES];
    const int tid = threadIdx.x, wave = tid / 64, lane = tid % 64;
    const int rounds = (entries + SORT_THREADS - 1) / SORT_THREADS, first = wave * rounds * 64 + lane;
    for (int e = tid; e < entries; e += SORT_THREADS * 8) {
        uint2 entry[8];
        load_entries(a, ids, ids_type, e, SORT_THREADS, entries, entry);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (e + j * SORT_THREADS < entries) word_s[e + j * SORT_THREADS] = entry[j].x << 14 | (e + j * SORT_THREADS);
    }
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = 14 + pass * bits, bins = 1 << bits;
        for (int i = tid; i < WAVES << bits; i += SORT_THREADS) count_s[i >> bits][i & (bins - 1)] = 0;
        __syncthreads();
        uint32_t word[ROUNDS / TOGETHER][TOGETHER], at[ROUNDS / TOGETHER][TOGETHER];
#pragma unroll
        for (int j = 0; j < ROUNDS / TOGETHER; ++j) {
            if (j * TOGETHER >= rounds) break;
            uint32_t digit[TOGETHER];
            bool live[TOGETHER];
#pragma unroll
            for (int u = 0; u < TOGETHER; ++u) {
                const int e = first + (j * TOGETHER + u) * 64;
                live[u] = j * TOGETHER + u < rounds && e < entries;
                word[j][u] = live[u] ? word_s[e] : 0;
                digit[u] = (word[j][u] >> shift) & (bins - 1);
            }
            places(count_s[wave], digit, live, bits, at[j]);
        }
        __syncthreads();
        uint32_t mine = 0;
        if (tid < bins) {
            uint32_t c[WAVES];
#pragma unroll
            for (int w = 0; w < WAVES; ++w) c[w] = count_s[w][tid];
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                count_s[w][tid] = mine;
                mine += c[w];
            }
        }
        const uint32_t before = sum_before<SORT_THREADS>(mine, wave_sums, nullptr);
        if (tid < bins) base_s[tid] = before;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < ROUNDS / TOGETHER; ++j)
#pragma unroll
            for (int u = 0; u < TOGETHER; ++u)
                if (j * TOGETHER + u < rounds && first + (j * TOGETHER + u) * 64 < entries) {
                    const uint32_t digit = (word[j][u] >> shift) & (bins - 1);
                    word_s[base_s[digit] + count_s[wave][digit] + at[j][u]] = word[j][u];
                }
        __syncthreads();
    }
    for (int i = tid; i < entries; i += SORT_THREADS) {
        const uint32_t w = word_s[i];
        rows_out[i] = w >> 14;
        tokens_out[i] = a.fields == 1 ? (w & (SORT_ONE - 1)) : (w & (SORT_ONE - 1)) / a.fields;
    }
}

// More entries: a pass is a count of every block's digits, one block's sums over all counts, and the placing.  A block owns
// `span` adjacent entries (a multiple of SORT_TILE, so that there are at most SORT_BLOCKS blocks).
constexpr int SORT_TILE = 4096, SORT_BLOCKS = 1024;

__global__ __launch_bounds__(THREADS) void embed_count_kernel(EmbedArgs a, const void *ids, int ids_type, const uint2 *from, int64_t entries, int span,
                                                              int shift, int bits, int blocks, uint32_t *counts, char *out, int64_t out_bytes) {
    __shared__ uint32_t count_s[MOST_BINS];
    const int bins = 1 << bits;
    if (static_cast<int>(blockIdx.x) >= blocks) return clear(out, out_bytes, blockIdx.x - blocks, gridDim.x - blocks);
    for (int i = threadIdx.x; i < bins; i += THREADS) count_s[i] = 0;
    __syncthreads();
    const int64_t lo = static_cast<int64_t>(blockIdx.x) * span, hi = min(lo + span, entries);
    for (int64_t e = lo + threadIdx.x; e < hi; e += THREADS * 8) {
        uint2 entry[8];
        if (from)
#pragma unroll
            for (int j = 0; j < 8; ++j) entry[j] = from[min(e + j * THREADS, hi - 1)];
        else
            load_entries(a, ids, ids_type, e, THREADS, hi, entry);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (e + j * THREADS < hi) atomicAdd(&count_s[(entry[j].x >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < bins; i += THREADS) counts[static_cast<int64_t>(i) * blocks + blockIdx.x] = count_s[i];
}

// One workgroup: 3.4 us for the counts of 32768 entries, 60 for those of 1000000 (62720), three quarters of their sort.
__global__ __launch_bounds__(SORT_THREADS) void embed_scan_kernel(uint32_t *counts, int n) {
    __shared__ uint32_t wave_sums[SORT_THREADS / 64];
    uint32_t done = 0;
    for (int i0 = 0; i0 < n; i0 += SORT_THREADS * 8) {  // eight adjacent numbers to a thread
        uint32_t v[8], mine = 0;
        const int at = i0 + threadIdx.x * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = at + j < n ? counts[at + j] : 0;
            mine += v[j];
        }
        uint32_t total;
        uint32_t before = done + sum_before<SORT_THREADS>(mine, wave_sums, &total);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (at + j < n) counts[at + j] = before;
            before += v[j];
        }
        done += total;
    }
}

__global__ __launch_bounds__(THREADS) void embed_place_kernel(EmbedArgs a, const void *ids, int ids_type, const uint2 *from, int64_t entries, int span,
                                                              int shift, int bits, const uint32_t *counts, uint2 *to, uint32_t *rows_out,
                                                              uint32_t *tokens_out) {
    constexpr int WAVES = THREADS / 64, ROUNDS = SORT_TILE / THREADS, TOGETHER = 4;
    __shared__ uint32_t count_s[WAVES][MOST_BINS], base_s[MOST_BINS];
    const int tid = threadIdx.x, wave = tid / 64, lane = tid % 64, bins = 1 << bits;
    for (int i = tid; i < bins; i += THREADS) base_s[i] = counts[static_cast<int64_t>(i) * gridDim.x + blockIdx.x];
    const int64_t lo = static_cast<int64_t>(blockIdx.x) * span, hi = min(lo + span, entries);
    for (int64_t e0 = lo; e0 < hi; e0 += SORT_TILE) {
        for (int i = tid; i < WAVES * MOST_BINS; i += THREADS) (&count_s[0][0])[i] = 0;
        __syncthreads();
        const int64_t first = e0 + wave * (SORT_TILE / WAVES) + lane;
        uint2 entry[ROUNDS];
        uint32_t at[ROUNDS / TOGETHER][TOGETHER];
        if (from)
#pragma unroll
            for (int j = 0; j < ROUNDS; ++j) entry[j] = from[min(first + j * 64, hi - 1)];
        else
            load_entries(a, ids, ids_type, first, 64, hi, entry);
#pragma unroll
        for (int j = 0; j < ROUNDS / TOGETHER; ++j) {
            uint32_t digit[TOGETHER];
            bool live[TOGETHER];
#pragma unroll
            for (int u = 0; u < TOGETHER; ++u) {
                digit[u] = (entry[j * TOGETHER + u].x >> shift) & (bins - 1);
                live[u] = first + (j * TOGETHER + u) * 64 < hi;
            }
            places(count_s[wave], digit, live, bits, at[j]);
        }
        __syncthreads();
        for (int i = tid; i < bins; i += THREADS) {
            uint32_t s = base_s[i];
            for (int w = 0; w < WAVES; ++w) {
                const uint32_t c = count_s[w][i];
                count_s[w][i] = s;
                s += c;
            }
            base_s[i] = s;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < ROUNDS; ++j)
            if (first + j * 64 < hi) {
                const uint32_t p = count_s[wave][(entry[j].x >> shift) & (bins - 1)] + at[j / TOGETHER][j % TOGETHER];
                if (to) {
                    to[p] = entry[j];
                } else {
                    rows_out[p] = entry[j].x;
                    tokens_out[p] = entry[j].y;
                }
            }
        __syncthreads();
    }
}

struct Sorted {
    const uint32_t *rows, *tokens;  // [entries], by row; a.rows behind the last row
    float *head, *tail;             // [chunks][dim]: what a chunk has of a run that an earlier chunk began / that goes on behind it
    int64_t entries;
    int32_t chunk, chunks;          // entries of a chunk, number of chunks
    int32_t lanes;                  // threads per chunk: a power of two, up to 64
};

template <class T>
__global__ __launch_bounds__(THREADS) void embed_runs_kernel(EmbedArgs a, Sorted s, const T *grad, T *out) {
    constexpr int V = WIDE<T>, AHEAD = 8;
    const int lane = threadIdx.x % s.lanes, group = threadIdx.x / s.lanes, groups = THREADS / s.lanes;
    const int d0 = (blockIdx.y * s.lanes + lane) * V, left = a.dim - d0, back = max(V - left, 0);
    if (left <= 0) return;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * groups + group;
    if (c >= s.chunks) return;
    const int64_t e0 = c * s.chunk, e1 = min(e0 + s.chunk, s.entries);
    const uint32_t none = a.rows;
    uint32_t row = s.rows[e0];
    bool begun = c > 0 && s.rows[e0 - 1] == row;
    float acc[V] = {};
    auto finish = [&](bool goes_on) {
        if (row == none) return;
        if (begun || goes_on) {
            store_part<float, V>((begun ? s.head : s.tail) + c * a.dim + d0, left, acc);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] *= a.scale;
            store_part<T, V>(out + static_cast<int64_t>(row) * a.dim + d0, left, acc);
        }
    };
    for (int64_t e = e0; e < e1; e += AHEAD) {
        uint32_t r[AHEAD], t[AHEAD], w[AHEAD][4];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {  // (behind the chunk its last entry again)
            const int64_t at = min(e + j, e1 - 1);
            r[j] = s.rows[at];
            t[j] = s.tokens[at];
        }
        if (a.dim >= V) {  // all of them under way, none behind a test; a column group that passes the row's end as in load_vectors
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) load_words<T, V>(grad + static_cast<int64_t>(t[j]) * a.row_stride + d0 - back, V, V, 0, w[j]);
            if (back > 0)
#pragma unroll
                for (int j = 0; j < AHEAD; ++j) move_down(w[j], back * 8 * static_cast<int>(sizeof(T)), 0);
        } else {
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) load_words<T, V>(grad + static_cast<int64_t>(t[j]) * a.row_stride + d0, left, a.dim, 0, w[j]);
        }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            if (e + j >= e1) break;
            if (r[j] != row) {
                finish(false);
                row = r[j];
                begun = false;
#pragma unroll
                for (int i = 0; i < V; ++i) acc[i] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] += element<T>(w[j], i);
        }
    }
    finish(e1 < s.entries && s.rows[e1] == row);
}

// Runs that pass chunk borders: the block of the chunk where one begins adds up its parts, the waves' shares of them in order.
template <class T>
__global__ __launch_bounds__(THREADS) void embed_span_kernel(EmbedArgs a, Sorted s, T *out) {
    constexpr int SPAN = 64;  // columns of a block
    __shared__ float sum_s[THREADS / SPAN][SPAN];
    const int64_t c = blockIdx.x, e0 = c * s.chunk, e1 = e0 + s.chunk;
    if (e1 >= s.entries) return;
    const uint32_t row = s.rows[e1 - 1], after = s.rows[e1], start = s.rows[e0], before = c > 0 ? s.rows[e0 - 1] : a.rows;
    if (row == static_cast<uint32_t>(a.rows) || after != row) return;  // nothing goes on here
    if (start == row && before == row) return;                         // an earlier chunk began it
    const int64_t lo = c + 1;
    int64_t hi = lo;  // chunks lo .. hi - 1 start with this row
    for (int more = THREADS; more == THREADS; hi += more) {
        const int64_t at = hi + threadIdx.x;
        more = __syncthreads_count(at < s.chunks && s.rows[at * s.chunk] == row);
    }
    const int col = threadIdx.x % SPAN, share = threadIdx.x / SPAN;
    const int64_t per = (hi - lo + THREADS / SPAN - 1) / (THREADS / SPAN);
    const int d = blockIdx.y * SPAN + col;
    float sum = 0.f;
    if (d < a.dim) {
        if (share == 0) sum = s.tail[c * a.dim + d];
        const int64_t from = lo + share * per, to = min(from + per, hi);
#pragma unroll 8
        for (int64_t i = from; i < to; ++i) sum += s.head[i * a.dim + d];
    }
    sum_s[share][col] = sum;
    __syncthreads();
    if (share == 0 && d < a.dim) {
        for (int w = 1; w < THREADS / SPAN; ++w) sum += sum_s[w][col];
        out[static_cast<int64_t>(row) * a.dim + d] = static_cast<T>(sum * a.scale);
    }
}

// ---- rows of few tokens --------------------------------------------------------------------------------------------

// Up to SHORT tokens (actions, not words) a thread has a row to itself, in registers: a wave's rows are adjacent in memory, so
// its unaligned 16-byte loads use every line they touch, and no lane waits for another.  K is 8, 16 or SHORT; the tests
// against the real number of tokens are the same for all lanes.  2^20 rows of 7 float32: draw 15 us, log-probabilities 14 and their
// gradient 22, adjustment with a history of 16 entries and a mask 26 (40 to 60 MB each); with eight threads to a row, as for
// longer ones, draw 100, log-probabilities 48, adjustment 101, and of 32 tokens still 90 against 55, 47 against 42, 99 against 87.
constexpr int SHORT = 32;
static_assert(SHORT == MG_LOGPROB_NO_STATS, "the gradient of a short row reads no statistics");

template <class T, int K>
__device__ __forceinline__ void load_row(const T *p, int k, float (&x)[K], uint32_t fill) {
    constexpr int V = WIDE<T>;
#pragma unroll
    for (int i = 0; i < K; i += V) {
        uint32_t w[4];
        load_words<T, V>(p + i, k - i, k, fill, w);
#pragma unroll
        for (int j = 0; j < V; ++j) x[i + j] = element<T>(w, j);
    }
}

template <class T, int K>
__device__ __forceinline__ void store_row(T *p, int k, const float (&x)[K]) {
    store_part<T, K>(p, k, x);
}

// ---- longer rows ---------------------------------------------------------------------------------------------------

// LANES threads (8 to 64: several rows to a block of THREADS; 256 and 512: a block to a row) hold a row of up to LANES * HELD
// 16-byte vectors in registers, vector j * LANES + lane with each: one pass over memory, whose loads are all under way at
// once; the maximum is known before the first exponential.  A row that no block holds is cut into pieces of
// PIECE_LANES * PIECE_HELD vectors, each taken as a row, and a second kernel joins what they give: many blocks to a row also
// where there are few rows.  At the border, 30011 bfloat16, one block to a row is faster still: one row 5.9 us against 9.4 in
// pieces (log-probabilities), 11.3 against 12 (draw); 4095 rows 55 against 60 and 136 against 170.
template <int LANES>
constexpr int BLOCK = LANES > THREADS ? LANES : THREADS;
constexpr int HELD_MOST = 4096, PIECE_LANES = 256, PIECE_HELD = 4;  // vectors of a row in one piece; a piece
template <class T>
constexpr int PIECE = PIECE_LANES * PIECE_HELD * WIDE<T>;  // tokens

template <class T, int LANES, int HELD>
struct Row {
    static constexpr int V = WIDE<T>;
    const T *x;
    int k, lane;
    uint32_t held[HELD][4];

    __device__ __forceinline__ Row(const T *row, int tokens, int thread) : x(row), k(tokens), lane(thread) {
        asm volatile("" : "+v"(lane));  // (else every token's number would wait in a register while rows go by)
        load_vectors<T, HELD>(x, k, 0, LANES, lane, NEG_INF_BITS<T>, held);
    }
    // f(number of the vector, its words) for all of this thread's vectors.  The empty statements keep a pass from sharing its
    // conversions with the next one and the barriers keep the vectors apart: either would take several times the registers.
    template <class F>
    __device__ __forceinline__ void each(F f) {
#pragma unroll
        for (int j = 0; j < HELD; ++j) {
            asm volatile("" : "+v"(held[j][0]), "+v"(held[j][1]), "+v"(held[j][2]), "+v"(held[j][3]));
            f(j, held[j]);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // vector j again, from the cache: an index into registers would cost more
    __device__ __forceinline__ void fetch(int j, uint32_t (&w)[4]) const {
        const int at = token(j, 0);
        load_words<T, V>(x + at, k - at, k, NEG_INF_BITS<T>, w);
    }
    __device__ __forceinline__ int token(int j, int i) const { return (j * LANES + lane) * V + i; }
};

// v of another lane, chosen by a DPP control (a row is 16 lanes): several times quicker than a shuffle through LDS
template <int CONTROL, class X>
__device__ __forceinline__ X of_lane(X v) {
    constexpr int N = sizeof(X) / 4;
    int w[N];
    __builtin_memcpy(w, &v, sizeof v);
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = __builtin_amdgcn_mov_dpp(w[i], CONTROL, 0xF, 0xF, true);
    __builtin_memcpy(&v, w, sizeof v);
    return v;
}
template <class X>
__device__ __forceinline__ X read_lane(X v, int lane) {
    constexpr int N = sizeof(X) / 4;
    int w[N];
    __builtin_memcpy(w, &v, sizeof v);
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = __builtin_amdgcn_readlane(w[i], lane);
    __builtin_memcpy(&v, w, sizeof v);
    return v;
}

template <class X>
__device__ __forceinline__ X other_half(X v) {  // of 32 lanes
    constexpr int N = sizeof(X) / 4;
    int w[N];
    __builtin_memcpy(w, &v, sizeof v);
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = __shfl_xor(w[i], 16, 64);
    __builtin_memcpy(&v, w, sizeof v);
    return v;
}

// f combined over the threads of a row, known to all of them; f is commutative.  `shared` holds one value a wave and is not to be
// used again before another barrier: callers take a slot of their own for each of a row's combinations.
template <int LANES, class X, class F>
__device__ __forceinline__ X over_row(X v, X *shared, F f) {
    v = f(v, of_lane<0xB1>(v));                    // the neighbour
    v = f(v, of_lane<0x4E>(v));                    // the other pair of four
    v = f(v, of_lane<0x141>(v));                   // mirrored in eight
    if constexpr (LANES > 8) v = f(v, of_lane<0x140>(v));  // mirrored in sixteen
    if constexpr (LANES == 32) v = f(v, other_half(v));
    if constexpr (LANES >= 64) v = f(f(read_lane(v, 0), read_lane(v, 16)), f(read_lane(v, 32), read_lane(v, 48)));
    if constexpr (LANES > 64) {
        if (threadIdx.x % 64 == 0) shared[threadIdx.x / 64] = v;
        __syncthreads();
        v = shared[0];
#pragma unroll
        for (int w = 1; w < LANES / 64; ++w) v = f(v, shared[w]);
    }
    return v;
}

__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }  // NaN if one of them is
template <class X>
__device__ __forceinline__ X sum_of(X a, X b) { return a + b; }

// exp(2 ln 2 * z) for z <= 0, NaN for NaN: the exponential instruction gives nothing below 2^-126, the square of half as much
// goes down to the smallest float.  For an exponent x it is off by up to 5 |x| + 5 half steps of float32, about twice as much as expf,
// which rows of up to SHORT tokens take.
__device__ __forceinline__ float exp_twice(float z) {
    const float h = __builtin_amdgcn_exp2f(z);
    return h * h;
}
constexpr float HALF_LOG2E = 0.72134752044448170368f, TWICE_LN2 = 1.38629436111989061883f;
constexpr float DEEP = -200.f;  // exp_twice of it is 0

// ---- adjustment of logits ------------------------------------------------------------------------------------------

// A repeated token's positive logit, or its gradient, is multiplied by 1 / repetition, rounded once for a row, instead of a division for
// a token.  No float holds the reciprocal of a repetition below 2^-126 with all its bits, or at all (and infinity times a gradient of 0
// would be NaN): they are multiplied by 2^24 first, and then by the reciprocal of 2^24 repetitions.
__device__ __forceinline__ float before_reciprocal(float repetition) { return repetition < 0x1p-126f ? 0x1p24f : 1.f; }
__device__ __forceinline__ float reciprocal(float repetition) { return 1.f / (repetition * before_reciprocal(repetition)); }

// frequency * c, and 0 for a token that is not there also if the frequency is infinite: this product is 0 where a factor is.  (With a test
// instead, at a token or once a wave, 256 rows x 128000 take 36.6 us, not 36.0.)
__device__ __forceinline__ float frequency_of(uint32_t c, float frequency) {
    float product;
    asm("v_mul_legacy_f32 %0, %1, %2" : "=v"(product) : "v"(frequency), "v"(static_cast<float>(c)));
    return product;
}

// A block counts a stretch of tokens' occurrences in their rows' histories in LDS, then the stretch streams through once: of
// `lanes` threads to a row (a power of two) each takes up to STRETCH 16-byte vectors, whose loads are under way while the
// history is counted.  Short rows share a block, a row longer than a block's stretch is cut, and each piece looks through the
// whole history (a few KB that the cache holds).  The counters have 16 bits where the history has no more entries than that, so
// that LDS holds eight blocks.  256 rows x 128000 bfloat16, 2048 entries, bits: 37.5 us (135 MB, 3.6 TB/s; 41 with 32-bit counters).
// What keeps it from a copy's 5.1 TB/s is the chain in each block: history, barrier, counting, barrier, output.
constexpr int STRETCH = 4;

template <class T, class H, bool GRAD, class C>
__global__ __launch_bounds__(THREADS) void adjust_kernel(MgAdjust a, int lanes, const T *logits, const T *grad, T *out) {
#pragma clang fp contract(off)
    constexpr int V = WIDE<T>, PIECE = THREADS * STRETCH * V, PER_WORD = 4 / static_cast<int>(sizeof(C)), WORDS = V / PER_WORD;
    __shared__ __align__(16) uint32_t counts_s[PIECE / PER_WORD];
    int lane = threadIdx.x & (lanes - 1);
    const int sub = threadIdx.x / lanes, per_block = THREADS / lanes, width = lanes * STRETCH * V;
    const int first = blockIdx.y * width;  // 0 where rows share a block
    const bool history = a.history_dev != nullptr && a.t > 0;
    uint32_t *counts = counts_s + sub * (width / PER_WORD);
    for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * per_block; row0 < a.n; row0 += static_cast<int64_t>(gridDim.x) * per_block) {
        const int64_t row = row0 + sub;
        const bool live = row < a.n;
        asm volatile("" : "+v"(lane));  // (else every token's number would wait in a register while rows go by)
        uint32_t x[STRETCH][4], g[STRETCH][4];
        if (live) {
            load_vectors<T, STRETCH>(logits + row * a.logits_stride, a.k, first, lanes, lane, 0, x);
            if (GRAD) load_vectors<T, STRETCH>(grad + row * a.grad_stride, a.k, first, lanes, lane, 0, g);
        }
        float rep = 1.f, presence = 0.f, frequency = 0.f;
        if (live) {
            rep = a.repetition_dev ? a.repetition_dev[row] : a.repetition;
            presence = a.presence_dev ? a.presence_dev[row] : a.presence;
            frequency = a.frequency_dev ? a.frequency_dev[row] : a.frequency;
        }
        if (history) {
            // the first entries before their number is known: they lie there whatever it is
            constexpr int AHEAD = 8;
            const H *h = static_cast<const H *>(a.history_dev) + (live ? row : 0) * a.history_stride;
            H entry[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) entry[u] = h[min(lane + u * lanes, a.t - 1)];
            const int len = !live ? 0 : (a.lengths_dev ? min(max(a.lengths_dev[row], 0), a.t) : a.t);
#pragma unroll
            for (int j = 0; j < STRETCH; ++j)
#pragma unroll
                for (int i = 0; i < WORDS; i += 2) *reinterpret_cast<uint2 *>(&counts[(j * lanes + lane) * WORDS + i]) = make_uint2(0, 0);
            __syncthreads();
            const int end = min(width, a.k - first);
            auto count = [&](int i, const H (&entry)[AHEAD]) {
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) {
                    const int64_t j = static_cast<int64_t>(entry[u]) - first;
                    if (i + u * lanes < len && j >= 0 && j < end) {
                        const uint32_t at = static_cast<uint32_t>(j);
                        atomicAdd(&counts[at / PER_WORD], PER_WORD == 1 ? 1u : 1u << (at % PER_WORD * 16));
                    }
                }
            };
            count(lane, entry);
            for (int i = lane + AHEAD * lanes; i < len; i += AHEAD * lanes) {
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) entry[u] = h[min(i + u * lanes, len - 1)];
                count(i, entry);
            }
            __syncthreads();
        }
        if (live) {
            const float inverse = reciprocal(rep);
            const bool some_small = __any(before_reciprocal(rep) != 1.f);  // (asked once a wave: with a factor for every token one row of 32000 takes 6.2 us, not 5.9)
#pragma unroll
            for (int j = 0; j < STRETCH; ++j) {
                const int at = first + (j * lanes + lane) * V;
                if (at >= a.k) break;
                const bool whole = at + V <= a.k;
                uint32_t allow = ~0u;  // bit i: token at + i
                if (a.mask_kind == MG_MASK_BITS) {  // `at` is a multiple of V, 4 or 8: its bits lie in one byte
                    allow = static_cast<const uint8_t *>(a.mask_dev)[4 * row * a.mask_stride + (at >> 3)] >> (at & 7);
                } else if (a.mask_kind == MG_MASK_BYTES) {
                    const uint8_t *m = static_cast<const uint8_t *>(a.mask_dev) + row * a.mask_stride + at;
                    allow = 0;
                    if (whole) {
                        const Vec<uint8_t, V> v = *reinterpret_cast<const Vec<uint8_t, V> *>(m);
#pragma unroll
                        for (int i = 0; i < V; ++i) allow |= (v.v[i] != 0) << i;
                    } else {
                        for (int i = 0; at + i < a.k; ++i) allow |= (m[i] != 0) << i;
                    }
                }
                uint32_t c[V] = {};
                if (history)
#pragma unroll
                    for (int i = 0; i < WORDS; i += 2) {
                        const uint2 q = *reinterpret_cast<const uint2 *>(&counts[(j * lanes + lane) * WORDS + i]);
                        const uint32_t w[2] = {q.x, q.y};
#pragma unroll
                        for (int o = 0; o < 2 * PER_WORD; ++o) c[i * PER_WORD + o] = PER_WORD == 1 ? w[o] : (w[o / PER_WORD] >> (16 * (o % PER_WORD))) & 0xFFFF;
                    }
                float y[V];
#pragma unroll
                for (int i = 0; i < V; ++i) y[i] = element<T>(GRAD ? g[j] : x[j], i);
                if (some_small) {
                    const float first = before_reciprocal(rep);
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        if (c[i] > 0 && element<T>(x[j], i) > 0.f) y[i] *= first;
                }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    if (GRAD) {
                        if (c[i] > 0) y[i] = y[i] * (element<T>(x[j], i) > 0.f ? inverse : rep);
                    } else {
                        if (c[i] > 0) y[i] = y[i] * (y[i] > 0.f ? inverse : rep) - presence;
                        y[i] = y[i] - frequency_of(c[i], frequency);
                    }
                }
                if (!GRAD && a.bias_dev) {
                    const float *b = a.bias_dev + row * a.bias_stride + at;
                    float v[V];
#pragma unroll
                    for (int i = 0; i < V; i += 4) {
                        uint32_t q[4];
                        if (whole) {
                            load_words<float, 4>(b + i, 4, 4, 0, q);
                        } else {
#pragma unroll
                            for (int o = 0; o < 4; ++o) q[o] = at + i + o < a.k ? __builtin_bit_cast(uint32_t, b[i + o]) : 0;
                        }
#pragma unroll
                        for (int o = 0; o < 4; ++o) v[i + o] = element<float>(q, o);
                    }
#pragma unroll
                    for (int i = 0; i < V; ++i) y[i] = y[i] + v[i];
                }
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (!((allow >> i) & 1)) y[i] = GRAD ? 0.f : NEG_INF;
                store_part<T, V>(out + row * a.out_stride + at, a.k - at, y);
                __builtin_amdgcn_sched_barrier(0);  // one vector after the other: fewer registers
            }
        }
        if (history) __syncthreads();  // the counters are read
    }
}

__device__ __forceinline__ uint32_t four_bytes(const uint8_t *p) {
    struct __attribute__((packed)) One {
        uint32_t w;
    };
    return reinterpret_cast<const One *>(p)->w;
}

// Rows of few tokens: every thread counts its own row's history in its own LDS counters (an odd number of words apart, so that
// lanes fall on different banks), which needs no barrier.
template <class T, class H, bool GRAD, int K>
__global__ __launch_bounds__(K <= 16 ? THREADS : 64) void adjust_short_kernel(MgAdjust a, const T *logits, const T *grad, T *out) {
#pragma clang fp contract(off)
    constexpr int ROWS = K <= 16 ? THREADS : 64;
    __shared__ uint32_t counts_s[ROWS][K + 1];
    uint32_t *counts = counts_s[threadIdx.x];
    const int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x;
    if (row >= a.n) return;
    const bool history = a.history_dev != nullptr && a.t > 0;
    float x[K], g[K];
    load_row<T, K>(logits + row * a.logits_stride, a.k, x, 0);
    if (GRAD) load_row<T, K>(grad + row * a.grad_stride, a.k, g, 0);
    const float rep = a.repetition_dev ? a.repetition_dev[row] : a.repetition;
    const float presence = a.presence_dev ? a.presence_dev[row] : a.presence;
    const float frequency = a.frequency_dev ? a.frequency_dev[row] : a.frequency;
    uint32_t allow = ~0u;
    if (a.mask_kind == MG_MASK_BYTES) {
        const uint8_t *m = static_cast<const uint8_t *>(a.mask_dev) + row * a.mask_stride;
        uint32_t w[K / 4];
#pragma unroll
        for (int j = 0; j < K; j += 4) {
            w[j / 4] = 0;
            if (j + 4 <= a.k)
                w[j / 4] = four_bytes(m + j);
            else if (j < a.k && a.k >= 4)
                w[j / 4] = four_bytes(m + a.k - 4) >> (8 * (4 - (a.k - j)));
            else
                for (int i = j; i < a.k; ++i) w[j / 4] |= static_cast<uint32_t>(m[i]) << (8 * (i - j));
        }
        allow = 0;
#pragma unroll
        for (int j = 0; j < K; ++j)
            if ((w[j / 4] >> (8 * (j % 4))) & 0xFF) allow |= 1u << j;
    } else if (a.mask_kind == MG_MASK_BITS) {
        allow = static_cast<const uint32_t *>(a.mask_dev)[row * a.mask_stride];
    }
    float bias[K];
    if (!GRAD && a.bias_dev) {
        if (a.bias_stride == 0) {  // the same for all rows: scalar loads
#pragma unroll
            for (int j = 0; j < K; ++j)
                if (j < a.k) bias[j] = a.bias_dev[j];
        } else {
            load_row<float, K>(a.bias_dev + row * a.bias_stride, a.k, bias, 0);
        }
    }
    if (history) {
#pragma unroll
        for (int j = 0; j < K; ++j) counts[j] = 0;
        constexpr int V = 16 / static_cast<int>(sizeof(H));
        const int len = a.lengths_dev ? min(max(a.lengths_dev[row], 0), a.t) : a.t;
        const H *h = static_cast<const H *>(a.history_dev) + row * a.history_stride;
        int i = 0;
        for (; i + V <= a.t && i < len; i += V) {
            const Vec<H, V> v = *reinterpret_cast<const Vec<H, V> *>(h + i);
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (i + j < len && v.v[j] >= 0 && v.v[j] < static_cast<H>(a.k)) atomicAdd(&counts[v.v[j]], 1u);
        }
        for (; i < len; ++i)
            if (h[i] >= 0 && h[i] < static_cast<H>(a.k)) atomicAdd(&counts[h[i]], 1u);
    }
    const float first = before_reciprocal(rep), inverse = reciprocal(rep);
#pragma unroll
    for (int j = 0; j < K; ++j) {
        if (j >= a.k) continue;
        const uint32_t c = history ? counts[j] : 0;
        const bool ok = (allow >> j) & 1;
        if (GRAD) {
            float v = g[j];
            if (c > 0) v = x[j] > 0.f ? v * first * inverse : v * rep;
            x[j] = ok ? v : 0.f;
        } else {
            float v = x[j];
            if (c > 0) v = (v > 0.f ? v * first * inverse : v * rep) - presence;
            v = v - frequency_of(c, frequency);
            if (a.bias_dev) v = v + bias[j];
            x[j] = ok ? v : NEG_INF;
        }
    }
    store_row<T, K>(out + row * a.out_stride, a.k, x);
}

// ---- draw ----------------------------------------------------------------------------------------------------------

__device__ __forceinline__ void put_token(void *tokens, int type, int64_t row, int64_t token) {
    if (type == MG_U8)
        static_cast<uint8_t *>(tokens)[row] = static_cast<uint8_t>(token);
    else if (type == MG_I32)
        static_cast<int32_t *>(tokens)[row] = static_cast<int32_t>(token);
    else
        static_cast<int64_t *>(tokens)[row] = token;
}

__device__ __forceinline__ int64_t get_token(const void *tokens, int type, int64_t row) {
    if (type == MG_U8) return static_cast<const uint8_t *>(tokens)[row];
    if (type == MG_I32) return static_cast<const int32_t *>(tokens)[row];
    return static_cast<const int64_t *>(tokens)[row];
}

// 2^t in 64 bits for t <= 0: the nearest whole number to the exponent, the rest, at most 1/2, through the polynomial of degree
// ten that meets 2^f at the Chebyshev points of that interval (3e-16 off; 1 at 0).  Half the instructions of a library
// exponential, which also has to deal with what does not come here.
__device__ __forceinline__ double exp2_64(double t) {
    t = fmax(t, -1100.0);  // nothing is left there, and -inf has no rest
    const double n = rint(t), f = t - n;
    double p = 7.072585949269224e-09;
    p = fma(p, f, 1.0208690299958306e-07);
    p = fma(p, f, 1.321544258792169e-06);
    p = fma(p, f, 1.5252657260200837e-05);
    p = fma(p, f, 0.0001540353044173605);
    p = fma(p, f, 0.0013333558230164974);
    p = fma(p, f, 0.009618129107606888);
    p = fma(p, f, 0.05550410866444772);
    p = fma(p, f, 0.24022650695910097);
    p = fma(p, f, 0.69314718055995);
    p = fma(p, f, 1.0);
    return ldexp(p, static_cast<int>(n));
}

// Of a row: a number on the device cannot be refused, one that is no temperature makes the row none that can be drawn from.
__device__ __forceinline__ float temperature_of(const MgLogits &l, int64_t row) {
    const float t = l.temperature_dev ? l.temperature_dev[row] : l.temperature;
    return t >= LEAST_TEMPERATURE && t < -NEG_INF ? t : __builtin_nanf("");
}

// A row as a distribution: its largest logit and log2(e) / temperature.
struct Spread {
    double m, c;
    __device__ __forceinline__ double p(float x) const { return exp2_64((static_cast<double>(x) - m) * c); }
    template <class T>
    __device__ __forceinline__ double of_vector(const uint32_t *v) const {
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < WIDE<T>; ++i) sum += p(element<T>(v, i));
        return sum;
    }
};
__device__ __forceinline__ Spread spread(const MgLogits &l, int64_t row, float m) {
    return Spread{m, 1.4426950408889634 / static_cast<double>(temperature_of(l, row))};
}
__device__ __forceinline__ bool drawable(float m, const Spread &s) { return fabsf(m) < -NEG_INF && s.c == s.c; }

// (outside of [0, 1] it is the nearest end, NaN the lower one)
__device__ __forceinline__ double uniform_at(const void *uniforms, int type, int64_t row) {
    const double u = type == MG_F64 ? static_cast<const double *>(uniforms)[row] : static_cast<double>(static_cast<const float *>(uniforms)[row]);
    return fmin(fmax(u, 0.0), 1.0);
}

// log p of a token from its logit; total - 1 is exact where little stands beside the maximum.  The logarithm has 32 bits, as the result.
__device__ __forceinline__ float drawn_logprob(float x, const Spread &s, double total) {
    return static_cast<float>((static_cast<double>(x) - s.m) * s.c * 0.6931471805599453 - log1pf(static_cast<float>(total - 1.0)));
}

struct DrawShared {
    double sums[HELD_MOST / 64], total[8];
    float most[8];
    int token;
};

// Many long rows: 4095 x 30011 bfloat16 141 us, the likeliest 130, where reading them takes 63 (log-probabilities); 53 are the issue of
// the exponentials in 64 bits, and in a block loads, maximum, exponentials and sums stand one behind the other.  Few are bound by
// latency: 64 rows x 128003 float16 in pieces 9.7 us and their join, which takes a piece's exponentials again, 7.1.
//
// The token of a row (or of a piece of one) at whose sum of probabilities the border lies, known to all of its threads, and
// the total.  `share`: the border is that share of the total; otherwise `border` is it, `before` what stands before the row.
template <class T, int LANES, int HELD>
__device__ __forceinline__ int find_border(Row<T, LANES, HELD> &row, DrawShared &sh, const Spread &s, bool share, double border, double before, double &total) {
    constexpr int V = WIDE<T>, SPAN = LANES < 64 ? LANES : 64, WAVES = LANES > 64 ? LANES / 64 : 1;
    const int wave = LANES > 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : 0, lane = row.lane % 64;
    double part[HELD];
    row.each([&](int j, const uint32_t *v) {
        part[j] = s.of_vector<T>(v);
        asm volatile("" : "+v"(part[j]));  // now, not where it is used
    });
    // inclusive sums over the threads of a wave (or of a shorter row)
    auto upto = [&](double v) {
#pragma unroll
        for (int by = 1; by < SPAN; by *= 2) {
            const double o = __shfl_up(v, by, SPAN);
            if ((lane & (SPAN - 1)) >= by) v += o;
        }
        return v;
    };
    int vec = -1, at_wave = 0;  // where the border lies
    if constexpr (WAVES > 1) {
        // the waves' sums of each vector: every exchange halves the vectors that a thread adds up
        int of = 0;
#pragma unroll
        for (int half = HELD / 2, by = 32; half > 0; half /= 2, by /= 2) {
            const bool upper = lane & by;
            of += upper ? half : 0;
#pragma unroll
            for (int j = 0; j < half; ++j) {
                const double give = upper ? part[j] : part[j + half], keep = upper ? part[j + half] : part[j];
                part[j] = keep + __shfl_xor(give, by, 64);
            }
        }
#pragma unroll
        for (int by = 32 / HELD; by > 0; by /= 2) part[0] += __shfl_xor(part[0], by, 64);
        if (lane % (64 / HELD) == 0) sh.sums[of * WAVES + wave] = part[0];
        __syncthreads();
        // in the order of the tokens: vectors, then waves; every wave does this by itself
        constexpr int N = HELD * WAVES, EACH = (N + 63) / 64;
        double own[EACH], run = 0.0;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            own[i] = lane * EACH + i < N ? sh.sums[lane * EACH + i] : 0.0;
            run += own[i];
        }
        const double end = upto(run);
        total = read_lane(end, 63);
        if (share) border *= total;
        double sum = before + (lane ? end - run : 0.0), start = 0.0;
        int found = N;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            if (found == N && own[i] > 0.0 && sum + own[i] > border) {  // (own: rounding may put the sum of one that has none above the last one's)
                found = lane * EACH + i;
                start = sum;
            }
            sum += own[i];
        }
        const uint64_t any = __ballot(found < N);
        if (any) {
            const int from = __builtin_ctzll(any);
            found = __shfl(found, from, 64);
            before = __shfl(start, from, 64);
            vec = found / WAVES;
            at_wave = found % WAVES;
        }
    } else {
        double sums[HELD];
        total = 0.0;
#pragma unroll
        for (int j = 0; j < HELD; ++j) {
            sums[j] = over_row<LANES>(part[j], sh.total, sum_of<double>);
            total += sums[j];
        }
        if (share) border *= total;
        double sum = before;
#pragma unroll
        for (int j = 0; j < HELD; ++j) {
            if (vec < 0 && sums[j] > 0.0 && sum + sums[j] > border) {
                vec = j;
                before = sum;
            }
            sum += sums[j];
        }
    }
    // the thread, then the token
    int token = -1;
    if (vec >= 0 && wave == at_wave) {
        uint32_t v[4];
        row.fetch(vec, v);
        const double here = s.of_vector<T>(v), end = before + upto(here);
        const int shift = (threadIdx.x % 64) / SPAN * SPAN;
        const uint64_t threads = (~0ull >> (64 - SPAN)) << shift;
        const uint64_t above = __ballot(end > border && here > 0.0) & threads, some = __ballot(here > 0.0) & threads;
        // rounding may leave none above it: the last one that has any then
        const int at = (above ? __builtin_ctzll(above) : (some ? 63 - __builtin_clzll(some) : shift)) - shift;
        if ((lane & (SPAN - 1)) == at) {
            double sum = at == 0 ? before : end - here;
            bool done = false;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const double q = s.p(element<T>(v, i));
                sum += q;
                if (!done && q > 0.0) token = row.token(vec, i);
                done |= sum > border;
            }
        }
        token = __shfl(token, shift + at, 64);
    }
    if (vec < 0 || WAVES > 1) {  // (the same for all threads of the row)
        if (vec < 0) {           // rounding left no sum above it: the last token that has any
            int last = -1;
            row.each([&](int j, const uint32_t *v) {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (s.p(element<T>(v, i)) > 0.0) last = max(last, row.token(j, i));
            });
#pragma unroll
            for (int by = SPAN / 2; by > 0; by /= 2) last = max(last, __shfl_xor(last, by, 64));
            token = last;
        }
        if constexpr (WAVES > 1) {
            if (threadIdx.x == 0) sh.token = -1;
            __syncthreads();
            if (lane == 0 && token >= 0) atomicMax(&sh.token, token);
            __syncthreads();
            token = sh.token;
        }
    }
    return token;
}

// the lowest token of the largest logit, and the total
template <class T, int LANES, int HELD>
__device__ __forceinline__ int find_largest(Row<T, LANES, HELD> &row, DrawShared &sh, const Spread &s, float m, double &total) {
    constexpr int WAVES = LANES > 64 ? LANES / 64 : 1;
    double sum = 0.0;
    int found = 0x7FFFFFFF;
    row.each([&](int j, const uint32_t *v) {
        sum += s.of_vector<T>(v);
#pragma unroll
        for (int i = 0; i < WIDE<T>; ++i)
            if (element<T>(v, i) == m) found = min(found, row.token(j, i));
    });
    total = over_row<LANES>(sum, sh.total, sum_of<double>);
#pragma unroll
    for (int by = (LANES < 64 ? LANES : 64) / 2; by > 0; by /= 2) found = min(found, __shfl_xor(found, by, 64));
    if constexpr (WAVES > 1) {
        if (threadIdx.x == 0) sh.token = 0x7FFFFFFF;
        __syncthreads();
        if (threadIdx.x % 64 == 0) atomicMin(&sh.token, found);
        __syncthreads();
        found = sh.token;
    }
    return found;
}

template <class T, int LANES, int HELD>
__device__ __forceinline__ float largest(Row<T, LANES, HELD> &row, float *shared) {
    float m = NEG_INF;
    row.each([&](int, const uint32_t *v) {
#pragma unroll
        for (int e = 0; e < WIDE<T>; ++e) m = larger(m, element<T>(v, e));
    });
    return over_row<LANES>(m, shared, larger);
}

__device__ __forceinline__ void put_drawn(const MgLogits &l, int64_t row, int token, float m, const Spread &s, float lp, void *tokens, float *logprob) {
    put_token(tokens, l.tokens_type, row, token);
    if (logprob) logprob[row] = token >= 0 ? lp : (m == NEG_INF && s.c == s.c ? NEG_INF : __builtin_nanf(""));
}

template <class T, int LANES, int HELD>
__global__ __launch_bounds__(BLOCK<LANES>, HELD == 8 ? 4 : 1) void draw_kernel(MgLogits l, const T *logits, const void *uniforms, int uniforms_type, void *tokens, float *logprob) {
    __shared__ DrawShared sh;
    constexpr int ROWS = BLOCK<LANES> / LANES;
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    const int64_t step = static_cast<int64_t>(gridDim.x) * ROWS;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * ROWS + sub; i < l.n; i += step) {
        Row<T, LANES, HELD> row(logits + i * l.stride, l.k, lane);
        const double u = uniforms ? uniform_at(uniforms, uniforms_type, i) : 0.0;
        const float m = largest(row, sh.most);
        const Spread s = spread(l, i, m);
        int token = -1;
        double total = 0.0;
        if (drawable(m, s)) token = uniforms ? find_border(row, sh, s, true, u, 0.0, total) : find_largest(row, sh, s, m, total);
        if (lane == 0) put_drawn(l, i, token, m, s, token >= 0 && logprob ? drawn_logprob(static_cast<float>(logits[i * l.stride + token]), s, total) : 0.f, tokens, logprob);
        if (LANES > 64 && i + step < l.n) __syncthreads();  // the shared values are read
    }
}

// A long row's pieces: each one's largest logit and its total relative to that.
struct DrawPiece {
    double total;
    float m, unused;
};

template <class T>
__global__ __launch_bounds__(PIECE_LANES) void draw_pieces_kernel(MgLogits l, const T *logits, DrawPiece *pieces) {
    __shared__ DrawShared sh;
    const int first = blockIdx.x * PIECE<T>;
    for (int64_t i = blockIdx.y; i < l.n; i += gridDim.y) {
        Row<T, PIECE_LANES, PIECE_HELD> row(logits + i * l.stride + first, min(PIECE<T>, l.k - first), threadIdx.x);
        const float m = largest(row, sh.most);
        double sum = m == NEG_INF ? 0.0 : __builtin_nan("");
        if (fabsf(m) < -NEG_INF) {
            const Spread s = spread(l, i, m);
            sum = 0.0;
            row.each([&](int, const uint32_t *v) { sum += s.of_vector<T>(v); });
            sum = over_row<PIECE_LANES>(sum, sh.total, sum_of<double>);
        }
        if (threadIdx.x == 0) pieces[i * gridDim.x + blockIdx.x] = DrawPiece{sum, m, 0.f};
        __syncthreads();
    }
}

// One block to a row: the pieces' totals, the piece in which the border lies, the token in that piece.  Every wave goes through
// the pieces by itself, a run of adjacent ones to each lane, and comes to the same.
template <class T>
__global__ __launch_bounds__(PIECE_LANES) void draw_join_kernel(MgLogits l, const T *logits, const void *uniforms, int uniforms_type, const DrawPiece *pieces,
                                                                int count, void *tokens, float *logprob) {
    __shared__ DrawShared sh;
    const int lane = threadIdx.x % 64, run = (count + 63) / 64, lo = min(lane * run, count), hi = min(lo + run, count);
    for (int64_t i = blockIdx.x; i < l.n; i += gridDim.x) {
        const DrawPiece *of = pieces + i * count;
        const double u = uniforms ? uniform_at(uniforms, uniforms_type, i) : 0.0;
        float m = NEG_INF;
        for (int p = lo; p < hi; ++p) m = larger(m, of[p].m);
        m = over_row<64>(m, sh.most, larger);
        const Spread s = spread(l, i, m);
        if (!drawable(m, s)) {
            if (threadIdx.x == 0) put_drawn(l, i, -1, m, s, 0.f, tokens, logprob);
            continue;
        }
        auto total_of = [&](int p) { return of[p].m == NEG_INF ? 0.0 : of[p].total * exp2_64((static_cast<double>(of[p].m) - s.m) * s.c); };
        double mine = 0.0;
        for (int p = lo; p < hi; ++p) mine += total_of(p);
        double end = mine;
#pragma unroll
        for (int by = 1; by < 64; by *= 2) {
            const double o = __shfl_up(end, by, 64);
            if (lane >= by) end += o;
        }
        const double total = read_lane(end, 63), border = u * total;
        // the lane whose pieces hold the border (rounding may leave none: the last one that has any), or the largest logit
        int piece = -1;
        double before = lane ? end - mine : 0.0;
        uint64_t there;
        if (uniforms) {
            const uint64_t above = __ballot(end > border && mine > 0.0), some = __ballot(mine > 0.0);
            there = above ? above & -above : 1ull << (63 - __builtin_clzll(some));
            double sum = before;
            bool done = false;
            for (int p = lo; p < hi && !done; ++p) {
                const double t = total_of(p);
                if (t > 0.0) {
                    piece = p;
                    before = sum;
                }
                sum += t;
                done = sum > border;
            }
        } else {
            for (int p = hi - 1; p >= lo; --p)
                if (of[p].m == m) piece = p;
            const uint64_t has = __ballot(piece >= 0);
            there = has & -has;
        }
        const int from = __builtin_ctzll(there);
        piece = __shfl(piece, from, 64);
        before = __shfl(before, from, 64);
        const int first = piece * PIECE<T>;
        Row<T, PIECE_LANES, PIECE_HELD> row(logits + i * l.stride + first, min(PIECE<T>, l.k - first), threadIdx.x);
        double unused;
        const int token = first + (uniforms ? find_border(row, sh, s, false, border, before, unused) : find_largest(row, sh, s, m, unused));
        if (threadIdx.x == 0) put_drawn(l, i, token, m, s, logprob ? drawn_logprob(static_cast<float>(logits[i * l.stride + token]), s, total) : 0.f, tokens, logprob);
        __syncthreads();
    }
}

// Rows of few tokens: one thread each.
template <class T, int K>
__global__ __launch_bounds__(THREADS) void draw_short_kernel(MgLogits l, const T *logits, const void *uniforms, int uniforms_type,
                                                             void *tokens, float *logprob) {
    const int64_t row = static_cast<int64_t>(blockIdx.x) * THREADS + threadIdx.x;
    if (row >= l.n) return;
    float x[K];
    load_row<T, K>(logits + row * l.stride, l.k, x, NEG_INF_BITS<T>);
    const double u = uniforms ? uniform_at(uniforms, uniforms_type, row) : 0.0;
    float m = x[0];
#pragma unroll
    for (int j = 1; j < K; ++j) m = larger(m, x[j]);
    const Spread s = spread(l, row, m);
    int token = -1;
    float lp = 0.f;
    if (drawable(m, s)) {
        // what is filled up behind the last token is -inf, so 0
        constexpr bool KEEP = K <= 16;
        double p[KEEP ? K : 1], total = 0.0;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            if (j >= l.k) break;
            const double v = s.p(x[j]);
            if (KEEP) p[j] = v;
            total += v;
        }
        float at = m;
        if (uniforms) {
            const double border = u * total;
            double upto = 0.0;
            bool done = false;
#pragma unroll
            for (int j = 0; j < K; ++j) {
                if (j >= l.k) break;
                const double v = KEEP ? p[KEEP ? j : 0] : s.p(x[j]);
                upto += v;
                if (!done && v > 0.0) {
                    token = j;
                    at = x[j];
                }
                done |= upto > border;
            }
        } else {
#pragma unroll
            for (int j = K - 1; j >= 0; --j)
                if (x[j] == m) token = j;
        }
        if (logprob) lp = drawn_logprob(at, s, total);
    }
    put_drawn(l, row, token, m, s, lp, tokens, logprob);
}

// ---- log-probabilities and entropies -------------------------------------------------------------------------------

// A part of a row: its maximum m, the sum of e = exp((x - m) / T) over its tokens LESS the one of the maximum itself (r), and
// the sum of e * (x - m) / T (t <= 0).  The maximum's own 1 is left out because what is wanted is log(1 + r): for a row whose
// maximum holds nearly everything, r is small and 1 + r would lose it.  Nothing seen yet: m = -inf, r = -1.
struct Soft {
    float m, r, t;
};

// Two parts of a row as one.
__device__ __forceinline__ Soft merge(Soft a, Soft b, float inv_t) {
    if (b.m > a.m || b.m != b.m) {
        const Soft c = a;
        a = b;
        b = c;
    }
    if (b.m == NEG_INF) {
        a.r += b.r + 1.f;  // 0, or NaN
        return a;
    }
    const float d = (b.m - a.m) * inv_t, e = expf(d), s = 1.f + b.r;
    a.r += s * e;
    if (e > 0.f) a.t += e * (b.t + s * d);
    return a;
}

__device__ __forceinline__ Soft merge_wave(Soft s, float inv_t) {
#pragma unroll
    for (int by = 32; by > 0; by /= 2) {
        Soft o;
        o.m = __shfl_down(s.m, by, 64);
        o.r = __shfl_down(s.r, by, 64);
        o.t = __shfl_down(s.t, by, 64);
        s = merge(s, o, inv_t);
    }
    return s;
}

// What the slope of a finished row needs: its maximum, the logarithm of its total, its entropy.
__device__ __forceinline__ float4 row_stats(const Soft &s) {
    const bool empty = s.m == NEG_INF && s.r == -1.f;
    const float log_total = s.m == -NEG_INF ? __builtin_nanf("") : log1pf(s.r);
    return make_float4(empty ? NEG_INF : (s.r == s.r ? s.m : s.r), log_total, empty ? 0.f : log_total - s.t / (1.f + s.r), 0.f);
}

// The token whose log-probability is wanted and its logit, read before anything is waited for; -1: none.
struct Taken {
    int64_t token;
    float x;
};
template <class T>
__device__ __forceinline__ Taken taken(const MgLogits &l, const T *x, int64_t row, const void *tokens, bool wanted) {
    Taken t{-1, 0.f};
    if (wanted) {
        t.token = get_token(tokens, l.tokens_type, row);
        if (t.token >= l.k) t.token = -1;
        if (t.token >= 0) t.x = static_cast<float>(x[t.token]);
    }
    return t;
}

// What a finished row gives.
__device__ __forceinline__ void row_result(int64_t row, const Soft &s, float inv_t, const Taken &t, float *logprob, float *entropy, float *stats) {
    const float4 st = row_stats(s);
    if (logprob) logprob[row] = t.token < 0 ? 0.f : (st.x == NEG_INF ? NEG_INF : (t.x - s.m) * inv_t - st.y);
    if (entropy) entropy[row] = st.z;
    if (stats) reinterpret_cast<float4 *>(stats)[row] = st;
}

struct SoftShared {
    float most[8];
    float2 sums[8], rest[8];
};

template <class T, int LANES, int HELD>
__device__ __forceinline__ Soft soft_of(Row<T, LANES, HELD> &row, SoftShared &sh, float inv_t) {
    const auto both = [](float2 a, float2 b) { return make_float2(a.x + b.x, a.y + b.y); };
    const float c = inv_t * HALF_LOG2E;
    Soft s{largest(row, sh.most), -1.f, 0.f};
    if (inv_t != inv_t) s.m = inv_t;  // no temperature: NaN throughout
    if (s.m > NEG_INF && s.m < -NEG_INF) {
        float sum = 0.f, slant = 0.f;
        row.each([&](int, const uint32_t *v) {
#pragma unroll
            for (int e = 0; e < WIDE<T>; ++e) {
                const float z = fmaxf((element<T>(v, e) - s.m) * c, DEEP), p = exp_twice(z);
                sum += p;
                slant = fmaf(p, z, slant);
            }
        });
        asm volatile("" : "+v"(sum), "+v"(slant));  // now, not where it is used: every p and z would wait for it
        const float2 sums = over_row<LANES>(make_float2(sum, slant), sh.sums, both);
        s.t = sums.y * TWICE_LN2;
        s.r = sums.x - 1.f;
        if (sums.x < 1.0625f) {  // little beside the maximum: the sum again without it, and how often it stands there
            float rest = 0.f, equal = 0.f;
            row.each([&](int, const uint32_t *v) {
#pragma unroll
                for (int e = 0; e < WIDE<T>; ++e) {
                    const float x = element<T>(v, e);
                    equal += x == s.m ? 1.f : 0.f;
                    rest += x == s.m ? 0.f : exp_twice((x - s.m) * c);
                }
            });
            const float2 r = over_row<LANES>(make_float2(rest, equal), sh.rest, both);
            s.r = r.x + (r.y - 1.f);
        }
    } else if (s.m != NEG_INF) {
        s.r = __builtin_nanf("");
    }
    return s;
}

template <class T, int LANES, int HELD>
__global__ __launch_bounds__(BLOCK<LANES>) void logprob_kernel(MgLogits l, const T *logits, const void *tokens, float *logprob, float *entropy, float *stats) {
    __shared__ SoftShared sh;
    constexpr int ROWS = BLOCK<LANES> / LANES;
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    const int64_t step = static_cast<int64_t>(gridDim.x) * ROWS;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * ROWS + sub; i < l.n; i += step) {
        Row<T, LANES, HELD> row(logits + i * l.stride, l.k, lane);
        const Taken t = taken(l, logits + i * l.stride, i, tokens, logprob != nullptr);
        const float inv_t = 1.f / temperature_of(l, i);
        const Soft s = soft_of(row, sh, inv_t);
        if (lane == 0) row_result(i, s, inv_t, t, logprob, entropy, stats);
        if (LANES > 64 && i + step < l.n) __syncthreads();  // the shared values are read
    }
}

// 4095 x 30011 bfloat16: 63 us (246 MB, 3.9 TB/s; a float32 sum over them 69), 82 behind the gradient of another batch.
//
// A long row's pieces, and their join by one wave.
template <class T>
__global__ __launch_bounds__(PIECE_LANES) void logprob_pieces_kernel(MgLogits l, const T *logits, float4 *pieces) {
    __shared__ SoftShared sh;
    const int first = blockIdx.x * PIECE<T>;
    for (int64_t i = blockIdx.y; i < l.n; i += gridDim.y) {
        Row<T, PIECE_LANES, PIECE_HELD> row(logits + i * l.stride + first, min(PIECE<T>, l.k - first), threadIdx.x);
        const Soft s = soft_of(row, sh, 1.f / temperature_of(l, i));
        if (threadIdx.x == 0) pieces[i * gridDim.x + blockIdx.x] = make_float4(s.m, s.r, s.t, 0.f);
        __syncthreads();
    }
}

template <class T>
__global__ __launch_bounds__(64) void logprob_join_kernel(MgLogits l, const T *logits, const float4 *pieces, int count, const void *tokens, float *logprob,
                                                          float *entropy, float *stats) {
    for (int64_t i = blockIdx.x; i < l.n; i += gridDim.x) {
        const Taken t = taken(l, logits + i * l.stride, i, tokens, logprob != nullptr);
        const float inv_t = 1.f / temperature_of(l, i);
        Soft s{NEG_INF, -1.f, 0.f};
        for (int p = threadIdx.x; p < count; p += 64) {
            const float4 q = pieces[i * count + p];
            s = merge(s, Soft{q.x, q.y, q.z}, inv_t);
        }
        s = merge_wave(s, inv_t);
        if (threadIdx.x == 0) row_result(i, s, inv_t, t, logprob, entropy, stats);
    }
}

// A row's incoming gradients g (of the log-probability) and h (of the entropy), divided by its temperature.  Where that could pass the
// largest float (a temperature below 1, and a gradient above 4 at the least one) they stay as they are and `after` is 1 / T: infinity
// times a probability of 0 would be NaN.  512 is more than |log p + entropy| comes to, see LEAST_LOGPROB.
struct Incoming {
    float g, h, after;
};
__device__ __forceinline__ Incoming incoming(float g, float h, float inv_t) {
    const bool fits = (fabsf(g) + 512.f * fabsf(h)) * inv_t < -NEG_INF;
    return fits ? Incoming{g * inv_t, h * inv_t, 1.f} : Incoming{g, h, inv_t};
}
// A log-probability where it multiplies: from here on p is 0, and 0 times -infinity (a logit of the type's lowest value at a temperature
// below 1) would be NaN.
constexpr float LEAST_LOGPROB = 2.f * DEEP;

// One product with p, the smallest factor, and that last: a p below 2^-126 has few bits left, which a second rounding would halve.
// (Where `after` is not 1, g or 512 h is above 4: their product with p has no fewer bits than p.)  A row that is NaN has it in st.z,
// which nothing clamps.
__device__ __forceinline__ float logprob_slope(float x, bool is_token, float4 st, float inv_t, const Incoming &in) {
    if (x == NEG_INF) return 0.f;
    const float lp = (x - st.x) * inv_t - st.y, p = expf(lp), hs = in.h * (fmaxf(lp, LEAST_LOGPROB) + st.z);
    return (is_token ? -in.g * expm1f(lp) - p * hs : -p * (in.g + hs)) * in.after;
}

// One pass over the logits, `lanes` threads (a power of two) to a row or to a piece of one.  Bound by memory: 4095 x 30011 bfloat16
// 104 us (492 MB, 4.7 TB/s), 87 behind the forward pass (part of the logits is still in the cache).
template <class T>
__global__ __launch_bounds__(THREADS) void logprob_grad_kernel(MgLogits l, int lanes, const T *logits, const void *tokens, const float *stats,
                                                               const float *grad_lp, int64_t lp_stride, const float *grad_h, int64_t h_stride, T *out) {
    constexpr int V = WIDE<T>, TAKES = 4;
    int lane = threadIdx.x & (lanes - 1);
    const int sub = threadIdx.x / lanes, per_block = THREADS / lanes, width = lanes * TAKES * V;
    const int first = blockIdx.y * width;
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * per_block + sub; row < l.n; row += static_cast<int64_t>(gridDim.x) * per_block) {
        const T *x = logits + row * l.stride;
        T *to = out + row * l.k;
        asm volatile("" : "+v"(lane));  // (else every token's number would wait in a register while rows go by)
        uint32_t w[TAKES][4];
        load_vectors<T, TAKES>(x, l.k, first, lanes, lane, NEG_INF_BITS<T>, w);
        // (none of these waits for another)
        const float temperature = temperature_of(l, row);
        const float4 st = reinterpret_cast<const float4 *>(stats)[row];
        const int64_t token = grad_lp ? get_token(tokens, l.tokens_type, row) : -1;
        const float grad_of_lp = grad_lp ? grad_lp[row * lp_stride] : 0.f, grad_of_h = grad_h ? grad_h[row * h_stride] : 0.f;
        const float inv_t = 1.f / temperature;
        const Incoming in = incoming(token >= 0 && token < l.k ? grad_of_lp : 0.f, grad_of_h, inv_t);
        // what a p of 0 must not hide: NaN where the row has one
        const float whole = fmaf(in.h, st.z, in.g);
#pragma unroll
        for (int j = 0; j < TAKES; ++j) {
            const int at = first + (j * lanes + lane) * V;
            if (at >= l.k) break;
            float v[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float at_i = element<T>(w[j], i), lp = fmaxf((at_i - st.x) * inv_t - st.y, LEAST_LOGPROB), p = exp_twice(lp * HALF_LOG2E);
                v[i] = at_i == NEG_INF ? 0.f : -p * fmaf(in.h, lp, whole) * in.after;
            }
            if (token >= at && token < at + V) {
                const float own = logprob_slope(static_cast<float>(x[token]), true, st, inv_t, in);
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (at + i == token) v[i] = own;
            }
            store_part<T, V>(to + at, l.k - at, v);
            __builtin_amdgcn_sched_barrier(0);  // one vector after the other: fewer registers
        }
    }
}

// Rows of few tokens: one thread each, the row in registers, its maximum known before the first exponential.  The backward pass
// works the row out again rather than reading what the forward pass could have kept (16 bytes, more than half of seven logits).
template <int K>
__device__ __forceinline__ Soft soft_short(const float (&x)[K], int k, float inv_t) {
    float m = x[0];
#pragma unroll
    for (int j = 1; j < K; ++j) m = __builtin_elementwise_maximum(m, x[j]);  // NaN if one is there
    if (inv_t != inv_t) m = inv_t;  // no temperature: NaN throughout
    Soft s{m, m == NEG_INF ? -1.f : 0.f, 0.f};
    bool passed = m == NEG_INF;
#pragma unroll
    for (int j = 0; j < K; ++j) {
        if (j >= k) break;
        const float z = (x[j] - m) * inv_t, e = expf(z);
        if (!passed && x[j] == m) {
            passed = true;
        } else if (m != NEG_INF) {
            s.r += e;
            if (e > 0.f) s.t += e * z;
        }
    }
    return s;
}

template <class T, int K>
__global__ __launch_bounds__(THREADS) void logprob_short_kernel(MgLogits l, const T *logits, const void *tokens, float *logprob,
                                                                float *entropy, float *stats) {
    const int64_t row = static_cast<int64_t>(blockIdx.x) * THREADS + threadIdx.x;
    if (row >= l.n) return;
    float x[K];
    load_row<T, K>(logits + row * l.stride, l.k, x, NEG_INF_BITS<T>);
    const Taken t = taken(l, logits + row * l.stride, row, tokens, logprob != nullptr);
    const float inv_t = 1.f / temperature_of(l, row);
    row_result(row, soft_short<K>(x, l.k, inv_t), inv_t, t, logprob, entropy, stats);
}

template <class T, int K>
__global__ __launch_bounds__(THREADS) void logprob_grad_short_kernel(MgLogits l, const T *logits, const void *tokens, const float *grad_lp,
                                                                     int64_t lp_stride, const float *grad_h, int64_t h_stride, T *out) {
    const int64_t row = static_cast<int64_t>(blockIdx.x) * THREADS + threadIdx.x;
    if (row >= l.n) return;
    float x[K];
    load_row<T, K>(logits + row * l.stride, l.k, x, NEG_INF_BITS<T>);
    const float temperature = temperature_of(l, row);
    const int64_t token = grad_lp ? get_token(tokens, l.tokens_type, row) : -1;
    const float grad_of_lp = grad_lp ? grad_lp[row * lp_stride] : 0.f, grad_of_h = grad_h ? grad_h[row * h_stride] : 0.f;
    const float inv_t = 1.f / temperature;
    const Incoming in = incoming(token >= 0 && token < l.k ? grad_of_lp : 0.f, grad_of_h, inv_t);
    const float4 st = row_stats(soft_short<K>(x, l.k, inv_t));
#pragma unroll
    for (int j = 0; j < K; ++j)
        if (j < l.k) x[j] = logprob_slope(x[j], j == token, st, inv_t, in);
    store_row<T, K>(out + row * l.k, l.k, x);
}

// ---- host side -----------------------------------------------------------------------------------------------------

using mgrid::refuse;

int launched(const char *who) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MG_OK : refuse(MG_EHIP, "%s: %s", who, hipGetErrorString(e));
}

unsigned blocks_for(int64_t items, int64_t most = 1 << 20) { return static_cast<unsigned>(items < most ? items : most); }

constexpr int64_t MOST_ROWS = (1ll << 31) - 1;
constexpr int32_t MOST_TOKENS = 1 << 24, MOST_COLUMNS = 1 << 20;  // (a grid's second dimension ends at 65535: 2^20 columns in blocks of 32)

bool workspace_ok(const char *who, const void *workspace, int64_t bytes, int64_t need) {
    if (need == 0 || (workspace && bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0)) return true;
    refuse(MG_EINVAL, "%s: needs a workspace of %lld bytes, 16-byte aligned", who, static_cast<long long>(need));
    return false;
}

bool dtype_ok(int32_t t) { return t == MG_F32 || t == MG_BF16 || t == MG_F16; }
bool int_ok(int32_t t) { return t == MG_U8 || t == MG_I32 || t == MG_I64; }

int embed_args(const char *who, const MgEmbed *e, EmbedArgs *a) {
    if (!e) return refuse(MG_EINVAL, "%s: null argument", who);
    if (e->n < 0 || e->n > MOST_ROWS) return refuse(MG_EINVAL, "%s: n %lld not supported (0..2^31 - 1)", who, static_cast<long long>(e->n));
    if (e->fields < 1 || e->fields > MG_MAX_FIELDS) return refuse(MG_EINVAL, "%s: %d fields not supported (1..%d)", who, e->fields, MG_MAX_FIELDS);
    if (e->dim < 1 || e->dim > MOST_COLUMNS) return refuse(MG_EINVAL, "%s: dim %d not supported (1..2^20)", who, e->dim);
    if (!int_ok(e->ids_type)) return refuse(MG_EINVAL, "%s: unknown type %d of the ids", who, e->ids_type);
    if (!dtype_ok(e->dtype)) return refuse(MG_EINVAL, "%s: unknown element type %d", who, e->dtype);
    if (e->ids_stride < 0 || e->field_stride < 0 || e->row_stride < 0) return refuse(MG_EINVAL, "%s: negative stride", who);
    if (e->reserved0 != 0) return refuse(MG_EINVAL, "%s: reserved0 must be 0", who);
    int64_t rows = 0;
    *a = EmbedArgs{e->n, e->ids_stride, e->field_stride, e->row_stride, e->fields, e->dim, 0, e->scale, {}};
    for (int f = 0; f < e->fields; ++f) {
        if (e->sizes[f] < 1) return refuse(MG_EINVAL, "%s: field %d has %d rows", who, f, e->sizes[f]);
        a->sizes[f] = e->sizes[f];
        rows += e->sizes[f];
    }
    if (e->n * e->fields > MOST_ROWS) return refuse(MG_EINVAL, "%s: n %lld times %d fields not supported (at most 2^31 - 1)", who, static_cast<long long>(e->n), e->fields);
    if (rows > 1ll << 30) return refuse(MG_EINVAL, "%s: %lld rows not supported (at most 2^30)", who, static_cast<long long>(rows));
    a->rows = static_cast<int32_t>(rows);
    return MG_OK;
}

// f(a value of the element type, a value of the ids' type)
template <class F>
void with_types(int32_t dtype, int32_t ints, F f) {
    auto inner = [&](auto t) {
        if (ints == MG_U8)
            f(t, uint8_t{});
        else if (ints == MG_I32)
            f(t, int32_t{});
        else
            f(t, int64_t{});
    };
    if (dtype == MG_F32)
        inner(float{});
    else if (dtype == MG_BF16)
        inner(bf16{});
    else
        inner(f16{});
}

// How a table gradient is taken: what it needs of the workspace, in order, each part 16-byte aligned.
struct GradPlan {
    bool few;
    // few rows
    int width, tiles, blocks;  // columns of a lane, tiles of 16 rows, blocks over the tokens
    // sorted
    bool one;                   // sorted by one workgroup
    int64_t entries;
    int bits, passes, sort_blocks, span;
    Sorted s;
    int64_t at_rows, at_tokens, at_head, at_tail, at_pairs, at_counts;
    int64_t bytes;
};

GradPlan plan_grad(const EmbedArgs &a, int wide) {
    GradPlan p{};
    auto take = [&](int64_t bytes) {
        const int64_t at = p.bytes;
        p.bytes += (bytes + 15) / 16 * 16;
        return at;
    };
    p.few = a.rows <= FEW && a.row_stride <= FAR_ROWS && a.n >= 64;  // (a wave takes 64 tokens at a time)
    if (p.few) {
        p.width = wide / 2;  // the narrowest that holds a token's columns at once, or 8 bytes: two sets of 16 loads are held
        while (p.width > 1 && (16 * (p.width / 2) >= a.dim || p.width > a.dim)) p.width /= 2;
        p.tiles = a.rows <= 32 ? 2 : 4;
        if (p.tiles > 2 && p.width > 2) p.width = 2;  // (the sums of four tiles and four columns leave no registers for the loads)
        const int64_t blocks = (a.n + THREADS - 1) / THREADS;
        const int64_t slabs = (a.dim + 16 * p.width - 1) / (16 * p.width), all = p.width > 2 ? FEW_BLOCKS * 2 / 3 : FEW_BLOCKS,
                      most = slabs < all / 64 ? all / slabs : 64;
        p.blocks = static_cast<int>(blocks < 1 ? 1 : (blocks < most ? blocks : most));
        if (p.blocks > 1) take(static_cast<int64_t>(p.blocks) * a.rows * a.dim * 4);
        return p;
    }
    p.entries = a.n * a.fields;
    int bits = 1;
    while ((a.rows >> bits) > 0) ++bits;  // the row numbers 0 .. rows
    p.passes = (bits + DIGIT - 1) / DIGIT;
    p.bits = (bits + p.passes - 1) / p.passes;
    p.one = p.entries <= SORT_ONE && a.rows <= SORT_ROWS;
    p.at_rows = take(p.entries * 4);
    p.at_tokens = take(p.entries * 4);
    // chunks of 16 entries until there are 4096 of them, longer ones then
    int64_t chunk = (p.entries + 4095) / 4096;
    chunk = chunk < 16 ? 16 : (chunk + 7) / 8 * 8;
    p.s.entries = p.entries;
    p.s.chunk = static_cast<int32_t>(chunk);
    p.s.chunks = static_cast<int32_t>((p.entries + chunk - 1) / chunk);
    p.at_head = take(static_cast<int64_t>(p.s.chunks) * a.dim * 4);
    p.at_tail = take(static_cast<int64_t>(p.s.chunks) * a.dim * 4);
    p.s.lanes = 1;
    while (p.s.lanes < 64 && p.s.lanes * wide < a.dim) p.s.lanes *= 2;
    if (!p.one) {
        int64_t span = (p.entries + SORT_BLOCKS - 1) / SORT_BLOCKS;
        span = (span + SORT_TILE - 1) / SORT_TILE * SORT_TILE;
        p.span = static_cast<int>(span);
        p.sort_blocks = static_cast<int>((p.entries + span - 1) / span);
        p.at_pairs = take(p.entries * 8 * (p.passes > 2 ? 2 : 1));
        p.at_counts = take(static_cast<int64_t>(p.sort_blocks) * (4 << p.bits));
    }
    return p;
}

template <class T, int W, int TILES>
void launch_few(const EmbedArgs &a, const GradPlan &p, const void *ids, int ids_type, const T *grad, T *out, float *parts, hipStream_t stream) {
    const dim3 grid(p.blocks, (a.dim + 16 * W - 1) / (16 * W));
    if (a.fields == 1)
        hipLaunchKernelGGL((embed_grad_few_kernel<T, W, TILES, 1>), grid, dim3(THREADS), 0, stream, a, ids, ids_type, grad, out, parts);
    else if (a.fields <= 3)
        hipLaunchKernelGGL((embed_grad_few_kernel<T, W, TILES, 3>), grid, dim3(THREADS), 0, stream, a, ids, ids_type, grad, out, parts);
    else
        hipLaunchKernelGGL((embed_grad_few_kernel<T, W, TILES, MG_MAX_FIELDS>), grid, dim3(THREADS), 0, stream, a, ids, ids_type, grad, out, parts);
}
template <class T, int W>
void launch_few(const EmbedArgs &a, const GradPlan &p, const void *ids, int ids_type, const T *grad, T *out, float *parts, hipStream_t stream) {
    if constexpr (W <= 2)
        if (p.tiles > 2) return launch_few<T, W, 4>(a, p, ids, ids_type, grad, out, parts, stream);
    launch_few<T, W, 2>(a, p, ids, ids_type, grad, out, parts, stream);
}

template <class T>
void launch_grad(const EmbedArgs &a, GradPlan p, const void *ids, int ids_type, const T *grad, T *out, char *ws, hipStream_t stream) {
    if (p.few) {
        float *parts = p.blocks > 1 ? reinterpret_cast<float *>(ws) : nullptr;
        if (p.width == 1)
            launch_few<T, 1>(a, p, ids, ids_type, grad, out, parts, stream);
        else if (p.width == 2)
            launch_few<T, 2>(a, p, ids, ids_type, grad, out, parts, stream);
        else if constexpr (sizeof(T) == 2)
            launch_few<T, 4>(a, p, ids, ids_type, grad, out, parts, stream);
        if (parts) {
            const int64_t elements = static_cast<int64_t>(a.rows) * a.dim;
            hipLaunchKernelGGL((embed_join_kernel<T>), dim3((elements + JOIN_COLS - 1) / JOIN_COLS), dim3(JOIN_COLS * JOIN_SHARES), 0, stream, parts, p.blocks,
                               elements, a.scale, out);
        }
        return;
    }
    uint32_t *rows = reinterpret_cast<uint32_t *>(ws + p.at_rows), *tokens = reinterpret_cast<uint32_t *>(ws + p.at_tokens);
    char *bytes = reinterpret_cast<char *>(out);
    const int64_t out_bytes = static_cast<int64_t>(a.rows) * a.dim * sizeof(T);
    if (p.one) {
        const int64_t fill = (out_bytes + SORT_THREADS * 64 - 1) / (SORT_THREADS * 64);  // four stores a thread, or a block to each compute unit
        hipLaunchKernelGGL(embed_sort_kernel, dim3(1 + static_cast<unsigned>(fill < 255 ? fill : 255)), dim3(SORT_THREADS), 0, stream, a, ids, ids_type,
                           static_cast<int>(p.entries), p.passes, p.bits, rows, tokens, bytes, out_bytes);
    } else {
        uint2 *pairs = reinterpret_cast<uint2 *>(ws + p.at_pairs);
        uint32_t *counts = reinterpret_cast<uint32_t *>(ws + p.at_counts);
        const uint2 *from = nullptr;
        for (int pass = 0; pass < p.passes; ++pass) {
            uint2 *to = pass + 1 < p.passes ? pairs + (pass & 1) * p.entries : nullptr;
            const int64_t fill = pass ? 0 : (out_bytes + THREADS * 64 - 1) / (THREADS * 64);
            hipLaunchKernelGGL(embed_count_kernel, dim3(p.sort_blocks + static_cast<unsigned>(fill < 2048 ? fill : 2048)), dim3(THREADS), 0, stream, a, ids, ids_type,
                               from, p.entries, p.span, pass * p.bits, p.bits, p.sort_blocks, counts, bytes, out_bytes);
            hipLaunchKernelGGL(embed_scan_kernel, dim3(1), dim3(SORT_THREADS), 0, stream, counts, p.sort_blocks << p.bits);
            hipLaunchKernelGGL(embed_place_kernel, dim3(p.sort_blocks), dim3(THREADS), 0, stream, a, ids, ids_type, from, p.entries, p.span, pass * p.bits, p.bits,
                               counts, to, rows, tokens);
            from = to;
        }
    }
    p.s.rows = rows;
    p.s.tokens = tokens;
    p.s.head = reinterpret_cast<float *>(ws + p.at_head);
    p.s.tail = reinterpret_cast<float *>(ws + p.at_tail);
    if (p.s.chunks == 0) return;
    const int groups = THREADS / p.s.lanes;
    const dim3 grid((p.s.chunks + groups - 1) / groups, (a.dim + p.s.lanes * WIDE<T> - 1) / (p.s.lanes * WIDE<T>));
    hipLaunchKernelGGL((embed_runs_kernel<T>), grid, dim3(THREADS), 0, stream, a, p.s, grad, out);
    if (p.s.chunks > 1) hipLaunchKernelGGL((embed_span_kernel<T>), dim3(p.s.chunks, (a.dim + 63) / 64), dim3(THREADS), 0, stream, a, p.s, out);
}

// f(the smallest of 8, 16, SHORT that holds k tokens), as a type with a constant `value`
template <int K>
struct Size {
    static constexpr int value = K;
};
template <class F>
void with_size(int k, F f) {
    if (k <= 8)
        f(Size<8>{});
    else if (k <= 16)
        f(Size<16>{});
    else
        f(Size<SHORT>{});
}

// f(threads to a row, vectors that each holds), for up to HELD_MOST vectors: the fewest threads that hold the row with one each, a
// wave up to four each, then blocks of 256 and of 512 up to eight
template <int LANES, int HELD>
struct Shape {
    static constexpr int lanes = LANES, held = HELD;
};
template <class F>
void with_shape(int64_t vecs, F f) {
    if (vecs <= 8)
        f(Shape<8, 1>{});
    else if (vecs <= 16)
        f(Shape<16, 1>{});
    else if (vecs <= 32)
        f(Shape<32, 1>{});
    else if (vecs <= 64)
        f(Shape<64, 1>{});
    else if (vecs <= 128)
        f(Shape<64, 2>{});
    else if (vecs <= 256)
        f(Shape<64, 4>{});
    else if (vecs <= 512)
        f(Shape<256, 2>{});
    else if (vecs <= 1024)
        f(Shape<256, 4>{});
    else if (vecs <= 2048)
        f(Shape<256, 8>{});
    else
        f(Shape<512, 8>{});
}

// pieces of a row that no block holds, 0 where one does
int64_t pieces_of(const MgLogits &l) {
    const int64_t wide = l.dtype == MG_F32 ? WIDE<float> : WIDE<bf16>, piece = PIECE_LANES * PIECE_HELD * wide;
    return l.k > HELD_MOST * wide ? (l.k + piece - 1) / piece : 0;
}

int adjust_args(const char *who, const MgAdjust *a) {
    if (!a) return refuse(MG_EINVAL, "%s: null argument", who);
    if (a->n < 0 || a->n > MOST_ROWS) return refuse(MG_EINVAL, "%s: n %lld not supported (0..2^31 - 1)", who, static_cast<long long>(a->n));
    if (a->k < 1 || a->k > MOST_TOKENS) return refuse(MG_EINVAL, "%s: k %d not supported (1..2^24)", who, a->k);
    if (!dtype_ok(a->dtype)) return refuse(MG_EINVAL, "%s: unknown element type %d", who, a->dtype);
    if (a->history_dev && (a->t < 0 || a->t > MOST_TOKENS || !int_ok(a->history_type)))
        return refuse(MG_EINVAL, "%s: history of %d entries of type %d not supported", who, a->t, a->history_type);
    if (a->mask_kind < MG_MASK_NONE || a->mask_kind > MG_MASK_BITS || (a->mask_kind != MG_MASK_NONE && !a->mask_dev))
        return refuse(MG_EINVAL, "%s: unknown kind of mask %d, or no mask", who, a->mask_kind);
    if (a->logits_stride < 0 || a->out_stride < 0 || a->grad_stride < 0 || a->history_stride < 0 || a->bias_stride < 0 || a->mask_stride < 0)
        return refuse(MG_EINVAL, "%s: negative stride", who);
    if (a->out_stride < a->k && a->n > 1) return refuse(MG_EINVAL, "%s: rows of the output overlap", who);
    if (!a->repetition_dev && !(a->repetition > 0.f && a->repetition < __builtin_inff()))
        return refuse(MG_EINVAL, "%s: repetition must be positive and finite", who);
    return MG_OK;
}

template <bool GRAD>
void launch_adjust(const MgAdjust &a, const void *logits, const void *grad, void *out, hipStream_t stream) {
    with_types(a.dtype, a.history_dev ? a.history_type : MG_U8, [&](auto t, auto h) {
        using T = decltype(t);
        using H = decltype(h);
        const T *x = static_cast<const T *>(logits), *g = static_cast<const T *>(grad);
        T *y = static_cast<T *>(out);
        if (a.k <= SHORT) {
            with_size(a.k, [&](auto size) {
                constexpr int K = decltype(size)::value, ROWS = K <= 16 ? THREADS : 64;
                hipLaunchKernelGGL((adjust_short_kernel<T, H, GRAD, K>), dim3((a.n + ROWS - 1) / ROWS), dim3(ROWS), 0, stream, a, x, g, y);
            });
        } else {
            constexpr int TAKES = STRETCH * WIDE<T>;
            int lanes = 8;  // the fewest that take a row at once
            while (lanes < THREADS && lanes * TAKES < a.k) lanes *= 2;
            const int64_t per_block = THREADS / lanes, pieces = (a.k + lanes * TAKES - 1) / (lanes * TAKES);
            const dim3 grid(blocks_for((a.n + per_block - 1) / per_block), pieces);
            if (a.history_dev && a.t > 0xFFFF)
                hipLaunchKernelGGL((adjust_kernel<T, H, GRAD, uint32_t>), grid, dim3(THREADS), 0, stream, a, lanes, x, g, y);
            else
                hipLaunchKernelGGL((adjust_kernel<T, H, GRAD, uint16_t>), grid, dim3(THREADS), 0, stream, a, lanes, x, g, y);
        }
    });
}

int logits_args(const char *who, const MgLogits *l) {
    if (!l) return refuse(MG_EINVAL, "%s: null argument", who);
    if (l->n < 0 || l->n > MOST_ROWS) return refuse(MG_EINVAL, "%s: n %lld not supported (0..2^31 - 1)", who, static_cast<long long>(l->n));
    if (l->k < 1 || l->k > MOST_TOKENS) return refuse(MG_EINVAL, "%s: k %d not supported (1..2^24)", who, l->k);
    if (!dtype_ok(l->dtype)) return refuse(MG_EINVAL, "%s: unknown element type %d", who, l->dtype);
    if (!int_ok(l->tokens_type) || (l->tokens_type == MG_U8 && l->k > 255))
        return refuse(MG_EINVAL, "%s: tokens of type %d not supported for k = %d", who, l->tokens_type, l->k);
    if (l->stride < 0) return refuse(MG_EINVAL, "%s: negative stride", who);
    if (!l->temperature_dev && !(l->temperature >= LEAST_TEMPERATURE && l->temperature < __builtin_inff()))
        return refuse(MG_EINVAL, "%s: temperature must be at least 2^-126 and finite", who);
    return MG_OK;
}

}  // namespace

extern "C" {

int mg_embed(const MgEmbed *e, const void *ids_dev, const void *table_dev, void *out_dev, void *stream) {
    EmbedArgs a;
    const int rc = embed_args("mg_embed", e, &a);
    if (rc != MG_OK || a.n == 0) return rc;
    if (!ids_dev || !table_dev || !out_dev) return refuse(MG_EINVAL, "mg_embed: null argument");
    with_types(e->dtype, e->ids_type, [&](auto t, auto i) {
        using T = decltype(t);
        using I = decltype(i);
        I *ids_copy = static_cast<I *>(e->ids_copy_dev);
        const int vecs = (a.dim + WIDE<T> - 1) / WIDE<T>, per_block = THREADS / (vecs < THREADS ? vecs : THREADS);
        const int64_t held = static_cast<int64_t>(a.rows + 1) * vecs * 16;
        // What a block prepares has to be little beside the tokens that it then writes.  Combinations: sixteen tokens for each, at a
        // block to a compute unit.  Microseconds by embed_combined_kernel and by embed_table_kernel where cells reach that, 2760000 of
        // them, without the ids' copy and with it: x 32 bfloat16 44.6 and 48.3, 40.7 and 50.1, x 16 26.6 and 28.4, 23.6 and 32.6, x 16
        // float32 46.8 and 41.2, 44.2 and 43.4, x 8 26.9 and 25.4, 23.2 and 29.5; half as many x 16 float32 27.9 and 21.2, 27.2 and 22.8.
        // A table: a full share of tokens for every compute unit (131072 cells x 32 bfloat16, where they begin: 6.6 us with it, 5.9 by
        // embed_kernel, x 64 float32 13.2 and 12.4; twice as many 8.7 and 9.5, 16.1 and 22.1).
        int64_t combined = 1;
        for (int f = 0; f < a.fields; ++f) combined = combined * (a.sizes[f] + 1) <= (1 << 15) ? combined * (a.sizes[f] + 1) : 1 << 15;
        const int64_t combined_bytes = (combined + a.rows + 1) * vecs * 16 + FAR * 2;
        if (a.dim % WIDE<T> == 0 && combined_bytes <= COMBINED_BYTES && a.n >= 16 * combined * UNITS) {
            hipLaunchKernelGGL((embed_combined_kernel<T, I>), dim3(blocks_for((a.n + FAR - 1) / FAR, COMBINED_BLOCKS)), dim3(COMBINED_THREADS),
                               combined_bytes, static_cast<hipStream_t>(stream), a, static_cast<int>(combined),
                               static_cast<const I *>(ids_dev), static_cast<const T *>(table_dev), static_cast<T *>(out_dev), ids_copy);
            return;
        }
        if (held <= TABLE_BYTES && a.n >= UNITS * FAR) {
            // as many tokens to a block as give every compute unit the same number of blocks
            const int64_t rounds = (a.n + UNITS * FAR - 1) / (UNITS * FAR), share = (a.n + UNITS * rounds - 1) / (UNITS * rounds);
            const int far = static_cast<int>(share + per_block - 1 < FAR ? (share + per_block - 1) / per_block * per_block : FAR);
            hipLaunchKernelGGL((embed_table_kernel<T, I>), dim3(blocks_for((a.n + far - 1) / far, TABLE_BLOCKS)), dim3(THREADS), held + a.fields * FAR * 2,
                               static_cast<hipStream_t>(stream), a, far, static_cast<const I *>(ids_dev), static_cast<const T *>(table_dev), static_cast<T *>(out_dev), ids_copy);
            return;
        }
        hipLaunchKernelGGL((embed_kernel<T, I>), dim3(blocks_for((a.n + per_block - 1) / per_block)), dim3(THREADS), 0,
                           static_cast<hipStream_t>(stream), a, static_cast<const I *>(ids_dev), static_cast<const T *>(table_dev),
                           static_cast<T *>(out_dev), ids_copy);
    });
    return launched("mg_embed");
}

int64_t mg_embed_grad_workspace(const MgEmbed *e) {
    EmbedArgs a;
    const int rc = embed_args("mg_embed_grad_workspace", e, &a);
    return rc != MG_OK ? rc : plan_grad(a, e->dtype == MG_F32 ? WIDE<float> : WIDE<bf16>).bytes;
}

int mg_embed_grad(const MgEmbed *e, const void *ids_dev, const void *grad_dev, void *table_grad_dev, void *workspace_dev,
                  int64_t workspace_bytes, void *stream) {
    EmbedArgs a;
    const int rc = embed_args("mg_embed_grad", e, &a);
    if (rc != MG_OK) return rc;
    if (((!ids_dev || !grad_dev) && a.n > 0) || !table_grad_dev) return refuse(MG_EINVAL, "mg_embed_grad: null argument");
    const GradPlan p = plan_grad(a, e->dtype == MG_F32 ? WIDE<float> : WIDE<bf16>);
    if (!workspace_ok("mg_embed_grad", workspace_dev, workspace_bytes, p.bytes)) return MG_EINVAL;
    with_types(e->dtype, MG_U8, [&](auto t, auto) {
        using T = decltype(t);
        launch_grad<T>(a, p, ids_dev, e->ids_type, static_cast<const T *>(grad_dev), static_cast<T *>(table_grad_dev), static_cast<char *>(workspace_dev),
                       static_cast<hipStream_t>(stream));
    });
    return launched("mg_embed_grad");
}

int mg_adjust_logits(const MgAdjust *a, const void *logits_dev, void *out_dev, void *stream) {
    const int rc = adjust_args("mg_adjust_logits", a);
    if (rc != MG_OK || a->n == 0) return rc;
    if (!logits_dev || !out_dev) return refuse(MG_EINVAL, "mg_adjust_logits: null argument");
    launch_adjust<false>(*a, logits_dev, nullptr, out_dev, static_cast<hipStream_t>(stream));
    return launched("mg_adjust_logits");
}

int mg_adjust_logits_grad(const MgAdjust *a, const void *logits_dev, const void *grad_dev, void *out_dev, void *stream) {
    const int rc = adjust_args("mg_adjust_logits_grad", a);
    if (rc != MG_OK || a->n == 0) return rc;
    if (!logits_dev || !grad_dev || !out_dev) return refuse(MG_EINVAL, "mg_adjust_logits_grad: null argument");
    launch_adjust<true>(*a, logits_dev, grad_dev, out_dev, static_cast<hipStream_t>(stream));
    return launched("mg_adjust_logits_grad");
}

int64_t mg_draw_workspace(const MgLogits *l) {
    const int rc = logits_args("mg_draw_workspace", l);
    return rc != MG_OK ? rc : l->n * pieces_of(*l) * static_cast<int64_t>(sizeof(DrawPiece));
}

int mg_draw(const MgLogits *l, const void *logits_dev, const void *uniforms_dev, int32_t uniforms_type, void *tokens_dev,
            float *logprob_dev, void *workspace_dev, int64_t workspace_bytes, void *stream) {
    const int rc = logits_args("mg_draw", l);
    if (rc != MG_OK || l->n == 0) return rc;
    if (!logits_dev || !tokens_dev) return refuse(MG_EINVAL, "mg_draw: null argument");
    if (uniforms_dev && uniforms_type != MG_F32 && uniforms_type != MG_F64) return refuse(MG_EINVAL, "mg_draw: unknown type %d of the uniform numbers", uniforms_type);
    const int64_t pieces = pieces_of(*l);
    if (!workspace_ok("mg_draw", workspace_dev, workspace_bytes, l->n * pieces * static_cast<int64_t>(sizeof(DrawPiece)))) return MG_EINVAL;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    with_types(l->dtype, MG_U8, [&](auto t, auto) {
        using T = decltype(t);
        const T *x = static_cast<const T *>(logits_dev);
        if (l->k <= SHORT) {
            with_size(l->k, [&](auto size) {
                hipLaunchKernelGGL((draw_short_kernel<T, decltype(size)::value>), dim3((l->n + THREADS - 1) / THREADS), dim3(THREADS), 0, s, *l, x, uniforms_dev,
                                   uniforms_type, tokens_dev, logprob_dev);
            });
        } else if (pieces == 0) {
            with_shape((l->k + WIDE<T> - 1) / WIDE<T>, [&](auto shape) {
                using S = decltype(shape);
                constexpr int ROWS = BLOCK<S::lanes> / S::lanes;
                hipLaunchKernelGGL((draw_kernel<T, S::lanes, S::held>), dim3(blocks_for((l->n + ROWS - 1) / ROWS)), dim3(BLOCK<S::lanes>), 0, s, *l, x, uniforms_dev,
                                   uniforms_type, tokens_dev, logprob_dev);
            });
        } else {
            DrawPiece *of = static_cast<DrawPiece *>(workspace_dev);
            hipLaunchKernelGGL((draw_pieces_kernel<T>), dim3(static_cast<unsigned>(pieces), blocks_for(l->n, 65535)), dim3(PIECE_LANES), 0, s, *l, x, of);
            hipLaunchKernelGGL((draw_join_kernel<T>), dim3(blocks_for(l->n)), dim3(PIECE_LANES), 0, s, *l, x, uniforms_dev, uniforms_type, of,
                               static_cast<int>(pieces), tokens_dev, logprob_dev);
        }
    });
    return launched("mg_draw");
}

int64_t mg_token_logprobs_workspace(const MgLogits *l) {
    const int rc = logits_args("mg_token_logprobs_workspace", l);
    return rc != MG_OK ? rc : l->n * pieces_of(*l) * static_cast<int64_t>(sizeof(float4));
}

int mg_token_logprobs(const MgLogits *l, const void *logits_dev, const void *tokens_dev, float *logprob_dev, float *entropy_dev,
                      float *stats_dev, void *workspace_dev, int64_t workspace_bytes, void *stream) {
    const int rc = logits_args("mg_token_logprobs", l);
    if (rc != MG_OK || l->n == 0) return rc;
    if (!logits_dev || (logprob_dev && !tokens_dev)) return refuse(MG_EINVAL, "mg_token_logprobs: null argument");
    if (reinterpret_cast<uintptr_t>(stats_dev) % 16) return refuse(MG_EINVAL, "mg_token_logprobs: stats_dev must be 16-byte aligned");
    const int64_t pieces = pieces_of(*l);
    if (!workspace_ok("mg_token_logprobs", workspace_dev, workspace_bytes, l->n * pieces * static_cast<int64_t>(sizeof(float4)))) return MG_EINVAL;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    with_types(l->dtype, MG_U8, [&](auto t, auto) {
        using T = decltype(t);
        const T *x = static_cast<const T *>(logits_dev);
        if (l->k <= SHORT) {
            with_size(l->k, [&](auto size) {
                hipLaunchKernelGGL((logprob_short_kernel<T, decltype(size)::value>), dim3((l->n + THREADS - 1) / THREADS), dim3(THREADS), 0, s, *l, x, tokens_dev,
                                   logprob_dev, entropy_dev, stats_dev);
            });
        } else if (pieces == 0) {
            with_shape((l->k + WIDE<T> - 1) / WIDE<T>, [&](auto shape) {
                using S = decltype(shape);
                constexpr int ROWS = BLOCK<S::lanes> / S::lanes;
                hipLaunchKernelGGL((logprob_kernel<T, S::lanes, S::held>), dim3(blocks_for((l->n + ROWS - 1) / ROWS)), dim3(BLOCK<S::lanes>), 0, s, *l, x, tokens_dev,
                                   logprob_dev, entropy_dev, stats_dev);
            });
        } else {
            float4 *of = static_cast<float4 *>(workspace_dev);
            hipLaunchKernelGGL((logprob_pieces_kernel<T>), dim3(static_cast<unsigned>(pieces), blocks_for(l->n, 65535)), dim3(PIECE_LANES), 0, s, *l, x, of);
            hipLaunchKernelGGL((logprob_join_kernel<T>), dim3(blocks_for(l->n)), dim3(64), 0, s, *l, x, of, static_cast<int>(pieces), tokens_dev, logprob_dev,
                               entropy_dev, stats_dev);
        }
    });
    return launched("mg_token_logprobs");
}

int mg_token_logprobs_grad(const MgLogits *l, const void *logits_dev, const void *tokens_dev, const float *stats_dev,
                           const float *grad_logprob_dev, int64_t grad_logprob_stride, const float *grad_entropy_dev,
                           int64_t grad_entropy_stride, void *out_dev, void *stream) {
    const int rc = logits_args("mg_token_logprobs_grad", l);
    if (rc != MG_OK || l->n == 0) return rc;
    if (!logits_dev || (!stats_dev && l->k > SHORT) || !out_dev || (grad_logprob_dev && !tokens_dev)) return refuse(MG_EINVAL, "mg_token_logprobs_grad: null argument");
    if (reinterpret_cast<uintptr_t>(stats_dev) % 16) return refuse(MG_EINVAL, "mg_token_logprobs_grad: stats_dev must be 16-byte aligned");
    if (grad_logprob_stride < 0 || grad_entropy_stride < 0) return refuse(MG_EINVAL, "mg_token_logprobs_grad: negative stride");
    with_types(l->dtype, MG_U8, [&](auto t, auto) {
        using T = decltype(t);
        if (l->k <= SHORT)
            return with_size(l->k, [&](auto size) {
                hipLaunchKernelGGL((logprob_grad_short_kernel<T, decltype(size)::value>), dim3((l->n + THREADS - 1) / THREADS), dim3(THREADS), 0,
                                   static_cast<hipStream_t>(stream), *l, static_cast<const T *>(logits_dev), tokens_dev, grad_logprob_dev, grad_logprob_stride,
                                   grad_entropy_dev, grad_entropy_stride, static_cast<T *>(out_dev));
            });
        constexpr int TAKES = 4 * WIDE<T>;
        int lanes = 8;
        while (lanes < THREADS && lanes * TAKES < l->k) lanes *= 2;
        const int64_t per_block = THREADS / lanes, pieces = (l->k + lanes * TAKES - 1) / (lanes * TAKES);
        hipLaunchKernelGGL((logprob_grad_kernel<T>), dim3(blocks_for((l->n + per_block - 1) / per_block), pieces), dim3(THREADS), 0,
                           static_cast<hipStream_t>(stream), *l, lanes, static_cast<const T *>(logits_dev), tokens_dev, stats_dev, grad_logprob_dev,
                           grad_logprob_stride, grad_entropy_dev, grad_entropy_stride, static_cast<T *>(out_dev));
    });
    return launched("mg_token_logprobs_grad");
}

}  // extern "C"
