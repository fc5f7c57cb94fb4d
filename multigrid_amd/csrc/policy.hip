// libmgrid_hip.so - what stands between the simulator and a policy network, for gfx950 (MI355X):
//   embedding of cells and tokens, and its gradient;
//   adjustment of logits (penalties, bias, mask), and its gradient;
//   draw of a token from logits;
//   log-probability and entropy of given tokens, and their gradient.
// The formulas stand in include/mgrid.h beside each entry point.
//
// Sums, maxima and probabilities are held in 32 bits (64 in the draw, where a token's borders decide); a value is
// rounded to its type once, when it is stored.

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "mgrid.h"
#include "mgrid_error.h"

namespace {

using bf16 = __bf16;
using f16 = _Float16;

constexpr int THREADS = 256;
constexpr float NEG_INF = -__builtin_inff();

// V elements at any element's alignment: global loads and stores of gfx950 take 16 bytes at any address
template <class T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Vec {
    T v[V];
};

template <class T, int V>
__device__ __forceinline__ void load(const T *p, float (&x)[V]) {
    const Vec<T, V> r = *reinterpret_cast<const Vec<T, V> *>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = static_cast<float>(r.v[i]);
}

template <class T, int V>
__device__ __forceinline__ void store(T *p, const float (&x)[V]) {
    Vec<T, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = static_cast<T>(x[i]);
    *reinterpret_cast<Vec<T, V> *>(p) = r;
}

// elements in 16 bytes
template <class T>
constexpr int WIDE = 16 / static_cast<int>(sizeof(T));

// ---- embedding -----------------------------------------------------------------------------------------------------

struct EmbedArgs {
    int64_t n, ids_stride, field_stride, row_stride;
    int32_t fields, dim, rows;
    float scale;
    int32_t sizes[MG_MAX_FIELDS];
};

// One thread per 16 bytes of output; the threads of a token share its ids.
template <class T, class I>
__global__ __launch_bounds__(THREADS) void embed_kernel(EmbedArgs a, const I *ids, const T *table, T *out) {
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
            const bool whole = d0 + V <= a.dim;
            float acc[V] = {};
            int64_t base = 0;
            for (int f = 0; f < a.fields; ++f) {
                const int64_t id = static_cast<int64_t>(id_at[f * a.field_stride]);
                if (id >= 0 && id < a.sizes[f]) {
                    const T *row = table + (base + id) * a.row_stride + d0;
                    if (whole) {
                        float x[V];
                        load<T, V>(row, x);
#pragma unroll
                        for (int i = 0; i < V; ++i) acc[i] += x[i];
                    } else {
#pragma unroll
                        for (int i = 0; i < V; ++i)
                            if (d0 + i < a.dim) acc[i] += static_cast<float>(row[i]);
                    }
                }
                base += a.sizes[f];
            }
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] *= a.scale;
            if (whole) {
                store<T, V>(to + d0, acc);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (d0 + i < a.dim) to[d0 + i] = static_cast<T>(acc[i]);
            }
        }
    }
}

// A block owns ROW_TILE rows and SLAB columns of the gradient, looks through all ids for those rows, in order, and adds up the
// tokens it finds in 32 bits; one thread per column and group of rows, so that no two threads share a sum.
constexpr int ROW_TILE = 16, SLAB = 256, SCAN = 1024;

template <class T, class I>
__global__ __launch_bounds__(THREADS) void embed_grad_scan_kernel(EmbedArgs a, const I *ids, const T *grad, T *out) {
    __shared__ float acc[ROW_TILE][SLAB];
    __shared__ uint32_t found[4][SCAN / 4];  // token of the segment in the low 16 bits, row of the tile above
    __shared__ int count[4];
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const int d0 = blockIdx.y * SLAB, width = min(SLAB, a.dim - d0);
    const int groups = THREADS / width, group = threadIdx.x / width, col = threadIdx.x - group * width;
    const int tiles = (a.rows + ROW_TILE - 1) / ROW_TILE;
    const int64_t entries = a.n * a.fields;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int row0 = tile * ROW_TILE;
        for (int i = threadIdx.x; i < ROW_TILE * SLAB; i += THREADS) (&acc[0][0])[i] = 0.f;
        for (int64_t e0 = 0; e0 < entries; e0 += SCAN) {
            __syncthreads();  // the last round's list is read, the sums are cleared
            int n_found = 0;
            for (int j = 0; j < SCAN / 4; j += 64) {
                const int64_t e = e0 + wave * (SCAN / 4) + j + lane;
                int row = -1;
                if (e < entries) {
                    const int64_t n = a.fields == 1 ? e : e / a.fields;
                    const int f = static_cast<int>(e - n * a.fields);
                    const int64_t id = static_cast<int64_t>(ids[n * a.ids_stride + f * a.field_stride]);
                    int base = 0;
                    for (int k = 0; k < f; ++k) base += a.sizes[k];
                    if (id >= 0 && id < a.sizes[f]) row = base + static_cast<int>(id) - row0;
                }
                const bool hit = row >= 0 && row < ROW_TILE;
                const uint64_t hits = __ballot(hit);
                if (hit) found[wave][n_found + __popcll(hits & ((1ull << lane) - 1))] = static_cast<uint32_t>(wave * (SCAN / 4) + j + lane) | static_cast<uint32_t>(row) << 16;
                n_found += __popcll(hits);
            }
            if (lane == 0) count[wave] = n_found;
            __syncthreads();
            if (group < groups)
                for (int w = 0; w < 4; ++w)
                    for (int i = 0; i < count[w]; ++i) {
                        const uint32_t what = found[w][i];
                        const int row = what >> 16;
                        if (row % groups != group) continue;
                        const int64_t e = e0 + (what & 0xFFFF);
                        const int64_t n = a.fields == 1 ? e : e / a.fields;
                        acc[row][col] += static_cast<float>(grad[n * a.row_stride + d0 + col]);
                    }
        }
        __syncthreads();
        if (group < groups)
            for (int r = group; r < ROW_TILE && row0 + r < a.rows; r += groups)
                out[static_cast<int64_t>(row0 + r) * a.dim + d0 + col] = static_cast<T>(acc[r][col] * a.scale);
        __syncthreads();
    }
}

// ---- adjustment of logits ------------------------------------------------------------------------------------------

// How often each token of a chunk stands in a row's history is counted in LDS (a chunk is what LDS holds counters for), then
// the chunk streams through once.
constexpr int CHUNK = 8192;

template <class H>
__device__ __forceinline__ void count_history(const MgAdjust &a, int64_t row, int first, int width, uint32_t *counts, int tid, int threads) {
    int len = a.lengths_dev ? min(max(a.lengths_dev[row], 0), a.t) : a.t;
    const H *h = static_cast<const H *>(a.history_dev) + row * a.history_stride;
    for (int i = tid; i < len; i += threads) {
        const int64_t j = static_cast<int64_t>(h[i]) - first;
        if (j >= 0 && j < width) atomicAdd(&counts[j], 1u);
    }
}

__device__ __forceinline__ bool allowed(const MgAdjust &a, int64_t row, int j) {
    if (a.mask_kind == MG_MASK_BYTES) return static_cast<const uint8_t *>(a.mask_dev)[row * a.mask_stride + j] != 0;
    if (a.mask_kind == MG_MASK_BITS) return (static_cast<const uint32_t *>(a.mask_dev)[row * a.mask_stride + (j >> 5)] >> (j & 31)) & 1;
    return true;
}

template <class T, class H, bool GRAD>
__global__ __launch_bounds__(THREADS) void adjust_kernel(MgAdjust a, const T *logits, const T *grad, T *out) {
#pragma clang fp contract(off)
    __shared__ uint32_t counts[CHUNK];
    const int chunks = (a.k + CHUNK - 1) / CHUNK;
    const int64_t items = a.n * chunks;
    const bool history = a.history_dev != nullptr && a.t > 0;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t row = item / chunks;
        const int first = static_cast<int>(item - row * chunks) * CHUNK, width = min(CHUNK, a.k - first);
        if (history) {
            __syncthreads();
            for (int i = threadIdx.x; i < width; i += THREADS) counts[i] = 0;
            __syncthreads();
            count_history<H>(a, row, first, width, counts, threadIdx.x, THREADS);
            __syncthreads();
        }
        const float rep = a.repetition_dev ? a.repetition_dev[row] : a.repetition;
        const float presence = a.presence_dev ? a.presence_dev[row] : a.presence;
        const float frequency = a.frequency_dev ? a.frequency_dev[row] : a.frequency;
        for (int i = threadIdx.x; i < width; i += THREADS) {
            const int j = first + i;
            const uint32_t c = history ? counts[i] : 0;
            float x = static_cast<float>(logits[row * a.logits_stride + j]);
            if (GRAD) {
                float g = static_cast<float>(grad[row * a.grad_stride + j]);
                if (c > 0) g = x > 0.f ? g / rep : g * rep;
                out[row * a.out_stride + j] = static_cast<T>(allowed(a, row, j) ? g : 0.f);
            } else {
                if (c > 0) x = (x > 0.f ? x / rep : x * rep) - presence;
                x = x - frequency * static_cast<float>(c);
                if (a.bias_dev) x = x + a.bias_dev[row * a.bias_stride + j];
                out[row * a.out_stride + j] = static_cast<T>(allowed(a, row, j) ? x : NEG_INF);
            }
        }
    }
}

// ---- draw ----------------------------------------------------------------------------------------------------------

template <class T>
__device__ __forceinline__ T shuffle_down(T v, int by) { return __shfl_down(v, by, 64); }

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

// One block per row: the maximum, then every thread's share of the total (a run of adjacent tokens), then the thread whose run
// holds the border walks it.
template <class T>
__global__ __launch_bounds__(THREADS) void draw_kernel(MgLogits l, const T *logits, const void *uniforms, int uniforms_type,
                                                       void *tokens, float *logprob) {
    __shared__ float best_s[THREADS];
    __shared__ int arg_s[THREADS];
    __shared__ double sum_s[THREADS];
    const int tid = threadIdx.x;
    const int run = (l.k + THREADS - 1) / THREADS;
    for (int64_t row = blockIdx.x; row < l.n; row += gridDim.x) {
        const T *x = logits + row * l.stride;
        const double inv_t = 1.0 / static_cast<double>(l.temperature_dev ? l.temperature_dev[row] : l.temperature);
        const int lo = min(tid * run, l.k), hi = min(lo + run, l.k);
        float best = NEG_INF;
        int arg = l.k;
        for (int j = lo; j < hi; ++j) {
            const float v = static_cast<float>(x[j]);
            if (v > best) {
                best = v;
                arg = j;
            }
        }
        __syncthreads();
        best_s[tid] = best;
        arg_s[tid] = arg;
        __syncthreads();
        for (int half = THREADS / 2; half > 0; half /= 2) {  // runs are in order: the left one wins a tie
            if (tid < half && (best_s[tid + half] > best_s[tid] || (best_s[tid + half] == best_s[tid] && arg_s[tid + half] < arg_s[tid]))) {
                best_s[tid] = best_s[tid + half];
                arg_s[tid] = arg_s[tid + half];
            }
            __syncthreads();
        }
        best = best_s[0];
        arg = arg_s[0];
        double sum = 0.0;
        if (best != NEG_INF)
            for (int j = lo; j < hi; ++j) sum += exp((static_cast<double>(static_cast<float>(x[j])) - best) * inv_t);
        else  // nothing to draw from, unless a NaN is among them
            for (int j = lo; j < hi; ++j)
                if (static_cast<float>(x[j]) != NEG_INF) sum = __builtin_nan("");
        sum_s[tid] = sum;
        __syncthreads();
        if (tid == 0) {
            double total = 0.0;
            for (int i = 0; i < THREADS; ++i) total += sum_s[i];
            int64_t token = -1;
            double lp = total == 0.0 ? -__builtin_inf() : __builtin_nan("");
            if (total > 0.0) {
                token = arg;
                if (uniforms) {
                    const double u = uniforms_type == MG_F64 ? static_cast<const double *>(uniforms)[row] : static_cast<double>(static_cast<const float *>(uniforms)[row]);
                    const double border = u * total;
                    double upto = 0.0;
                    int last = arg;
                    bool done = false;
                    for (int i = 0; i < THREADS && !done; ++i) {
                        if (!(upto + sum_s[i] > border) && i * run + run < l.k) {
                            upto += sum_s[i];
                            continue;
                        }
                        for (int j = i * run; j < min(i * run + run, l.k); ++j) {
                            const double p = exp((static_cast<double>(static_cast<float>(x[j])) - best) * inv_t);
                            upto += p;
                            if (p > 0.0) last = j;
                            if (upto > border) {
                                done = true;
                                break;
                            }
                        }
                    }
                    token = last;
                }
                lp = (static_cast<double>(static_cast<float>(x[token])) - best) * inv_t - log(total);
            }
            put_token(tokens, l.tokens_type, row, token);
            if (logprob) logprob[row] = static_cast<float>(lp);
        }
    }
}

// ---- log-probabilities and entropies -------------------------------------------------------------------------------

// A part of a row: its maximum m, the sum of e = exp((x - m) / T) over its tokens LESS the one of the maximum itself (r), and
// the sum of e * (x - m) / T (t <= 0).  The maximum's own 1 is left out because what is wanted is log(1 + r): for a row whose
// maximum holds nearly everything, r is small and 1 + r would lose it.  Nothing seen yet: m = -inf, r = -1.
struct Soft {
    float m, r, t;
};

__device__ __forceinline__ void take(Soft &s, float x, float inv_t) {
    if (x > s.m) {
        if (s.m == NEG_INF) {
            s.r += 1.f;  // 0, or NaN if a NaN came before
        } else {
            const float d = (s.m - x) * inv_t, e = expf(d);
            s.t = e > 0.f ? e * (s.t + (1.f + s.r) * d) : 0.f;
            s.r = (1.f + s.r) * e;
        }
        s.m = x;
    } else if (x != NEG_INF) {
        const float z = (x - s.m) * inv_t, e = expf(z);
        s.r += e;
        if (e > 0.f) s.t += e * z;
    }
}

__device__ __forceinline__ Soft merge(Soft a, Soft b, float inv_t) {
    if (b.m > a.m) {
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
        o.m = shuffle_down(s.m, by);
        o.r = shuffle_down(s.r, by);
        o.t = shuffle_down(s.t, by);
        s = merge(s, o, inv_t);
    }
    return s;
}

// What a finished row gives.
template <class T>
__device__ __forceinline__ void row_result(const MgLogits &l, const T *x, int64_t row, const Soft &s, float inv_t, const void *tokens,
                                           float *logprob, float *entropy, float *stats) {
    const bool empty = s.m == NEG_INF && s.r == -1.f;
    const float log_total = s.m == -NEG_INF ? __builtin_nanf("") : log1pf(s.r), h = empty ? 0.f : log_total - s.t / (1.f + s.r);
    if (logprob) {
        const int64_t token = get_token(tokens, l.tokens_type, row);
        float lp = 0.f;
        if (token >= 0 && token < l.k) lp = empty ? NEG_INF : (static_cast<float>(x[token]) - s.m) * inv_t - log_total;
        logprob[row] = lp;
    }
    if (entropy) entropy[row] = h;
    if (stats) reinterpret_cast<float4 *>(stats)[row] = make_float4(empty ? NEG_INF : s.m, log_total, h, 0.f);
}

template <class T>
__global__ __launch_bounds__(THREADS) void logprob_kernel(MgLogits l, const T *logits, const void *tokens, float *logprob,
                                                          float *entropy, float *stats) {
    __shared__ Soft part[THREADS / 64];
    for (int64_t row = blockIdx.x; row < l.n; row += gridDim.x) {
        const T *x = logits + row * l.stride;
        const float inv_t = 1.f / (l.temperature_dev ? l.temperature_dev[row] : l.temperature);
        Soft s{NEG_INF, -1.f, 0.f};
        for (int j = threadIdx.x; j < l.k; j += THREADS) take(s, static_cast<float>(x[j]), inv_t);
        s = merge_wave(s, inv_t);
        __syncthreads();
        if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = s;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < THREADS / 64; ++w) s = merge(s, part[w], inv_t);
            row_result(l, x, row, s, inv_t, tokens, logprob, entropy, stats);
        }
    }
}

// g, h: the row's gradients divided by its temperature.  One product with p, the smallest factor, and that last: a p below
// 2^-126 has few bits left, which a second rounding would halve.
__device__ __forceinline__ float logprob_slope(float x, bool is_token, float4 st, float inv_t, float g, float h) {
    if (x == NEG_INF) return 0.f;
    const float lp = (x - st.x) * inv_t - st.y, p = expf(lp), hs = h * (lp + st.z);
    return is_token ? -g * expm1f(lp) - p * hs : -p * (g + hs);
}

template <class T>
__global__ __launch_bounds__(THREADS) void logprob_grad_kernel(MgLogits l, const T *logits, const void *tokens, const float *stats,
                                                               const float *grad_lp, int64_t lp_stride, const float *grad_h,
                                                               int64_t h_stride, T *out) {
    for (int64_t row = blockIdx.x; row < l.n; row += gridDim.x) {
        const T *x = logits + row * l.stride;
        const float inv_t = 1.f / (l.temperature_dev ? l.temperature_dev[row] : l.temperature);
        const float4 st = reinterpret_cast<const float4 *>(stats)[row];
        const int64_t token = grad_lp ? get_token(tokens, l.tokens_type, row) : -1;
        const float g = token >= 0 && token < l.k ? grad_lp[row * lp_stride] * inv_t : 0.f;
        const float h = grad_h ? grad_h[row * h_stride] * inv_t : 0.f;
        for (int j = threadIdx.x; j < l.k; j += THREADS)
            out[row * l.k + j] = static_cast<T>(logprob_slope(static_cast<float>(x[j]), j == token, st, inv_t, g, h));
    }
}

// ---- host side -----------------------------------------------------------------------------------------------------

using mgrid::refuse;

int launched(const char *who) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MG_OK : refuse(MG_EHIP, "%s: %s", who, hipGetErrorString(e));
}

unsigned blocks_for(int64_t items, int64_t most = 1 << 20) { return static_cast<unsigned>(items < most ? items : most); }

constexpr int64_t MOST_ROWS = (1ll << 31) - 1;
constexpr int32_t MOST_TOKENS = 1 << 24;

bool dtype_ok(int32_t t) { return t == MG_F32 || t == MG_BF16 || t == MG_F16; }
bool int_ok(int32_t t) { return t == MG_U8 || t == MG_I32 || t == MG_I64; }

int embed_args(const char *who, const MgEmbed *e, EmbedArgs *a) {
    if (!e) return refuse(MG_EINVAL, "%s: null argument", who);
    if (e->n < 0 || e->n > MOST_ROWS) return refuse(MG_EINVAL, "%s: n %lld not supported (0..2^31 - 1)", who, static_cast<long long>(e->n));
    if (e->fields < 1 || e->fields > MG_MAX_FIELDS) return refuse(MG_EINVAL, "%s: %d fields not supported (1..%d)", who, e->fields, MG_MAX_FIELDS);
    if (e->dim < 1 || e->dim > MOST_TOKENS) return refuse(MG_EINVAL, "%s: dim %d not supported (1..2^24)", who, e->dim);
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

int logits_args(const char *who, const MgLogits *l) {
    if (!l) return refuse(MG_EINVAL, "%s: null argument", who);
    if (l->n < 0 || l->n > MOST_ROWS) return refuse(MG_EINVAL, "%s: n %lld not supported (0..2^31 - 1)", who, static_cast<long long>(l->n));
    if (l->k < 1 || l->k > MOST_TOKENS) return refuse(MG_EINVAL, "%s: k %d not supported (1..2^24)", who, l->k);
    if (!dtype_ok(l->dtype)) return refuse(MG_EINVAL, "%s: unknown element type %d", who, l->dtype);
    if (!int_ok(l->tokens_type) || (l->tokens_type == MG_U8 && l->k > 255))
        return refuse(MG_EINVAL, "%s: tokens of type %d not supported for k = %d", who, l->tokens_type, l->k);
    if (l->stride < 0) return refuse(MG_EINVAL, "%s: negative stride", who);
    if (!l->temperature_dev && !(l->temperature > 0.f && l->temperature < __builtin_inff()))
        return refuse(MG_EINVAL, "%s: temperature must be positive and finite", who);
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
        const int vecs = (a.dim + WIDE<T> - 1) / WIDE<T>, per_block = THREADS / (vecs < THREADS ? vecs : THREADS);
        hipLaunchKernelGGL((embed_kernel<T, I>), dim3(blocks_for((a.n + per_block - 1) / per_block)), dim3(THREADS), 0,
                           static_cast<hipStream_t>(stream), a, static_cast<const I *>(ids_dev), static_cast<const T *>(table_dev),
                           static_cast<T *>(out_dev));
    });
    return launched("mg_embed");
}

int64_t mg_embed_grad_workspace(const MgEmbed *e) {
    EmbedArgs a;
    return embed_args("mg_embed_grad_workspace", e, &a);
}

int mg_embed_grad(const MgEmbed *e, const void *ids_dev, const void *grad_dev, void *table_grad_dev, void *workspace_dev,
                  int64_t workspace_bytes, void *stream) {
    EmbedArgs a;
    const int rc = embed_args("mg_embed_grad", e, &a);
    if (rc != MG_OK) return rc;
    if (((!ids_dev || !grad_dev) && a.n > 0) || !table_grad_dev) return refuse(MG_EINVAL, "mg_embed_grad: null argument");
    (void)workspace_dev;
    (void)workspace_bytes;
    with_types(e->dtype, e->ids_type, [&](auto t, auto i) {
        using T = decltype(t);
        using I = decltype(i);
        const int64_t tiles = (static_cast<int64_t>(a.rows) + ROW_TILE - 1) / ROW_TILE;
        hipLaunchKernelGGL((embed_grad_scan_kernel<T, I>), dim3(blocks_for(tiles, 1 << 16), (a.dim + SLAB - 1) / SLAB), dim3(THREADS), 0,
                           static_cast<hipStream_t>(stream), a, static_cast<const I *>(ids_dev), static_cast<const T *>(grad_dev),
                           static_cast<T *>(table_grad_dev));
    });
    return launched("mg_embed_grad");
}

int mg_adjust_logits(const MgAdjust *a, const void *logits_dev, void *out_dev, void *stream) {
    const int rc = adjust_args("mg_adjust_logits", a);
    if (rc != MG_OK || a->n == 0) return rc;
    if (!logits_dev || !out_dev) return refuse(MG_EINVAL, "mg_adjust_logits: null argument");
    with_types(a->dtype, a->history_type, [&](auto t, auto h) {
        using T = decltype(t);
        const int64_t chunks = (a->k + CHUNK - 1) / CHUNK;
        hipLaunchKernelGGL((adjust_kernel<T, decltype(h), false>), dim3(blocks_for(a->n * chunks)), dim3(THREADS), 0,
                           static_cast<hipStream_t>(stream), *a, static_cast<const T *>(logits_dev), static_cast<const T *>(nullptr), static_cast<T *>(out_dev));
    });
    return launched("mg_adjust_logits");
}

int mg_adjust_logits_grad(const MgAdjust *a, const void *logits_dev, const void *grad_dev, void *out_dev, void *stream) {
    const int rc = adjust_args("mg_adjust_logits_grad", a);
    if (rc != MG_OK || a->n == 0) return rc;
    if (!logits_dev || !grad_dev || !out_dev) return refuse(MG_EINVAL, "mg_adjust_logits_grad: null argument");
    with_types(a->dtype, a->history_type, [&](auto t, auto h) {
        using T = decltype(t);
        const int64_t chunks = (a->k + CHUNK - 1) / CHUNK;
        hipLaunchKernelGGL((adjust_kernel<T, decltype(h), true>), dim3(blocks_for(a->n * chunks)), dim3(THREADS), 0,
                           static_cast<hipStream_t>(stream), *a, static_cast<const T *>(logits_dev), static_cast<const T *>(grad_dev), static_cast<T *>(out_dev));
    });
    return launched("mg_adjust_logits_grad");
}

int64_t mg_draw_workspace(const MgLogits *l) { return logits_args("mg_draw_workspace", l); }

int mg_draw(const MgLogits *l, const void *logits_dev, const void *uniforms_dev, int32_t uniforms_type, void *tokens_dev,
            float *logprob_dev, void *workspace_dev, int64_t workspace_bytes, void *stream) {
    const int rc = logits_args("mg_draw", l);
    if (rc != MG_OK || l->n == 0) return rc;
    if (!logits_dev || !tokens_dev) return refuse(MG_EINVAL, "mg_draw: null argument");
    if (uniforms_dev && uniforms_type != MG_F32 && uniforms_type != MG_F64) return refuse(MG_EINVAL, "mg_draw: unknown type %d of the uniform numbers", uniforms_type);
    (void)workspace_dev;
    (void)workspace_bytes;
    with_types(l->dtype, MG_U8, [&](auto t, auto) {
        using T = decltype(t);
        hipLaunchKernelGGL((draw_kernel<T>), dim3(blocks_for(l->n)), dim3(THREADS), 0, static_cast<hipStream_t>(stream), *l,
                           static_cast<const T *>(logits_dev), uniforms_dev, uniforms_type, tokens_dev, logprob_dev);
    });
    return launched("mg_draw");
}

int64_t mg_token_logprobs_workspace(const MgLogits *l) { return logits_args("mg_token_logprobs_workspace", l); }

int mg_token_logprobs(const MgLogits *l, const void *logits_dev, const void *tokens_dev, float *logprob_dev, float *entropy_dev,
                      float *stats_dev, void *workspace_dev, int64_t workspace_bytes, void *stream) {
    const int rc = logits_args("mg_token_logprobs", l);
    if (rc != MG_OK || l->n == 0) return rc;
    if (!logits_dev || (logprob_dev && !tokens_dev)) return refuse(MG_EINVAL, "mg_token_logprobs: null argument");
    if (reinterpret_cast<uintptr_t>(stats_dev) % 16) return refuse(MG_EINVAL, "mg_token_logprobs: stats_dev must be 16-byte aligned");
    (void)workspace_dev;
    (void)workspace_bytes;
    with_types(l->dtype, MG_U8, [&](auto t, auto) {
        using T = decltype(t);
        hipLaunchKernelGGL((logprob_kernel<T>), dim3(blocks_for(l->n)), dim3(THREADS), 0, static_cast<hipStream_t>(stream), *l,
                           static_cast<const T *>(logits_dev), tokens_dev, logprob_dev, entropy_dev, stats_dev);
    });
    return launched("mg_token_logprobs");
}

int mg_token_logprobs_grad(const MgLogits *l, const void *logits_dev, const void *tokens_dev, const float *stats_dev,
                           const float *grad_logprob_dev, int64_t grad_logprob_stride, const float *grad_entropy_dev,
                           int64_t grad_entropy_stride, void *out_dev, void *stream) {
    const int rc = logits_args("mg_token_logprobs_grad", l);
    if (rc != MG_OK || l->n == 0) return rc;
    if (!logits_dev || !stats_dev || !out_dev || (grad_logprob_dev && !tokens_dev)) return refuse(MG_EINVAL, "mg_token_logprobs_grad: null argument");
    if (reinterpret_cast<uintptr_t>(stats_dev) % 16) return refuse(MG_EINVAL, "mg_token_logprobs_grad: stats_dev must be 16-byte aligned");
    if (grad_logprob_stride < 0 || grad_entropy_stride < 0) return refuse(MG_EINVAL, "mg_token_logprobs_grad: negative stride");
    with_types(l->dtype, MG_U8, [&](auto t, auto) {
        using T = decltype(t);
        hipLaunchKernelGGL((logprob_grad_kernel<T>), dim3(blocks_for(l->n)), dim3(THREADS), 0, static_cast<hipStream_t>(stream), *l,
                           static_cast<const T *>(logits_dev), tokens_dev, stats_dev, grad_logprob_dev, grad_logprob_stride, grad_entropy_dev,
                           grad_entropy_stride, static_cast<T *>(out_dev));
    });
    return launched("mg_token_logprobs_grad");
}

}  // extern "C"
