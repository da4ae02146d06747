// Paged key-value cache: appending tokens, reading them back, and eviction by
// accumulated attention weight.  All three are bound by the rows they move.
#include <atomic>
#include <cmath>
#include <cstdint>

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <cuda_runtime.h>

#include "rans_kv_common.h"

namespace rb200kv {
namespace {

constexpr int kThreads = 256;

// ------------------------------------------------------------------ append, read
// One thread per 8 values of a row: 16 bytes of a 16-bit row, one word of a 4-bit
// row (a quarter of a block of 32, so four neighbouring lanes share a scale).  A
// thread keeps its column (head and part of the row) and goes through the block's
// tokens, whose places are found once: what is left per 8 values is the rounding.
// 10127 tokens of 8 heads of 128 into 4 bits and back: 28 us together, bound by
// instructions; one token each of 4 sequences 3.1 us.

struct RowArgs {
    RansKvCache c;
    Divider page;
    const char* k_in;
    const char* v_in;
    int64_t k_token, k_head, v_token, v_head;      // bytes
    uint4* k_out;
    uint4* v_out;
    const int32_t* starts;
    int tokens;
    int part_shift;                                // log2 of a row's threads
    Divider columns;                               // by the threads of one token, or the block's if they are fewer
};

// Tokens of a block: a warp each to find out where they are.
constexpr int kTokens = kThreads / 32;

struct Where {
    int64_t k, v;              // where the token's first key and value row lies, in bytes
    int64_t place;             // and its books: of head 0
    int position;
    int ok;                    // 0: nowhere
};

// Sequence b's rows, as far as there are any.
__device__ __forceinline__ int rows_of(const RowArgs& a, int b) {
    return a.starts == nullptr ? 1 : max(min(a.starts[b + 1], a.tokens) - min(max(a.starts[b], 0), a.tokens), 0);
}

// Whether the rows are ranges that rise from 0 to `tokens`; a block asks, and raises what is wrong.  true: they rise, if not
// between those two.
__device__ __forceinline__ bool check_starts(const RowArgs& a) {
    if (a.starts == nullptr) return true;
    bool falls = false;
    for (int b = threadIdx.x; b < a.c.batch; b += kThreads) falls |= a.starts[b + 1] < a.starts[b];
    falls = __syncthreads_or(falls);
    if (threadIdx.x == 0 && (falls || a.starts[0] != 0 || a.starts[a.c.batch] != a.tokens)) raise(a.c, RANS_KV_BAD_STARTS);
    return !falls;
}

// The sequence b with starts[b] <= token < starts[b + 1], by the 32 lanes of a warp, and its first row; -1 if there is none.
__device__ __forceinline__ int sequence_of(const RowArgs& a, int token, int lane, int& first) {
    first = token;
    if (a.starts == nullptr) return token < a.c.batch ? token : -1;
    const int edge = a.starts[lane == 0 ? 0 : a.c.batch];
    int lo = 0, hi = a.c.batch, step;
    do {
        step = (hi - lo + 31) / 32;
        const int at = lo + lane * step, start = a.starts[min(at, hi)];
        const unsigned below = __ballot_sync(~0u, at < hi && start <= token);
        const int of = below == 0 ? 0 : 31 - __clz(below);
        first = __shfl_sync(~0u, start, of);
        lo += of * step;
        hi = min(lo + step, hi);
    } while (hi - lo > 1);
    first = max(first, 0);
    return __any_sync(~0u, lane == 0 ? token < edge : token >= edge) ? -1 : lo;
}

// Where the block's tokens lie, or are to lie: `last` 0 for tokens that follow what is there, 1 for the last ones there.
__device__ __forceinline__ void find_tokens(const RowArgs& a, Where* where, bool last) {
    const RansKvCache& c = a.c;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, token = blockIdx.x * kTokens + warp;
    if (token < a.tokens) {
        int first;
        const int b = sequence_of(a, token, lane, first);
        if (lane == 0) {
            Where w{};
            if (b < 0) {
                raise(c, RANS_KV_BAD_STARTS);
            } else {
                const int number = token - first, rows = last ? rows_of(a, b) : 0;
                const int place = checked_length(c, b) + number - rows;
                w.position = c.seen[b] + number;
                if (place < 0 || (last && number >= rows)) {
                    raise(c, RANS_KV_BAD_STARTS);
                } else if (place >= (int64_t)c.table_cols * c.page) {
                    raise(c, RANS_KV_BAD_LENGTH);
                } else {
                    const int in_page = a.page(place), page = checked_page(c, b, in_page), slot = place - in_page * c.page;
                    if (page >= 0) {
                        w.ok = 1;
                        w.k = page * c.k_page + slot * c.k_slot;
                        w.v = page * c.v_page + slot * c.v_slot;
                        w.place = (int64_t)page * c.kv_heads * c.page + slot;
                    }
                }
            }
            where[warp] = w;
        }
    }
    __syncthreads();
}

// 8 values as they are given.
template <int GIVEN>
struct Given8 {
    uint4 w[GIVEN == RANS_KV_FP32 ? 2 : 1];
};

// (Plain loads: the kernel before may still write rows when this one starts, so they are not constant while it lives.)
template <int GIVEN>
__device__ __forceinline__ void load8(Given8<GIVEN>& x, const char* p) {
    x.w[0] = *reinterpret_cast<const uint4*>(p);
    if constexpr (GIVEN == RANS_KV_FP32) x.w[1] = *(reinterpret_cast<const uint4*>(p) + 1);
}

template <int GIVEN>
__device__ __forceinline__ void to_float(float (&x)[8], const Given8<GIVEN>& y) {
    if constexpr (GIVEN == RANS_KV_FP32) {
        x[0] = __uint_as_float(y.w[0].x); x[1] = __uint_as_float(y.w[0].y); x[2] = __uint_as_float(y.w[0].z); x[3] = __uint_as_float(y.w[0].w);
        x[4] = __uint_as_float(y.w[1].x); x[5] = __uint_as_float(y.w[1].y); x[6] = __uint_as_float(y.w[1].z); x[7] = __uint_as_float(y.w[1].w);
    } else {
        const uint32_t u[4] = {y.w[0].x, y.w[0].y, y.w[0].z, y.w[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = GIVEN == RANS_KV_FP16 ? __half22float2(*reinterpret_cast<const __half2*>(&u[i]))
                                                   : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u[i]));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
}

__device__ __forceinline__ uint4 pack8(const float (&x)[8], int kind) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (kind == RANS_KV_FP16) {
            const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
            u[i] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            u[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
}

// 8 values in the cache's 16-bit type.
template <int GIVEN>
__device__ __forceinline__ uint4 rounded8(const Given8<GIVEN>& y, int kind) {
    if (kind == GIVEN) return y.w[0];
    float x[8];
    to_float(x, y);
    return pack8(x, kind);
}

// Four pairs of values as e2m1 codes, the first of a pair in a byte's low half.
__device__ __forceinline__ uint32_t to_e2m1(const float (&x)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r) : "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]));
    return r;
}

// 8 values of a block of 32 that lies over 4 neighbouring lanes -> 8 codes; `byte` the block's scale.
template <int GIVEN>
__device__ __forceinline__ uint32_t quantise8(const Given8<GIVEN>& y, uint32_t& byte) {
    float x[8];
    uint32_t top;          // the largest magnitude's bits: magnitudes compare as integers, an infinity or NaN as the largest
    if constexpr (GIVEN == RANS_KV_BF16) {
        const uint32_t abs = 0x7fff7fffu;
        uint32_t m = __vmaxu2(__vimax3_u16x2(y.w[0].x & abs, y.w[0].y & abs, y.w[0].z & abs), y.w[0].w & abs);
        m = __vmaxu2(m, __shfl_xor_sync(~0u, m, 1));
        m = __vmaxu2(m, __shfl_xor_sync(~0u, m, 2));
        top = max(m & 0xffff0000u, m << 16);
    } else {
        to_float(x, y);
        top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
        top = max(top, __shfl_xor_sync(~0u, top, 1));
        top = max(top, __shfl_xor_sync(~0u, top, 2));
    }
    if (top >= 0x7f800000u) {
        byte = 255;
        return 0;
    }
    const int e = min(max((int)(top >> 23) - 127 - 2, -63), 63);
    byte = (uint32_t)(e + 127);
    const float f = __uint_as_float((uint32_t)(127 - e) << 23);      // 2^-e: the division is exact
    if constexpr (GIVEN == RANS_KV_BF16) to_float(x, y);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= f;
    return to_e2m1(x);
}

template <int GIVEN, bool FP4>
__global__ void __launch_bounds__(kThreads, GIVEN == RANS_KV_FP32 ? 4 : 5) append_kernel(const __grid_constant__ RowArgs a) {
    __shared__ Where where[kTokens];
    __shared__ bool last;
    const RansKvCache& c = a.c;
    wait_for_previous();
    let_next_start();
    const int tokens = min(kTokens, a.tokens - (int)blockIdx.x * kTokens), columns = c.kv_heads << a.part_shift;
    const int wide = min(columns, kThreads), t0 = a.columns(threadIdx.x), c0 = threadIdx.x - t0 * wide, step = a.columns(kThreads);
    constexpr int kAtOnce = 2;                     // (5 blocks an SM with 2 rows each at once: 28.3 us for the case above, 4 with 4: 29.7; in bf16 17.3 and 18.2)
    Given8<GIVEN> in[kAtOnce][2];
    // token t0 + (first + u) * step of the block, column `col`; threads beyond step * wide have no token
    auto token_of = [&](int first, int u, int col) {
        const int t = t0 + (first + u) * step;
        return t0 < step && col < columns && t < tokens ? t : -1;
    };
    auto load = [&](int first, int col) {
        const int h = col >> a.part_shift;
        const int64_t at = (int64_t)(col & ((1 << a.part_shift) - 1)) * sizeof(Given8<GIVEN>);
        const char *k = a.k_in + h * a.k_head + at, *v = a.v_in + h * a.v_head + at;
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const int t = token_of(first, u, col);
            in[u][0] = in[u][1] = Given8<GIVEN>{};
            if (t < 0) continue;
            const int64_t token = blockIdx.x * kTokens + t;
            load8(in[u][0], k + token * a.k_token);
            load8(in[u][1], v + token * a.v_token);
        }
    };
    load(0, c0);                                   // on their way while the block finds out where they go
    find_tokens(a, where, false);
    // The block has read its lengths; the last one to say so moves them on below.
    int* counter = static_cast<int*>(c.workspace);
    if (threadIdx.x == 0) {
        last = atomicAdd(counter, 1) == (int)gridDim.x - 1;
        if (last) *counter = 0;
    }
    // (all lanes take every turn: a row has 8 threads or more, so a block of 32 values lies in four lanes that have a token
    // or none together)
    for (int col0 = 0; col0 < columns; col0 += wide) {
        const int col = c0 + col0, h = col >> a.part_shift, part = col & ((1 << a.part_shift) - 1);
        char *k = static_cast<char*>(c.k) + h * c.k_head, *v = static_cast<char*>(c.v) + h * c.v_head;
        const int in_row = FP4 ? (part % 4 << a.part_shift) + part / 4 * 4 : part * 16;
        for (int first = 0; first * step < tokens; first += kAtOnce) {
            if (col0 != 0 || first != 0) load(first, col);
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                if ((first + u) * step >= tokens) break;
                const int t = token_of(first, u, col);
                const Where& w = where[max(t, 0)];
                const bool stored = t >= 0 && w.ok;
                const int64_t place = w.place + h * c.page;
                if constexpr (FP4) {
                    uint32_t byte[2];
                    const uint32_t k_code = quantise8(in[u][0], byte[0]), v_code = quantise8(in[u][1], byte[1]);
                    if (stored) {
                        *reinterpret_cast<uint32_t*>(k + w.k + in_row) = k_code;
                        *reinterpret_cast<uint32_t*>(v + w.v + in_row) = v_code;
                        if (part % 4 == 0) {
                            const int64_t at = (place << (a.part_shift - 2)) + part / 4;
                            c.k_scale[at] = (uint8_t)byte[0];
                            c.v_scale[at] = (uint8_t)byte[1];
                        }
                    }
                } else if (stored) {
                    *reinterpret_cast<uint4*>(k + w.k + in_row) = rounded8(in[u][0], c.kind);
                    *reinterpret_cast<uint4*>(v + w.v + in_row) = rounded8(in[u][1], c.kind);
                }
                if (stored && part == 0) {
                    if (c.position != nullptr) c.position[place] = w.position;
                    if (c.weight != nullptr) c.weight[place] = 0.0f;
                }
            }
        }
    }
    __syncthreads();
    // (where the ranges fall, nobody can say which rows are whose: what was stored lies behind the lengths and stays there)
    if (last && check_starts(a))
        for (int b = threadIdx.x; b < c.batch; b += kThreads) {
            const int n = rows_of(a, b);
            c.length[b] = (int)min((int64_t)checked_length(c, b) + n, (int64_t)c.table_cols * c.page);
            c.seen[b] += n;
        }
}

// What 8 codes and their block's scale byte stand for, in bf16 (exact).
__device__ __forceinline__ uint4 values8(uint32_t code, uint32_t byte) {
    const float f = byte == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23);
    float y[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const __half2_raw r = __nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)((code >> (8 * e)) & 255), __NV_E2M1);
        const float2 z = __half22float2(__half2(r));
        y[2 * e] = z.x * f;
        y[2 * e + 1] = z.y * f;
    }
    return pack8(y, RANS_KV_BF16);
}

// (Six blocks an SM for 4-bit rows; 16-bit ones then spill, and take five: 10127 tokens of 8 heads of 128 18.8 -> 16.3 us, 20000 of
// 2 heads of 64 9.4 -> 9.2, the same as with four and 9.9.)
template <bool FP4>
__global__ void __launch_bounds__(kThreads, FP4 ? 6 : 5) read_kernel(const __grid_constant__ RowArgs a) {
    __shared__ Where where[kTokens];
    const RansKvCache& c = a.c;
    wait_for_previous();
    let_next_start();
    find_tokens(a, where, true);
    if (blockIdx.x == 0) check_starts(a);
    const int tokens = min(kTokens, a.tokens - (int)blockIdx.x * kTokens), columns = c.kv_heads << a.part_shift;
    const int wide = min(columns, kThreads), t0 = a.columns(threadIdx.x), c0 = threadIdx.x - t0 * wide, step = a.columns(kThreads);
    if (t0 >= step) return;
    const int64_t out0 = (int64_t)blockIdx.x * kTokens * columns;
    constexpr int kAtOnce = 4;
    for (int col = c0; col < columns; col += wide) {
        const int h = col >> a.part_shift, part = col & ((1 << a.part_shift) - 1);
        const char *k = static_cast<const char*>(c.k) + h * c.k_head, *v = static_cast<const char*>(c.v) + h * c.v_head;
        for (int first = t0; first < tokens; first += step * kAtOnce) {
            uint4 x[kAtOnce][2];           // 4 bits: the codes in .x, the scale byte in .y
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int t = first + u * step;
                x[u][0] = x[u][1] = make_uint4(0, 0, 0, 0);
                if (t >= tokens || !where[t].ok) continue;
                const Where& w = where[t];
                if constexpr (FP4) {
                    const int in_row = (part % 4 << a.part_shift) + part / 4 * 4;
                    const int64_t at = ((w.place + h * c.page) << (a.part_shift - 2)) + part / 4;
                    x[u][0].x = *reinterpret_cast<const uint32_t*>(k + w.k + in_row);
                    x[u][0].y = c.k_scale[at];
                    x[u][1].x = *reinterpret_cast<const uint32_t*>(v + w.v + in_row);
                    x[u][1].y = c.v_scale[at];
                } else {
                    x[u][0] = *reinterpret_cast<const uint4*>(k + w.k + part * 16);
                    x[u][1] = *reinterpret_cast<const uint4*>(v + w.v + part * 16);
                }
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int t = first + u * step;
                if (t >= tokens) continue;
                const int64_t at = out0 + (int64_t)t * columns + col;
                a.k_out[at] = FP4 ? values8(x[u][0].x, x[u][0].y) : x[u][0];
                a.v_out[at] = FP4 ? values8(x[u][1].x, x[u][1].y) : x[u][1];
            }
        }
    }
}

// ------------------------------------------------------------------ evict
// Per (sequence, kv head) a cluster of blocks: find the key of the budget-th heaviest token by radix selection over 32-bit
// keys (passes of 11, 11 and 10 bits, of which the last is seldom needed; the blocks' histograms are added up through the
// cluster's shared memory), mark what stays, pair
// the i-th kept place at or above the budget with the i-th freed place below it, and move the rows.  Sources lie at or above
// the budget and destinations below it, so moves never meet.  Bound by the passes' latency (32 x 2 heads of 4160 tokens: 13.5 us)
// and, where much moves, by rows of 256 bytes read and written (8 heads of 65536 to 16384, 50 MB: 22 us to select, 24 to move).
// Clusters, shared memory and the kernel of the moves are chosen by the table's room: these figures are of tables as long as the
// sequences.  In tables 8 times as long 32 x 8 heads of 4160 tokens take 43 us instead of 24, 8 heads of 16385 10.4 instead of 9.2.

// Threads of a block: many for a head's latency, fewer where there are more heads than SMs, so that four blocks share one (392 heads
// of 147 tokens 18.2 -> 7.3 us, of 4200 51.3 -> 37.6; 160 of 4200 28.6 -> 26.3; but 128 of 4160 16.2 -> 22.5).
constexpr int kSelect = 1024, kSelectMany = 256;
constexpr int kBins = 2048;
constexpr int kFew = 4;                                    // tokens over the budget that are searched for one by one
constexpr int kMaxCluster = 8;                             // the portable size; of 16, seven at most run at a time
constexpr int kPlaces = 4096;                              // a block takes before there are more of them
constexpr int kMaxSharedKeys = 40 * 1024;                  // of a block; more are kept in the workspace

struct EvictArgs {
    RansKvCache c;
    Divider page;
    int budget, recent;
    int* counter;                // [batch], zero between calls
    int* to;                     // [batch * kv_heads][lists]: place of each move's destination
    int* from;                   // and source
    int lists;                   // the moves that the table has room for
    uint32_t* keys;              // [batch * kv_heads][table_cols * page], or NULL: in shared memory
    int* moves;                  // [batch * kv_heads]: how many, for move_kernel, or NULL: moved here
    int row_shift;               // log2 of the 16-byte pieces of a row
};

// Order-preserving key of a weight; the newest tokens come first, then NaN.
__device__ __forceinline__ uint32_t key_of(float w, bool late) {
    if (late) return 0xffffffffu;
    if (w != w) return 0xfffffffeu;
    const uint32_t u = __float_as_uint(w + 0.0f);          // -0 -> +0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int warp_sum(int x) { return __reduce_add_sync(~0u, x); }

// Moves m0 .. m1 - 1 of one (sequence, kv head), by a block of THREADS threads.
template <int THREADS>
__device__ __forceinline__ void move_rows(const EvictArgs& a, int b, int h, const int* to, const int* from, int m0, int m1, int4* moving) {
    const RansKvCache& c = a.c;
    const int tid = threadIdx.x;
            for (int m = m0; m < m1; m += THREADS) {
                // a thread per move: its pages, and what goes with the rows
                const int here = min(THREADS, m1 - m);
                if (tid < here) {
                    const int to_t = to[m + tid], from_t = from[m + tid];
                    const int to_page = a.page(to_t), from_page = a.page(from_t);
            const int4 mv = make_int4(checked_page(c, b, to_page), to_t - to_page * c.page, checked_page(c, b, from_page), from_t - from_page * c.page);
                    moving[tid] = mv;
                    if (mv.x >= 0 && mv.z >= 0) {
                        const int64_t x = ((int64_t)mv.x * c.kv_heads + h) * c.page + mv.y, y = ((int64_t)mv.z * c.kv_heads + h) * c.page + mv.w;
                        c.weight[x] = c.weight[y];
                        c.position[x] = c.position[y];
                        if (c.kind == RANS_KV_MXFP4) {
                            if (c.dim == 64) {
                                reinterpret_cast<uint16_t*>(c.k_scale)[x] = reinterpret_cast<uint16_t*>(c.k_scale)[y];
                                reinterpret_cast<uint16_t*>(c.v_scale)[x] = reinterpret_cast<uint16_t*>(c.v_scale)[y];
                            } else if (c.dim == 128) {
                                reinterpret_cast<uint32_t*>(c.k_scale)[x] = reinterpret_cast<uint32_t*>(c.k_scale)[y];
                                reinterpret_cast<uint32_t*>(c.v_scale)[x] = reinterpret_cast<uint32_t*>(c.v_scale)[y];
                            } else {
                                reinterpret_cast<uint64_t*>(c.k_scale)[x] = reinterpret_cast<uint64_t*>(c.k_scale)[y];
                                reinterpret_cast<uint64_t*>(c.v_scale)[x] = reinterpret_cast<uint64_t*>(c.v_scale)[y];
                            }
                        }
                    }
                }
                __syncthreads();
                const int all = here << (a.row_shift + 1);                       // pieces of the key and value rows
                constexpr int kAtOnce = 4;
                for (int i0 = tid; i0 < all; i0 += THREADS * kAtOnce) {
                    uint4 x[kAtOnce];
                    char* dst[kAtOnce];
    #pragma unroll
                    for (int u = 0; u < kAtOnce; ++u) {
                        const int i = i0 + u * THREADS, part = i & ((1 << a.row_shift) - 1);
                        const bool is_k = (i >> a.row_shift & 1) == 0;
                        dst[u] = nullptr;
                        if (i >= all) continue;
                        const int4 mv = moving[i >> (a.row_shift + 1)];
                        if (mv.x < 0 || mv.z < 0) continue;                      // (a bad page: reported above)
                        char* base = static_cast<char*>(is_k ? c.k : c.v) + h * (is_k ? c.k_head : c.v_head) + part * 16;
                        const int64_t page = is_k ? c.k_page : c.v_page, slot = is_k ? c.k_slot : c.v_slot;
                        x[u] = *reinterpret_cast<const uint4*>(base + mv.z * page + mv.w * slot);
                        dst[u] = base + mv.x * page + mv.y * slot;
                    }
    #pragma unroll
                    for (int u = 0; u < kAtOnce; ++u)
                        if (dst[u] != nullptr) *reinterpret_cast<uint4*>(dst[u]) = x[u];
                }
                __syncthreads();
            }
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) evict_kernel(const __grid_constant__ EvictArgs a) {
    constexpr int kWarps = THREADS / 32, kPer = kBins / THREADS;
    extern __shared__ uint32_t shared_keys[];
    __shared__ __align__(8) int hist[2][kBins];
    __shared__ int digit_s, rank_s, count_s;
    __shared__ uint2 lightest[kFew];                       // the block's lightest token of each turn: key, place
    __shared__ int wsum[2][kWarps];
    __shared__ int block_sum[3];                           // ties, holes, movers of the block's places
    __shared__ int4 moving[THREADS];                       // (page, slot) to and from
    const cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    const RansKvCache& c = a.c;
    const int blocks = cluster.num_blocks(), block = cluster.block_rank(), bh = blockIdx.x / blocks;
    const int h = bh % c.kv_heads, b = bh / c.kv_heads;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    wait_for_previous();
    let_next_start();
    const int n = checked_length(c, b), k = a.budget;
    if (n > k) {
        // each block has a run of 32-place words, each warp a run of the block's
        const int words = (n + 31) / 32, bw0 = (int)((int64_t)words * block / blocks), bw1 = (int)((int64_t)words * (block + 1) / blocks);
        const int w0 = bw0 + (bw1 - bw0) * warp / kWarps, w1 = bw0 + (bw1 - bw0) * (warp + 1) / kWarps;
        uint32_t* keys = a.keys != nullptr ? a.keys + (int64_t)bh * c.table_cols * c.page : shared_keys - (int64_t)bw0 * 32;
        const int first_late = c.seen[b] - a.recent;
        const int t_end = min(bw1 * 32, n);
        constexpr int kLoads = 4;
        for (int t0 = bw0 * 32 + tid; t0 < t_end; t0 += THREADS * kLoads) {
            int64_t at[kLoads];
            float weight[kLoads];
            int position[kLoads];
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int t = t0 + i * THREADS, in_page = a.page(t), p = t < t_end ? checked_page(c, b, in_page) : -1;
                at[i] = p >= 0 ? ((int64_t)p * c.kv_heads + h) * c.page + (t - in_page * c.page) : -1;
            }
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                weight[i] = at[i] >= 0 ? c.weight[at[i]] : 0.0f;
                position[i] = at[i] >= 0 ? c.position[at[i]] : 0;
            }
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                if (t0 + i * THREADS < t_end) keys[t0 + i * THREADS] = at[i] >= 0 ? key_of(weight[i], position[i] >= first_late) : 0;
        }
        auto sync = [&]() {
            if (blocks == 1) __syncthreads(); else cluster.sync();
        };
        int *to = a.to + (int64_t)bh * a.lists, *from = a.from + (int64_t)bh * a.lists;
        int moves = 0;
        if (n - k <= kFew) {
            // A few too many, as in a loop that evicts as it appends: the lightest (of equals the last) goes, n - k times.
            int gone[kFew];
#pragma unroll
            for (int turn = 0; turn < kFew; ++turn) {
                gone[turn] = -1;
                if (turn >= n - k) continue;
                __syncthreads();
                uint32_t key = 0xffffffffu;
                int place = -1;
                for (int t = w0 * 32 + lane; t < min(w1 * 32, n); t += 32) {
                    bool out = false;
#pragma unroll
                    for (int i = 0; i < turn; ++i) out |= t == gone[i];
                    if (!out && keys[t] <= key) {
                        key = keys[t];
                        place = t;
                    }
                }
                uint32_t least = __reduce_min_sync(~0u, key);
                int last = __reduce_max_sync(~0u, key == least ? place : -1);
                if (lane == 0) {
                    wsum[0][warp] = (int)least;
                    wsum[1][warp] = last;
                }
                __syncthreads();
                key = lane < kWarps ? (uint32_t)wsum[0][lane] : 0xffffffffu;
                place = lane < kWarps ? wsum[1][lane] : -1;
                least = __reduce_min_sync(~0u, place >= 0 ? key : 0xffffffffu);
                last = __reduce_max_sync(~0u, key == least ? place : -1);
                if (blocks > 1) {
                    if (tid == 0) lightest[turn] = make_uint2(least, (uint32_t)last);
                    cluster.sync();
                    const uint2 x = lane < blocks ? *cluster.map_shared_rank(&lightest[turn], lane) : make_uint2(0xffffffffu, (uint32_t)-1);
                    least = __reduce_min_sync(~0u, (int)x.y >= 0 ? x.x : 0xffffffffu);
                    last = __reduce_max_sync(~0u, x.x == least ? (int)x.y : -1);
                }
                gone[turn] = last;
            }
            if (block == 0 && tid == 0) {
                // the freed places below the budget, rising, and the kept ones above it
                int holes = 0, kept = 0;
                for (int above = -1;;) {
                    int next = k;
#pragma unroll
                    for (int i = 0; i < kFew; ++i)
                        if (gone[i] > above && gone[i] < next) next = gone[i];
                    if (next == k) break;
                    to[holes++] = above = next;
                }
                for (int t = k; t < n; ++t) {
                    bool out = false;
#pragma unroll
                    for (int i = 0; i < kFew; ++i) out |= t == gone[i];
                    if (!out) from[kept++] = t;
                }
                block_sum[1] = holes;
            }
            sync();
            moves = *cluster.map_shared_rank(&block_sum[1], 0);
            if (blocks > 1) cluster.sync();                // block 0 stays until all have read
        } else {
            uint32_t prefix = 0;
            int rank = k;                                      // of the threshold among the keys that share the prefix
#pragma unroll 1
            for (int pass = 0; pass < 3; ++pass) {
                const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
                const uint32_t mask = pass == 0 ? 0u : pass == 1 ? ~0u << 21 : ~0u << 10;        // of the digits found
                int* mine = hist[pass & 1];
#pragma unroll
                for (int i = 0; i < kPer; ++i) mine[tid + i * THREADS] = 0;
                __syncthreads();
                for (int w = w0; w < w1; ++w) {
                    const int t = w * 32 + lane;
                    const uint32_t key = t < n ? keys[t] : 0;
                    if (t < n && (key & mask) == prefix) atomicAdd(&mine[(key >> shift) & (kBins - 1)], 1);
                }
                sync();
                // thread i: kPer bins of all blocks, falling from kBins - 1 - kPer i
                int sum[kPer];
#pragma unroll
                for (int i = 0; i < kPer; ++i) sum[i] = 0;
                for (int r = 0; r < blocks; ++r) {
                    const int2* x = reinterpret_cast<const int2*>(cluster.map_shared_rank(mine, r)) + (THREADS - 1 - tid) * (kPer / 2);
#pragma unroll
                    for (int i = 0; i < kPer; i += 2) {
                        const int2 y = x[kPer / 2 - 1 - i / 2];
                        sum[i] += y.y;
                        sum[i + 1] += y.x;
                    }
                }
                int own = 0;
#pragma unroll
                for (int i = 0; i < kPer; ++i) own += sum[i];
                int inc = own;
#pragma unroll
                for (int i = 1; i < 32; i *= 2) {
                    const int y = __shfl_up_sync(~0u, inc, i);
                    if (lane >= i) inc += y;
                }
                if (lane == 31) wsum[pass & 1][warp] = inc;
                __syncthreads();
                int before = inc - own + warp_sum(lane < warp ? wsum[pass & 1][lane] : 0);
                if (before < rank && rank <= before + own) {
                    bool found = false;
#pragma unroll
                    for (int i = 0; i < kPer; ++i) {
                        if (!found && rank <= before + sum[i]) {
                            digit_s = kBins - 1 - kPer * tid - i;
                            rank_s = rank - before;
                            count_s = sum[i];
                            found = true;
                        }
                        before += sum[i];
                    }
                }
                __syncthreads();
                prefix |= (uint32_t)digit_s << shift;
                rank = rank_s;
                if (rank == count_s) {
                    // all that share these digits stay: no ties to part.  (prefix > 0, for n > budget keys are not all kept.)
                    --prefix;
                    rank = 0;
                    break;
                }
            }
            // Keys above `prefix` stay, and the first `rank` places whose key equals it.
            int tie0 = 0;
            if (rank > 0) {
                int ties = 0;
                for (int w = w0; w < w1; ++w) {
                    const int t = w * 32 + lane;
                    ties += __popc(__ballot_sync(~0u, t < n && keys[t] == prefix));
                }
                __syncthreads();
                if (lane == 0) wsum[0][warp] = ties;
                __syncthreads();
                tie0 = warp_sum(lane < warp ? wsum[0][lane] : 0);
                if (tid == THREADS - 1) block_sum[0] = tie0 + ties;
                sync();
                tie0 += warp_sum(lane < block ? *cluster.map_shared_rank(&block_sum[0], lane) : 0);
            }
            auto kept = [&](int w, int& tie) {
                const int t = w * 32 + lane;
                const uint32_t key = t < n ? keys[t] : 0;
                const unsigned equal = __ballot_sync(~0u, t < n && key == prefix);
                const bool keep = t < n && (key > prefix || (key == prefix && tie + __popc(equal & ((1u << lane) - 1)) < rank));
                tie += __popc(equal);
                return keep;
            };
            int holes = 0, movers = 0, tie = tie0;
            for (int w = w0; w < w1; ++w) {
                const int t = w * 32 + lane;
                const bool keep = kept(w, tie);
                holes += __popc(__ballot_sync(~0u, t < k && !keep));
                movers += __popc(__ballot_sync(~0u, t >= k && keep));
            }
            __syncthreads();
            if (lane == 0) {
                wsum[0][warp] = holes;
                wsum[1][warp] = movers;
            }
            __syncthreads();
            int hole = warp_sum(lane < warp ? wsum[0][lane] : 0), mover = warp_sum(lane < warp ? wsum[1][lane] : 0);
            if (tid == THREADS - 1) {
                block_sum[1] = hole + holes;
                block_sum[2] = mover + movers;
            }
            sync();
            const int block_holes = lane < blocks ? *cluster.map_shared_rank(&block_sum[1], lane) : 0;
            const int block_movers = lane < blocks ? *cluster.map_shared_rank(&block_sum[2], lane) : 0;
            hole += warp_sum(lane < block ? block_holes : 0);
            mover += warp_sum(lane < block ? block_movers : 0);
            moves = warp_sum(block_holes);
            tie = tie0;
            for (int w = w0; w < w1; ++w) {
                const int t = w * 32 + lane;
                const bool keep = kept(w, tie);
                const unsigned is_hole = __ballot_sync(~0u, t < k && !keep), is_mover = __ballot_sync(~0u, t >= k && keep);
                const unsigned below = (1u << lane) - 1;
                if (is_hole >> lane & 1) to[hole + __popc(is_hole & below)] = t;
                if (is_mover >> lane & 1) from[mover + __popc(is_mover & below)] = t;
                hole += __popc(is_hole);
                mover += __popc(is_mover);
            }
            sync();                                            // the lists are whole; nobody reads another block's memory from here on
        }

        if (a.moves != nullptr) {
            if (block == 0 && tid == 0) a.moves[bh] = moves;
        } else {
            move_rows<THREADS>(a, b, h, to, from, (int)((int64_t)moves * block / blocks), (int)((int64_t)moves * (block + 1) / blocks), moving);
        }
    } else if (a.moves != nullptr && block == 0 && tid == 0) {
        a.moves[bh] = 0;
    }
    // The last block of a sequence (all have read its length by then) shortens it.
    __syncthreads();
    if (tid == 0) {
        __threadfence();
        if (atomicAdd(a.counter + b, 1) == blocks * c.kv_heads - 1) {
            a.counter[b] = 0;
            if (n > k) c.length[b] = k;
        }
    }
}

__global__ void __launch_bounds__(kThreads) move_kernel(const __grid_constant__ EvictArgs a) {
    __shared__ int4 moving[kThreads];
    wait_for_previous();
    let_next_start();
    const int bh = blockIdx.y, moves = a.moves[bh];
    const int m0 = (int)((int64_t)moves * blockIdx.x / gridDim.x), m1 = (int)((int64_t)moves * (blockIdx.x + 1) / gridDim.x);
    move_rows<kThreads>(a, bh / a.c.kv_heads, bh % a.c.kv_heads, a.to + (int64_t)bh * a.lists, a.from + (int64_t)bh * a.lists, m0, m1, moving);
}

struct EvictPlan {
    int64_t to, from, moves, keys, bytes;
    int lists;                       // most moves of a (sequence, kv head)
    bool apart;                      // moves in a kernel of their own
    int blocks, shared_keys;         // of a (sequence, kv head); keys a block holds in shared memory (0: in the workspace)
};

bool plan_evict(const RansKvCache& c, int budget, EvictPlan& p) {
    if (budget < 1) return false;
    auto up = [](int64_t x) { return (x + 255) & ~(int64_t)255; };
    const int64_t heads = (int64_t)c.batch * c.kv_heads, room = (int64_t)c.table_cols * c.page;
    // as many blocks as fill the SMs once, but no more than have a few places for each thread
    p.blocks = 1;
    while (p.blocks < kMaxCluster && heads * p.blocks * 2 <= kSms && room > (int64_t)p.blocks * kPlaces) p.blocks *= 2;
    const int64_t most = ((room + 31) / 32 / p.blocks + 1) * 32;
    p.shared_keys = most <= kMaxSharedKeys ? (int)most : 0;
    p.lists = room > budget ? (int)(budget < room - budget ? budget : room - budget) : 0;
    p.to = counter_bytes(c);
    p.from = p.to + up(heads * p.lists * 4);
    p.moves = p.from + up(heads * p.lists * 4);
    p.keys = p.moves + up(heads * 4);
    // Few heads leave SMs without a block of the selection: from 32 MB on, the moves get a grid of their own.
    const int64_t row = c.kind == RANS_KV_MXFP4 ? c.dim / 2 : c.dim * 2;
    p.apart = heads * p.blocks < kSms && heads * p.lists * row * 2 >= (32 << 20);
    p.bytes = p.keys + (p.shared_keys ? 0 : up(heads * room * 4));
    return true;
}

void set_rows(RowArgs& a, const RansKvCache& c, const int32_t* starts, int tokens) {
    a.c = c;
    fill_strides(a.c);
    a.page = Divider::of((uint32_t)c.page);
    a.starts = starts;
    a.tokens = tokens;
    a.part_shift = c.dim == 64 ? 3 : c.dim == 128 ? 4 : 5;
    const int columns = c.kv_heads << a.part_shift;
    a.columns = Divider::of((uint32_t)(columns < kThreads ? columns : kThreads));
}

int row_grid(const RowArgs& a) { return (a.tokens + kTokens - 1) / kTokens; }

}  // namespace
}  // namespace rb200kv

using namespace rb200kv;

extern "C" int rans_kv_append(const RansKvCache* cache, const void* k, const void* v, int given, int64_t k_token, int64_t k_head,
                              int64_t v_token, int64_t v_head, const int32_t* starts, int tokens, cudaStream_t stream) {
    const int rc = check_cache(cache);
    if (rc != 0) return rc;
    if (given != RANS_KV_BF16 && given != RANS_KV_FP16 && given != RANS_KV_FP32) return -1;
    if (tokens < 0 || (starts == nullptr && tokens != cache->batch)) return -2;
    if (tokens == 0) return 0;
    if (k == nullptr || v == nullptr || !aligned16(k) || !aligned16(v) || ((k_token | k_head | v_token | v_head) & 15)) return -2;
    RowArgs a{};
    set_rows(a, *cache, starts, tokens);
    a.k_in = static_cast<const char*>(k);
    a.v_in = static_cast<const char*>(v);
    a.k_token = k_token; a.k_head = k_head; a.v_token = v_token; a.v_head = v_head;
    const bool fp4 = cache->kind == RANS_KV_MXFP4;
    auto kernel = given == RANS_KV_FP32   ? (fp4 ? append_kernel<RANS_KV_FP32, true> : append_kernel<RANS_KV_FP32, false>)
                  : given == RANS_KV_FP16 ? (fp4 ? append_kernel<RANS_KV_FP16, true> : append_kernel<RANS_KV_FP16, false>)
                                          : (fp4 ? append_kernel<RANS_KV_BF16, true> : append_kernel<RANS_KV_BF16, false>);
    return launch_after(kernel, dim3(row_grid(a)), kThreads, 0, 1, stream, a);
}

extern "C" int rans_kv_read(const RansKvCache* cache, void* k_out, void* v_out, const int32_t* starts, int tokens,
                            cudaStream_t stream) {
    const int rc = check_cache(cache);
    if (rc != 0) return rc;
    if (tokens < 0 || (starts == nullptr && tokens != cache->batch)) return -2;
    if (tokens == 0) return 0;
    if (k_out == nullptr || v_out == nullptr || !aligned16(k_out) || !aligned16(v_out)) return -2;
    RowArgs a{};
    set_rows(a, *cache, starts, tokens);
    a.k_out = static_cast<uint4*>(k_out);
    a.v_out = static_cast<uint4*>(v_out);
    return launch_after(cache->kind == RANS_KV_MXFP4 ? read_kernel<true> : read_kernel<false>, dim3(row_grid(a)), kThreads, 0, 1, stream, a);
}

extern "C" int64_t rans_kv_evict_bytes(const RansKvCache* c, int budget) {
    if (rans_kv_counter_bytes(c) < 0 || c->table_cols < 1 || c->page < 16) return -2;
    EvictPlan p;
    return plan_evict(*c, budget, p) ? p.bytes : -2;
}

extern "C" int rans_kv_evict(const RansKvCache* cache, int budget, int recent, cudaStream_t stream) {
    const int rc = check_cache(cache);
    if (rc != 0) return rc;
    EvictPlan p;
    if (cache->weight == nullptr || cache->position == nullptr || recent < 0 || recent > budget || !plan_evict(*cache, budget, p)) return -2;
    if (cache->workspace_bytes < p.bytes) return -3;
    EvictArgs a{};
    a.c = *cache;
    fill_strides(a.c);
    a.page = Divider::of((uint32_t)cache->page);
    char* ws = static_cast<char*>(cache->workspace);
    a.budget = budget;
    a.recent = recent;
    a.lists = p.lists;
    a.counter = reinterpret_cast<int*>(ws + 256);
    a.to = reinterpret_cast<int*>(ws + p.to);
    a.from = reinterpret_cast<int*>(ws + p.from);
    a.keys = p.shared_keys ? nullptr : reinterpret_cast<uint32_t*>(ws + p.keys);
    for (int pieces = cache->kind == RANS_KV_MXFP4 ? cache->dim / 32 : cache->dim / 8; pieces > 1; pieces /= 2) ++a.row_shift;
    a.moves = p.apart ? reinterpret_cast<int*>(ws + p.moves) : nullptr;
    static std::atomic<uint64_t> told{0};      // per device: the kernel may use this much shared memory
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return (int)e;
    const uint64_t bit = (uint64_t)1 << (device & 63);
    if ((told.load(std::memory_order_relaxed) & bit) == 0) {
        e = cudaFuncSetAttribute(evict_kernel<kSelect>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSharedKeys * 4);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(evict_kernel<kSelectMany>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSharedKeys * 4);
        if (e != cudaSuccess) return (int)e;
        told.fetch_or(bit, std::memory_order_relaxed);
    }
    const int heads = cache->batch * cache->kv_heads;
    const bool many = heads > kSms;
    const int rc2 = launch_after(many ? evict_kernel<kSelectMany> : evict_kernel<kSelect>, dim3(heads * p.blocks), many ? kSelectMany : kSelect, (size_t)p.shared_keys * 4, p.blocks, stream, a);
    if (rc2 != 0 || !p.apart) return rc2;
    return launch_after(move_kernel, dim3((4 * kSms + heads - 1) / heads, heads), kThreads, 0, 1, stream, a);
}
