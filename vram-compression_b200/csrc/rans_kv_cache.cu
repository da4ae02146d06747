// Paged key-value cache: appending tokens, reading them back, and eviction by
// accumulated attention weight.  All three are bound by the rows they move.
#include <cmath>
#include <cstdint>

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
// row (a quarter of a block of 32, so four neighbouring lanes share a scale).

struct RowArgs {
    RansKvCache c;
    const char* k_in;
    const char* v_in;
    int64_t k_token, k_head, v_token, v_head;      // bytes
    uint4* k_out;
    uint4* v_out;
    const int32_t* starts;
    int tokens;
    int given;
};

// The sequence that row `token` belongs to, or -1, and the row's number within it.
__device__ __forceinline__ int sequence_of(const RowArgs& a, int token, int& number) {
    if (a.starts == nullptr) {
        number = 0;
        return token < a.c.batch ? token : -1;
    }
    int lo = 0, hi = a.c.batch;                    // starts[lo] <= token < starts[hi]
    if (token < a.starts[0] || token >= a.starts[a.c.batch]) return -1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.starts[mid] <= token) lo = mid; else hi = mid;
    }
    number = token - a.starts[lo];
    return lo;
}

__device__ __forceinline__ int rows_of(const RowArgs& a, int b) {
    return a.starts == nullptr ? 1 : max(a.starts[b + 1] - a.starts[b], 0);
}

__device__ __forceinline__ void load8(float (&x)[8], const char* p, int given) {
    if (given == RANS_KV_FP32) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
        return;
    }
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = given == RANS_KV_FP16 ? __half22float2(*reinterpret_cast<const __half2*>(&u[i]))
                                               : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
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

// 8 values of a block of 32 that lies over 4 neighbouring lanes -> 8 codes; `byte` the block's scale.
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], uint32_t& byte) {
    // magnitudes compare as integers, and an infinity or NaN as the largest
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(~0u, top, 1));
    top = max(top, __shfl_xor_sync(~0u, top, 2));
    if (top >= 0x7f800000u) {
        byte = 255;
        return 0;
    }
    const int e = min(max((int)(top >> 23) - 127 - 2, -63), 63);
    byte = (uint32_t)(e + 127);
    const float f = __uint_as_float((uint32_t)(127 - e) << 23);      // 2^-e: the division is exact
    uint32_t code = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        code |= (uint32_t)__nv_cvt_float2_to_fp4x2(make_float2(x[2 * i] * f, x[2 * i + 1] * f), __NV_E2M1, cudaRoundNearest) << (8 * i);
    return code;
}

__global__ void __launch_bounds__(kThreads) append_kernel(const __grid_constant__ RowArgs a) {
    const RansKvCache& c = a.c;
    const int per_row = c.dim / 8;
    const int64_t all = (int64_t)a.tokens * c.kv_heads * per_row;
    // dim / 8 is a multiple of 8, so the 4 lanes of a block are in or out of range together
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i - (threadIdx.x & 31) < all; i += (int64_t)gridDim.x * kThreads) {
        const int part = (int)(i % per_row);
        const int64_t row = i / per_row;
        const int h = (int)(row % c.kv_heads), token = (int)(row / c.kv_heads);
        const bool in = i < all;
        int number = 0, p = -1, slot = 0, place = 0, b = -1;
        if (in) {
            b = sequence_of(a, token, number);
            if (b < 0) {
                raise(c, RANS_KV_BAD_STARTS);
            } else {
                place = checked_length(c, b) + number;
                if (place >= (int64_t)c.table_cols * c.page) {
                    raise(c, RANS_KV_BAD_LENGTH);
                } else {
                    p = checked_page(c, b, place / c.page);
                    slot = place % c.page;
                }
            }
        }
        float x[8];
        uint32_t byte;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const char* src = w == 0 ? a.k_in + token * a.k_token + h * a.k_head : a.v_in + token * a.v_token + h * a.v_head;
            if (in) {
                load8(x, src + (int64_t)part * (a.given == RANS_KV_FP32 ? 32 : 16), a.given);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = 0.0f;
            }
            char* base = static_cast<char*>(w == 0 ? c.k : c.v);
            const int64_t at = (int64_t)p * (w == 0 ? c.k_page : c.v_page) + h * (w == 0 ? c.k_head : c.v_head) + slot * (w == 0 ? c.k_slot : c.v_slot);
            if (c.kind == RANS_KV_MXFP4) {
                const uint32_t code = quantise8(x, byte);
                if (p >= 0) {
                    const int n = part / 4, q = part % 4;
                    *reinterpret_cast<uint32_t*>(base + at + q * per_row + n * 4) = code;
                    if (q == 0) (w == 0 ? c.k_scale : c.v_scale)[(((int64_t)p * c.kv_heads + h) * c.page + slot) * (c.dim / 32) + n] = (uint8_t)byte;
                }
            } else if (p >= 0) {
                *reinterpret_cast<uint4*>(base + at + part * 16) = pack8(x, c.kind);
            }
        }
        if (p >= 0 && part == 0) {
            const int64_t at = ((int64_t)p * c.kv_heads + h) * c.page + slot;
            if (c.position != nullptr) c.position[at] = c.seen[b] + number;
            if (c.weight != nullptr) c.weight[at] = 0.0f;
        }
    }
    // The last block to get here (all have read the lengths by then) moves them on.
    __shared__ bool last;
    __syncthreads();
    int* counter = static_cast<int*>(c.workspace);
    if (threadIdx.x == 0) {
        __threadfence();
        last = atomicAdd(counter, 1) == (int)gridDim.x - 1;
        if (last) *counter = 0;
    }
    __syncthreads();
    if (last)
        for (int b = threadIdx.x; b < c.batch; b += kThreads) {
            const int n = rows_of(a, b);
            c.length[b] = (int)min((int64_t)checked_length(c, b) + n, (int64_t)c.table_cols * c.page);
            c.seen[b] += n;
        }
}

__global__ void __launch_bounds__(kThreads) read_kernel(const __grid_constant__ RowArgs a) {
    const RansKvCache& c = a.c;
    const int per_row = c.dim / 8;
    const int64_t all = (int64_t)a.tokens * c.kv_heads * per_row;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < all; i += (int64_t)gridDim.x * kThreads) {
        const int part = (int)(i % per_row);
        const int64_t row = i / per_row;
        const int h = (int)(row % c.kv_heads), token = (int)(row / c.kv_heads);
        int number = 0, p = -1, slot = 0;
        const int b = sequence_of(a, token, number);
        if (b < 0) {
            raise(c, RANS_KV_BAD_STARTS);
        } else {
            const int place = checked_length(c, b) - rows_of(a, b) + number;
            if (place < 0) {
                raise(c, RANS_KV_BAD_STARTS);
            } else {
                p = checked_page(c, b, place / c.page);
                slot = place % c.page;
            }
        }
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const char* base = static_cast<const char*>(w == 0 ? c.k : c.v);
            const int64_t at = (int64_t)p * (w == 0 ? c.k_page : c.v_page) + h * (w == 0 ? c.k_head : c.v_head) + slot * (w == 0 ? c.k_slot : c.v_slot);
            uint4 out = make_uint4(0, 0, 0, 0);
            if (p >= 0) {
                if (c.kind == RANS_KV_MXFP4) {
                    const int n = part / 4, q = part % 4;
                    const uint32_t code = *reinterpret_cast<const uint32_t*>(base + at + q * per_row + n * 4);
                    const uint32_t byte = (w == 0 ? c.k_scale : c.v_scale)[(((int64_t)p * c.kv_heads + h) * c.page + slot) * (c.dim / 32) + n];
                    const float f = byte == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23);
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const __half2_raw r = __nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)((code >> (8 * e)) & 255), __NV_E2M1);
                        const float2 y = __half22float2(__half2(r));
                        x[2 * e] = y.x * f;
                        x[2 * e + 1] = y.y * f;
                    }
                    out = pack8(x, RANS_KV_BF16);
                } else {
                    out = *reinterpret_cast<const uint4*>(base + at + part * 16);
                }
            }
            (w == 0 ? a.k_out : a.v_out)[i] = out;
        }
    }
}

// ------------------------------------------------------------------ evict
// Per (sequence, kv head): find the key T of the budget-th heaviest token by
// radix selection over 32-bit keys, mark what stays, and list the moves
// (i-th kept place >= budget -> i-th freed place < budget).  A second kernel
// copies the listed rows: sources lie at or above the budget and destinations
// below it, so moves never meet.

constexpr int kSelect = 1024;
constexpr int kSelectWarps = kSelect / 32;

struct EvictArgs {
    RansKvCache c;
    int budget, recent;
    int* moves;                  // [batch * kv_heads]: number of moves
    int2* list;                  // [batch * kv_heads][budget]: (to, from)
    uint32_t* keys;              // [batch * kv_heads][table_cols * page]
};

// Order-preserving key of a weight; the newest tokens come first, then NaN.
__device__ __forceinline__ uint32_t key_of(float w, bool late) {
    if (late) return 0xffffffffu;
    if (w != w) return 0xfffffffeu;
    const uint32_t u = __float_as_uint(w + 0.0f);          // -0 -> +0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kSelect) select_kernel(const __grid_constant__ EvictArgs a) {
    const RansKvCache& c = a.c;
    const int h = blockIdx.x % c.kv_heads, b = blockIdx.x / c.kv_heads;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    __shared__ int hist[256];
    __shared__ int digit_s, rank_s;
    __shared__ int wsum[kSelectWarps + 1], wsum2[kSelectWarps + 1];
    const int n = checked_length(c, b), k = a.budget;
    if (n <= k) {
        if (tid == 0) a.moves[blockIdx.x] = 0;
        return;
    }
    uint32_t* keys = a.keys + (int64_t)blockIdx.x * c.table_cols * c.page;
    const int first_late = c.seen[b] - a.recent;
    for (int t = tid; t < n; t += kSelect) {
        const int p = checked_page(c, b, t / c.page);
        uint32_t key = 0;
        if (p >= 0) {
            const int64_t at = ((int64_t)p * c.kv_heads + h) * c.page + t % c.page;
            key = key_of(c.weight[at], c.position[at] >= first_late);
        }
        keys[t] = key;
    }
    __syncthreads();
    uint32_t prefix = 0;
    int rank = k;                                          // of the threshold among the keys that share the prefix
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += kSelect) hist[i] = 0;
        __syncthreads();
        const uint32_t mask = shift == 24 ? 0u : ~0u << (shift + 8);
        for (int t = tid; t < n; t += kSelect) {
            const uint32_t key = keys[t];
            if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1);
        }
        __syncthreads();
        if (warp == 0) {
            // lane l: digits 255 - 8 l downwards
            int own = 0;
            for (int i = 0; i < 8; ++i) own += hist[255 - 8 * lane - i];
            int inc = own;
#pragma unroll
            for (int i = 1; i < 32; i *= 2) {
                const int y = __shfl_up_sync(~0u, inc, i);
                if (lane >= i) inc += y;
            }
            int before = inc - own;
            if (before < rank && rank <= inc)
                for (int i = 0; i < 8; ++i) {
                    const int d = 255 - 8 * lane - i;
                    if (rank <= before + hist[d]) { digit_s = d; rank_s = rank - before; break; }
                    before += hist[d];
                }
        }
        __syncthreads();
        prefix |= (uint32_t)digit_s << shift;
        rank = rank_s;
    }
    // Keys above `prefix` stay, and the first `rank` that equal it.  Each warp has a run of places.
    const int words = (n + 31) / 32, w0 = (int)((int64_t)words * warp / kSelectWarps), w1 = (int)((int64_t)words * (warp + 1) / kSelectWarps);
    int ties = 0;
    for (int w = w0; w < w1; ++w) {
        const int t = w * 32 + lane;
        ties += __popc(__ballot_sync(~0u, t < n && keys[t] == prefix));
    }
    if (lane == 0) wsum[warp] = ties;
    __syncthreads();
    int tie0 = 0;
    for (int w = 0; w < warp; ++w) tie0 += wsum[w];
    __syncthreads();
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
    if (lane == 0) { wsum[warp] = holes; wsum2[warp] = movers; }
    __syncthreads();
    int hole = 0, mover = 0;
    for (int w = 0; w < warp; ++w) { hole += wsum[w]; mover += wsum2[w]; }
    int2* list = a.list + (int64_t)blockIdx.x * a.budget;
    tie = tie0;
    for (int w = w0; w < w1; ++w) {
        const int t = w * 32 + lane;
        const bool keep = kept(w, tie);
        const unsigned is_hole = __ballot_sync(~0u, t < k && !keep), is_mover = __ballot_sync(~0u, t >= k && keep);
        const unsigned below = (1u << lane) - 1;
        if (is_hole >> lane & 1) list[hole + __popc(is_hole & below)].x = t;
        if (is_mover >> lane & 1) list[mover + __popc(is_mover & below)].y = t;
        hole += __popc(is_hole);
        mover += __popc(is_mover);
    }
    if (tid == kSelect - 1) a.moves[blockIdx.x] = mover;
}

__global__ void __launch_bounds__(kThreads) move_kernel(const __grid_constant__ EvictArgs a) {
    const RansKvCache& c = a.c;
    const int bh = blockIdx.y, h = bh % c.kv_heads, b = bh / c.kv_heads;
    const int count = a.moves[bh];
    const int2* list = a.list + (int64_t)bh * a.budget;
    const int row = c.kind == RANS_KV_MXFP4 ? c.dim / 32 : c.dim / 8;      // 16-byte pieces of a row
    const int64_t all = (int64_t)count * row;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < all; i += (int64_t)gridDim.x * kThreads) {
        const int m = (int)(i / row), part = (int)(i % row);
        const int2 move = list[m];
        const int pt = checked_page(c, b, move.x / c.page), pf = checked_page(c, b, move.y / c.page);
        if (pt < 0 || pf < 0) continue;
        const int st = move.x % c.page, sf = move.y % c.page;
        const char* k = static_cast<const char*>(c.k) + h * c.k_head + part * 16;
        const char* v = static_cast<const char*>(c.v) + h * c.v_head + part * 16;
        const uint4 x = *reinterpret_cast<const uint4*>(k + pf * c.k_page + sf * c.k_slot);
        const uint4 y = *reinterpret_cast<const uint4*>(v + pf * c.v_page + sf * c.v_slot);
        *reinterpret_cast<uint4*>(const_cast<char*>(k) + pt * c.k_page + st * c.k_slot) = x;
        *reinterpret_cast<uint4*>(const_cast<char*>(v) + pt * c.v_page + st * c.v_slot) = y;
        const int64_t to = ((int64_t)pt * c.kv_heads + h) * c.page + st, from = ((int64_t)pf * c.kv_heads + h) * c.page + sf;
        if (c.kind == RANS_KV_MXFP4) {
            c.k_scale[to * row + part] = c.k_scale[from * row + part];     // dim / 32 scale bytes, as many as pieces
            c.v_scale[to * row + part] = c.v_scale[from * row + part];
        }
        if (part == 0) {
            c.weight[to] = c.weight[from];
            c.position[to] = c.position[from];
        }
    }
    if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) c.length[b] = min(checked_length(c, b), a.budget);
}

struct EvictPlan {
    int64_t moves, list, keys, bytes;
};

bool plan_evict(const RansKvCache& c, int budget, EvictPlan& p) {
    if (budget < 1) return false;
    auto up = [](int64_t x) { return (x + 255) & ~(int64_t)255; };
    const int64_t heads = (int64_t)c.batch * c.kv_heads;
    p.moves = counter_bytes(c);
    p.list = p.moves + up(heads * 4);
    p.keys = p.list + up(heads * budget * 8);
    p.bytes = p.keys + up(heads * c.table_cols * c.page * 4);
    return true;
}

int row_grid(const RowArgs& a) {
    const int64_t blocks = ((int64_t)a.tokens * a.c.kv_heads * (a.c.dim / 8) + kThreads - 1) / kThreads;
    return (int)(blocks < kSms * 8 ? blocks : kSms * 8);
}

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
    a.c = *cache;
    fill_strides(a.c);
    a.k_in = static_cast<const char*>(k);
    a.v_in = static_cast<const char*>(v);
    a.k_token = k_token; a.k_head = k_head; a.v_token = v_token; a.v_head = v_head;
    a.starts = starts;
    a.tokens = tokens;
    a.given = given;
    append_kernel<<<row_grid(a), kThreads, 0, stream>>>(a);
    return (int)cudaGetLastError();
}

extern "C" int rans_kv_read(const RansKvCache* cache, void* k_out, void* v_out, const int32_t* starts, int tokens,
                            cudaStream_t stream) {
    const int rc = check_cache(cache);
    if (rc != 0) return rc;
    if (tokens < 0 || (starts == nullptr && tokens != cache->batch)) return -2;
    if (tokens == 0) return 0;
    if (k_out == nullptr || v_out == nullptr || !aligned16(k_out) || !aligned16(v_out)) return -2;
    RowArgs a{};
    a.c = *cache;
    fill_strides(a.c);
    a.k_out = static_cast<uint4*>(k_out);
    a.v_out = static_cast<uint4*>(v_out);
    a.starts = starts;
    a.tokens = tokens;
    read_kernel<<<row_grid(a), kThreads, 0, stream>>>(a);
    return (int)cudaGetLastError();
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
    char* ws = static_cast<char*>(cache->workspace);
    a.budget = budget;
    a.recent = recent;
    a.moves = reinterpret_cast<int*>(ws + p.moves);
    a.list = reinterpret_cast<int2*>(ws + p.list);
    a.keys = reinterpret_cast<uint32_t*>(ws + p.keys);
    const int heads = cache->batch * cache->kv_heads;
    select_kernel<<<heads, kSelect, 0, stream>>>(a);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return (int)e;
    const int chunks = heads >= kSms * 8 ? 1 : (kSms * 8 + heads - 1) / heads;
    move_kernel<<<dim3(chunks, heads), kThreads, 0, stream>>>(a);
    return (int)cudaGetLastError();
}
