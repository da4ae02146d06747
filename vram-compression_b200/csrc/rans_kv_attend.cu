// Attention of one new token per sequence over a paged key-value cache, split
// over the cache's length and joined.
//
// For a kv head and its group of query heads q_0..q_{G-1} the kernel computes,
// over tiles of 16 tokens and with the running maximum m and sum l of a softmax,
//
//     S^T = K Q^T            (tokens x heads)
//     P^T = exp2(S^T c - m)  (c = scale * log2 e; for 16-bit rows the sum of two operands, high and low)
//     O^T = O^T 2^(m_old - m) + V^T P^T   (dim x heads)
//
// Both products take the cache as the 16-row operand of mma.m16n8k16 and the
// heads as its 8 columns, so a group of 8 heads wastes no tensor work and a tile's
// scores lie in four registers.  The work is bound by reading K and V once (4 G
// flops a byte at 16 bits, far below the tensor rate even of this instruction).
//
// Operands go from global memory straight to registers, 16 bytes a lane: the
// order of the contraction index is free, so a lane's 8 consecutive values of a
// key row are its operands of two consecutive k-steps, with Q's words loaded in the
// same order; and a lane that reads the same 8 columns of four value rows gets V^T's
// operands by one byte permute each.
// Nothing is staged, so no warp waits for another while it streams.  4-bit rows are
// staged instead (their loop is bound by instructions and has no registers to spare).
//
// Work is shared out by tiles: the grid's warps get equal runs of the list of all
// (sequence, kv head, tile), whatever the lengths are.  A warp that has a whole
// (sequence, kv head) writes its output; else the block joins its warps' parts in
// shared memory, and the last block to finish a (sequence, kv head) joins the
// blocks' parts (always in the order of the tiles, so results do not depend on
// which block that is).
//
// Measured on one B200, 64 query heads on 8 of size 128: 48 uneven sequences in bf16
// (1.58 GB) 236 us, 6.7 TB/s, the rate of a plain copy; one of 32768 tokens 30 us, of
// which 18 us stream at 7.3 TB/s and the rest is launch, page lookups and joins; one of
// 131071 tokens in 4 bits (143 MB) 48 us, about 425 instructions per 16 tokens, issued
// in 55 % of the cycles; one of 777 tokens on 2 heads 8.7 us.
#include <atomic>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <cuda_runtime.h>

#include "rans_kv_common.h"

namespace rb200kv {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTile = 16;
constexpr int kGrid = kSms;
// A group's first tile waits for its page number and queries, and its end is written out: in the shares of work it
// counts as this many tiles more (places without a tile behind the group's last one).  With 1, 2, 4: 200 sequences of 20
// tokens 17.2, 16.5, 15.6 us; 32 uneven ones in 4 bits 78.7, 77.3, 76.6 (now 79); one long one the same.
constexpr int kStart = 4;
// Probabilities are 2^(score - m) for a reference m that follows the running maximum from a distance: when a score passes
// m + kHigh, m becomes the maximum - kRest, and most tiles leave O alone.  For fp16 operands the largest probability lies
// between 2^11 and 2^15, so that they keep probabilities down to 2^-36 of the largest instead of 2^-25.  bf16 operands need no
// such help, and bf16 values may be as large as fp32 sums: there the largest lies between 2^-4 and 1, and sum and O are held in
// units of 2^-30, so that no sum over the 2^30 tokens that a table may have passes the largest value among them.
template <int KIND>
struct Reference {
    static constexpr bool kBf16 = KIND == RANS_KV_BF16;
    static constexpr float kHigh = kBf16 ? 0.0f : 15.0f, kRest = kBf16 ? -4.0f : 11.0f, kUnits = kBf16 ? 1073741824.0f : 1.0f;
};

// The maximum before there is a score: finite, so that no difference of two of them is NaN, and no finite score is below it.
constexpr float kNothing = -3.402823466e38f;

struct AttendArgs {
    RansKvCache c;
    Divider page;
    const char* q;
    int64_t q_batch, q_head;     // bytes
    void* out;
    float* log_sum;
    float scale_log2;
    int heads, group;            // group = heads / kv_heads
    int subs, sub_heads;         // a group is cut into `subs` parts of at most sub_heads
    int q_half;                  // q and out are fp16 (else bf16)
    int weigh;
    int* counter;                // [batch * kv_heads * subs]
    float2* stats;               // [batch * heads]: maximum (log2) and 1 / sum
    float* part;                 // [grid][2] Attend::Part: what a block has of its first and last group
    float* first;                // 4 bits: [grid][warps] Attend::Part
    float* scores;               // [tile][16][HP], scaled, log2
    int score_tiles;
};

// (Not the path for data that is constant while the kernel lives: the kernel before may still write rows when this one starts.
// volatile: stays behind wait_for_previous().)
__device__ __forceinline__ uint4 load16(const void* p) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
    return r;
}

// 16 bytes into shared memory, the first `size` of them from global memory, the rest zero.
__device__ __forceinline__ void copy16(void* to, const void* from, int size) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                 :: "r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "r"(size) : "memory");
}
__device__ __forceinline__ void copy16(void* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory"); }

template <bool HALF>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    if constexpr (HALF)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <bool HALF>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (HALF) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}

template <bool HALF>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
    return HALF ? __half22float2(*reinterpret_cast<const __half2*>(&w)) : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}

__device__ __forceinline__ uint32_t pack_as(int half, float lo, float hi) {
    return half ? pack2<true>(lo, hi) : pack2<false>(lo, hi);
}

// The e2m1 codes of a word's four bytes as four fp16 pairs (low half, high half of the byte), exact.
__device__ __forceinline__ void e2m1_to_half(uint32_t (&r)[4], uint32_t w) {
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(w));
}

__device__ __forceinline__ uint32_t multiply2(uint32_t x, uint32_t f) {
    const __half2 z = __hmul2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&f));
    return *reinterpret_cast<const uint32_t*>(&z);
}

// (1 + 2^-23) 2^e of byte k of a word, a scale byte e + 127, or NaN for 255: the lowest bit of the fraction, set in all, makes
// a NaN of what would be infinity (the mask takes it along; a comparison would be two instructions more for each scale).  kOne
// takes the factor out again.
__device__ __forceinline__ float scale_of(uint32_t w, int k) {
    return __uint_as_float(((k < 3 ? w << (23 - 8 * k) : w >> 1) & 0x7f800000u) | 1u);
}
constexpr float kOne = 1.0f - 1.1920928955078125e-7f;

// 2^e for -126 <= e <= 127.
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

__device__ __forceinline__ float join_factor(float m, float top) { return m == -INFINITY ? 0.0f : exp2_fast(m - top); }

template <int KIND, int D, int NT>
struct Attend {
    static constexpr bool kFp4 = KIND == RANS_KV_MXFP4;
    static constexpr float kHigh = Reference<KIND>::kHigh, kRest = Reference<KIND>::kRest, kUnits = Reference<KIND>::kUnits;
    static constexpr int HP = NT * 8;                         // heads of a tile, padded
    static constexpr int kChunks = D / 32;                    // 32 values of a row
    // One block of an SM's whole register file: fewer parts to join than from several blocks.  As many warps as the registers
    // for rows, O and statistics allow: nothing is spilled but 4 to 24 bytes a thread where 16 heads of 64 or 4-bit rows are
    // worked on, 40 for 4-bit rows in groups of 9 to 16 heads of 128.  4-bit rows are not held in registers (12 against 8
    // warps: 16 x 8000 tokens of 8 heads in 4 bits, groups of 12 heads of 128: 79 -> 68 us, of 8 heads of 256: 93 -> 83, now 85).
    static constexpr bool kLarge = (NT == 2 && D == 128) || D == 256;
    static constexpr int kWarps = kLarge ? (kFp4 ? 12 : 8) : D == 128 && !kFp4 ? 12 : 16;
    static constexpr int kRow = D + 4;                        // a head's part in shared memory

    // What is left of a run of tiles of one group: O, and the running maximum and sum of each head; a warp's in shared
    // memory, a block's in the workspace.
    struct alignas(16) Part {
        float o[HP][kRow];
        float2 ml[HP];
    };

    // 4-bit tiles as they lie in the pages, copied ahead of their use; kSub of them are worked on at a time, as many as the
    // registers allow (the loop then turns less often, and several chains of instructions run side by side: with 1 and
    // these, 16 x 8000 tokens of 8 heads, groups of 12 heads of 128 67 -> 64 us, now 65, of 16 of 64 45 -> 42, of 8 of 64 38 -> 33).
    static constexpr int kSub = !kFp4 || D == 256 ? 1 : NT == 1 && D == 64 ? 4 : 2;
    static constexpr int kStages = kSub > 1 ? 2 : 3;
    struct alignas(16) Stage {
        uint8_t k[kTile * D / 2], v[kTile * D / 2], ks[kTile * kChunks], vs[kTile * kChunks];
    };
    // A warp's second part is written when its last tile is done, in the place of its stages.  A first part, which only a
    // warp at a group's end has, goes to shared memory, or for 4 bits, whose stages leave no room, to the workspace.
    union Late {
        Part part;
        Stage stage[kFp4 ? kStages : 1][kSub];
    };

    struct Smem {
        Part part[kFp4 ? 1 : kWarps];        // the warps' first parts
        Late late[kWarps];                   // their second ones
        uint4 q[kWarps][NT * kChunks * 32];  // the queries that they work on
        int tag[kWarps * 2];                 // the group of each part
        int first_block[2], last_block[2], last[2];      // of the block's first and last group, if it has only some of it
        int warp_sum[kWarps];
        int pre[RANS_KV_MAX_BATCH + 1];      // places of one head in front of each sequence
    };

    // One tile's rows in registers, 16 bits a value ..
    struct RawK {
        uint4 k[2][kChunks];                                  // rows g, g + 8
    };
    struct RawV {
        uint4 v[4][D / 64];
    };
    // .. or 4: words of 8 codes, and scale bytes
    struct CodeK {
        uint32_t w[2][kChunks], s[2][(D + 127) / 128];        // word n = block n
    };
    struct CodeV {
        uint32_t w[4][D / 64], s[4];
    };

    // A lane's place in the tiles of one (sequence, kv head).  Within a page it steps by 16 rows; the number of the following
    // page is fetched a page ahead.
    struct Cursor {
        const char *k, *v;                       // 16 bits: the lane's first key and value row of the tile
        int64_t row;                             // 4 bits: the tile's first row
        int slot, ahead, next, left, valid;      // left: tokens from the tile's first one on; valid: of them in the tile

        __device__ __forceinline__ void at_page(const RansKvCache& c, int h, int p, int lane) {
            const int g = lane >> 2, q4 = lane & 3;
            const bool ok = p >= 0 && p < c.pages;
            if (!ok) raise(c, RANS_KV_BAD_PAGE);
            valid = ok ? min(left, kTile) : 0;
            const int64_t pg = ok ? p : 0;
            if constexpr (kFp4) {
                row = (pg * c.kv_heads + h) * c.page + slot;
            } else {
                k = static_cast<const char*>(c.k) + pg * c.k_page + h * c.k_head + (slot + g) * c.k_slot + q4 * 16;
                v = static_cast<const char*>(c.v) + pg * c.v_page + h * c.v_head + (slot + 2 * q4) * c.v_slot + g * 16;
            }
        }
        __device__ __forceinline__ void fetch_next(const RansKvCache& c, int b) {
            ++ahead;
            // only a page that holds tokens is looked up (n <= table_cols * page, so `ahead` is then inside the table)
            next = left > c.page - slot ? c.table[(int64_t)b * c.table_cols + ahead] : -1;
        }
        __device__ __forceinline__ void begin(const RansKvCache& c, const Divider& page, int b, int h, int n, int tile, int lane) {
            const int t0 = tile * kTile;
            ahead = page(t0);
            slot = t0 - ahead * c.page;
            left = n - t0;
            at_page(c, h, c.table[(int64_t)b * c.table_cols + ahead], lane);
            fetch_next(c, b);
        }
        __device__ __forceinline__ void advance(const RansKvCache& c, int b, int h, int lane) {
            left -= kTile;
            slot += kTile;
            if (slot == c.page) {
                slot = 0;
                at_page(c, h, next, lane);
                fetch_next(c, b);
                return;
            }
            if (valid > 0) valid = min(left, kTile);
            if constexpr (kFp4) {
                row += kTile;
            } else {
                k += kTile * c.k_slot;
                v += kTile * c.v_slot;
            }
        }
    };

    template <bool FULL>
    static __device__ __forceinline__ void load_k(RawK& r, const RansKvCache& c, const char* k, int valid, int lane) {
        const int g = lane >> 2;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const bool in = FULL || g + 8 * i < valid;
            const char* p = k + 8 * i * c.k_slot;
#pragma unroll
            for (int j = 0; j < kChunks; ++j) r.k[i][j] = in ? load16(p + j * 64) : make_uint4(0, 0, 0, 0);
        }
    }
    template <bool FULL>
    static __device__ __forceinline__ void load_v(RawV& r, const RansKvCache& c, const char* v, int valid, int lane) {
        const int q4 = lane & 3;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = (i & 1) + 8 * (i >> 1);
            const bool in = FULL || 2 * q4 + row < valid;
            const char* p = v + row * c.v_slot;
#pragma unroll
            for (int j = 0; j < D / 64; ++j) r.v[i][j] = in ? load16(p + j * 128) : make_uint4(0, 0, 0, 0);
        }
    }
    static __device__ __forceinline__ void load_k(RawK& r, const RansKvCache& c, const Cursor& u, int lane) {
        if (u.valid == kTile) load_k<true>(r, c, u.k, u.valid, lane); else load_k<false>(r, c, u.k, u.valid, lane);
    }
    static __device__ __forceinline__ void load_v(RawV& r, const RansKvCache& c, const Cursor& u, int lane) {
        if (u.valid == kTile) load_v<true>(r, c, u.v, u.valid, lane); else load_v<false>(r, c, u.v, u.valid, lane);
    }

    // Starts a 4-bit tile's copy into shared memory, 16 bytes a lane; what lies behind its last token becomes zero.
    static __device__ __forceinline__ void copy_tile(Stage& st, const RansKvCache& c, const Cursor& u, int lane) {
        constexpr int kScaleLanes = kTile * kChunks / 16;        // of the keys; as many lanes copy the values' scales
        const int at = lane * 16;
        const bool is_k = lane < kScaleLanes;
        const int from = at - (is_k ? 0 : kTile * kChunks);
        const uint8_t* k = static_cast<const uint8_t*>(c.k) + u.row * (D / 2) + at;
        const uint8_t* v = static_cast<const uint8_t*>(c.v) + u.row * (D / 2) + at;
        const uint8_t* s = (is_k ? c.k_scale : c.v_scale) + u.row * kChunks + from;
        if (u.valid == kTile) {
#pragma unroll
            for (int i = 0; i < kTile * D / 2; i += 512) {
                copy16(st.k + at + i, k + i);
                copy16(st.v + at + i, v + i);
            }
            if (lane < 2 * kScaleLanes) copy16(st.ks + at, s);
        } else {
#pragma unroll
            for (int i = 0; i < kTile * D / 2; i += 512) {
                const int size = min(max(u.valid * (D / 2) - at - i, 0), 16);
                copy16(st.k + at + i, k + i, size);
                copy16(st.v + at + i, v + i, size);
            }
            if (lane < 2 * kScaleLanes) copy16(st.ks + at, s, min(max(u.valid * kChunks - from, 0), 16));
        }
    }

    static __device__ __forceinline__ void read_k(CodeK& r, const Stage& st, int lane) {
        const int g = lane >> 2, q4 = lane & 3;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = g + 8 * i;
            const uint8_t* p = st.k + row * (D / 2) + q4 * (D / 8);
            if constexpr (D == 64) {
                const uint2 w = *reinterpret_cast<const uint2*>(p);
                r.w[i][0] = w.x; r.w[i][1] = w.y;
                r.s[i][0] = *reinterpret_cast<const uint16_t*>(st.ks + row * kChunks);
            } else {
#pragma unroll
                for (int j = 0; j < kChunks; j += 4) {
                    const uint4 w = *reinterpret_cast<const uint4*>(p + j * 4);
                    r.w[i][j] = w.x; r.w[i][j + 1] = w.y; r.w[i][j + 2] = w.z; r.w[i][j + 3] = w.w;
                    r.s[i][j / 4] = *reinterpret_cast<const uint32_t*>(st.ks + row * kChunks + j);
                }
            }
        }
    }
    static __device__ __forceinline__ void read_v(CodeV& r, const Stage& st, int lane) {
        const int g = lane >> 2, q4 = lane & 3;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = 2 * q4 + (i & 1) + 8 * (i >> 1);
            const uint8_t* p = st.v + row * (D / 2) + g * (D / 16);
            const uint8_t* s = st.vs + row * kChunks + (g & 1) * (D / 64);
            if constexpr (D == 256) {
                const uint4 w = *reinterpret_cast<const uint4*>(p);
                r.w[i][0] = w.x; r.w[i][1] = w.y; r.w[i][2] = w.z; r.w[i][3] = w.w;
                r.s[i] = *reinterpret_cast<const uint32_t*>(s);
            } else if constexpr (D == 128) {
                const uint2 w = *reinterpret_cast<const uint2*>(p);
                r.w[i][0] = w.x; r.w[i][1] = w.y;
                r.s[i] = *reinterpret_cast<const uint16_t*>(s);
            } else {
                r.w[i][0] = *reinterpret_cast<const uint32_t*>(p);
                r.s[i] = *s;
            }
        }
    }

    struct State {
        float o[D / 16][NT][4];
        float m[NT][2], l[NT][2];
        float qs[kFp4 ? NT : 1][2];      // 4-bit: the powers of two taken out of the two heads' queries, times scale
        // 4-bit: O of the lane's D / 64 words is held in units of 2^(unit - 127), a power near the words' scales, so that
        // the values' operands fit fp16 (exactly: they have two significant bits).
        int unit[kFp4 ? D / 64 : 1];
    };

    // The queries of a head group, in the order of load_k()'s values, to the warp's place in shared memory
    // ([NT][kChunks][32 lanes]; 16 registers less than keeping them, for four wide reads a tile).  For 4-bit
    // keys they become fp16: each head's largest value is first brought to [2^14, 2^15) by a power of two, so that nothing
    // overflows and what is lost is below 2^-38 of it.
    static __device__ __forceinline__ void begin(State& s, uint4* qs, const AttendArgs& a, int b, int head0, int heads, int lane) {
        const int g = lane >> 2, q4 = lane & 3;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const bool in = t * 8 + g < heads;
            const char* qp = a.q + b * a.q_batch + (int64_t)(head0 + t * 8 + g) * a.q_head + q4 * 16;
            float top = 0.0f;
            uint4 q[kChunks];
#pragma unroll
            for (int j = 0; j < kChunks; ++j) q[j] = in ? load16(qp + j * 64) : make_uint4(0, 0, 0, 0);
            if constexpr (kFp4) {
                auto unpack = [&](uint32_t w) {
                    return a.q_half ? __half22float2(*reinterpret_cast<__half2*>(&w))
                                    : __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&w));
                };
#pragma unroll
                for (int j = 0; j < kChunks; ++j)
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const float2 f = unpack((&q[j].x)[w]);
                        top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
                    }
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
                const int e = top > 0.0f && top <= 3.4e38f ? min(max((int)(__float_as_uint(top) >> 23) - 127 - 14, -100), 113) : 0;
                const float down = __uint_as_float((uint32_t)(127 - e) << 23), up = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
                for (int j = 0; j < kChunks; ++j)
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const float2 f = unpack((&q[j].x)[w]);
                        (&q[j].x)[w] = pack2<true>(f.x * down, f.y * down);
                    }
                // a lane's scores are of heads 2 q4 and 2 q4 + 1
                s.qs[t][0] = __shfl_sync(~0u, up, (2 * q4) * 4) * (a.scale_log2 * kOne);
                s.qs[t][1] = __shfl_sync(~0u, up, (2 * q4 + 1) * 4) * (a.scale_log2 * kOne);
            }
#pragma unroll
            for (int j = 0; j < kChunks; ++j) qs[(t * kChunks + j) * 32 + lane] = q[j];
            s.m[t][0] = s.m[t][1] = kNothing;
            if constexpr (kFp4) {
#pragma unroll
                for (int j = 0; j < D / 64; ++j) s.unit[j] = 0;
            }
            s.l[t][0] = s.l[t][1] = 0.0f;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) s.o[i][t][0] = s.o[i][t][1] = s.o[i][t][2] = s.o[i][t][3] = 0.0f;
        }
        __syncwarp();
    }

    // S^T of a tile, scaled to powers of two.
    static __device__ __forceinline__ void scores(const State& s, const uint4* qs, const RawK& r, const AttendArgs& a,
                                                  float (&sc)[NT][4], int lane) {
#pragma unroll
        for (int t = 0; t < NT; ++t) sc[t][0] = sc[t][1] = sc[t][2] = sc[t][3] = 0.0f;
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            const uint4 k0 = r.k[0][j], k1 = r.k[1][j];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const uint4 q = qs[(t * kChunks + j) * 32 + lane];
                mma<KIND == RANS_KV_FP16>(sc[t], k0.x, k1.x, k0.y, k1.y, q.x, q.y);
                mma<KIND == RANS_KV_FP16>(sc[t], k0.z, k1.z, k0.w, k1.w, q.z, q.w);
            }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[t][i] *= a.scale_log2;
    }
    static __device__ __forceinline__ void scores(const State& s, const uint4* qs, const CodeK& r, const AttendArgs& a,
                                                  float (&sc)[NT][4], int lane) {
#pragma unroll
        for (int t = 0; t < NT; ++t) sc[t][0] = sc[t][1] = sc[t][2] = sc[t][3] = 0.0f;
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            uint32_t w0[4], w1[4];
            e2m1_to_half(w0, r.w[0][j]);
            e2m1_to_half(w1, r.w[1][j]);
            const float f0 = scale_of(r.s[0][j / 4], j % 4);
            const float f1 = scale_of(r.s[1][j / 4], j % 4);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                const uint4 q = qs[(t * kChunks + j) * 32 + lane];
                mma<true>(d, w0[0], w1[0], w0[1], w1[1], q.x, q.y);
                mma<true>(d, w0[2], w1[2], w0[3], w1[3], q.z, q.w);
                sc[t][0] = fmaf(d[0], f0, sc[t][0]);
                sc[t][1] = fmaf(d[1], f0, sc[t][1]);
                sc[t][2] = fmaf(d[2], f1, sc[t][2]);
                sc[t][3] = fmaf(d[3], f1, sc[t][3]);
            }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            sc[t][0] *= s.qs[t][0]; sc[t][1] *= s.qs[t][1];
            sc[t][2] *= s.qs[t][0]; sc[t][3] *= s.qs[t][1];
        }
    }

    // The softmax's part of SUB tiles with `valid` tokens each: scores become probabilities, the maximum, the sum and O follow.
    template <int SUB>
    static __device__ __forceinline__ void probabilities(State& s, float (&sc)[SUB][NT][4], const AttendArgs& a, int x,
                                                         const int (&valid)[SUB], int lane) {
        const int q4 = lane & 3, row = lane >> 2;
        bool raise_max = false;
#pragma unroll
        for (int i = 0; i < SUB; ++i)
            if (valid[i] < kTile) {
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    if (row >= valid[i]) sc[i][t][0] = sc[i][t][1] = -INFINITY;
                    if (row + 8 >= valid[i]) sc[i][t][2] = sc[i][t][3] = -INFINITY;
                }
            }
        if (a.weigh) {
#pragma unroll
            for (int i = 0; i < SUB; ++i) {
                if (valid[i] == 0 || x + i >= a.score_tiles) continue;
                float* p = a.scores + ((int64_t)(x + i) * kTile + row) * HP + 2 * q4;
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    *reinterpret_cast<float2*>(p + t * 8) = make_float2(sc[i][t][0], sc[i][t][1]);
                    *reinterpret_cast<float2*>(p + t * 8 + 8 * HP) = make_float2(sc[i][t][2], sc[i][t][3]);
                }
            }
        }
        float top[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                top[t][e] = fmaxf(sc[0][t][e], sc[0][t][e + 2]);
#pragma unroll
                for (int i = 1; i < SUB; ++i) top[t][e] = fmaxf(top[t][e], fmaxf(sc[i][t][e], sc[i][t][e + 2]));
                raise_max |= top[t][e] > s.m[t][e] + kHigh;
            }
        if (__any_sync(~0u, raise_max)) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float m = top[t][e];
                    m = fmaxf(m, __shfl_xor_sync(~0u, m, 4));
                    m = fmaxf(m, __shfl_xor_sync(~0u, m, 8));
                    m = fmaxf(m, __shfl_xor_sync(~0u, m, 16));
                    m = fmaxf(m - kRest, s.m[t][e]);
                    const float f = exp2_fast(s.m[t][e] - m);
                    s.m[t][e] = m;
                    s.l[t][e] *= f;
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        s.o[i][t][e] *= f;
                        s.o[i][t][e + 2] *= f;
                    }
                }
        }
#pragma unroll
        for (int i = 0; i < SUB; ++i)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[i][t][e] = exp2_fast(sc[i][t][e] - s.m[t][e & 1]) * (1.0f / kUnits);
                s.l[t][0] += sc[i][t][0] + sc[i][t][2];
                s.l[t][1] += sc[i][t][1] + sc[i][t][3];
            }
    }

    // P^T's operands from a tile's probabilities, rounded once.  For 4-bit values: to 2^-11, where the values themselves have
    // two bits, outputs are mostly bf16 (2^-8), and the loop is short of instructions.
    template <bool HALF>
    static __device__ __forceinline__ void pack_probabilities(uint32_t (&pb)[NT][2], const float (&p)[NT][4]) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            pb[t][0] = transpose8x8(pack2<HALF>(p[t][0], p[t][1]));
            pb[t][1] = transpose8x8(pack2<HALF>(p[t][2], p[t][3]));
        }
    }

    // The same as sums of two operands, p to 2^-16 (bf16) or 2^-22 (fp16) of itself: the output's own rounding is then the
    // only one that shows.  (One bf16 operand alone adds a quarter to the error's root mean square.)
    template <bool HALF>
    static __device__ __forceinline__ void split_probabilities(uint32_t (&high)[NT][2], uint32_t (&low)[NT][2], const float (&p)[NT][4]) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t w = pack2<HALF>(p[t][2 * i], p[t][2 * i + 1]);
                const float2 f = unpack2<HALF>(w);
                high[t][i] = transpose8x8(w);
                low[t][i] = transpose8x8(pack2<HALF>(p[t][2 * i] - f.x, p[t][2 * i + 1] - f.y));
            }
    }

    // O^T += V^T P^T.
    static __device__ __forceinline__ void accumulate(State& s, const RawV& r, const float (&p)[NT][4]) {
        uint32_t high[NT][2], low[NT][2];
        split_probabilities<KIND == RANS_KV_FP16>(high, low, p);
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
            const uint32_t* v0 = &r.v[0][j].x;
            const uint32_t* v1 = &r.v[1][j].x;
            const uint32_t* v2 = &r.v[2][j].x;
            const uint32_t* v3 = &r.v[3][j].x;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t a0 = __byte_perm(v0[i], v1[i], 0x5410), a1 = __byte_perm(v0[i], v1[i], 0x7632);
                const uint32_t a2 = __byte_perm(v2[i], v3[i], 0x5410), a3 = __byte_perm(v2[i], v3[i], 0x7632);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    mma<KIND == RANS_KV_FP16>(s.o[j * 4 + i][t], a0, a1, a2, a3, high[t][0], high[t][1]);
                    mma<KIND == RANS_KV_FP16>(s.o[j * 4 + i][t], a0, a1, a2, a3, low[t][0], low[t][1]);
                }
            }
        }
    }

    // fp16 factors 2^(scale byte - unit) of a lane's words, for bytes from unit - 7 to unit + 8; nonzero bits under 0xfff0fff0
    // where some are outside.
    static __device__ __forceinline__ uint32_t factors(uint32_t (&f)[D / 64][2], const State& s, const CodeV& r) {
        uint32_t outside = 0;
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
            const uint32_t low = (uint32_t)(s.unit[j] - 7) * 0x10001u;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                // the two tokens' scale bytes, one in each half (byte 3 is zero where a lane has fewer than four)
                const uint32_t u = D == 256 ? __byte_perm(r.s[2 * k], r.s[2 * k + 1], j | (j << 4) | ((4 + j) << 8) | ((4 + j) << 12)) & 0x00ff00ffu
                                            : __byte_perm(r.s[2 * k], r.s[2 * k + 1], j | (3 << 4) | ((4 + j) << 8) | (7 << 12));
                const uint32_t in = u - low;
                outside |= in;
                f[j][k] = in * 1024u + 0x20002000u;
            }
        }
        return outside;
    }

    // Rows behind a tile's last token hold zeros, their scale bytes too: these become the units, so that a group's last tile
    // is like any other.
    static __device__ __forceinline__ void fill_scales(CodeV& r, const State& s, int valid, int q4) {
        uint32_t units = 0;
#pragma unroll
        for (int j = 0; j < D / 64; ++j) units |= (uint32_t)s.unit[j] << (8 * j);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (2 * q4 + (i & 1) + 8 * (i >> 1) >= valid) r.s[i] = units;
    }

    // O^T += V^T P^T over the first `count` of kSub tiles.
    static __device__ __forceinline__ void accumulate(State& s, CodeV (&r)[kSub], const float (&p)[kSub][NT][4],
                                                      const int (&valid)[kSub], int count, int lane) {
        uint32_t f[kSub][D / 64][2];
        auto wide = [&]() {
#pragma unroll
            for (int i = 0; i < kSub; ++i)
                if (valid[i] < kTile) fill_scales(r[i], s, valid[i], lane & 3);
            uint32_t outside = factors(f[0], s, r[0]);
#pragma unroll
            for (int i = 1; i < kSub; ++i) {
                const uint32_t more = factors(f[i], s, r[i]);
                if (i < count) outside |= more;
            }
            return __any_sync(~0u, (outside & 0xfff0fff0u) != 0);
        };
        bool any_wide = wide();
        if (any_wide) {
#pragma unroll
            for (int i = 0; i < kSub; ++i)
                if (i < count) raise_unit(s, r[i]);
            any_wide = wide();
        }
        if (any_wide) {
#pragma unroll
            for (int i = 0; i < kSub; ++i)
                if (i < count) accumulate_wide(s, r[i], p[i]);
            return;
        }
#pragma unroll
        for (int i = 0; i < kSub; ++i) {
            if (i >= count) break;
            uint32_t pb[NT][2];
            pack_probabilities<true>(pb, p[i]);
#pragma unroll
            for (int j = 0; j < D / 64; ++j) {
                // two tokens' codes of one column next to each other: columns 0, 2, 4, 6 and 1, 3, 5, 7
                const uint32_t even0 = (r[i].w[0][j] & 0x0f0f0f0fu) | ((r[i].w[1][j] << 4) & 0xf0f0f0f0u);
                const uint32_t odd0 = ((r[i].w[0][j] >> 4) & 0x0f0f0f0fu) | (r[i].w[1][j] & 0xf0f0f0f0u);
                const uint32_t even1 = (r[i].w[2][j] & 0x0f0f0f0fu) | ((r[i].w[3][j] << 4) & 0xf0f0f0f0u);
                const uint32_t odd1 = ((r[i].w[2][j] >> 4) & 0x0f0f0f0fu) | (r[i].w[3][j] & 0xf0f0f0f0u);
                uint32_t e0[4], o0[4], e1[4], o1[4];
                e2m1_to_half(e0, even0);
                e2m1_to_half(o0, odd0);
                e2m1_to_half(e1, even1);
                e2m1_to_half(o1, odd1);
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const uint32_t a0 = multiply2(e0[d], f[i][j][0]), a1 = multiply2(o0[d], f[i][j][0]);
                    const uint32_t a2 = multiply2(e1[d], f[i][j][1]), a3 = multiply2(o1[d], f[i][j][1]);
#pragma unroll
                    for (int t = 0; t < NT; ++t) mma<true>(s.o[j * 4 + d][t], a0, a1, a2, a3, pb[t][0], pb[t][1]);
                }
            }
        }
    }

    // 4-bit: a new unit for words whose scales are above what the present one takes, from their largest scale.
    static __device__ __forceinline__ void raise_unit(State& s, const CodeV& r) {
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
            int top = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int byte = (int)((r.s[i] >> (8 * j)) & 255);
                top = byte == 255 ? top : max(top, byte);
            }
            top = max(top, __shfl_xor_sync(~0u, top, 1));        // over the tile's tokens, of one lane group's words
            top = max(top, __shfl_xor_sync(~0u, top, 2));
            if (top <= (s.unit[j] == 0 ? 0 : s.unit[j] + 8)) continue;
            const float down = s.unit[j] - top < -126 ? 0.0f : power_of_two(s.unit[j] - top);
            s.unit[j] = top;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s.o[j * 4 + i][t][e] *= down;
        }
    }

    // 4-bit: a tile whose scales are too far apart for fp16 (or that has a block of NaN): bf16 operands, any scale.
    static __device__ __forceinline__ void accumulate_wide(State& s, const CodeV& r, const float (&p)[NT][4]) {
        uint32_t high[NT][2], low[NT][2];
        split_probabilities<false>(high, low, p);
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
            float f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int byte = (int)((r.s[i] >> (8 * j)) & 255);
                f[i] = byte == 255 ? __uint_as_float(0x7fc00000u) : power_of_two(max(byte - s.unit[j], -126));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                auto value = [&](int token, int d) {
                    const uint32_t code = (r.w[token][j] >> (4 * d)) & 15, n = code & 7;
                    // 2^(n / 2 - 1) (1 + n % 2 / 2), or 0 and 0.5
                    const float v = n < 2 ? 0.5f * (float)n : power_of_two((int)(n >> 1) - 1) * (n & 1 ? 1.5f : 1.0f);
                    return (code & 8 ? -v : v) * f[token];
                };
                const uint32_t a0 = pack2<false>(value(0, 2 * i), value(1, 2 * i)), a1 = pack2<false>(value(0, 2 * i + 1), value(1, 2 * i + 1));
                const uint32_t a2 = pack2<false>(value(2, 2 * i), value(3, 2 * i)), a3 = pack2<false>(value(2, 2 * i + 1), value(3, 2 * i + 1));
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    mma<false>(s.o[j * 4 + i][t], a0, a1, a2, a3, high[t][0], high[t][1]);
                    mma<false>(s.o[j * 4 + i][t], a0, a1, a2, a3, low[t][0], low[t][1]);
                }
            }
        }
    }

    // First of the 8 consecutive values that o[j * 4 .. j * 4 + 3] of lane group g hold, two each.
    static __device__ __forceinline__ int first_d(int j, int g) {
        if constexpr (!kFp4) return j * 64 + g * 8;
        const int w = g * (D / 64) + j;
        return (w % kChunks) * 32 + (w / kChunks) * 8;
    }
    static __device__ __forceinline__ float value_of(const State& s, int j, int t, int head, int e) {
        return s.o[j * 4 + (e >> 1)][t][head + 2 * (e & 1)];
    }

    static __device__ __forceinline__ void finish_head(const AttendArgs& a, int b, int head, float m, float l) {
        const int64_t i = (int64_t)b * a.heads + head;
        l *= kUnits;
        if (a.log_sum != nullptr) a.log_sum[i] = l > 0.0f || l != l ? m * 0.6931471805599453f + logf(l) : -INFINITY;
        if (a.weigh) a.stats[i] = make_float2(m == -INFINITY ? 0.0f : m, l > 0.0f || l != l ? 1.0f / l : 0.0f);
    }

    // A warp's state once its tiles are done: sums over the lanes, O in units of one.  It goes into a part, or to the output
    // when it is the whole of a group.
    static __device__ __forceinline__ void finish(State& s) {
        if constexpr (kFp4) {
#pragma unroll
            for (int j = 0; j < D / 64; ++j) {
                const float up = s.unit[j] == 0 ? 1.0f : power_of_two(s.unit[j] - 127);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s.o[j * 4 + i][t][e] *= up;
            }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                s.l[t][e] += __shfl_xor_sync(~0u, s.l[t][e], 4);
                s.l[t][e] += __shfl_xor_sync(~0u, s.l[t][e], 8);
                s.l[t][e] += __shfl_xor_sync(~0u, s.l[t][e], 16);
            }
    }

    static __device__ __forceinline__ void write_out(const State& s, const AttendArgs& a, int b, int head0, int heads, int lane) {
        const int g = lane >> 2, q4 = lane & 3;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int head = t * 8 + 2 * q4 + e;
                if (head >= heads) continue;
                const float l = s.l[t][e], f = l > 0.0f || l != l ? 1.0f / l : 0.0f;
                char* o = static_cast<char*>(a.out) + ((int64_t)b * a.heads + head0 + head) * D * 2;
#pragma unroll
                for (int j = 0; j < D / 64; ++j) {
                    uint4 w;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        (&w.x)[i] = pack_as(a.q_half, value_of(s, j, t, e, 2 * i) * f, value_of(s, j, t, e, 2 * i + 1) * f);
                    *reinterpret_cast<uint4*>(o + first_d(j, g) * 2) = w;
                }
                if (g == 0) finish_head(a, b, head0 + head, s.m[t][e], l);
            }
    }

    static __device__ __forceinline__ void write_part(const State& s, Part& part, int lane) {
        const int g = lane >> 2, q4 = lane & 3;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int head = t * 8 + 2 * q4 + e;
#pragma unroll
                for (int j = 0; j < D / 64; ++j)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        *reinterpret_cast<float4*>(&part.o[head][first_d(j, g) + 4 * i]) =
                            make_float4(value_of(s, j, t, e, 4 * i), value_of(s, j, t, e, 4 * i + 1),
                                        value_of(s, j, t, e, 4 * i + 2), value_of(s, j, t, e, 4 * i + 3));
                if (g == 0) part.ml[head] = make_float2(s.m[t][e], s.l[t][e]);
            }
    }

    // Joins four values of one head over n parts, in their order, many parts' loads at once (8 groups over 148 blocks: two trips).  Every column's thread works
    // out the factors for itself: that costs a few exponentials, and no barrier and no second trip to memory.
    template <bool SHARED, class PartAt>
    static __device__ __forceinline__ void join(PartAt part_at, int n, int head, int d, float4& o, float& top, float& l) {
        constexpr int kAtOnce = SHARED ? 8 : 10;
        o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        top = -INFINITY;
        l = 0.0f;
        for (int k = 0; k < n; k += kAtOnce) {
            float4 y[kAtOnce];
            float2 ml[kAtOnce];
            float m = top;
#pragma unroll
            for (int e = 0; e < kAtOnce; ++e) {
                y[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                ml[e] = make_float2(-INFINITY, 0.0f);
                if (k + e < n) {
                    const Part* p = part_at(k + e);
                    if constexpr (SHARED) {
                        ml[e] = p->ml[head];
                        y[e] = *reinterpret_cast<const float4*>(&p->o[head][d]);
                    } else {
                        ml[e] = __ldcg(&p->ml[head]);
                        y[e] = __ldcg(reinterpret_cast<const float4*>(&p->o[head][d]));
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < kAtOnce; ++e) m = fmaxf(m, ml[e].x);
            const float down = join_factor(top, m);
            o.x *= down; o.y *= down; o.z *= down; o.w *= down; l *= down;
            top = m;
#pragma unroll
            for (int e = 0; e < kAtOnce; ++e) {
                const float f = join_factor(ml[e].x, m);
                o.x = fmaf(y[e].x, f, o.x); o.y = fmaf(y[e].y, f, o.y); o.z = fmaf(y[e].z, f, o.z); o.w = fmaf(y[e].w, f, o.w);
                l = fmaf(ml[e].y, f, l);
            }
        }
    }

    static __device__ __forceinline__ void store_joined(const AttendArgs& a, int b, int head, int d, float4 o, float m, float l) {
        const float f = l > 0.0f || l != l ? 1.0f / l : 0.0f;
        uint2 w;
        w.x = pack_as(a.q_half, o.x * f, o.y * f);
        w.y = pack_as(a.q_half, o.z * f, o.w * f);
        *reinterpret_cast<uint2*>(static_cast<char*>(a.out) + (((int64_t)b * a.heads + head) * D + d) * 2) = w;
        if (d == 0) finish_head(a, b, head, m, l);
    }
};


// Places of one head's group of a sequence of n tokens in the shares of work.
__device__ __forceinline__ int places_of(int n) { return n > 0 ? (n + kTile - 1) / kTile + kStart : 0; }

// Adds one and returns what was there: the parts written before the barrier in front of it are seen by whoever finds
// the last count, and that one sees everybody's.
__device__ __forceinline__ int count_up(int* p) {
    int old;
    asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(old) : "l"(p) : "memory");
    return old;
}

// A (sequence, kv head, part of its group) in one word: at most 2048, 1024 and 16 of them.
struct Group {
    int b, h, sub;
    __device__ __forceinline__ int pack() const { return (b << 14) | (h << 4) | sub; }
    static __device__ __forceinline__ Group of(int tag) { return {tag >> 14, (tag >> 4) & 1023, tag & 15}; }
};

template <int KIND, int D, int NT>
__global__ void __launch_bounds__(Attend<KIND, D, NT>::kWarps * 32, 1)
attend_kernel(const __grid_constant__ AttendArgs a) {
    using A = Attend<KIND, D, NT>;
    constexpr int HP = A::HP, W = A::kWarps, kThreads = W * 32;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    typename A::Smem& sm = *reinterpret_cast<typename A::Smem*>(smem_raw);
    const RansKvCache& c = a.c;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int segs = c.kv_heads * a.subs;               // groups of one sequence

    wait_for_previous();
    let_next_start();
    // Places in front of each sequence.
    {
        const int per = (c.batch + kThreads - 1) / kThreads, b0 = min(tid * per, c.batch), b1 = min(b0 + per, c.batch);
        int sum = 0;
        for (int b = b0; b < b1; ++b) sum += places_of(checked_length(c, b));
        int inc = sum;
#pragma unroll
        for (int i = 1; i < 32; i *= 2) {
            const int y = __shfl_up_sync(~0u, inc, i);
            if (lane >= i) inc += y;
        }
        if (lane == 31) sm.warp_sum[warp] = inc;
        if (lane < 2) sm.tag[lane * W + warp] = -1;
        __syncthreads();
        int at = inc - sum;
        for (int w = 0; w < warp; ++w) at += sm.warp_sum[w];
        for (int b = b0; b < b1; ++b) {
            sm.pre[b] = at;
            at += places_of(checked_length(c, b));
        }
        if (b1 == c.batch && b0 < b1) sm.pre[c.batch] = at;
        __syncthreads();
    }
    const int total = sm.pre[c.batch] * segs;

    // Sequences without tokens.
    for (int b = blockIdx.x; b < c.batch; b += gridDim.x)
        if (sm.pre[b + 1] == sm.pre[b])
            for (int i = tid; i < a.heads * (D / 8); i += kThreads) {
                reinterpret_cast<uint4*>(a.out)[(int64_t)b * a.heads * (D / 8) + i] = make_uint4(0, 0, 0, 0);
                if (i < a.heads && a.log_sum != nullptr) a.log_sum[(int64_t)b * a.heads + i] = -INFINITY;
            }

    static_assert(sizeof(typename A::Smem) <= 227 * 1024, "a block's shared memory");
    static_assert(sizeof(typename A::Part) == sizeof(float) * HP * (D + 6), "make_plan's size of a part");
    static_assert(kThreads >= kGrid, "a thread for every block");
    // Equal runs of places: per block, and in it per warp.
    const int blocks = min((int)gridDim.x, (total + W - 1) / W);       // each of their warps has a tile
    if ((int)blockIdx.x >= blocks) return;
    const int per_block = total / blocks, longer = total - per_block * blocks;       // the first `longer` have one more
    auto first_of = [&](int block) { return per_block * block + min(block, longer); };
    const int x0 = first_of(blockIdx.x), x1 = first_of(blockIdx.x + 1);
    const int per_warp = (x1 - x0) / W, warps_longer = x1 - x0 - per_warp * W;
    int x = x0 + per_warp * warp + min(warp, warps_longer);
    const int xe = x + per_warp + (warp < warps_longer ? 1 : 0);
    auto tiles_of = [&](int b) { return sm.pre[b + 1] - sm.pre[b] - kStart; };
    auto heads_of = [&](const Group& s) { return min(a.sub_heads, a.group - s.sub * a.sub_heads); };
    auto head0_of = [&](const Group& s) { return s.h * a.group + s.sub * a.sub_heads; };

    auto first_part = [&](int w) {
        if constexpr (A::kFp4) return reinterpret_cast<typename A::Part*>(a.first) + blockIdx.x * W + w;
        else return &sm.part[w];
    };
    Group s{};
    int nt = 0, tile = 0;
    auto next_group = [&](Group& s, int& nt, int& tile) {
        tile = 0;
        if (++s.sub < a.subs) return;
        s.sub = 0;
        if (++s.h < c.kv_heads) return;
        s.h = 0;
        do ++s.b; while (s.b < c.batch && sm.pre[s.b + 1] == sm.pre[s.b]);
        if (s.b < c.batch) nt = tiles_of(s.b);
    };
    if (x < xe) {
        int lo = 0, hi = c.batch;                       // the sequence of place x: pre[lo] * segs <= x < pre[lo + 1] * segs
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (sm.pre[mid] * segs <= x) lo = mid; else hi = mid;
        }
        nt = tiles_of(lo);
        const int in = x - sm.pre[lo] * segs, seg = in / (nt + kStart);
        tile = in - seg * (nt + kStart);
        s.b = lo;
        s.h = seg / a.subs;
        s.sub = seg - s.h * a.subs;
        if (tile >= nt) {                               // behind a group's last tile
            x += nt + kStart - tile;
            next_group(s, nt, tile);
        }
    }
    if (x < xe) {
        uint4* qs = sm.q[warp];
        typename A::State st;
        typename A::Cursor u;
        int flushed = 0;
        bool whole = tile == 0;
        auto flush = [&](const Group& of, bool ends) {
            A::finish(st);
            __syncwarp();
            if (whole && ends) {
                A::write_out(st, a, of.b, head0_of(of), heads_of(of), lane);
            } else {
                A::write_part(st, flushed == 0 ? *first_part(warp) : sm.late[warp].part, lane);
                if (lane == 0) sm.tag[flushed * W + warp] = of.pack();
                ++flushed;
            }
        };
        if constexpr (A::kFp4) {
            // The copies run kStages - 1 turns ahead, in places of their own (`ahead`).  A turn takes kSub tiles of a group, or
            // what is left of it.
            constexpr int kStages = A::kStages, kSub = A::kSub;
            auto stages = sm.late[warp].stage;
            Group ahead = s;
            int ahead_nt = nt, ahead_tile = tile, ahead_x = x;
            std::conditional_t<(kStages * kSub > 6), uint64_t, uint32_t> valid = 0;      // tokens of each stage's tiles, 5 bits each
            bool fresh = true, ahead_fresh = true;
            auto copy = [&](int stage) {
#pragma unroll
                for (int i = 0; i < kSub; ++i) {
                    if (ahead_x >= xe || (i > 0 && ahead_fresh)) break;
                    if (ahead_fresh) u.begin(c, a.page, ahead.b, ahead.h, checked_length(c, ahead.b), ahead_tile, lane);
                    else u.advance(c, ahead.b, ahead.h, lane);
                    const int at = (stage * kSub + i) * 5;
                    valid = (valid & ~(decltype(valid)(31) << at)) | decltype(valid)(u.valid) << at;
                    A::copy_tile(stages[stage][i], c, u, lane);
                    ++ahead_x;
                    ahead_fresh = ++ahead_tile == ahead_nt;
                }
                if (ahead_fresh && ahead_tile == ahead_nt) {
                    ahead_x += kStart;
                    if (ahead_x < xe) next_group(ahead, ahead_nt, ahead_tile); else ahead_tile = 0;
                }
                copies_end();
            };
#pragma unroll 1
            for (int i = 0; i < kStages - 1; ++i) copy(i);
#pragma unroll 1
            for (int stage = 0, free = kStages - 1;; free = stage, stage = stage == kStages - 1 ? 0 : stage + 1) {
                if (fresh) A::begin(st, qs, a, s.b, head0_of(s), heads_of(s), lane);
                copies_wait<kStages - 2>();
                __syncwarp();                            // all lanes' copies of these tiles are there, and those before are read
                copy(free);
                const int count = kSub == 1 ? 1 : min(min(kSub, nt - tile), xe - x);
                float sc[kSub][NT][4];
                int tokens[kSub];
#pragma unroll
                for (int i = 0; i < kSub; ++i) {
                    tokens[i] = i < count ? (int)(valid >> ((stage * kSub + i) * 5)) & 31 : 0;
                    typename A::CodeK ck;
                    A::read_k(ck, stages[stage][i], lane);   // (of a missing tile: whatever is there, masked below)
                    A::scores(st, qs, ck, a, sc[i], lane);
                }
                A::probabilities(st, sc, a, x, tokens, lane);
                typename A::CodeV cv[kSub];
#pragma unroll
                for (int i = 0; i < kSub; ++i) A::read_v(cv[i], stages[stage][i], lane);
                A::accumulate(st, cv, sc, tokens, count, lane);
                tile += count;
                fresh = tile == nt;
                x += count + (fresh ? kStart : 0);
                if (fresh || x >= xe) flush(s, fresh);
                if (x >= xe) break;
                if (fresh) {
                    next_group(s, nt, tile);
                    whole = true;
                }
            }
        } else {
            // Keys of the next tile are on their way while this tile's softmax and values are worked on, and values while the
            // next scores are: the same registers, refilled as soon as their contents are used.
            typename A::RawK rk;
            typename A::RawV rv;
            bool have = false, fresh = true;
#pragma unroll 1
            while (true) {
                float sc[1][NT][4];
                bool more = true, ends = false;
                const Group now = s;
                int next = x, valid[1] = {0};
                if (have) {
                    A::scores(st, qs, rk, a, sc[0], lane);
                    ends = ++tile == nt;
                    next = x + 1 + (ends ? kStart : 0);
                    more = next < xe;
                    valid[0] = u.valid;
                    fresh = ends;
                    if (ends && more) next_group(s, nt, tile);
                }
                if (more) {
                    if (fresh) u.begin(c, a.page, s.b, s.h, checked_length(c, s.b), tile, lane); else u.advance(c, s.b, s.h, lane);
                    A::load_k(rk, c, u, lane);
                }
                if (have) {
                    A::probabilities(st, sc, a, x, valid, lane);
                    A::accumulate(st, rv, sc[0]);
                    x = next;
                    if (ends || !more) flush(now, ends);
                }
                if (!more) break;
                if (fresh) {
                    whole = tile == 0;
                    A::begin(st, qs, a, s.b, head0_of(s), heads_of(s), lane);
                    fresh = false;
                }
                A::load_v(rv, c, u, lane);
                have = true;
            }
        }
    }
    __syncthreads();

    // Join the warps' parts group by group; what the block has not all of goes to the workspace.  Each warp finds the groups
    // for itself, and the warps take turns at 32 columns of a group.
    static_assert(W * 2 <= 32, "one lane per part");
    constexpr int kVec = HP * (D / 4);
    typename A::Part* parts = reinterpret_cast<typename A::Part*>(a.part);
    int open0 = -1, open1 = -1;                          // groups that the block has only some of: its first, its last
    const int my_tag = lane < W * 2 ? sm.tag[lane] : -1;
    constexpr int kSlices = kVec / 32;
    int turn = warp;                                     // of this group's slices: turn, turn + W, ..
    for (unsigned left = __ballot_sync(~0u, my_tag >= 0); left != 0;) {
        const int tag = __shfl_sync(~0u, my_tag, __ffs(left) - 1);
        const unsigned run = __ballot_sync(~0u, my_tag == tag);
        left &= ~run;
        const Group s = Group::of(tag);
        const int nt = tiles_of(s.b), start = sm.pre[s.b] * segs + (s.h * a.subs + s.sub) * (nt + kStart);
        const bool whole = start >= x0 && start + nt <= x1;
        const int slot = start <= x0 ? 0 : 1, heads = heads_of(s);
        if (!whole) {
            if (slot == 0) open0 = tag; else open1 = tag;
            // which blocks share the group: every thread looks at one block (no division)
            if (tid < blocks) {
                const int f0 = first_of(tid), f1 = first_of(tid + 1);
                if (f0 <= start && start < f1) sm.first_block[slot] = tid;
                if (f0 < start + nt && start + nt <= f1) sm.last_block[slot] = tid;
            }
        }
        for (; turn < kSlices; turn += W) {
            const int v = turn * 32 + lane, head = v / (D / 4), d = v % (D / 4) * 4;
            if (head >= heads) continue;
            float4 o;
            float top, l;
            unsigned rest = run;
            A::template join<true>([&](int) { const int e = __ffs(rest) - 1; rest &= rest - 1; return e < W ? (const typename A::Part*)first_part(e) : &sm.late[e - W].part; }, __popc(run), head, d, o, top, l);
            if (whole) {
                A::store_joined(a, s.b, head0_of(s) + head, d, o, top, l);
            } else {
                typename A::Part* mine = parts + blockIdx.x * 2 + slot;
                __stcg(reinterpret_cast<float4*>(&mine->o[head][d]), o);
                if (d == 0) __stcg(&mine->ml[head], make_float2(top, l));
            }
        }
        turn -= kSlices;
    }

    // The last block of a group to get here joins the blocks' parts.
    if (open0 < 0 && open1 < 0) return;
    __syncthreads();
    if (tid < 2) {
        const int tag = tid == 0 ? open0 : open1;
        bool last = false;
        if (tag >= 0) {
            const Group s = Group::of(tag);
            int* counter = a.counter + s.b * segs + s.h * a.subs + s.sub;
            last = count_up(counter) == sm.last_block[tid] - sm.first_block[tid];
            if (last) *counter = 0;
        }
        sm.last[tid] = last;
    }
    __syncthreads();
    const int first_slices = sm.last[0] ? kSlices : 0, slices = first_slices + (sm.last[1] ? kSlices : 0);
#pragma unroll 1
    for (int slice = warp; slice < slices; slice += W) {
        const int i = slice < first_slices ? 0 : 1, v = (slice - (i == 0 ? 0 : first_slices)) * 32 + lane, head = v / (D / 4), d = v % (D / 4) * 4;
        const Group s = Group::of(i == 0 ? open0 : open1);
        if (head >= heads_of(s)) continue;
        const int nt = tiles_of(s.b), start = sm.pre[s.b] * segs + (s.h * a.subs + s.sub) * (nt + kStart);
        const int c0 = sm.first_block[i], second = first_of(c0) == start ? 0 : 1;    // only a group's first block has it as its second
        float4 o;
        float top, l;
        A::template join<false>([&](int k) { return parts + (c0 + k) * 2 + (k == 0 ? second : 0); }, sm.last_block[i] - c0 + 1, head, d, o, top, l);
        A::store_joined(a, s.b, head0_of(s) + head, d, o, top, l);
    }
}

// weight[t] += sum over a kv head's query heads of exp2(score - m) / l.  A warp takes 64 tokens of a head at a time, each lane
// two of them: scores are read 32 bytes a lane, the heads' m and 1 / l by one lane each.  Bound by reading the scores (4 bytes
// a token and query head, mostly from L2): with the stores of attend_kernel 13 us of a step of 16 x 4097 tokens on 64 heads.
constexpr int kWeighThreads = 256;
constexpr int kSpan = 64;
constexpr int kWeighBlocks = 6;          // an SM

template <int HP>
__global__ void __launch_bounds__(kWeighThreads) weigh_kernel(const __grid_constant__ AttendArgs a) {
    __shared__ int places[RANS_KV_MAX_BATCH + 1], spans[RANS_KV_MAX_BATCH + 1];      // of one head, in front of each sequence
    __shared__ int warp_sum[2][kWeighThreads / 32];
    const RansKvCache& c = a.c;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    wait_for_previous();
    let_next_start();
    {
        const int per = (c.batch + kWeighThreads - 1) / kWeighThreads, b0 = min(tid * per, c.batch), b1 = min(b0 + per, c.batch);
        int sum[2] = {0, 0};
        for (int b = b0; b < b1; ++b) {
            const int n = checked_length(c, b);
            sum[0] += places_of(n);
            sum[1] += (n + kSpan - 1) / kSpan;
        }
        int inc[2] = {sum[0], sum[1]};
#pragma unroll
        for (int i = 1; i < 32; i *= 2) {
            const int x = __shfl_up_sync(~0u, inc[0], i), y = __shfl_up_sync(~0u, inc[1], i);
            if (lane >= i) {
                inc[0] += x;
                inc[1] += y;
            }
        }
        if (lane == 31) {
            warp_sum[0][warp] = inc[0];
            warp_sum[1][warp] = inc[1];
        }
        __syncthreads();
        int at[2] = {inc[0] - sum[0], inc[1] - sum[1]};
        for (int w = 0; w < warp; ++w) {
            at[0] += warp_sum[0][w];
            at[1] += warp_sum[1][w];
        }
        for (int b = b0; b < b1; ++b) {
            const int n = checked_length(c, b);
            places[b] = at[0];
            spans[b] = at[1];
            at[0] += places_of(n);
            at[1] += (n + kSpan - 1) / kSpan;
        }
        if (b1 == c.batch && b0 < b1) spans[c.batch] = at[1];
        __syncthreads();
    }
    const int total = spans[c.batch] * c.kv_heads;
    for (int i = blockIdx.x * (kWeighThreads / 32) + warp; i < total; i += gridDim.x * (kWeighThreads / 32)) {
        int b = 0, hi = c.batch;
        while (hi - b > 1) {
            const int mid = (b + hi) / 2;
            if (spans[mid] * c.kv_heads <= i) b = mid; else hi = mid;
        }
        const int per_head = spans[b + 1] - spans[b], in = i - spans[b] * c.kv_heads, h = in / per_head, t0 = (in - h * per_head) * kSpan;
        const int n = checked_length(c, b), per_group = places_of(n);
        int64_t at[2];
        float add[2] = {0.0f, 0.0f}, before[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int t = t0 + e * 32 + lane, in_page = a.page(t), p = t < n ? checked_page(c, b, in_page) : -1;
            at[e] = p >= 0 ? ((int64_t)p * c.kv_heads + h) * c.page + (t - in_page * c.page) : -1;
        }
        for (int sub = 0; sub < a.subs; ++sub) {
            const int first = sub * a.sub_heads, heads = min(a.sub_heads, a.group - first);
            const int64_t x = (int64_t)places[b] * c.kv_heads * a.subs + (int64_t)(h * a.subs + sub) * per_group + t0 / kTile;
            if (x + (min(t0 + kSpan, n) - 1 - t0) / kTile >= a.score_tiles) {
                raise(c, RANS_KV_BAD_LENGTH);
                break;
            }
            const float2 ml = lane < heads ? a.stats[(int64_t)b * a.heads + h * a.group + first + lane] : make_float2(0.0f, 0.0f);
            float4 s[2][HP / 4];
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int k = 0; k < HP / 4; ++k)
                    s[e][k] = at[e] >= 0 ? __ldcg(reinterpret_cast<const float4*>(a.scores + (x * kTile + e * 32 + lane) * HP) + k) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (sub == 0)
#pragma unroll
                for (int e = 0; e < 2; ++e) before[e] = at[e] >= 0 ? c.weight[at[e]] : 0.0f;
#pragma unroll
            for (int k = 0; k < HP; ++k) {
                if (k >= heads) break;
                const float m = __shfl_sync(~0u, ml.x, k), l = __shfl_sync(~0u, ml.y, k);
#pragma unroll
                for (int e = 0; e < 2; ++e) add[e] = fmaf(exp2_fast((&s[e][k / 4].x)[k % 4] - m), l, add[e]);
            }
            if (sub == a.subs - 1)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (at[e] >= 0) c.weight[at[e]] = before[e] + add[e];
        }
    }
}

struct Plan {
    int nt, subs, sub_heads;
    int64_t counter, stats, part, first, scores, bytes, score_tiles;
};

bool make_plan(const RansKvCache& c, int heads, int weigh, Plan& p) {
    if (heads < 1 || heads % c.kv_heads != 0) return false;
    const int group = heads / c.kv_heads, most = c.dim == 256 ? 8 : 16;
    p.subs = (group + most - 1) / most;
    if (p.subs > kMaxSubgroups) return false;
    p.sub_heads = (group + p.subs - 1) / p.subs;
    p.nt = p.sub_heads > 8 ? 2 : 1;
    // places are counted in 32 bits
    if (((int64_t)c.table_cols * c.page / kTile + kStart) * c.batch * c.kv_heads * p.subs > 0x7fffffff) return false;
    auto up = [](int64_t x) { return (x + 255) & ~(int64_t)255; };
    p.counter = 256;
    p.stats = counter_bytes(c);
    p.part = p.stats + up((int64_t)c.batch * heads * 8);
    const int64_t part = (int64_t)p.nt * 8 * (c.dim + 4 + 2) * 4;            // sizeof(Attend::Part)
    p.first = p.part + up(kGrid * 2 * part);
    p.scores = p.first + (c.kind == RANS_KV_MXFP4 ? up(kGrid * 16 * part) : 0);
    // every token of every page, and the places behind the groups' last tiles
    p.score_tiles = weigh ? ((int64_t)c.pages * c.page / kTile + (int64_t)c.batch * kStart) * c.kv_heads * p.subs : 0;
    if (p.score_tiles > 0x7fffffff) return false;
    p.bytes = p.scores + up(p.score_tiles * kTile * p.nt * 8 * 4);
    return true;
}

template <int KIND, int D, int NT>
int launch(const AttendArgs& a, cudaStream_t stream) {
    using A = Attend<KIND, D, NT>;
    auto kernel = attend_kernel<KIND, D, NT>;
    // once per device (a repetition by another thread does no harm)
    static std::atomic<uint64_t> told{0};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return (int)e;
    const uint64_t bit = (uint64_t)1 << (device & 63);
    if ((told.load(std::memory_order_relaxed) & bit) == 0) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(typename A::Smem));
        if (e != cudaSuccess) return (int)e;
        told.fetch_or(bit, std::memory_order_relaxed);
    }
    return launch_after(kernel, dim3(kGrid), A::kWarps * 32, sizeof(typename A::Smem), 1, stream, a);
}

template <int KIND>
int launch_kind(const AttendArgs& a, int nt, cudaStream_t stream) {
    switch (a.c.dim) {
        case 64: return nt == 1 ? launch<KIND, 64, 1>(a, stream) : launch<KIND, 64, 2>(a, stream);
        case 128: return nt == 1 ? launch<KIND, 128, 1>(a, stream) : launch<KIND, 128, 2>(a, stream);
        case 256: return launch<KIND, 256, 1>(a, stream);
        default: return -1;
    }
}

}  // namespace
}  // namespace rb200kv

using namespace rb200kv;

extern "C" int64_t rans_kv_counter_bytes(const RansKvCache* c) {
    if (c == nullptr || c->batch < 1 || c->batch > RANS_KV_MAX_BATCH || c->kv_heads < 1) return -2;
    return counter_bytes(*c);
}

extern "C" int64_t rans_kv_attend_bytes(const RansKvCache* c, int heads, int weigh) {
    if (rans_kv_counter_bytes(c) < 0 || c->pages < 1 || c->page < 16) return -2;
    Plan p;
    return make_plan(*c, heads, weigh, p) ? p.bytes : -2;
}

extern "C" int rans_kv_attend(const RansKvCache* cache, const void* q, int q_kind, int64_t q_batch, int64_t q_head, int heads,
                              float scale, void* out, float* log_sum, int weigh, cudaStream_t stream) {
    const int rc = check_cache(cache);
    if (rc != 0) return rc;
    if (q_kind != RANS_KV_BF16 && q_kind != RANS_KV_FP16) return -1;
    if (cache->kind != RANS_KV_MXFP4 && q_kind != cache->kind) return -1;
    Plan p;
    if (!make_plan(*cache, heads, weigh, p)) return -2;
    if (q == nullptr || out == nullptr || !aligned16(q) || !aligned16(out) || ((q_batch | q_head) & 15)) return -2;
    if (weigh && cache->weight == nullptr) return -2;
    if (cache->workspace_bytes < p.bytes) return -3;
    AttendArgs a{};
    a.c = *cache;
    fill_strides(a.c);
    a.page = Divider::of((uint32_t)cache->page);
    char* ws = static_cast<char*>(cache->workspace);
    a.q = static_cast<const char*>(q);
    a.q_batch = q_batch;
    a.q_head = q_head;
    a.out = out;
    a.log_sum = log_sum;
    a.scale_log2 = scale * kLog2e;
    a.heads = heads;
    a.group = heads / cache->kv_heads;
    a.subs = p.subs;
    a.sub_heads = p.sub_heads;
    a.q_half = q_kind == RANS_KV_FP16;
    a.weigh = weigh != 0;
    a.counter = reinterpret_cast<int*>(ws + p.counter);
    a.stats = reinterpret_cast<float2*>(ws + p.stats);
    a.part = reinterpret_cast<float*>(ws + p.part);
    a.scores = reinterpret_cast<float*>(ws + p.scores);
    a.first = reinterpret_cast<float*>(ws + p.first);
    a.score_tiles = (int)p.score_tiles;
    int e;
    switch (cache->kind) {
        case RANS_KV_BF16: e = launch_kind<RANS_KV_BF16>(a, p.nt, stream); break;
        case RANS_KV_FP16: e = launch_kind<RANS_KV_FP16>(a, p.nt, stream); break;
        default: e = launch_kind<RANS_KV_MXFP4>(a, p.nt, stream); break;
    }
    if (e != 0 || !weigh) return e;
    return launch_after(p.nt == 1 ? weigh_kernel<8> : weigh_kernel<16>, dim3(kSms * kWeighBlocks), kWeighThreads, 0, 1, stream, a);
}
