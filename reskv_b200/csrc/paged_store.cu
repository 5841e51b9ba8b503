// The 4-bit paged cache takes tokens, gives them back, and moves pages.
//
// Storing: of a token's vector of one head, every group of 64 coordinates becomes offset = min, scale = (max - min) / 15
// rounded to the model's type, code = round((x - offset) / scale) to the nearest, ties to even, at most 15 (0 where the scale
// is 0).  512 bytes of K and V become 144.  Four lanes hold a row of one side,
// sixteen coordinates of either group each, eight rows (K and V of four heads) to a warp; a lane's words of a key row are then 16
// bytes in a row of their own.  Extremes of both groups travel together as 16-bit pairs.  A warp looks up by itself where its tokens
// go, while their rows are on the way.
//
// 8 x 4000 tokens, 8 heads: written in 36 us (168 MB, 4.7 TB/s, 0.72 of the copy rate), read back in 30 us (5.6 TB/s, 0.87); 65 and 59 % of
// the issue slots are taken: writing is bound by neither alone, reading nearly by bytes.  Loads that ask to leave L2 first: 34.6 us, but attention over the prompt reads the same rows.
// Eight lanes to a row: 46 and 32 us, sixteen: 91 and 51 us.  Ties and what is near them left to the division: 2 us more, with six BF16
// prompts of 4546 tokens 11 us for 7.9.  Places looked up by a few threads for the block: 0.2 to 0.9 us more on small calls.
#include <algorithm>
#include <new>
#include <vector>

#include "paged_int4.cuh"

namespace reskv {
namespace {

constexpr int kStoreWarps = 4, kStoreThreads = kStoreWarps * 32;
constexpr int kPassRows = 4;  // (token, head) rows that a warp takes at once
// Passes of a warp that are in flight together, where there are enough rows.  8 x 4000 tokens, us written and read, by passes: 1 37.5 and
// 32.9, 2 36.4 and 30.2, 4 42.6 and 32.0; 8 warps a block at 2 passes 39.7 and 30.2, 2 warps 35.9 and 29.9 (small calls slower).
constexpr int kPasses = 2;
// Blocks that an SM is to hold: registers against rows in flight.  6 prompts of 4546 BF16 tokens, us written: left to the compiler (71
// registers) 7.2, 8 blocks 6.4, 10 (spills) 8.1; read: left to the compiler 6.4, 10 blocks 6.1, 14 blocks 5.6, 16 blocks 5.6.
template <bool WRITE>
constexpr int kBlocksPerSm = WRITE ? 8 : 14;

struct StoreParams {
    PagedPlace at;
    unsigned char* pages;            // of the layer
    const unsigned short *k, *v;     // write: sources
    unsigned short *k_out, *v_out;   // read: destinations [total, heads, 128]
    int64_t k_token, k_head, v_token, v_head;  // elements
    int total, heads;
    uint32_t* status;
};

// Where token i goes: byte of its block in the pool for head 0 (below 0: nowhere), and row of the block.
struct TokenPlace {
    int64_t block;
    int row;
};
__device__ __forceinline__ TokenPlace place_of(const StoreParams& p, int token) {
    // Of a step with one token for each sequence it is the token's number (32 sequences: 2.3 us for 2.7); otherwise a search for the
    // number of sequences that end at the token or in front of it.
    int low = min(token, p.at.sequences - 1);
    if (token < p.at.cu[low] || token >= p.at.cu[low + 1]) {
        low = 0;
        for (int high = p.at.sequences; low < high;) {
            const int mid = (low + high) >> 1;
            if (p.at.cu[mid + 1] <= token) low = mid + 1; else high = mid;
        }
        if (low >= p.at.sequences || token < p.at.cu[low]) return {-1, 0};
    }
    const int number = p.at.starts[low] + token - p.at.cu[low], slot = number / kPageTokens;
    const int page = number >= 0 && slot < p.at.width ? p.at.table[static_cast<int64_t>(low) * p.at.width + slot] : -1;
    if (page < 0 || page >= p.at.pages) {  // outside the table or the pool
        atomicOr(p.status, RESKV_STATUS_STATE_RANGE);
        return {-1, 0};
    }
    return {static_cast<int64_t>(page) * p.heads * kPageHeadBytes + (number / kBlockTokens & 3) * kBlockBytes, number & (kBlockTokens - 1)};
}

// The larger / smaller numbers of two pairs, NaN if one of the two is.
template <bool BF16>
__device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b) {
    uint32_t r;
    if (BF16) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <bool BF16>
__device__ __forceinline__ uint32_t min_pair(uint32_t a, uint32_t b) {
    uint32_t r;
    if (BF16) asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Codes of eight numbers; `scale` as stored, `low` the offset.
//
// The quotient by the reciprocal, corrected by its remainder, is the one that IEEE division gives: the correction leaves a relative
// error below 2^-40, while a quotient of a 24-bit number and an 11-bit scale is never nearer than 2^-37 to the middle of two FP32
// numbers.  That holds as long as the remainder does not underflow, hence kLeast.  Ties are common (one in
// seven groups of 64 normal BF16 numbers has one), so they are not left to the division.
struct Codes {
    uint32_t a, b;
};
template <bool BF16>
__device__ __forceinline__ Codes codes_of(const uint4& x, const uint4& y, float low, float scale) {
    constexpr float kRound = 12582912.f;  // 1.5 * 2^23: a sum with it is rounded to a whole number
    constexpr float kLeast = BF16 ? 0x1p-90f : 0x1p-14f, kMost = BF16 ? 0x1p125f : 65504.f;
    const uint32_t pairs[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    float inverse;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(scale));
    const float2 minus_low = make_float2(-low, -low), inverses = make_float2(inverse, inverse), minus_scale = make_float2(-scale, -scale),
                 up = make_float2(kRound, kRound);
    const bool usual = scale >= kLeast && scale <= kMost;
    uint32_t words[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        uint32_t word = 0;
#pragma unroll
        for (int e = 4 * w + 3; e >= 4 * w; --e) {
            const float2 above = add2(make_float2(low_of<BF16>(pairs[e]), high_of<BF16>(pairs[e])), minus_low), first = mul2(above, inverses);
            const float2 rounded = add2(fma2(fma2(minus_scale, first, above), inverses, first), up);
            word = (word * 16u + __float_as_uint(rounded.y)) * 16u + __float_as_uint(rounded.x);  // the constant part goes below
        }
        words[w] = word - 0x4B400000u * 0x11111111u;
    }
    if (!usual) {  // scales that rounding may have made much too small (below the normal numbers, 0), and what is not finite
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            words[w] = 0;
#pragma unroll
            for (int e = 4 * w + 3; e >= 4 * w; --e)
#pragma unroll
                for (int half = 1; half >= 0; --half) {  // a NaN becomes 0: the scale says it
                    const float quotient = ((half ? high_of<BF16>(pairs[e]) : low_of<BF16>(pairs[e])) - low) / scale;
                    words[w] = words[w] * 16u + (scale > 0.f ? static_cast<uint32_t>(fminf(fmaxf(rintf(quotient), 0.f), 15.f)) : 0u);
                }
        }
    }
    return {words[0], words[1]};
}

// x / 15 as IEEE division rounds it (x finite): the quotient by the reciprocal, corrected by its remainder.
__device__ __forceinline__ float fifteenth(float x) {
    constexpr float kInverse = 1.f / 15.f;
    const float q = x * kInverse;
    return fmaf(fmaf(-15.f, q, x), kInverse, q);
}

template <bool BF16, bool WRITE, int PASSES>
__global__ void __launch_bounds__(kStoreThreads, kBlocksPerSm<WRITE>) paged_store_kernel(const StoreParams p) {
    wait_for_previous_launch();
    let_next_launch_start();
    const int lane = threadIdx.x & 31, side = lane >> 2 & 1, c = lane & 3;
    // a warp's rows lie next to each other
    const int64_t first = (static_cast<int64_t>(blockIdx.x) * kStoreWarps + (threadIdx.x >> 5)) * (PASSES * kPassRows);
    int token[PASSES], head[PASSES];
    uint4 x[PASSES][4];
    {
        const int before = static_cast<int>(first / p.heads), row = static_cast<int>(first - static_cast<int64_t>(before) * p.heads) + (lane >> 3);
        int t = before + row / p.heads, h = row % p.heads;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            token[i] = t < p.total ? t : -1, head[i] = h;
            if (WRITE && token[i] >= 0) {
                const uint4* from = reinterpret_cast<const uint4*>(side ? p.v + t * p.v_token + h * p.v_head : p.k + t * p.k_token + h * p.k_head);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[i][j] = from[c + 4 * j];
            }
            for (h += kPassRows; h >= p.heads; h -= p.heads) ++t;
        }
    }
    unsigned char* block[PASSES];  // of the row's side, or null
    int row[PASSES];
    TokenPlace to{-1, 0};
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        block[i] = nullptr, row[i] = 0;
        if (token[i] < 0) continue;
        if (i == 0 || token[i] != token[i - 1]) to = place_of(p, token[i]);
        if (to.block >= 0) block[i] = p.pages + to.block + static_cast<int64_t>(head[i]) * kPageHeadBytes + side * kBlockSide;
        row[i] = to.row;
    }
    if (WRITE) {
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            // (group 0, group 1) extremes; rows without a place take part in the exchange with whatever they hold
            if (token[i] < 0) x[i][0] = x[i][1] = x[i][2] = x[i][3] = make_uint4(0, 0, 0, 0);
            uint32_t top[2], bottom[2];
#pragma unroll
            for (int group = 0; group < 2; ++group) {
                const uint4 &v = x[i][2 * group], &w = x[i][2 * group + 1];
                top[group] = max_pair<BF16>(max_pair<BF16>(max_pair<BF16>(v.x, v.y), max_pair<BF16>(v.z, v.w)),
                                            max_pair<BF16>(max_pair<BF16>(w.x, w.y), max_pair<BF16>(w.z, w.w)));
                bottom[group] = min_pair<BF16>(min_pair<BF16>(min_pair<BF16>(v.x, v.y), min_pair<BF16>(v.z, v.w)),
                                               min_pair<BF16>(min_pair<BF16>(w.x, w.y), min_pair<BF16>(w.z, w.w)));
            }
            uint32_t high = max_pair<BF16>(__byte_perm(top[0], top[1], 0x5410), __byte_perm(top[0], top[1], 0x7632));
            uint32_t low = min_pair<BF16>(__byte_perm(bottom[0], bottom[1], 0x5410), __byte_perm(bottom[0], bottom[1], 0x7632));
#pragma unroll
            for (int off = 1; off < 4; off <<= 1) {
                high = max_pair<BF16>(high, __shfl_xor_sync(0xffffffffu, high, off));
                low = min_pair<BF16>(low, __shfl_xor_sync(0xffffffffu, low, off));
            }
            if (!block[i]) continue;
            const float low0 = low_of<BF16>(low), low1 = high_of<BF16>(low);
            const uint32_t scales = pack2<BF16>(fifteenth(low_of<BF16>(high) - low0), fifteenth(high_of<BF16>(high) - low1));
            const Codes first_group = codes_of<BF16>(x[i][0], x[i][1], low0, low_of<BF16>(scales)),
                        second_group = codes_of<BF16>(x[i][2], x[i][3], low1, high_of<BF16>(scales));
            if (side) {
                *reinterpret_cast<uint2*>(block[i] + value_word(row[i], c)) = make_uint2(first_group.a, second_group.a);
                *reinterpret_cast<uint2*>(block[i] + value_word(row[i], c + 4)) = make_uint2(first_group.b, second_group.b);
            } else {
                *reinterpret_cast<uint4*>(block[i] + key_word(row[i], c)) = make_uint4(first_group.a, first_group.b, second_group.a, second_group.b);
            }
            if (c == 0) *reinterpret_cast<uint2*>(block[i] + kBlockCodes + row[i] * 8) = make_uint2(scales, low);
        }
    } else {
        uint4 words[PASSES];  // c, c + 4, c + 8, c + 12
        uint2 params[PASSES];
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            if (!block[i]) continue;
            if (side) {
                const uint2 a = *reinterpret_cast<const uint2*>(block[i] + value_word(row[i], c)),
                            b = *reinterpret_cast<const uint2*>(block[i] + value_word(row[i], c + 4));
                words[i] = make_uint4(a.x, b.x, a.y, b.y);
            } else {
                words[i] = *reinterpret_cast<const uint4*>(block[i] + key_word(row[i], c));
            }
            params[i] = *reinterpret_cast<const uint2*>(block[i] + kBlockCodes + row[i] * 8);
        }
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            if (!block[i]) continue;
            uint4* to = reinterpret_cast<uint4*>((side ? p.v_out : p.k_out) + (static_cast<int64_t>(token[i]) * p.heads + head[i]) * 128);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float scale = j >> 1 ? high_of<BF16>(params[i].x) : low_of<BF16>(params[i].x);
                const float low = j >> 1 ? high_of<BF16>(params[i].y) : low_of<BF16>(params[i].y);
                const uint32_t word = j == 0 ? words[i].x : j == 1 ? words[i].y : j == 2 ? words[i].z : words[i].w;
                const float2 scales = make_float2(scale, scale), lows = make_float2(low, low), down = make_float2(-8388608.f, -8388608.f);
                uint4 y;
                uint32_t* pairs = reinterpret_cast<uint32_t*>(&y);
#pragma unroll
                for (int e = 0; e < 4; ++e) {  // codes as the low bits of 2^23 + code
                    const float2 code = add2(make_float2(__uint_as_float((word >> (8 * e) & 15u) | 0x4B000000u),
                                                         __uint_as_float((word >> (8 * e + 4) & 15u) | 0x4B000000u)), down);
                    const float2 v = fma2(scales, code, lows);
                    pairs[e] = pack2<BF16>(v.x, v.y);
                }
                to[4 * j + c] = y;
            }
        }
    }
}

// ---- pages ----------------------------------------------------------------------------------------------------------------
constexpr int kPairsPerLaunch = 480;  // pairs travel as launch parameters: no copy to the device, and a captured launch keeps them
constexpr int kCopyThreads = 256;
constexpr int kCopyPiece = kCopyThreads * 16 * 4;

struct PagePairs {
    int src[kPairsPerLaunch], dst[kPairsPerLaunch];
};

// Bound by bytes: 192 pages in 32 layers of 8 heads, 906 MB, 138 us = 6.6 TB/s, 1.02 of the copy rate.
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(unsigned char* pages, int64_t layer_bytes, int64_t page_bytes, const PagePairs pairs) {
    wait_for_previous_launch();
    let_next_launch_start();
    unsigned char* layer = pages + blockIdx.z * layer_bytes;
    const uint4* from = reinterpret_cast<const uint4*>(layer + pairs.src[blockIdx.y] * page_bytes);
    uint4* to = reinterpret_cast<uint4*>(layer + pairs.dst[blockIdx.y] * page_bytes);
    const int64_t n = page_bytes / 16, at = static_cast<int64_t>(blockIdx.x) * (kCopyPiece / 16) + threadIdx.x;
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (at + i * kCopyThreads < n) v[i] = from[at + i * kCopyThreads];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (at + i * kCopyThreads < n) to[at + i * kCopyThreads] = v[i];
}

int check_place(const char* who, const int32_t* cu, const int32_t* starts, const int32_t* table, int sequences, int width, int total,
                int heads, const void* pages, int page_count, const uint32_t* status) {
    if (sequences < 0 || width < 0 || total < 0 || heads < 1 || page_count < 0)
        return fail(RESKV_ERR_INVALID, "%s: %d sequences, table of %d pages, %d tokens, %d heads, %d pages", who, sequences, width, total, heads, page_count);
    if (sequences == 0 || total == 0) return RESKV_OK;
    if (!cu || !starts || (!table && width > 0) || !pages || !status) return fail(RESKV_ERR_INVALID, "%s: null pointer", who);
    if (!aligned16(pages)) return fail(RESKV_ERR_INVALID, "%s: pages must start on a 16-byte boundary", who);
    if (int rc = check_device_pointer(pages, who, "pages")) return rc;
    if (int rc = check_device_pointer(cu, who, "cu_seqlens")) return rc;
    if (int rc = check_device_pointer(starts, who, "starts")) return rc;
    if (int rc = check_device_pointer(status, who, "status")) return rc;
    return width > 0 ? check_device_pointer(table, who, "table") : RESKV_OK;
}

template <bool BF16, bool WRITE, int PASSES>
int launch_store(const StoreParams& p, cudaStream_t stream) {
    constexpr int per = kStoreWarps * kPassRows * PASSES;
    const int64_t blocks = (static_cast<int64_t>(p.total) * p.heads + per - 1) / per;
    if (blocks > 0x7fffffff) return fail(RESKV_ERR_LIMIT, "paged cache: too many tokens for one call");
    return check_cuda(launch_overlapped(paged_store_kernel<BF16, WRITE, PASSES>, dim3(static_cast<unsigned>(blocks)), kStoreThreads, 0, stream, true, p),
                      WRITE ? "paged_write launch" : "paged_read launch");
}
// One pass per warp up to eight blocks per SM.  us written and read with one pass and with two, 8 heads: 64 tokens 2.0 and 2.0, 2.7 and
// 2.5; 800 tokens 2.7 and 2.7, 3.2 and 3.0; 1600 tokens 3.8 and 3.2, 3.6 and 3.4; 4546 tokens 6.4 and 5.5, 5.9 and 5.4.
template <bool WRITE>
int run_store(const StoreParams& p, int bf16, cudaStream_t stream) {
    const bool many = static_cast<int64_t>(p.total) * p.heads > 8 * static_cast<int64_t>(sm_count()) * kStoreWarps * kPassRows;
    return bf16 ? many ? launch_store<true, WRITE, kPasses>(p, stream) : launch_store<true, WRITE, 1>(p, stream)
                : many ? launch_store<false, WRITE, kPasses>(p, stream) : launch_store<false, WRITE, 1>(p, stream);
}

}  // namespace
}  // namespace reskv

using namespace reskv;

extern "C" int reskv_paged_write(const void* k, const void* v, int bf16, int64_t k_token, int64_t k_head, int64_t v_token, int64_t v_head,
                                 const int32_t* cu_seqlens, const int32_t* starts, const int32_t* table, int sequences, int width, int total,
                                 int kv_heads, void* pages, int page_count, uint32_t* status, void* stream) {
    if (int rc = check_place("paged_write", cu_seqlens, starts, table, sequences, width, total, kv_heads, pages, page_count, status)) return rc;
    if (sequences == 0 || total == 0) return RESKV_OK;
    if (!k || !v) return fail(RESKV_ERR_INVALID, "paged_write: null pointer");
    if (!aligned16(k) || !aligned16(v) || k_token % 8 || k_head % 8 || v_token % 8 || v_head % 8 || k_token < 0 || k_head < 0 || v_token < 0 || v_head < 0)
        return fail(RESKV_ERR_INVALID, "paged_write: k and v must start on 16-byte boundaries, their strides be multiples of 8 elements");
    if (int rc = check_device_pointer(k, "paged_write", "k")) return rc;
    if (int rc = check_device_pointer(v, "paged_write", "v")) return rc;
    StoreParams p{};
    p.at = {cu_seqlens, starts, table, sequences, width, page_count};
    p.pages = static_cast<unsigned char*>(pages);
    p.k = static_cast<const unsigned short*>(k), p.v = static_cast<const unsigned short*>(v);
    p.k_token = k_token, p.k_head = k_head, p.v_token = v_token, p.v_head = v_head, p.total = total, p.heads = kv_heads, p.status = status;
    return run_store<true>(p, bf16, static_cast<cudaStream_t>(stream));
}

extern "C" int reskv_paged_read(void* k, void* v, int bf16, const int32_t* cu_seqlens, const int32_t* starts, const int32_t* table,
                                int sequences, int width, int total, int kv_heads, const void* pages, int page_count, uint32_t* status,
                                void* stream) {
    if (int rc = check_place("paged_read", cu_seqlens, starts, table, sequences, width, total, kv_heads, pages, page_count, status)) return rc;
    if (sequences == 0 || total == 0) return RESKV_OK;
    if (!k || !v || !aligned16(k) || !aligned16(v)) return fail(RESKV_ERR_INVALID, "paged_read: k and v must start on 16-byte boundaries");
    if (int rc = check_device_pointer(k, "paged_read", "k")) return rc;
    if (int rc = check_device_pointer(v, "paged_read", "v")) return rc;
    StoreParams p{};
    p.at = {cu_seqlens, starts, table, sequences, width, page_count};
    p.pages = const_cast<unsigned char*>(static_cast<const unsigned char*>(pages));
    p.k_out = static_cast<unsigned short*>(k), p.v_out = static_cast<unsigned short*>(v);
    p.total = total, p.heads = kv_heads, p.status = status;
    return run_store<false>(p, bf16, static_cast<cudaStream_t>(stream));
}

extern "C" int reskv_copy_pages(void* pages, int layers, int page_count, int64_t page_bytes, const int32_t* src, const int32_t* dst, int count,
                                void* stream) {
    if (layers < 0 || page_count < 0 || page_bytes < 0 || page_bytes % 16 || count < 0)
        return fail(RESKV_ERR_INVALID, "copy_pages: %d layers, %d pages, %d pairs", layers, page_count, count);
    if (layers > 65535) return fail(RESKV_ERR_LIMIT, "copy_pages: more than 65535 layers");
    if (layers == 0 || page_bytes == 0 || count == 0) return RESKV_OK;
    if (!pages || !src || !dst || !aligned16(pages)) return fail(RESKV_ERR_INVALID, "copy_pages: null or misaligned pointer");
    // all copies run at the same time: no page may be a destination twice, or a source and a destination
    try {
        std::vector<int32_t> to(dst, dst + count);
        std::sort(to.begin(), to.end());
        for (int i = 0; i < count; ++i) {
            if (src[i] < 0 || src[i] >= page_count || dst[i] < 0 || dst[i] >= page_count)
                return fail(RESKV_ERR_INVALID, "copy_pages: pair %d -> %d of %d pages", src[i], dst[i], page_count);
            if (i > 0 && to[i] == to[i - 1]) return fail(RESKV_ERR_INVALID, "copy_pages: page %d is a destination twice", to[i]);
            if (std::binary_search(to.begin(), to.end(), src[i]))
                return fail(RESKV_ERR_INVALID, "copy_pages: page %d is a source and a destination", src[i]);
        }
    } catch (const std::bad_alloc&) {
        return fail(RESKV_ERR_LIMIT, "copy_pages: no host memory for %d pairs", count);
    }
    if (int rc = check_device_pointer(pages, "copy_pages", "pages")) return rc;
    const int64_t pieces = (page_bytes + kCopyPiece - 1) / kCopyPiece;
    if (pieces > 0x7fffffff) return fail(RESKV_ERR_LIMIT, "copy_pages: pages too large");
    for (int i = 0; i < count; i += kPairsPerLaunch) {
        const int n = count - i < kPairsPerLaunch ? count - i : kPairsPerLaunch;
        PagePairs pairs{};
        std::copy(src + i, src + i + n, pairs.src);
        std::copy(dst + i, dst + i + n, pairs.dst);
        const dim3 grid(static_cast<unsigned>(pieces), static_cast<unsigned>(n), static_cast<unsigned>(layers));
        if (int rc = check_cuda(launch_overlapped(copy_pages_kernel, grid, kCopyThreads, 0, static_cast<cudaStream_t>(stream), true,
                                                  static_cast<unsigned char*>(pages), page_bytes * page_count, page_bytes, pairs),
                                "copy_pages launch"))
            return rc;
    }
    return RESKV_OK;
}
