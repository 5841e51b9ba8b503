// The 4-bit paged cache takes tokens, gives them back, and moves pages.
//
// Storing: of a token's vector of one head, every group of 64 coordinates becomes offset = min, scale = (max - min) / 15
// rounded to the model's type, code = round((x - offset) / scale) to the nearest, ties to even, at most 15 (0 where the scale
// is 0).  512 bytes of K and V become 144.  Bound by bytes, and close to that by instructions.  Eight lanes hold a row of one side,
// eight coordinates of either group each, four rows (K and V of two heads) to a warp; extremes of both groups travel together as
// 16-bit pairs; a code is the low bits of (x - offset) * (1 / scale) + 1.5 * 2^23, and only where that lies within 1e-5 of a half
// the division itself decides.  A block first looks up where its tokens go, while their rows are on the way.
//
// 8 x 4000 tokens, 8 heads: written in 53 us (168 MB, 3.2 TB/s, half of the copy rate; 150 instructions per token and head), read back
// in 33 us.  With half a warp to a row and the division always: 91 and 51 us.
#include <algorithm>
#include <new>
#include <vector>

#include "paged_int4.cuh"

namespace reskv {
namespace {

constexpr int kStoreWarps = 4, kStoreThreads = kStoreWarps * 32;
// Pairs of (token, head) rows of a warp that are in flight together, where there are enough of them.  8 x 4000 tokens, us written and
// read, pairs at 4 warps a block: 2 / 2 53.1 and 35.5, 4 / 4 54.8 and 32.9; at 8 warps 4 / 4 59.4 and 33.8, 8 / 8 73.4 and 37.0.
template <bool WRITE>
constexpr int kPairsAtOnce = WRITE ? 2 : 4;

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
    int low = 0, high = p.at.sequences;  // the number of sequences that end at the token or in front of it
    while (low < high) {
        const int mid = (low + high) >> 1;
        if (p.at.cu[mid + 1] <= token) low = mid + 1; else high = mid;
    }
    if (low >= p.at.sequences || token < p.at.cu[low]) return {-1, 0};
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
template <bool BF16>
__device__ __forceinline__ uint32_t codes_of(const uint4& x, float low, float scale) {
    constexpr float kRound = 12582912.f;  // 1.5 * 2^23: a sum with it is rounded to a whole number
    constexpr float kNormal = BF16 ? 0x1p-126f : 0x1p-14f;
    const uint32_t pairs[4] = {x.x, x.y, x.z, x.w};
    float inverse, far = 0.f;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(scale));
    const float2 minus_low = make_float2(-low, -low), inverses = make_float2(inverse, inverse), up = make_float2(kRound, kRound),
                 down = make_float2(-kRound, -kRound);
    float2 above[4];
    uint32_t word = 0;
#pragma unroll
    for (int e = 3; e >= 0; --e) {
        above[e] = add2(make_float2(low_of<BF16>(pairs[e]), high_of<BF16>(pairs[e])), minus_low);
        const float2 quotient = mul2(above[e], inverses), rounded = add2(quotient, up), whole = add2(rounded, down);
        const float2 off = fma2(whole, make_float2(-1.f, -1.f), quotient);
        far = max3_nan(far, fabsf(off.x), fabsf(off.y));
        word = (word * 16u + __float_as_uint(rounded.y)) * 16u + __float_as_uint(rounded.x);  // the constant part goes below
    }
    word -= 0x4B400000u * 0x11111111u;
    // By the reciprocal a quotient is off by less than 1e-5.  A quotient that near to a half, a scale that rounding has made much
    // smaller than it should be (below the normal numbers, 0) and what is not finite: by the division.
    if (far <= 0.49999f && scale >= kNormal) return word;
    word = 0;
#pragma unroll
    for (int e = 7; e >= 0; --e) {
        const float code = fminf(fmaxf(rintf((e & 1 ? above[e >> 1].y : above[e >> 1].x) / scale), 0.f), 15.f);  // a NaN becomes 0:
        word = word * 16u + (scale > 0.f ? static_cast<uint32_t>(code) : 0u);                                   // the scale says it
    }
    return word;
}

// x / 15 as IEEE division rounds it (x finite): the quotient by the reciprocal, corrected by its remainder.
__device__ __forceinline__ float fifteenth(float x) {
    constexpr float kInverse = 1.f / 15.f;
    const float q = x * kInverse;
    return fmaf(fmaf(-15.f, q, x), kInverse, q);
}

template <bool BF16, bool WRITE, int PAIRS>
__global__ void __launch_bounds__(kStoreThreads) paged_store_kernel(const StoreParams p) {
    constexpr int kRows = kStoreWarps * 2 * PAIRS;  // of a block
    __shared__ TokenPlace places[kRows];
    wait_for_previous_launch();
    let_next_launch_start();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, side = lane >> 3 & 1, c = lane & 7;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kRows;
    const int token0 = static_cast<int>(first / p.heads), head0 = static_cast<int>(first - static_cast<int64_t>(token0) * p.heads);
    // a warp's pairs of rows lie next to each other
    int token[PAIRS], head[PAIRS];
    uint4 x[PAIRS][2];
    {
        const int row = warp * PAIRS * 2 + (lane >> 4);
        int t = token0 + (head0 + row) / p.heads, h = (head0 + row) % p.heads;
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            token[i] = t < p.total ? t : -1, head[i] = h;
            if (WRITE && token[i] >= 0) {
                const uint4* from = reinterpret_cast<const uint4*>(side ? p.v + t * p.v_token + h * p.v_head : p.k + t * p.k_token + h * p.k_head);
                x[i][0] = from[c], x[i][1] = from[8 + c];
            }
            for (h += 2; h >= p.heads; h -= p.heads) ++t;
        }
    }
    for (int i = threadIdx.x; i < kRows && token0 + i < p.total && i <= (head0 + kRows - 1) / p.heads; i += kStoreThreads)
        places[i] = place_of(p, token0 + i);
    __syncthreads();
    unsigned char* block[PAIRS];  // of the row's side, or null
    int row[PAIRS];
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
        block[i] = nullptr, row[i] = 0;
        if (token[i] < 0) continue;
        const TokenPlace to = places[token[i] - token0];
        if (to.block >= 0) block[i] = p.pages + to.block + static_cast<int64_t>(head[i]) * kPageHeadBytes + side * kBlockSide;
        row[i] = to.row;
    }
    if (WRITE) {
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            // (group 0, group 1) extremes; rows without a place take part in the exchange with whatever they hold
            if (token[i] < 0) x[i][0] = x[i][1] = make_uint4(0, 0, 0, 0);
            uint32_t top[2], bottom[2];
#pragma unroll
            for (int group = 0; group < 2; ++group) {
                const uint4& v = x[i][group];
                top[group] = max_pair<BF16>(max_pair<BF16>(v.x, v.y), max_pair<BF16>(v.z, v.w));
                bottom[group] = min_pair<BF16>(min_pair<BF16>(v.x, v.y), min_pair<BF16>(v.z, v.w));
            }
            uint32_t high = max_pair<BF16>(__byte_perm(top[0], top[1], 0x5410), __byte_perm(top[0], top[1], 0x7632));
            uint32_t low = min_pair<BF16>(__byte_perm(bottom[0], bottom[1], 0x5410), __byte_perm(bottom[0], bottom[1], 0x7632));
#pragma unroll
            for (int off = 1; off < 8; off <<= 1) {
                high = max_pair<BF16>(high, __shfl_xor_sync(0xffffffffu, high, off));
                low = min_pair<BF16>(low, __shfl_xor_sync(0xffffffffu, low, off));
            }
            if (!block[i]) continue;
            const float low0 = low_of<BF16>(low), low1 = high_of<BF16>(low);
            const uint32_t scales = pack2<BF16>(fifteenth(low_of<BF16>(high) - low0), fifteenth(high_of<BF16>(high) - low1));
            const uint32_t w0 = codes_of<BF16>(x[i][0], low0, low_of<BF16>(scales)), w1 = codes_of<BF16>(x[i][1], low1, high_of<BF16>(scales));
            if (side) {
                *reinterpret_cast<uint2*>(block[i] + value_word(row[i], c)) = make_uint2(w0, w1);
            } else {
                *reinterpret_cast<uint32_t*>(block[i] + key_word(row[i], c)) = w0;
                *reinterpret_cast<uint32_t*>(block[i] + key_word(row[i], c + 8)) = w1;
            }
            if (c == 0) *reinterpret_cast<uint2*>(block[i] + kBlockCodes + row[i] * 8) = make_uint2(scales, low);
        }
    } else {
        uint2 words[PAIRS], params[PAIRS];
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            if (!block[i]) continue;
            if (side)
                words[i] = *reinterpret_cast<const uint2*>(block[i] + value_word(row[i], c));
            else
                words[i] = make_uint2(*reinterpret_cast<const uint32_t*>(block[i] + key_word(row[i], c)),
                                      *reinterpret_cast<const uint32_t*>(block[i] + key_word(row[i], c + 8)));
            params[i] = *reinterpret_cast<const uint2*>(block[i] + kBlockCodes + row[i] * 8);
        }
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            if (!block[i]) continue;
            uint4* to = reinterpret_cast<uint4*>((side ? p.v_out : p.k_out) + (static_cast<int64_t>(token[i]) * p.heads + head[i]) * 128);
#pragma unroll
            for (int group = 0; group < 2; ++group) {
                const float scale = group ? high_of<BF16>(params[i].x) : low_of<BF16>(params[i].x);
                const float low = group ? high_of<BF16>(params[i].y) : low_of<BF16>(params[i].y);
                const uint32_t word = group ? words[i].y : words[i].x;
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
                to[8 * group + c] = y;
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

template <bool BF16, bool WRITE, int PAIRS>
int launch_store(const StoreParams& p, cudaStream_t stream) {
    constexpr int per = kStoreWarps * 2 * PAIRS;
    const int64_t blocks = (static_cast<int64_t>(p.total) * p.heads + per - 1) / per;
    if (blocks > 0x7fffffff) return fail(RESKV_ERR_LIMIT, "paged cache: too many tokens for one call");
    return check_cuda(launch_overlapped(paged_store_kernel<BF16, WRITE, PAIRS>, dim3(static_cast<unsigned>(blocks)), kStoreThreads, 0, stream, true, p),
                      WRITE ? "paged_write launch" : "paged_read launch");
}
// One pair of rows per warp as long as that leaves SMs without a block.
template <bool WRITE>
int run_store(const StoreParams& p, int bf16, cudaStream_t stream) {
    const bool many = static_cast<int64_t>(p.total) * p.heads > static_cast<int64_t>(sm_count()) * kStoreWarps * 2;
    return bf16 ? many ? launch_store<true, WRITE, kPairsAtOnce<WRITE>>(p, stream) : launch_store<true, WRITE, 1>(p, stream)
                : many ? launch_store<false, WRITE, kPairsAtOnce<WRITE>>(p, stream) : launch_store<false, WRITE, 1>(p, stream);
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
