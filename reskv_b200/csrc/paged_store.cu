// The 4-bit paged cache takes tokens, gives them back, and moves pages.
//
// Storing: of a token's vector of one head, every group of 64 coordinates becomes offset = min, scale = (max - min) / 15
// rounded to the model's type, code = round((x - offset) / scale) to the nearest, ties to even, at most 15 (0 where the scale
// is 0).  512 bytes of K and V become 144.  Bound by bytes: half a warp holds a row (16 bytes a lane), the other half the same
// row of the other side; extremes meet in three shuffles, every lane writes the word of its eight coordinates.  Several rows
// are requested before the first is used.
#include <algorithm>
#include <new>
#include <vector>

#include "paged_int4.cuh"

namespace reskv {
namespace {

constexpr int kRowsAtOnce = 4;       // (token, head) rows of a warp that are in flight together
constexpr int kStoreThreads = 256;

struct StoreParams {
    PagedPlace at;
    unsigned char* pages;            // of the layer
    const unsigned short *k, *v;     // write: sources
    unsigned short *k_out, *v_out;   // read: destinations [total, heads, 128]
    int64_t k_token, k_head, v_token, v_head;  // elements
    int total, heads;
    uint32_t* status;
};

// Sequence of token i and its number in it; false: in none.  Whole warp.
__device__ __forceinline__ bool place_of(const PagedPlace& at, int token, int lane, int& sequence, int& number) {
    int before = 0;  // ends that lie at the token or in front of it
    for (int s = lane; s < at.sequences; s += 32) before += at.cu[s + 1] <= token;
    sequence = __reduce_add_sync(0xffffffffu, before);
    if (sequence >= at.sequences) return false;
    number = at.starts[sequence] + token - at.cu[sequence];
    return token >= at.cu[sequence];
}

// Block of the pool that holds token `number` of a sequence for one head, and its row there; null (and a status bit): outside
// the table or the pool.
__device__ __forceinline__ unsigned char* block_of(const StoreParams& p, int sequence, int number, int head, int lane) {
    const int slot = number / kPageTokens;
    const bool inside = number >= 0 && slot < p.at.width;
    const int page = inside ? p.at.table[static_cast<int64_t>(sequence) * p.at.width + slot] : -1;
    if (page < 0 || page >= p.at.pages) {
        if (lane == 0) atomicOr(p.status, RESKV_STATUS_STATE_RANGE);
        return nullptr;
    }
    return p.pages + (static_cast<int64_t>(page) * p.heads + head) * kPageHeadBytes + (number / kBlockTokens & 3) * kBlockBytes;
}

__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

template <bool BF16, bool WRITE>
__global__ void __launch_bounds__(kStoreThreads) paged_store_kernel(const StoreParams p) {
    wait_for_previous_launch();
    let_next_launch_start();
    const int lane = threadIdx.x & 31, side = lane >> 4, c = lane & 15;
    const int64_t rows = static_cast<int64_t>(p.total) * p.heads;
    const int64_t first = (static_cast<int64_t>(blockIdx.x) * (kStoreThreads / 32) + (threadIdx.x >> 5)) * kRowsAtOnce;
    if (first >= rows) return;
    int token = static_cast<int>(first / p.heads), head = static_cast<int>(first - static_cast<int64_t>(token) * p.heads);
    unsigned char* row_at[kRowsAtOnce];
    int block_row[kRowsAtOnce];
    uint4 x[kRowsAtOnce];
    int tokens[kRowsAtOnce], heads[kRowsAtOnce];
    if (WRITE) {
        int t = token, h = head;
#pragma unroll
        for (int r = 0; r < kRowsAtOnce; ++r) {
            if (first + r < rows)
                x[r] = *reinterpret_cast<const uint4*>(side ? p.v + t * p.v_token + h * p.v_head + 8 * c : p.k + t * p.k_token + h * p.k_head + 8 * c);
            if (++h == p.heads) h = 0, ++t;
        }
    }
    int known = -1, sequence = 0, number = 0;
    bool placed = false;
#pragma unroll
    for (int r = 0; r < kRowsAtOnce; ++r) {
        row_at[r] = nullptr;
        tokens[r] = token, heads[r] = head;
        if (first + r < rows) {
            if (token != known) placed = place_of(p.at, token, lane, sequence, number), known = token;
            if (placed) row_at[r] = block_of(p, sequence, number, head, lane);
            block_row[r] = number & (kBlockTokens - 1);
        }
        if (++head == p.heads) head = 0, ++token;
    }
    if (WRITE) {
#pragma unroll
        for (int r = 0; r < kRowsAtOnce; ++r) {
            if (!row_at[r]) continue;
            const uint32_t* pairs = reinterpret_cast<const uint32_t*>(&x[r]);
            float v[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[2 * e] = low_of<BF16>(pairs[e]), v[2 * e + 1] = high_of<BF16>(pairs[e]);
            float low = v[0], high = v[0];
#pragma unroll
            for (int e = 1; e < 8; ++e) low = min_nan(low, v[e]), high = max_nan(high, v[e]);
#pragma unroll
            for (int off = 1; off < 8; off <<= 1) {
                low = min_nan(low, __shfl_xor_sync(0xffffffffu, low, off));
                high = max_nan(high, __shfl_xor_sync(0xffffffffu, high, off));
            }
            const unsigned short scale_bits = narrow<BF16>((high - low) / 15.f);
            const float scale = widen<BF16>(scale_bits);
            uint32_t word = 0;
            const float inverse = __frcp_rn(scale);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                // by the reciprocal (off by less than 1e-5), unless that lies so near to a half that the quotient has to decide;
                // a NaN (of an infinite or NaN group) becomes 0 here: the group's values are NaN by its scale
                const float above = v[e] - low, quotient = above * inverse;
                float code = rintf(quotient);
                if (!(fabsf(quotient - code) <= 0.4999f)) code = rintf(above / scale);
                code = fminf(fmaxf(code, 0.f), 15.f);
                word |= (scale > 0.f ? static_cast<uint32_t>(code) : 0u) << (4 * e);
            }
            unsigned char* codes = row_at[r] + side * kBlockSide;
            *reinterpret_cast<uint32_t*>(codes + (side ? value_word(block_row[r], c) : key_word(block_row[r], c))) = word;
            if ((c & 7) == 0) {
                unsigned short* params = reinterpret_cast<unsigned short*>(codes + kBlockCodes + block_row[r] * 8);
                params[c >> 3] = scale_bits;
                params[2 + (c >> 3)] = narrow<BF16>(low);
            }
        }
    } else {
        uint32_t word[kRowsAtOnce];
        uint2 params[kRowsAtOnce];
#pragma unroll
        for (int r = 0; r < kRowsAtOnce; ++r) {
            if (!row_at[r]) continue;
            const unsigned char* codes = row_at[r] + side * kBlockSide;
            word[r] = *reinterpret_cast<const uint32_t*>(codes + (side ? value_word(block_row[r], c) : key_word(block_row[r], c)));
            params[r] = *reinterpret_cast<const uint2*>(codes + kBlockCodes + block_row[r] * 8);
        }
#pragma unroll
        for (int r = 0; r < kRowsAtOnce; ++r) {
            if (!row_at[r]) continue;
            const float scale = c < 8 ? low_of<BF16>(params[r].x) : high_of<BF16>(params[r].x);
            const float low = c < 8 ? low_of<BF16>(params[r].y) : high_of<BF16>(params[r].y);
            uint4 y;
            uint32_t* pairs = reinterpret_cast<uint32_t*>(&y);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                pairs[e] = pack2<BF16>(fmaf(scale, static_cast<float>(word[r] >> (8 * e) & 15u), low),
                                       fmaf(scale, static_cast<float>(word[r] >> (8 * e + 4) & 15u), low));
            *reinterpret_cast<uint4*>((side ? p.v_out : p.k_out) + (static_cast<int64_t>(tokens[r]) * p.heads + heads[r]) * 128 + 8 * c) = y;
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

template <bool WRITE>
int run_store(const StoreParams& p, int bf16, cudaStream_t stream) {
    const int64_t rows = static_cast<int64_t>(p.total) * p.heads, per = kRowsAtOnce * (kStoreThreads / 32), blocks = (rows + per - 1) / per;
    if (blocks > 0x7fffffff) return fail(RESKV_ERR_LIMIT, "paged cache: too many tokens for one call");
    const dim3 grid(static_cast<unsigned>(blocks));
    return check_cuda(bf16 ? launch_overlapped(paged_store_kernel<true, WRITE>, grid, kStoreThreads, 0, stream, true, p)
                           : launch_overlapped(paged_store_kernel<false, WRITE>, grid, kStoreThreads, 0, stream, true, p),
                      WRITE ? "paged_write launch" : "paged_read launch");
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
