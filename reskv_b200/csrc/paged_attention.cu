// One query token of every sequence against its pages of the 4-bit cache.
//
// out[h] = sum_j softmax_j(q_h . k_j * scaling) v_j with k_j = offset + scale * code per group of 64 coordinates, v_j the same.
// The codes go to the tensor cores as they are: four bits in a 16-bit lane are a subnormal FP16 number, code * 2^-24 in the low
// nibble, code * 2^-20 in the next one, exactly; scales and offsets enter outside of the product,
//     q . k_j   = sum_groups scale_j,g * (q_g . code_j,g) + offset_j,g * sum(q_g)
//     sum p v   = sum_j (p_j scale_j,g) code_j,g + sum_j p_j offset_j,g
// with p * scale rounded to FP16 once as the product's operand.  Bound by the cache's bytes as long as a token costs less than
// its 144 bytes take to arrive.
//
// Work: the pages of all (sequence, KV head) units lie end to end and every CTA takes an equal share; a unit that lies in one
// CTA is finished there, the parts of the others are added by a second kernel.  Eight warps take a segment's blocks of 16 tokens
// in turn, each through a ring of its own (one bulk copy of 2304 bytes per block) with a running softmax of its own; they meet
// in shared memory at a segment's end.
#include "paged_int4.cuh"

namespace reskv {
namespace {

constexpr int kPaWarps = 8;
constexpr int kPaThreads = kPaWarps * 32;
constexpr int kPaStages = 4;
constexpr int kPaPerSm = 2;                       // CTAs of an SM
constexpr int kPaLeast = 2;                       // pages of a share, at least: one block for every warp
constexpr int kPaSumBytes = kPaWarps * kPagedGroup * kHeadDim * 4;
constexpr int kPaSmem = kPaWarps * kPaStages * kBlockBytes + kPaSumBytes;
constexpr int kPartialFloats = kPagedGroup * (kHeadDim + 2);  // of a part: outputs [8][128], maxima [8], sums [8]

struct PagedParams {
    const unsigned char* pages;  // of the layer
    int page_count;
    const int *table, *lengths;
    int sequences, width, heads, group;
    const unsigned short* q;
    int64_t q_sequence, q_head;  // elements
    float scale_log2;
    unsigned short* out;         // [sequences, heads * group, 128]
    float* lse;                  // [sequences, heads * group] or null
    float* parts;                // two per CTA
    int ctas;
    uint32_t* status;
};

__device__ __forceinline__ int length_of(const PagedParams& p, int s) {
    const int n = p.lengths[s], most = p.width * kPageTokens;
    return n < 0 ? 0 : n > most ? most : n;
}
__device__ __forceinline__ int pages_of(int length) { return (length + kPageTokens - 1) / kPageTokens; }

// How the pages of all units, laid end to end, are dealt out; the same for both kernels.
struct Shares {
    int64_t pages;
    int ctas;
    __device__ __forceinline__ int64_t begin(int cta) const { return cta * pages / ctas; }
    __device__ __forceinline__ int owner(int64_t page) const { return static_cast<int>(((page + 1) * ctas - 1) / pages); }
};
__device__ __forceinline__ Shares shares_of(const PagedParams& p, int lane) {
    int64_t n = 0;
    for (int s = lane; s < p.sequences; s += 32) n += pages_of(length_of(p, s));
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) n += __shfl_xor_sync(0xffffffffu, n, off);
    n *= p.heads;
    const int64_t most = (n + kPaLeast - 1) / kPaLeast;
    return {n, static_cast<int>(most < p.ctas ? most : p.ctas)};
}

// A unit's consecutive pages inside a share, one segment after the other.
struct Segments {
    int sequence, head, length, first, last;
    int64_t left;  // pages of the share behind this segment
    // The segment that holds page `page` of all; whole warp.
    __device__ __forceinline__ void start(const PagedParams& p, int64_t page, int64_t count, int lane) {
        int64_t before = 0;
        for (int s0 = 0; s0 < p.sequences; s0 += 32) {
            const int n = s0 + lane < p.sequences ? length_of(p, s0 + lane) : 0;
            const int64_t mine = static_cast<int64_t>(pages_of(n)) * p.heads;
            int64_t upto = mine;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int64_t other = __shfl_up_sync(0xffffffffu, upto, off);
                if (lane >= off) upto += other;
            }
            const uint32_t mask = __ballot_sync(0xffffffffu, before + upto > page);
            if (mask) {
                const int owner = __ffs(mask) - 1;
                length = __shfl_sync(0xffffffffu, n, owner);
                const int64_t at = page - (before + __shfl_sync(0xffffffffu, upto - mine, owner));
                const int per = pages_of(length);
                sequence = s0 + owner, head = static_cast<int>(at / per), first = static_cast<int>(at - static_cast<int64_t>(head) * per);
                last = static_cast<int64_t>(per - first) < count ? per : first + static_cast<int>(count);
                left = count - (last - first);
                return;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
        left = -1;  // not reached: the page lies in some sequence
    }
    __device__ __forceinline__ bool next(const PagedParams& p) {
        if (left <= 0) return false;
        if (++head == p.heads) {
            head = 0;
            do {
                if (++sequence >= p.sequences) return false;
                length = length_of(p, sequence);
            } while (length == 0);
        }
        first = 0;
        const int per = pages_of(length);
        last = per < left ? per : static_cast<int>(left);
        left -= last;
        return true;
    }
    __device__ __forceinline__ int first_block() const { return first * (kPageTokens / kBlockTokens); }
    __device__ __forceinline__ int last_block() const {
        const int all = (length + kBlockTokens - 1) / kBlockTokens, end = last * (kPageTokens / kBlockTokens);
        return all < end ? all : end;
    }
};

__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127
__device__ __forceinline__ int exponent_of(float x) { return static_cast<int>(__float_as_uint(x) >> 23 & 255u) - 127; }
__device__ __forceinline__ int clamped(int x, int low, int high) { return x < low ? low : x > high ? high : x; }

__device__ __forceinline__ void ctas_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kPaThreads) : "memory"); }

template <bool BF16>
__device__ __forceinline__ uint32_t larger_pair(uint32_t a, uint32_t b) {
    uint32_t r;
    if (BF16)
        asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else
        asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

template <bool BF16>
__global__ void __launch_bounds__(kPaThreads, kPaPerSm) paged_attention_kernel(const PagedParams p) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ uint64_t bar_full[kPaWarps][kPaStages];
    __shared__ float s_max[kPaWarps][kPagedGroup], s_sum[kPaWarps][kPagedGroup], s_top[kPagedGroup];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    unsigned char* ring = smem + warp * kPaStages * kBlockBytes;
    float* sums = reinterpret_cast<float*>(smem + kPaWarps * kPaStages * kBlockBytes);  // [warp][head][128]
    if (lane == 0) {
        for (int s = 0; s < kPaStages; ++s) mbar_init(&bar_full[warp][s], 1);
        mbar_fence_init();
    }
    __syncwarp();
    wait_for_previous_launch();
    let_next_launch_start();
    const Shares shares = shares_of(p, lane);
    if (static_cast<int>(blockIdx.x) >= shares.ctas) return;
    const int64_t begin = shares.begin(blockIdx.x), count = shares.begin(blockIdx.x + 1) - begin;
    Segments at;  // being worked on
    at.start(p, begin, count, lane);
    Segments ahead = at;  // being requested
    int ahead_block = ahead.first_block() + warp, ahead_end = ahead.last_block();
    bool more = true, lost = false;
    int page = -1;
    const auto look = [&] {  // the page of the block that is requested next
        while (more && ahead_block >= ahead_end) {
            more = ahead.next(p);
            ahead_block = ahead.first_block() + warp, ahead_end = ahead.last_block();
        }
        if (more) page = p.table[static_cast<int64_t>(ahead.sequence) * p.width + ahead_block / (kPageTokens / kBlockTokens)];
    };
    const auto request = [&](int stage) {
        if (!more) return;
        if (page < 0 || page >= p.page_count) {
            if (lane == 0) atomicOr(p.status, RESKV_STATUS_STATE_RANGE);
            page = 0;
        }
        if (lane == 0) {
            mbar_arrive_expect_tx(&bar_full[warp][stage], kBlockBytes);
            bulk_g2s(ring + stage * kBlockBytes, p.pages + (static_cast<int64_t>(page) * p.heads + ahead.head) * kPageHeadBytes +
                                                     (ahead_block & (kPageTokens / kBlockTokens - 1)) * kBlockBytes,
                     kBlockBytes, &bar_full[warp][stage]);
        }
        ahead_block += kPaWarps;
        look();
    };
    look();
#pragma unroll
    for (int s = 0; s < kPaStages; ++s) request(s);

    // rows of a block that this lane's columns 2t, 2t + 1 of the scores stand for: a score tile's column n is row
    // n / 2 (n even) or 4 + (n / 2 ^ 1) (n odd) of its eight
    const int row_even = t, row_odd = 4 + (t ^ 1), key_row = (g >> 1) ^ (g & 1 ? 5 : 0);
    int stage = 0, phase = 0;
    bool first_segment = true;
    for (bool any = true; any; any = at.next(p), first_segment = false) {
        // ---- the query: head g's coordinates 32 j + 8 t .. + 7, scaled by a power of two that makes the largest about 2^9 ------
        uint32_t q_low[4][2], q_high[4][2];
        float q_sum[2] = {0.f, 0.f}, q_scale;
        {
            float v[4][8], top = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint4 raw = make_uint4(0, 0, 0, 0);
                if (g < p.group)
                    raw = *reinterpret_cast<const uint4*>(p.q + at.sequence * p.q_sequence + (at.head * p.group + g) * p.q_head + 32 * j + 8 * t);
                const uint32_t* pairs = reinterpret_cast<const uint32_t*>(&raw);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[j][2 * e] = low_of<BF16>(pairs[e]), v[j][2 * e + 1] = high_of<BF16>(pairs[e]);
                    top = fmaxf(top, fmaxf(fabsf(v[j][2 * e]), fabsf(v[j][2 * e + 1])));
                    q_sum[j >> 1] += v[j][2 * e] + v[j][2 * e + 1];
                }
            }
#pragma unroll
            for (int off = 1; off < 4; off <<= 1) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
                q_sum[0] += __shfl_xor_sync(0xffffffffu, q_sum[0], off);
                q_sum[1] += __shfl_xor_sync(0xffffffffu, q_sum[1], off);
            }
            const int up = clamped(9 - exponent_of(top), -118, 100);
            const float by = power_of_two(up);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {  // coordinates 2e, 2e + 4: low nibbles of the codes; 2e + 1, 2e + 5: the next ones
                    q_low[j][e] = pack2<false>(v[j][2 * e] * by, v[j][2 * e + 4] * by);
                    q_high[j][e] = pack2<false>(v[j][2 * e + 1] * by * 0.0625f, v[j][2 * e + 5] * by * 0.0625f);
                }
            q_scale = p.scale_log2 * power_of_two(24) / by;
            q_sum[0] *= p.scale_log2, q_sum[1] *= p.scale_log2;
        }

        float m = -INFINITY, l = 0.f, flat[2] = {0.f, 0.f};  // of head g: maximum, sum, sum of p * offset
        float acc[8][4];                                    // outputs: rows = coordinates, columns = heads 2t, 2t + 1
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
        float value_scale = 1.f, scale_limit = -1.f;        // p * scale * value_scale stays in FP16's range up to that scale
        const int end = at.last_block();
        for (int block = at.first_block() + warp; block < end; block += kPaWarps) {
            if (!lost) lost = !mbar_wait(&bar_full[warp][stage], phase);
            const unsigned char* keys = ring + stage * kBlockBytes;
            const unsigned char* values = keys + kBlockSide;
            // ---- scores of 2 x 8 tokens ---------------------------------------------------------------------------------
            float s[2][2];
            const int tokens = at.length - block * kBlockTokens;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint4 w = *reinterpret_cast<const uint4*>(keys + (8 * i + key_row) * 64 + 16 * t);
                const uint32_t words[4] = {w.x, w.y, w.z, w.w};
                float c[2][4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float(&d)[4] = c[j >> 1];
                    if ((j & 1) == 0) d[0] = d[1] = d[2] = d[3] = 0.f;
                    const uint32_t next = words[j] >> 8;
                    mma_16816(d, q_low[j][0], 0u, q_high[j][0], 0u, words[j] & 0x000F000Fu, words[j] & 0x00F000F0u);
                    mma_16816(d, q_low[j][1], 0u, q_high[j][1], 0u, next & 0x000F000Fu, next & 0x00F000F0u);
                }
                const unsigned char* params = keys + kBlockCodes + 64 * i;
                const uint2 even = *reinterpret_cast<const uint2*>(params + 8 * row_even), odd = *reinterpret_cast<const uint2*>(params + 8 * row_odd);
                s[i][0] = (c[0][0] * low_of<BF16>(even.x) + c[1][0] * high_of<BF16>(even.x)) * q_scale +
                          (q_sum[0] * low_of<BF16>(even.y) + q_sum[1] * high_of<BF16>(even.y));
                s[i][1] = (c[0][1] * low_of<BF16>(odd.x) + c[1][1] * high_of<BF16>(odd.x)) * q_scale +
                          (q_sum[0] * low_of<BF16>(odd.y) + q_sum[1] * high_of<BF16>(odd.y));
            }
            uint2 params[2][2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                params[i][0] = *reinterpret_cast<const uint2*>(values + kBlockCodes + 8 * (8 * i + row_even));
                params[i][1] = *reinterpret_cast<const uint2*>(values + kBlockCodes + 8 * (8 * i + row_odd));
            }
            if (tokens < kBlockTokens) {  // behind the sequence's end: whatever lies there counts for nothing
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        if (8 * i + (e ? row_odd : row_even) >= tokens) s[i][e] = -INFINITY, params[i][e] = make_uint2(0, 0);
            }
            // ---- running softmax --------------------------------------------------------------------------------------------
            float top = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            if (__any_sync(0xffffffffu, top > m)) {
                const float next = fmaxf(m, top), factor = m == next ? 1.f : fast_exp2(m - next);
                m = next, l *= factor, flat[0] *= factor, flat[1] *= factor;
                const float f0 = __shfl_sync(0xffffffffu, factor, 8 * t), f1 = __shfl_sync(0xffffffffu, factor, 8 * t + 4);
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[i][0] *= f0, acc[i][1] *= f1, acc[i][2] *= f0, acc[i][3] *= f1;
            }
            // ---- the scales of the values: a power of two keeps p * scale where FP16 is exact to half a step -------------------
            {
                const uint32_t pair = larger_pair<BF16>(larger_pair<BF16>(params[0][0].x, params[0][1].x), larger_pair<BF16>(params[1][0].x, params[1][1].x));
                float most = fmaxf(low_of<BF16>(pair), high_of<BF16>(pair));
                if (__any_sync(0xffffffffu, most > scale_limit)) {
                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                    const int e = clamped(exponent_of(most), -100, 126);
                    const float now = power_of_two(14 - e > 126 ? 126 : 14 - e), change = scale_limit < 0.f ? 0.f : now / value_scale;
                    value_scale = now, scale_limit = power_of_two(e + 1 > 127 ? 127 : e + 1);
                    if (scale_limit < 0.f) scale_limit = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) acc[i][0] *= change, acc[i][1] *= change, acc[i][2] *= change, acc[i][3] *= change;
                }
            }
            uint32_t weights[2][2];  // [group][half of the tokens]
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float p0 = fast_exp2(s[i][0] - m), p1 = fast_exp2(s[i][1] - m);
                l += p0 + p1;
                const float n0 = p0 * value_scale, n1 = p1 * value_scale;
                weights[0][i] = pack2<false>(n0 * low_of<BF16>(params[i][0].x), n1 * low_of<BF16>(params[i][1].x));
                weights[1][i] = pack2<false>(n0 * high_of<BF16>(params[i][0].x), n1 * high_of<BF16>(params[i][1].x));
                flat[0] = fmaf(p0, low_of<BF16>(params[i][0].y), fmaf(p1, low_of<BF16>(params[i][1].y), flat[0]));
                flat[1] = fmaf(p0, high_of<BF16>(params[i][0].y), fmaf(p1, high_of<BF16>(params[i][1].y), flat[1]));
            }
            // ---- outputs ------------------------------------------------------------------------------------------------------
            uint2 rows[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = 8 * (i >> 1) + (i & 1 ? row_odd : row_even);
                rows[i] = *reinterpret_cast<const uint2*>(values + row * 64 + 8 * (g ^ ((row >> 1 & 1) << 2)));
            }
#pragma unroll
            for (int group = 0; group < 2; ++group)
#pragma unroll
                for (int half = 0; half < 2; ++half) {  // bytes 0, 1 and 2, 3 of the words
                    const uint32_t pick = half ? 0x7632u : 0x5410u;
                    const uint32_t a = __byte_perm(group ? rows[0].y : rows[0].x, group ? rows[1].y : rows[1].x, pick);
                    const uint32_t b = __byte_perm(group ? rows[2].y : rows[2].x, group ? rows[3].y : rows[3].x, pick);
                    const uint32_t a8 = a >> 8, b8 = b >> 8;
                    mma_16816(acc[group * 4 + half * 2], a & 0x000F000Fu, a & 0x00F000F0u, b & 0x000F000Fu, b & 0x00F000F0u, weights[group][0], weights[group][1]);
                    mma_16816(acc[group * 4 + half * 2 + 1], a8 & 0x000F000Fu, a8 & 0x00F000F0u, b8 & 0x000F000Fu, b8 & 0x00F000F0u, weights[group][0], weights[group][1]);
                }
            __syncwarp();
            request(stage);
            if (++stage == kPaStages) stage = 0, phase ^= 1;
        }
        // ---- the warps' parts of the segment ------------------------------------------------------------------------------------
#pragma unroll
        for (int off = 1; off < 4; off <<= 1) {
            l += __shfl_xor_sync(0xffffffffu, l, off);
            flat[0] += __shfl_xor_sync(0xffffffffu, flat[0], off), flat[1] += __shfl_xor_sync(0xffffffffu, flat[1], off);
        }
        if (t == 0) s_max[warp][g] = m;
        ctas_sync();
        const int active = min(kPaWarps, end - at.first_block());
        float top = s_max[0][g];
        for (int w = 1; w < active; ++w) top = fmaxf(top, s_max[w][g]);
        if (warp < active) {
            const float weight = m == top ? 1.f : fast_exp2(m - top);
            if (t == 0) s_sum[warp][g] = l * weight;
            const float w0 = __shfl_sync(0xffffffffu, weight, 8 * t), w1 = __shfl_sync(0xffffffffu, weight, 8 * t + 4);
            float flats[2][2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
                flats[i][0] = __shfl_sync(0xffffffffu, flat[i], 8 * t), flats[i][1] = __shfl_sync(0xffffffffu, flat[i], 8 * t + 4);
            const float unit = 1.f / value_scale;
            float* mine = sums + warp * kPagedGroup * kHeadDim;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int d = (i >> 2) * 64 + 8 * g + (i & 3) * 2;
                constexpr float low = 1 << 24, high = 1 << 20;  // of codes in the low and in the next nibbles
                if (2 * t < p.group)
                    *reinterpret_cast<float2*>(mine + 2 * t * kHeadDim + d) =
                        make_float2(fmaf(acc[i][0] * low, unit, flats[i >> 2][0]) * w0, fmaf(acc[i][2] * high, unit, flats[i >> 2][0]) * w0);
                if (2 * t + 1 < p.group)
                    *reinterpret_cast<float2*>(mine + (2 * t + 1) * kHeadDim + d) =
                        make_float2(fmaf(acc[i][1] * low, unit, flats[i >> 2][1]) * w1, fmaf(acc[i][3] * high, unit, flats[i >> 2][1]) * w1);
            }
        }
        if (warp == 0 && t == 0) s_top[g] = top;
        ctas_sync();
        const bool whole = at.first == 0 && at.last == pages_of(at.length);
        float* part = p.parts + (2 * static_cast<int64_t>(blockIdx.x) + (first_segment ? 0 : 1)) * kPartialFloats;
        for (int i = threadIdx.x * 4; i < p.group * kHeadDim; i += kPaThreads * 4) {
            const int head = i / kHeadDim;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
            float total = 0.f;
            for (int w = 0; w < active; ++w) {
                const float4 x = *reinterpret_cast<const float4*>(sums + w * kPagedGroup * kHeadDim + i);
                sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
                total += s_sum[w][head];
            }
            if (whole) {
                const float inv = 1.f / total;
                const int64_t row = static_cast<int64_t>(at.sequence) * p.heads * p.group + at.head * p.group;
                *reinterpret_cast<uint2*>(p.out + row * kHeadDim + i) =
                    make_uint2(pack2<BF16>(sum.x * inv, sum.y * inv), pack2<BF16>(sum.z * inv, sum.w * inv));
                if (p.lse && i % kHeadDim == 0) p.lse[row + head] = s_top[head] * kLn2 + logf(total);
            } else {
                *reinterpret_cast<float4*>(part + i) = sum;
                if (i % kHeadDim == 0) part[kPagedGroup * kHeadDim + head] = s_top[head], part[kPagedGroup * (kHeadDim + 1) + head] = total;
            }
        }
        // the next segment's sums and s_top are written behind its first barrier
    }
    if (lost) {  // no copy may land after the block's end
        for (int s = 0; s < kPaStages; ++s) mbar_wait(&bar_full[warp][s], s < stage ? phase ^ 1 : phase);
        if (lane == 0) atomicOr(p.status, RESKV_STATUS_WAIT_TIMEOUT);
    }
}

// Adds the parts of a unit that lies in several CTAs; a unit without tokens gets zeros.  Warp = query head.
template <bool BF16>
__global__ void __launch_bounds__(kPagedGroup * 32) paged_merge_kernel(const PagedParams p) {
    const int lane = threadIdx.x & 31, head = threadIdx.x >> 5, unit = blockIdx.x;
    wait_for_previous_launch();
    let_next_launch_start();
    const int sequence = unit / p.heads, kv_head = unit - sequence * p.heads;
    const int length = length_of(p, sequence);
    const int64_t row = static_cast<int64_t>(sequence) * p.heads * p.group + kv_head * p.group + head;
    if (length == 0) {
        *reinterpret_cast<uint2*>(p.out + row * kHeadDim + 4 * lane) = make_uint2(0, 0);
        if (p.lse && lane == 0) p.lse[row] = -INFINITY;
        return;
    }
    const Shares shares = shares_of(p, lane);
    int64_t before = 0;
    for (int s = lane; s < sequence; s += 32) before += pages_of(length_of(p, s));
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) before += __shfl_xor_sync(0xffffffffu, before, off);
    const int per = pages_of(length);
    const int64_t a = before * p.heads + static_cast<int64_t>(kv_head) * per;
    const int from = shares.owner(a), to = shares.owner(a + per - 1);
    if (from == to) return;
    const int count = to - from + 1;
    const int skip = shares.begin(from) == a ? 0 : 1;  // the unit begins behind another one in its first CTA: that CTA's second part
    const float* parts = p.parts + 2 * static_cast<int64_t>(from) * kPartialFloats;
    const auto part = [&](int i) { return parts + (2 * i + (i == 0 ? skip : 0)) * kPartialFloats; };
    float top = -INFINITY;
    for (int i = lane; i < count; i += 32) top = fmaxf(top, part(i)[kPagedGroup * kHeadDim + head]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float total = 0.f;
#pragma unroll 8
    for (int i = 0; i < count; ++i) {
        const float* from_part = part(i);
        const float m = from_part[kPagedGroup * kHeadDim + head], l = from_part[kPagedGroup * (kHeadDim + 1) + head];
        const float4 x = *reinterpret_cast<const float4*>(from_part + head * kHeadDim + 4 * lane);
        const float weight = m == top ? 1.f : fast_exp2(m - top);
        sum.x = fmaf(x.x, weight, sum.x), sum.y = fmaf(x.y, weight, sum.y), sum.z = fmaf(x.z, weight, sum.z), sum.w = fmaf(x.w, weight, sum.w);
        total = fmaf(l, weight, total);
    }
    const float inv = 1.f / total;
    *reinterpret_cast<uint2*>(p.out + row * kHeadDim + 4 * lane) =
        make_uint2(pack2<BF16>(sum.x * inv, sum.y * inv), pack2<BF16>(sum.z * inv, sum.w * inv));
    if (p.lse && lane == 0) p.lse[row] = top * kLn2 + logf(total);
}

// CTAs of the first kernel for as many pages as there may be.
int paged_ctas(int sequences, int width, int heads) {
    const int64_t most = (static_cast<int64_t>(sequences) * width * heads + kPaLeast - 1) / kPaLeast, room = kPaPerSm * sm_count();
    return static_cast<int>(most < room ? most : room);
}

template <bool BF16>
int launch(const PagedParams& p, cudaStream_t stream) {
    static std::atomic<unsigned long long> done{0};
    if (int rc = allow_smem(paged_attention_kernel<BF16>, kPaSmem, done, "cudaFuncSetAttribute(paged_attention)")) return rc;
    if (p.ctas > 0)
        if (int rc = check_cuda(launch_overlapped(paged_attention_kernel<BF16>, dim3(static_cast<unsigned>(p.ctas)), kPaThreads, kPaSmem, stream, true, p),
                                "paged_attention launch"))
            return rc;
    return check_cuda(launch_overlapped(paged_merge_kernel<BF16>, dim3(static_cast<unsigned>(p.sequences * p.heads)), p.group * 32, 0, stream, true, p),
                      "paged_attention merge launch");
}

}  // namespace
}  // namespace reskv

using namespace reskv;

extern "C" size_t reskv_paged_attention_workspace_bytes(int sequences, int width, int kv_heads) {
    if (sequences < 0 || width < 0 || kv_heads < 1) return 0;
    return static_cast<size_t>(paged_ctas(sequences, width, kv_heads)) * 2 * kPartialFloats * sizeof(float) + 256;
}

extern "C" int reskv_paged_attention(const void* q, int bf16, int64_t q_sequence, int64_t q_head, const int32_t* lengths, const int32_t* table,
                                     int sequences, int width, int kv_heads, int q_heads, const void* pages, int page_count, float scaling,
                                     void* workspace, size_t workspace_bytes, void* out, float* lse, uint32_t* status, void* stream) {
    if (sequences < 0 || width < 0 || kv_heads < 1 || q_heads < 1 || q_heads % kv_heads || page_count < 0)
        return fail(RESKV_ERR_INVALID, "paged_attention: %d sequences, table of %d pages, %d KV and %d query heads, %d pages", sequences, width,
                    kv_heads, q_heads, page_count);
    if (q_heads / kv_heads > kPagedGroup) return fail(RESKV_ERR_LIMIT, "paged_attention: more than %d query heads per KV head", kPagedGroup);
    if (!(scaling > 0.f) || !(scaling < 3.0e38f)) return fail(RESKV_ERR_INVALID, "paged_attention: scaling must be positive and finite");
    if (static_cast<int64_t>(sequences) * kv_heads > 0x7fffffff || width > (1 << 24))
        return fail(RESKV_ERR_LIMIT, "paged_attention: %d sequences of up to %d pages", sequences, width);
    if (sequences == 0) return RESKV_OK;
    if (!q || !lengths || !out || !status || (width > 0 && (!table || !pages))) return fail(RESKV_ERR_INVALID, "paged_attention: null pointer");
    if (width > 0 && page_count == 0) return fail(RESKV_ERR_INVALID, "paged_attention: a table, but no pages");
    if (!aligned16(q) || !aligned16(out) || !aligned16(pages) || !aligned16(workspace) || q_sequence % 8 || q_head % 8 || q_sequence < 0 || q_head < 0)
        return fail(RESKV_ERR_INVALID, "paged_attention: q, out, pages and workspace must start on 16-byte boundaries, q's strides be multiples of 8 elements");
    if (!workspace || workspace_bytes < reskv_paged_attention_workspace_bytes(sequences, width, kv_heads))
        return fail(RESKV_ERR_WORKSPACE, "paged_attention: workspace of %zu bytes, needs %zu", workspace_bytes,
                    reskv_paged_attention_workspace_bytes(sequences, width, kv_heads));
    if (int rc = check_device_pointer(q, "paged_attention", "q")) return rc;
    if (int rc = check_device_pointer(lengths, "paged_attention", "lengths")) return rc;
    if (int rc = check_device_pointer(workspace, "paged_attention", "workspace")) return rc;
    if (int rc = check_device_pointer(out, "paged_attention", "out")) return rc;
    if (width > 0) {
        if (int rc = check_device_pointer(table, "paged_attention", "table")) return rc;
        if (int rc = check_device_pointer(pages, "paged_attention", "pages")) return rc;
    }
    PagedParams p{};
    p.pages = static_cast<const unsigned char*>(pages), p.page_count = page_count, p.table = table, p.lengths = lengths;
    p.sequences = sequences, p.width = width, p.heads = kv_heads, p.group = q_heads / kv_heads;
    p.q = static_cast<const unsigned short*>(q), p.q_sequence = q_sequence, p.q_head = q_head, p.scale_log2 = scaling * kLog2e;
    p.out = static_cast<unsigned short*>(out), p.lse = lse, p.parts = static_cast<float*>(workspace);
    p.ctas = paged_ctas(sequences, width, kv_heads), p.status = status;
    return bf16 ? launch<true>(p, static_cast<cudaStream_t>(stream)) : launch<false>(p, static_cast<cudaStream_t>(stream));
}
