// One query token of every sequence against its pages of the 4-bit cache.
//
// out[h] = sum_j softmax_j(q_h . k_j * scaling) v_j with k_j = offset + scale * code per group of 64 coordinates, v_j the same.
// The codes go to the tensor cores as they are: four bits in a 16-bit lane are a subnormal FP16 number, code * 2^-24 in the low
// nibble, code * 2^-20 in the next one, exactly; scales and offsets enter outside of the product,
//     q . k_j   = sum_groups scale_j,g * (q_g . code_j,g) + offset_j,g * sum(q_g)
//     sum p v   = sum_j (p_j scale_j,g) (code_j,g - 8) + sum_j p_j (offset_j,g + 8 scale_j,g)
// with p * scale in FP16 as the product's operand, for FP16 models in two parts.
//
// 32 x 8128 tokens, 32 / 8 heads: 71 us for 300 MB, 4.2 TB/s (0.65 of the copy rate).  Neither bytes nor issue slots (57 %) nor a pipe
// (integer 48 %: masks and shifts that bring the codes into operands) are full: 20 instructions of a warp per token and KV head, most of
// them in chains, and the registers leave 16 warps an SM to cover them.  Small calls are bound by latency: one sequence of 300 tokens
// 6.9 us, of 8128 10.4 us, nine ragged BF16 ones with eight query heads 16 us (28 MB), of which two dependent launches, look-ups of
// lengths and pages, a copy, a chunk, two meetings of the warps and the merge follow one another.
//
// Work: the pages of all (sequence, KV head) units lie end to end and every CTA takes an equal share; a unit that lies in one
// CTA is finished there, the parts of the others are added by a second kernel.  Eight warps take a segment's chunks of 32 tokens
// in turn, each through a ring of its own (one bulk copy of 4608 bytes per chunk) with a running softmax of its own; they meet
// in shared memory at a segment's end.
#include <algorithm>

#include "paged_int4.cuh"

namespace reskv {
namespace {

constexpr int kPaWarps = 8;
constexpr int kPaThreads = kPaWarps * 32;
constexpr int kPaStages = 2;
constexpr int kChunkBlocks = 2, kChunkTokens = kChunkBlocks * kBlockTokens, kChunkBytes = kChunkBlocks * kBlockBytes;  // a warp's turn
constexpr int kPaPerSm = 2;                       // CTAs of an SM
constexpr int kPageChunks = kPageTokens / kChunkTokens;
// A segment costs as much as kPaCharge pages besides its own.  us at charges of 2, 5, 8, 12: nine ragged sequences 21.5, 18.0, 16.8,
// 17.5; 64 ragged ones 33.0, 26.1, 25.7, 26.6; 32 x 2000 tokens 26.4, 26.1, 25.7, 25.2.
constexpr int kPaCharge = 8;
// A share is at least two pages long, four or eight (one or two turns of the eight warps) where the average stretch of a unit is
// longer: parts cost time when they are added.  us at 2, 4, 8: 1 x 1000 tokens 7.0, 7.6, 8.7; 1 x 3000 9.1, 8.2, 9.1; 1 x 8128 11.3,
// 10.9, 10.2.
__host__ __device__ constexpr int least_share(int average) { return average > 90 ? 8 : average > 40 ? 4 : 2; }
constexpr int kPaMergeWarps = 16;                 // of a query head at most
constexpr int kPaSumBytes = kPaWarps * kPagedGroup * kHeadDim * 4;
constexpr int kPaSmem = kPaWarps * kPaStages * kChunkBytes + kPaSumBytes;
constexpr float kCodeMiddle = 8.f;
constexpr uint32_t kMiddleLow = 0x80088008u, kMiddleByte = 0x80888088u;  // pairs of -8 * 2^-24 and -(8 + 16 * 8) * 2^-24
constexpr int kPaSlack = 5;
constexpr float kPaNear = 8192.f;                 // a maximum up to here has a rounding of 2^-12 at most
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

// How the work is dealt out; the same for both kernels.  All units are laid end to end, each with its pages behind a charge of
// kPaCharge (what a segment costs besides them: the query, the first chunk's latency, the meeting of the warps), and every CTA
// takes an equal stretch (the first `extra` one more).  The host refuses what does not fit 31 bits.
__device__ __forceinline__ int stretch_of(int length) { return length > 0 ? pages_of(length) + kPaCharge : 0; }
struct Shares {
    int ctas, each, extra;
    __device__ __forceinline__ Shares(const PagedParams& p, int all) {
        const int least = least_share(all / (p.heads * p.sequences));
        ctas = min(p.ctas, (all + least - 1) / least);
        each = ctas ? all / ctas : 0, extra = all - each * ctas;
    }
    __device__ __forceinline__ int begin(int cta) const { return cta * each + min(cta, extra); }
    __device__ __forceinline__ int owner(int place) const {
        const int longer = extra * (each + 1);
        return place < longer ? place / (each + 1) : extra + (place - longer) / each;
    }
};

// The stretches of the sequences, one after the other, of one head.
struct Lengths {
    int mine, upto, all;  // of the lane's sequence among the first 32: its length, the stretches up to its end; all stretches
    __device__ __forceinline__ Lengths(const PagedParams& p, int lane) {
        mine = lane < p.sequences ? length_of(p, lane) : 0;
        upto = running_sum(stretch_of(mine), lane);
        all = __shfl_sync(0xffffffffu, upto, 31);
        if (p.sequences > 32) {
            int rest = 0;
            for (int s = 32 + lane; s < p.sequences; s += 32) rest += stretch_of(length_of(p, s));
            all += __reduce_add_sync(0xffffffffu, rest);
        }
    }
    static __device__ __forceinline__ int running_sum(int x, int lane) {
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, x, off);
            if (lane >= off) x += other;
        }
        return x;
    }
};

// The segments of a share, one after the other: consecutive pages of a unit.
struct Segments {
    int sequence, head, length, first, last;
    int left;  // of the share behind this segment
    // From place `place` on, `count` long; whole warp.  The first segment may be empty (first == last).
    __device__ __forceinline__ void start(const PagedParams& p, const Lengths& known, int place, int count, int lane) {
        int before = 0, n = known.mine, upto = known.upto;
        left = -1;
        for (int s0 = 0; s0 < p.sequences; s0 += 32) {
            if (s0 > 0) {
                n = s0 + lane < p.sequences ? length_of(p, s0 + lane) : 0;
                upto = Lengths::running_sum(stretch_of(n), lane);
            }
            const uint32_t mask = __ballot_sync(0xffffffffu, (before + upto) * p.heads > place);
            if (mask) {
                const int owner = __ffs(mask) - 1;
                length = __shfl_sync(0xffffffffu, n, owner);
                const int per = stretch_of(length);
                const int at = place - (before + __shfl_sync(0xffffffffu, upto, owner) - per) * p.heads;
                sequence = s0 + owner, head = at / per;
                take(at - head * per, count);
                return;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
    }
    // What `count` from offset `from` of the unit's stretch on holds of it.
    __device__ __forceinline__ void take(int from, int count) {
        const int per = stretch_of(length), to = min(per, from + count);
        first = from > kPaCharge ? from - kPaCharge : 0, last = to > kPaCharge ? to - kPaCharge : 0;
        left = count - (to - from);
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
        take(0, left);
        return true;
    }
    __device__ __forceinline__ int first_chunk() const { return first * kPageChunks; }
    __device__ __forceinline__ int last_chunk() const {
        const int all = (length + kChunkTokens - 1) / kChunkTokens, end = last * kPageChunks;
        return all < end ? all : end;
    }
};

__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127
__device__ __forceinline__ int exponent_of(float x) { return static_cast<int>(__float_as_uint(x) >> 23 & 255u) - 127; }
__device__ __forceinline__ int clamped(int x, int low, int high) { return x < low ? low : x > high ? high : x; }

__device__ __forceinline__ void ctas_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kPaThreads) : "memory"); }

// mma_16816 with nothing to add to.
__device__ __forceinline__ void mma_16816_start(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// Tokens' offsets (a0: token g, a1: token g + 8, groups 0 and 1, the same in every lane of a quad) times the parts of the sums of q
// that the lanes of a quad hold, in the type of the model.
template <bool BF16>
__device__ __forceinline__ void mma_offsets(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
                     : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                     : "r"(a0), "r"(a1), "r"(b0), "f"(0.f));
    else
        asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
                     : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                     : "r"(a0), "r"(a1), "r"(b0), "f"(0.f));
}

// The larger numbers of two pairs (a NaN counts for nothing).
template <bool BF16>
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    uint32_t r;
    if (BF16) asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// An 8 x 8 matrix of 16-bit numbers, two of a row per lane, with rows and columns exchanged.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

struct Requests {
    Segments segment;           // behind the one that is being requested; left < 0: none
    const int* entry;           // in the table, of the chunk that is looked up next
    const unsigned char* base;  // of the head and the chunk's place in page 0
    int chunks;                 // left to look up of the segment (-1: none at all)
    int page[kPaStages];        // looked up: pages, and `base` (null: there is no further chunk)
    const unsigned char* at[kPaStages];
    int stage, phase;           // of the wait that ran out
};

// The warp's next segment, in shared memory; whole warp.  The first barrier keeps the record until every lane has read it, the second
// puts lane 0's stores before the other lanes' loads: an exchange between lanes alone orders no memory.
__device__ __forceinline__ bool next_segment(const PagedParams& p, Segments& at, int lane) {
    bool any = false;
    __syncwarp();
    if (lane == 0) any = at.next(p);
    __syncwarp();
    return __shfl_sync(0xffffffffu, any, 0);
}

// How p * scale goes into the product with the codes.  Rounded to FP16 once it is off by as much as an FP16 result, so FP16 models add
// what the rounding took: in columns 4 to 7, which hold the heads once more, as long as there are four heads at most, otherwise by a
// second product.  Error of the result over that of its own rounding, 32 x 8128 tokens: 1.45 rounded once, 1.00 with the rest.  That
// costs 67.8 to 71.2 us there, 27.0 to 30.1 us with 32 x 2000 tokens of eight heads.  BF16 results are rounded eight times as far: 1.01.
enum class Weights { kOnce, kBeside, kTwice };

template <bool BF16, Weights WEIGHTS>
__global__ void __launch_bounds__(kPaThreads, kPaPerSm) paged_attention_kernel(const PagedParams p) {
    constexpr bool kBeside = WEIGHTS == Weights::kBeside, kTwice = WEIGHTS == Weights::kTwice;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ uint64_t bar_full[kPaWarps][kPaStages];
    __shared__ float s_max[kPaWarps][kPagedGroup], s_sum[kPaWarps][kPagedGroup], s_top[kPagedGroup];
    __shared__ Segments s_at[kPaWarps];
    __shared__ Requests s_ahead[kPaWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    unsigned char* ring = smem + warp * kPaStages * kChunkBytes;
    float* sums = reinterpret_cast<float*>(smem + kPaWarps * kPaStages * kChunkBytes);  // [warp][head][128]
    if (lane == 0) {
        for (int s = 0; s < kPaStages; ++s) mbar_init(&bar_full[warp][s], 1);
        mbar_fence_init();
    }
    __syncwarp();
    wait_for_previous_launch();
    let_next_launch_start();
    const Lengths lengths(p, lane);
    const Shares shares(p, lengths.all * p.heads);
    if (static_cast<int>(blockIdx.x) >= shares.ctas) return;
    const int begin = shares.begin(blockIdx.x), count = shares.begin(blockIdx.x + 1) - begin;
    // A warp's places in its list of segments, the one that is worked on and the one whose chunks are requested, are in shared
    // memory: registers are scarce.
    Segments& at = s_at[warp];
    Requests& ahead = s_ahead[warp];
    {
        Segments first{};
        first.start(p, lengths, begin, count, lane);
        if (lane == 0) at = first, ahead.segment = first, ahead.chunks = 0;
        __syncwarp();
    }
    // Requests run ahead of the work (lane 0).  A warp's chunks are kPaWarps apart, so they lie at the same place of their pages.
    // The numbers of the next two pages are under way into shared memory while a chunk is worked on.
    const auto look = [&](int slot) {
        while (ahead.chunks == 0) {
            if (ahead.segment.left < 0) {
                ahead.chunks = -1;
                break;
            }
            const int first = ahead.segment.first_chunk() + warp, end = ahead.segment.last_chunk();
            if (end > first) {
                ahead.chunks = (end - first + kPaWarps - 1) / kPaWarps;
                ahead.entry = p.table + static_cast<int64_t>(ahead.segment.sequence) * p.width + first / kPageChunks;
                ahead.base = p.pages + static_cast<int64_t>(ahead.segment.head) * kPageHeadBytes + (first & (kPageChunks - 1)) * kChunkBytes;
            }
            if (!ahead.segment.next(p)) ahead.segment.left = -1;
        }
        ahead.at[slot] = nullptr;
        if (ahead.chunks > 0) {
            ahead.at[slot] = ahead.base;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(&ahead.page[slot])), "l"(ahead.entry) : "memory");
            ahead.entry += kPaWarps / kPageChunks;
            --ahead.chunks;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const auto request = [&](int stage) {  // page slots and stages go round together
        const unsigned char* from = ahead.at[stage];
        if (!from) return;
        asm volatile("cp.async.wait_group %0;" ::"n"(kPaStages - 1) : "memory");
        int page = *static_cast<volatile int*>(&ahead.page[stage]);
        if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.page_count)) {
            atomicOr(p.status, RESKV_STATUS_STATE_RANGE);
            page = 0;
        }
        mbar_arrive_expect_tx(&bar_full[warp][stage], kChunkBytes);
        bulk_g2s(ring + stage * kChunkBytes, from + page * (static_cast<int64_t>(p.heads) * kPageHeadBytes), kChunkBytes, &bar_full[warp][stage]);
        look(stage);
    };
    bool lost = false;
    if (lane == 0) {
#pragma unroll 1
        for (int s = 0; s < kPaStages; ++s) look(s);
#pragma unroll 1
        for (int s = 0; s < kPaStages; ++s) request(s);
    }

    // Row n of a tile of eight tokens is row n / 2 (n even) or 4 + (n / 2 ^ 1) (n odd) of the block's eight: the rows that the lanes
    // of a quad read together (tokens 2t, 2t + 1 of the contraction with the values) lie on different banks.
    const int row_even = t, row_odd = 4 + (t ^ 1), own_row = (g >> 1) ^ (g & 1 ? 5 : 0);
    const float takes = kTwice || t >= 2 ? -1.f : 0.f;  // whether the lane's columns hold what the rounding took
    int stage = 0, phase = 0;
    bool first_segment = true;
    for (bool any = true; any; any = next_segment(p, at, lane)) {
        if (at.first == at.last) continue;
        // ---- the query: head g's coordinates 32 j + 8 t .. + 7, scaled by a power of two that makes the largest about 2^9 ------
        uint32_t q_low[4][2], q_high[4][2], q_sums;
        float q_scale[2];  // of heads 2t, 2t + 1: of the scores as they come from the products
        {
            float v[4][8], top = 0.f, sum[2] = {0.f, 0.f};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint4 raw = make_uint4(0, 0, 0, 0);
                const int head = kBeside ? g & 3 : g;
                if (head < p.group)
                    raw = *reinterpret_cast<const uint4*>(p.q + at.sequence * p.q_sequence + (at.head * p.group + head) * p.q_head + 32 * j + 8 * t);
                const uint32_t* pairs = reinterpret_cast<const uint32_t*>(&raw);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[j][2 * e] = low_of<BF16>(pairs[e]), v[j][2 * e + 1] = high_of<BF16>(pairs[e]);
                    top = fmaxf(top, fmaxf(fabsf(v[j][2 * e]), fabsf(v[j][2 * e + 1])));
                    sum[j >> 1] += v[j][2 * e] + v[j][2 * e + 1];
                }
            }
#pragma unroll
            for (int off = 1; off < 4; off <<= 1) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
                sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], off);
                sum[1] += __shfl_xor_sync(0xffffffffu, sum[1], off);
            }
            const int up = clamped(9 - exponent_of(top), -100, 100);
            const float by = power_of_two(up);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {  // coordinates 2e, 2e + 4: low nibbles of the codes; 2e + 1, 2e + 5: the next ones
                    q_low[j][e] = pack2<false>(v[j][2 * e] * by, v[j][2 * e + 4] * by);
                    q_high[j][e] = pack2<false>(v[j][2 * e + 1] * by * 0.0625f, v[j][2 * e + 5] * by * 0.0625f);
                }
            // A quarter of the sums (below 2^14), against the offsets: the lanes of a quad hold what one 16-bit number leaves of
            // them (FP16: two parts, BF16: three), each against the same offsets
            sum[0] *= 0.25f * by, sum[1] *= 0.25f * by;
            q_sums = 0;
#pragma unroll
            for (int part = 0; part < (BF16 ? 3 : 2); ++part) {
                const uint32_t pair = pack2<BF16>(sum[0], sum[1]);
                if (t == part) q_sums = pair;
                sum[0] -= low_of<BF16>(pair), sum[1] -= high_of<BF16>(pair);
            }
            // not below the normal numbers, which leave scores as good as 0: a factor of 0 (a query of zeros, a tiny scaling) would make
            // masked scores NaN
            const float mine = fmaxf(4.f * p.scale_log2 / by, 0x1p-126f);
            q_scale[0] = __shfl_sync(0xffffffffu, mine, 8 * t), q_scale[1] = __shfl_sync(0xffffffffu, mine, 8 * t + 4);
        }

        // Of heads 2t and 2t + 1, over the lane's tokens: sums of p and per group of p * middle.  They and the outputs are in units of
        // 2^-unit_up, which keeps p * scale where FP16 is exact to half a step.
        // m may lag behind the maximum by kPaSlack powers of two: fewer rescalings.
        // It starts at the lowest finite number: scores of -infinity (BF16 offsets so large that their products leave FP32) have weights
        // of 0 then, where a maximum of -infinity would make them NaN.
        constexpr float kNone = -3.402823466e38f;
        float m[2] = {kNone, kNone};  // times q_scale
        bool far = false;  // one of the warp's is far from 0
        float unit_up = 0.f, unit_limit = -1.f;
        // Powers of the weights: s * q_scale - m + unit_up in one step where m is near 0, otherwise rounded in front of the subtraction, as
        // m was: in one step the largest score's power would be m's rounding, 2^6 for scores of 2^30, and unit_up lost beside m.
        const auto powers_of = [&](float(&power)[kChunkBlocks][4], const float(&s)[kChunkBlocks][4]) {
            const float shift[2] = {unit_up - m[0], unit_up - m[1]};
#pragma unroll
            for (int b = 0; b < kChunkBlocks; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) power[b][i] = fmaf(s[b][i], q_scale[i & 1], shift[i & 1]);
            if (far) {
#pragma unroll
                for (int b = 0; b < kChunkBlocks; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (fabsf(m[i & 1]) > kPaNear) power[b][i] = __fadd_rn(__fadd_rn(__fmul_rn(s[b][i], q_scale[i & 1]), -m[i & 1]), unit_up);
            }
        };
        float2 l = make_float2(0.f, 0.f), flat[2] = {l, l};
        float acc[8][4];  // rows = coordinates, columns = heads 2t, 2t + 1
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
        const int end = at.last_chunk(), start = at.first_chunk() + warp;
        int tokens = at.length - start * kChunkTokens;  // from this chunk on
        for (int chunks = end - start; chunks > 0; chunks -= kPaWarps, tokens -= kPaWarps * kChunkTokens) {
            if (!lost && !mbar_wait(&bar_full[warp][stage], phase)) {
                lost = true;
                if (lane == 0) {  // nothing more is asked for: a stage whose copy has not arrived must not be armed again
#pragma unroll
                    for (int s = 0; s < kPaStages; ++s) ahead.at[s] = nullptr;
                    ahead.stage = stage, ahead.phase = phase;
                }
            }
            unsigned char* const chunk = ring + stage * kChunkBytes;
            // ---- scores: rows = tokens g, g + 8 of a block, columns = heads: (scale . (q . code) 2^22 + offset . sum(q) / 4) * q_scale ----
            float s[kChunkBlocks][4];
#pragma unroll
            for (int b = 0; b < kChunkBlocks; ++b) {
                const unsigned char* keys = chunk + b * kBlockBytes + own_row * 64 + 16 * t;
                const unsigned char* own = chunk + b * kBlockBytes + kBlockCodes + own_row * 8;
                const uint4 w0 = *reinterpret_cast<const uint4*>(keys), w1 = *reinterpret_cast<const uint4*>(keys + 8 * 64);
                const uint32_t words[2][4] = {{w0.x, w0.y, w0.z, w0.w}, {w1.x, w1.y, w1.z, w1.w}};
                const uint2 param[2] = {*reinterpret_cast<const uint2*>(own), *reinterpret_cast<const uint2*>(own + 64)};
                float c[2][4], offsets[4];
                mma_offsets<BF16>(offsets, param[0].y, param[1].y, q_sums);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float(&d)[4] = c[j >> 1];
                    const uint32_t x = words[0][j], y = words[1][j], x8 = x >> 8, y8 = y >> 8;
                    if (j & 1)
                        mma_16816(d, x & 0x000F000Fu, y & 0x000F000Fu, x & 0x00F000F0u, y & 0x00F000F0u, q_low[j][0], q_high[j][0]);
                    else
                        mma_16816_start(d, x & 0x000F000Fu, y & 0x000F000Fu, x & 0x00F000F0u, y & 0x00F000F0u, q_low[j][0], q_high[j][0]);
                    mma_16816(d, x8 & 0x000F000Fu, y8 & 0x000F000Fu, x8 & 0x00F000F0u, y8 & 0x00F000F0u, q_low[j][1], q_high[j][1]);
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float scale0 = low_of<BF16>(param[i].x), scale1 = high_of<BF16>(param[i].x);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        s[b][2 * i + h] = fmaf(fmaf(c[0][2 * i + h], scale0, c[1][2 * i + h] * scale1), 1 << 22, offsets[2 * i + h]);
                }
            }
            if (tokens < kChunkTokens) {  // behind the sequence's end: whatever lies there counts for nothing
                __syncwarp();
                if (lane >= tokens) {
                    *reinterpret_cast<uint2*>(chunk + (lane >> 4) * kBlockBytes + kBlockSide + kBlockCodes + (lane & 15) * 8) = make_uint2(0, 0);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the next copy to this place comes behind it
                }
                __syncwarp();
#pragma unroll
                for (int b = 0; b < kChunkBlocks; ++b) {
                    if (16 * b + own_row >= tokens) s[b][0] = s[b][1] = -INFINITY;
                    if (16 * b + own_row + 8 >= tokens) s[b][2] = s[b][3] = -INFINITY;
                }
            }
            // ---- running softmax; the unit follows the largest scale (BF16: or 2^-30 of an offset, so that a sum of offsets stays in
            // range where all scales are 0) ----------------------------------------------------------------------------------------
            uint2 params[kChunkBlocks][2];  // of the lane's tokens: scales, offsets
#pragma unroll
            for (int b = 0; b < kChunkBlocks; ++b)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    params[b][i] = *reinterpret_cast<const uint2*>(chunk + b * kBlockBytes + kBlockSide + kBlockCodes + (own_row + 8 * i) * 8);
            float most;
            {
                const uint32_t pair = larger<BF16>(larger<BF16>(params[0][0].x, params[0][1].x), larger<BF16>(params[1][0].x, params[1][1].x));
                most = fmaxf(low_of<BF16>(pair), high_of<BF16>(pair));
                if (BF16) {
                    constexpr uint32_t kPlus = 0x7FFF7FFFu;
                    const uint32_t off = larger<BF16>(larger<BF16>(params[0][0].y & kPlus, params[0][1].y & kPlus), larger<BF16>(params[1][0].y & kPlus, params[1][1].y & kPlus));
                    most = fmaxf(most, 0x1p-30f * fmaxf(low_of<BF16>(off), high_of<BF16>(off)));
                }
            }
            float power[kChunkBlocks][4], highest = -INFINITY;
            powers_of(power, s);
#pragma unroll
            for (int b = 0; b < kChunkBlocks; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) highest = fmaxf(highest, power[b][i]);
            if (__any_sync(0xffffffffu, highest > unit_up + kPaSlack || most > unit_limit)) {
                float top[2] = {fmaxf(fmaxf(s[0][0], s[0][2]), fmaxf(s[1][0], s[1][2])), fmaxf(fmaxf(s[0][1], s[0][3]), fmaxf(s[1][1], s[1][3]))};
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) {
                    top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], off));
                    top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], off));
                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
                }
                float up = unit_up;
                if (most > unit_limit) {  // the same in every lane
                    const int e = clamped(exponent_of(most), -60, 100);
                    up = 14 - kPaSlack - e;  // a scale up to 2^(e + 1) times a p up to 2^kPaSlack, 2^15 at most
                    unit_limit = power_of_two(e + 1);
                }
                const float change = power_of_two(clamped(static_cast<int>(up - unit_up), -126, 126));
                float factor[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float next = fmaxf(m[h], __fmul_rn(top[h], q_scale[h]));
                    factor[h] = (m[h] == next ? 1.f : fast_exp2(m[h] - next)) * change;
                    m[h] = next;
                }
                unit_up = up;
                far = __any_sync(0xffffffffu, fmaxf(fabsf(m[0]), fabsf(m[1])) > kPaNear);
                powers_of(power, s);
                l.x *= factor[0], l.y *= factor[1];
#pragma unroll
                for (int i = 0; i < 2; ++i) flat[i].x *= factor[0], flat[i].y *= factor[1];
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[i][0] *= factor[0], acc[i][1] *= factor[1], acc[i][2] *= factor[0], acc[i][3] *= factor[1];
            }
            float eights[2][4];
#pragma unroll
            for (int b = 0; b < kChunkBlocks; ++b) {
                const unsigned char* values = chunk + b * kBlockBytes + kBlockSide;
                // ---- weights: rows = tokens, turned round for the contraction over them --------------------------------------------
                uint32_t weights[2][2], rest[2][2];  // [group][half of the block's tokens]
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float2 weight = make_float2(fast_exp2(power[b][2 * i]), fast_exp2(power[b][2 * i + 1]));
                    l = add2(l, weight);
#pragma unroll
                    for (int group = 0; group < 2; ++group) {
                        const float scale = group ? high_of<BF16>(params[b][i].x) : low_of<BF16>(params[b][i].x);
                        const float offset = group ? high_of<BF16>(params[b][i].y) : low_of<BF16>(params[b][i].y);
                        const float2 exact = make_float2(weight.x * scale, weight.y * scale);
                        uint32_t pair = pack2<false>(exact.x, exact.y);
                        if (kBeside || kTwice) {
                            const float2 left = fma2(make_float2(low_of<false>(pair), high_of<false>(pair)), make_float2(takes, takes), exact);
                            const uint32_t other = pack2<false>(left.x, left.y);
                            if (kBeside) pair = other; else rest[group][i] = transposed(other);
                        }
                        weights[group][i] = transposed(pair);
                        const float middle = fmaf(scale, kCodeMiddle, offset);
                        flat[group].x = fmaf(weight.x, middle, flat[group].x), flat[group].y = fmaf(weight.y, middle, flat[group].y);
                    }
                }
                // ---- outputs: a value is offset + 8 scale (its middle) + (code - 8) scale.  With the codes alone the sum would be many times
                // the result, most of it taken back by the offsets, and its rounding with it: eight times the weights are taken off again
                // after every chunk.
#pragma unroll
                for (int group = 0; group < 2; ++group) {
                    if (b == 0)
                        mma_16816_start(eights[group], kMiddleLow, kMiddleByte, kMiddleLow, kMiddleByte, weights[group][0], weights[group][1]);
                    else
                        mma_16816(eights[group], kMiddleLow, kMiddleByte, kMiddleLow, kMiddleByte, weights[group][0], weights[group][1]);
                    if (kTwice) mma_16816(eights[group], kMiddleLow, kMiddleByte, kMiddleLow, kMiddleByte, rest[group][0], rest[group][1]);
                }
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
                        const uint32_t x = __byte_perm(group ? rows[0].y : rows[0].x, group ? rows[1].y : rows[1].x, pick), x8 = __byte_perm(x, 0, 0x4341);
                        const uint32_t y = __byte_perm(group ? rows[2].y : rows[2].x, group ? rows[3].y : rows[3].x, pick), y8 = __byte_perm(y, 0, 0x4341);
                        const auto add = [&](const uint32_t(&w)[2]) {
                            mma_16816(acc[group * 4 + half * 2], x & 0x000F000Fu, x & 0x00FF00FFu, y & 0x000F000Fu, y & 0x00FF00FFu, w[0], w[1]);
                            mma_16816(acc[group * 4 + half * 2 + 1], x8 & 0x000F000Fu, x8, y8 & 0x000F000Fu, y8, w[0], w[1]);
                        };
                        add(weights[group]);
                        if (kTwice) add(rest[group]);
                    }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 x = add2(make_float2(acc[i][0], acc[i][1]), make_float2(eights[i >> 2][0], eights[i >> 2][1]));
                const float2 y = add2(make_float2(acc[i][2], acc[i][3]), make_float2(eights[i >> 2][2], eights[i >> 2][3]));
                acc[i][0] = x.x, acc[i][1] = x.y, acc[i][2] = y.x, acc[i][3] = y.y;
            }
            __syncwarp();
            if (lane == 0) request(stage);
            if (++stage == kPaStages) stage = 0, phase ^= 1;
        }
        // ---- the warps' parts of the segment ------------------------------------------------------------------------------------
        const auto over_tokens = [](float2 x) {
#pragma unroll
            for (int off = 4; off < 32; off <<= 1)
                x.x += __shfl_xor_sync(0xffffffffu, x.x, off), x.y += __shfl_xor_sync(0xffffffffu, x.y, off);
            return x;
        };
        l = over_tokens(l);
        if (g == 0) s_max[warp][2 * t] = m[0], s_max[warp][2 * t + 1] = m[1];
        ctas_sync();
        const int active = min(kPaWarps, end - at.first_chunk());
        float top[2] = {s_max[0][2 * t], s_max[0][2 * t + 1]};
        for (int w = 1; w < active; ++w) top[0] = fmaxf(top[0], s_max[w][2 * t]), top[1] = fmaxf(top[1], s_max[w][2 * t + 1]);
        if (warp < active) {
            const float unit = power_of_two(-static_cast<int>(unit_up));
            const float weight[2] = {m[0] == top[0] ? 1.f : fast_exp2(m[0] - top[0]), m[1] == top[1] ? 1.f : fast_exp2(m[1] - top[1])};
            if (g == 0) s_sum[warp][2 * t] = l.x * unit * weight[0], s_sum[warp][2 * t + 1] = l.y * unit * weight[1];
            float base[2][2];  // [group][head]
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float2 f = over_tokens(flat[i]);
                base[i][0] = f.x * unit, base[i][1] = f.y * unit;
                if (kBeside && t >= 2) base[i][0] = base[i][1] = 0.f;
            }
            float* mine = sums + warp * kPagedGroup * kHeadDim + 2 * t * kHeadDim;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                constexpr float low = 1 << 24, high = 1 << 20;  // of codes alone, and of what they leave of their bytes
                const int d = (i >> 2) * 64 + 8 * g + (i & 3) * 2;
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if ((kBeside ? (2 * t + h) & 3 : 2 * t + h) < p.group)
                        *reinterpret_cast<float2*>(mine + h * kHeadDim + d) = make_float2(fmaf(acc[i][h] * low, unit, base[i >> 2][h]) * weight[h],
                                                                                       fmaf((acc[i][2 + h] - acc[i][h]) * high, unit, base[i >> 2][h]) * weight[h]);
            }
        }
        if (warp == 0 && g == 0) s_top[2 * t] = top[0], s_top[2 * t + 1] = top[1];
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
                if (kBeside) {
                    const float4 y = *reinterpret_cast<const float4*>(sums + (w * kPagedGroup + 4) * kHeadDim + i);
                    sum.x += y.x, sum.y += y.y, sum.z += y.z, sum.w += y.w;
                }
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
        first_segment = false;
    }
    if (lost && lane == 0) {  // no copy may land after the block's end: those from the lost one on, once round the ring
#pragma unroll 1
        for (int s = 0; s < kPaStages; ++s) mbar_wait(&bar_full[warp][s], s < ahead.stage ? ahead.phase ^ 1 : ahead.phase);
        asm volatile("cp.async.wait_all;" ::: "memory");
        atomicOr(p.status, RESKV_STATUS_WAIT_TIMEOUT);
    }
}

// Adds the parts of a unit that lies in several CTAs; a unit without tokens gets zeros.  Bound by latency: `split` warps per query
// head take the parts in turn, each with a running maximum of its own, and meet in shared memory.
template <bool BF16>
__global__ void __launch_bounds__(1024) paged_merge_kernel(const PagedParams p, int split) {
    __shared__ float4 s_out[32][32];
    __shared__ float2 s_stats[32];  // maximum, sum
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, turn = warp % split, unit = blockIdx.x;
    const int head = blockIdx.y * (blockDim.x / 32 / split) + warp / split;
    // The lengths may be read at once: this kernel starts when every CTA of the first one has seen the end of what came before
    // (without pages there is no first one, and the lengths count as 0).
    const int sequence = unit / p.heads, kv_head = unit - sequence * p.heads;
    const int64_t row = static_cast<int64_t>(sequence) * p.heads * p.group + kv_head * p.group + head;
    int all = 0, before = 0;
    for (int s = lane; s < p.sequences; s += 32) {
        const int n = stretch_of(length_of(p, s));
        all += n, before += s < sequence ? n : 0;
    }
    all = __reduce_add_sync(0xffffffffu, all), before = __reduce_add_sync(0xffffffffu, before);
    const int length = length_of(p, sequence), per = stretch_of(length);
    const Shares shares(p, all * p.heads);
    const int a = before * p.heads + kv_head * per;
    const int from = length ? shares.owner(a + kPaCharge) : 0, to = length ? shares.owner(a + per - 1) : 0;
    wait_for_previous_launch();
    let_next_launch_start();
    if (length == 0) {
        if (turn == 0) *reinterpret_cast<uint2*>(p.out + row * kHeadDim + 4 * lane) = make_uint2(0, 0);
        if (p.lse && turn == 0 && lane == 0) p.lse[row] = -INFINITY;
        return;
    }
    if (from == to) return;
    const int count = to - from + 1;
    const int skip = shares.begin(from) < a ? 1 : 0;  // the last page of another unit lies in front of it in its first CTA: that CTA's second part
    const float* parts = p.parts + 2 * static_cast<int64_t>(from) * kPartialFloats;
    float top = -INFINITY, total = 0.f;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    const auto add = [&](float m, float l, const float4& x) {
        const float next = fmaxf(top, m), old = top == next ? 1.f : fast_exp2(top - next), now = m == next ? 1.f : fast_exp2(m - next);
        top = next;
        sum.x = fmaf(x.x, now, sum.x * old), sum.y = fmaf(x.y, now, sum.y * old), sum.z = fmaf(x.z, now, sum.z * old), sum.w = fmaf(x.w, now, sum.w * old);
        total = fmaf(l, now, total * old);
    };
#pragma unroll 4
    for (int i = turn; i < count; i += split) {
        const float* part = parts + (2 * i + (i == 0 ? skip : 0)) * kPartialFloats;
        add(part[kPagedGroup * kHeadDim + head], part[kPagedGroup * (kHeadDim + 1) + head], *reinterpret_cast<const float4*>(part + head * kHeadDim + 4 * lane));
    }
    if (split > 1) {
        s_out[warp][lane] = sum;
        if (lane == 0) s_stats[warp] = make_float2(top, total);
        __syncthreads();
        if (turn > 0) return;
        for (int w = 1; w < min(split, count); ++w) add(s_stats[warp + w].x, s_stats[warp + w].y, s_out[warp + w][lane]);
    }
    const float inv = 1.f / total;
    *reinterpret_cast<uint2*>(p.out + row * kHeadDim + 4 * lane) =
        make_uint2(pack2<BF16>(sum.x * inv, sum.y * inv), pack2<BF16>(sum.z * inv, sum.w * inv));
    if (p.lse && lane == 0) p.lse[row] = top * kLn2 + logf(total);
}

int most_shares(int sequences, int width, int heads, int least) {
    const int64_t most = (static_cast<int64_t>(sequences) * (width + kPaCharge) * heads + least - 1) / least;
    return static_cast<int>(std::min<int64_t>(most, kPaPerSm * sm_count()));
}

// CTAs of the first kernel for as many pages as there may be.  No more than will have a share: those without one displace others
// (1 x 8128 tokens: 12.6 us with 296 CTAs for 135 shares, 10.2 with 135).
int paged_ctas(int sequences, int width, int heads) {
    return width == 0 ? 0 : most_shares(sequences, width, heads, least_share(width + kPaCharge));
}

template <bool BF16, Weights WEIGHTS>
int launch(const PagedParams& p, cudaStream_t stream) {
    static std::atomic<unsigned long long> done{0};
    if (int rc = allow_smem(paged_attention_kernel<BF16, WEIGHTS>, kPaSmem, done, "cudaFuncSetAttribute(paged_attention)")) return rc;
    if (p.ctas > 0)
        if (int rc = check_cuda(launch_overlapped(paged_attention_kernel<BF16, WEIGHTS>, dim3(static_cast<unsigned>(p.ctas)), kPaThreads, kPaSmem, stream, true, p),
                                "paged_attention launch"))
            return rc;
    const int units = p.sequences * p.heads;
    // As many warps per query head as the SMs hold at once; one, and all heads in a block, where that would be two: 16, 8 and 1
    // for nine sequences of eight heads with eight query heads each 16.7, 15.7 and 19 us, for 64 with four each 22 (8) and 18.4 (1) us.
    int split = kPaMergeWarps;
    while (split > 1 && static_cast<int64_t>(units) * p.group * split > 32 * sm_count()) split /= 2;
    const bool few = split >= 4;
    const dim3 grid(static_cast<unsigned>(units), static_cast<unsigned>(few ? p.group : 1));
    return check_cuda(launch_overlapped(paged_merge_kernel<BF16>, grid, (few ? split : p.group) * 32, 0, stream, true, p, few ? split : 1),
                      "paged_attention merge launch");
}

}  // namespace
}  // namespace reskv

using namespace reskv;

extern "C" size_t reskv_paged_attention_workspace_bytes(int sequences, int width, int kv_heads) {
    if (sequences < 0 || width < 0 || kv_heads < 1) return 0;
    // for the shortest shares, so that what is enough for a wide table is enough for a narrow one
    return static_cast<size_t>(width == 0 ? 0 : most_shares(sequences, width, kv_heads, least_share(0))) * 2 * kPartialFloats * sizeof(float) + 256;
}

extern "C" int reskv_paged_attention(const void* q, int bf16, int64_t q_sequence, int64_t q_head, const int32_t* lengths, const int32_t* table,
                                     int sequences, int width, int kv_heads, int q_heads, const void* pages, int page_count, float scaling,
                                     void* workspace, size_t workspace_bytes, void* out, float* lse, uint32_t* status, void* stream) {
    if (sequences < 0 || width < 0 || kv_heads < 1 || q_heads < 1 || q_heads % kv_heads || page_count < 0)
        return fail(RESKV_ERR_INVALID, "paged_attention: %d sequences, table of %d pages, %d KV and %d query heads, %d pages", sequences, width,
                    kv_heads, q_heads, page_count);
    if (q_heads / kv_heads > kPagedGroup) return fail(RESKV_ERR_LIMIT, "paged_attention: more than %d query heads per KV head", kPagedGroup);
    if (!(scaling > 0.f) || !(scaling < 3.0e38f)) return fail(RESKV_ERR_INVALID, "paged_attention: scaling must be positive and finite");
    if (static_cast<int64_t>(sequences) * kv_heads * (static_cast<int64_t>(width) + kPaCharge) > 0x3fffffff || width > (1 << 24))
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
    if (int rc = check_device_pointer(status, "paged_attention", "status")) return rc;
    if (lse)
        if (int rc = check_device_pointer(lse, "paged_attention", "lse")) return rc;
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
    const cudaStream_t on = static_cast<cudaStream_t>(stream);
    if (bf16) return launch<true, Weights::kOnce>(p, on);
    return p.group <= kPagedGroup / 2 ? launch<false, Weights::kBeside>(p, on) : launch<false, Weights::kTwice>(p, on);
}
