// Attention over whole prompts that lie one behind the other in packed tensors: for token i of a sequence and every query
// head, out_i = sum_j softmax_j(q_i . k_j * scaling) v_j over the keys j <= i (causal) or over all keys of the sequence.
//
// Both products run on tcgen05.mma.  A row tile is 128 rows: the query heads of one KV head for as many tokens as fit, so that
// grouped heads share the keys and a short sequence still fills rows; an item is two row tiles, in short calls one.  Per tile of 80
// keys: scores S = Q K^T into tensor memory, one thread per row forms the weights P with a running maximum (it lags by up to 2^8, so
// that the output is rarely rescaled), and the output accumulates P V with P read from tensor memory.  A row tile's scores (80
// columns) and weights (40) lie side by side in 128 columns, which is why a tile has 80 keys: the next scores do not wait for the
// product with the weights in front.  A warp issues the scores' products, another one the outputs', so neither waits for the other's
// operands.  Tiles arrive by TMA through a ring of eight.
//
// Items are ordered by their place in their sequence, last ones first, which with causal attention are the longest; the grid has
// a CTA for every item that there may be, and a CTA that has finished takes over one that has not started (cluster launch
// control), so it keeps its tensor memory and its ring.
//
// What is masked counts for nothing: masked scores are replaced, rows of V behind the sequence are cleared in shared memory, and
// infinities or NaN in rows of V that only part of a row tile sees are cleared there too and added where they are seen.
//
// Bound (1 x 8192 tokens, 32 / 8 heads, 550 GFLOP): 460 us = 1.20 PFLOP/s in short runs, 521 to 531 us = 1.05 PFLOP/s in long ones under
// the power cap; seven ragged prompts of 84 GFLOP 101 us in short runs, 108 with cold inputs, five short ones of 0.9 GFLOP 13 us.  (Without
// the way for scores far from 0 454 and 517 us, 99 and 107.)  A row tile's softmax is what takes longest: 2070 cycles per tile of 80
// keys, of them 1230 forming weights (16 exponentials per clock and SM, two row tiles: 1280 for both), 180 and 280 waiting for scores
// and for the product in front, 150 the maximum; per item another 1300 waiting for the last product, 2300 storing, 1000 until the first
// scores.  An item has all keys of its rows, so a call of few items takes as long as its longest one: one sequence of 2000 tokens with
// one head keeps 16 SMs busy, 31 us.  What was measured besides, on 1 x 8192 in short runs of the form that took 449 us:
//   128 keys a tile, weights in the scores' place, one warp for both products, ring of five: 463 us (seven ragged: 100 us)
//   a quarter of the exponentials by a polynomial: 447 us, not worth its code; a half: no faster
//   two threads per row (16 softmax warps): 502 us
//   the wait for the product in front behind all exponentials: 490 us; one lane polling for its warp: 490 us
//   descriptors that the compiler does not see as uniform: 550 us for 463; the products issued from a loop in one thread: 512 us
//   a fourth warpgroup that stores the outputs while the others go on: 458 us, seven ragged prompts 95 us for 96; the row tiles' warps of
//   an SM quarter taking turns at the exponentials: 472 us
//   the product begun with the weights of the first 16, 32 or 48 keys of a tile: no faster, seven ragged prompts 96 us for 94
//   outputs stored by row, 16 bytes a lane, instead of by lines: seven ragged prompts 106 us for 100
#include "pairs.cuh"
#include "tensor_map.cuh"
#include "tmem.cuh"
#include "umma.cuh"

namespace reskv {
namespace {

constexpr int kPKeys = 80;                      // keys of a tile
constexpr int kPChunks = kPKeys / 16;           // of a row of scores
constexpr int kPQHalf = 128 * 128, kPQTile = 2 * kPQHalf;        // bytes of 128 rows x 64 coordinates, and of all coordinates
constexpr int kPKHalf = kPKeys * 128, kPKTile = 2 * kPKHalf;     // the same of a tile of keys or values
constexpr int kPStages = 8;                     // ring of K and V tiles
constexpr int kPThreads = 384;                  // two softmax warpgroups; a warp each for scores, outputs and copies, one idle
// A row of scores and what becomes of it take more than the 168 registers that the launch gives a thread (the most for 384); the last
// warpgroup hands back what the softmax warpgroups take: 2 x 208 + 88 = 3 x 168.
constexpr int kPLaunchRegs = 168, kPSoftmaxRegs = 208, kPOtherRegs = 88;
static_assert(2 * kPSoftmaxRegs + kPOtherRegs <= 3 * kPLaunchRegs, "the shares come out of the launch's registers");
constexpr int kPSmem = 2 * kPQTile + kPStages * kPKTile + 1024;  // + room to start on a 1024-byte boundary
// Tensor memory, columns of the two row tiles: scores (80), weights (40, two to a column), outputs (128).
__host__ __device__ constexpr uint32_t score_column(int i) { return i * 128; }
__host__ __device__ constexpr uint32_t weight_column(int i) { return i * 128 + kPKeys; }
__host__ __device__ constexpr uint32_t output_column(int i) { return 256 + i * 128; }
static_assert(kPKeys + kPKeys / 2 <= 128 && kPKeys % 16 == 0, "scores and weights of a row tile share 128 columns");
constexpr float kPSlack = 8.f;                  // the running maximum lags by at most this (in powers of two)
// Where the maximum times the scale is beyond this, it is taken off the scores in front of the multiplication: the rounding of the
// product (2^-12 here) would be the largest score's power, 2^6 for scores of 2^30.
constexpr float kPNear = 8192.f;
constexpr float kPLowest = -0x1.ffffp127f;      // the running maximum of a row whose scores have all been -infinity

__device__ uint32_t g_prompt_status;  // RESKV_STATUS_* bits of calls without a word of their own

struct PromptParams {
    const int* cu;      // [sequences + 1]
    int sequences, total, kv_heads, group, tile_tokens;  // tile_tokens: tokens of 128 rows
    int64_t most_single;  // items have one row tile each if there are no more than that many of them
    const unsigned short* v;      // the values once more, for the outputs that infinities and NaN reach
    int64_t v_token, v_head;      // elements between its tokens and heads
    void* out;          // [total, query heads, 128]
    float* lse;         // [total, query heads] or null
    float scale_log2;
    int causal;
    uint32_t* status;   // or null: g_prompt_status
};

// A work item: one or two row tiles of one sequence and KV head.
struct PromptItem {
    int start, len, token0, head, tiles0, tiles1;  // tiles0 / tiles1: key tiles that the first / second row tile needs
};

__device__ __forceinline__ int clamped(int x, int low, int high) { return x < low ? low : x > high ? high : x; }

struct SequenceSpan {
    int start, len;
};
__device__ __forceinline__ SequenceSpan span_of(const PromptParams& p, int s) {
    const int a = clamped(p.cu[s], 0, p.total), b = clamped(p.cu[s + 1], a, p.total);
    return {a, b - a};
}

// Number of pieces of `per` tokens of all sequences whose place in the sequence is `level` or behind it; whole warp.
__device__ __forceinline__ int items_from(const PromptParams& p, int per, int level, int lane) {
    int n = 0;
#pragma unroll 4
    for (int s = lane; s < p.sequences; s += 32) {
        const int tiles = (span_of(p, s).len + per - 1) / per;
        n += tiles > level ? tiles - level : 0;
    }
    return __reduce_add_sync(0xffffffffu, n);
}

// Items are ordered by their place in their sequence, last ones first: with causal attention the longest ones.  The items that a CTA
// takes come as a rule in this order, so the search for one begins at the level of the one before.
struct ItemSearch {
    int per, all, level, before, upto;  // tokens of an item; all pieces; the level's are those from `before` to `upto`
    __device__ __forceinline__ ItemSearch(const PromptParams& p, int lane) : per(p.tile_tokens), all(0), before(0), upto(0) {
        if (p.most_single) all = items_from(p, per, 0, lane);
        if (!p.most_single || static_cast<int64_t>(all) * p.kv_heads > p.most_single) per *= 2, all = items_from(p, per, 0, lane);
        level = highest(p);
    }
    __device__ __forceinline__ int highest(const PromptParams& p) const { return (p.total + per - 1) / per; }
    // Item `index`.  tiles0 = 0 in the result: there is none.  Whole warp.
    __device__ PromptItem find(const PromptParams& p, int index, int lane) {
        PromptItem it{};
        const int pos = index / p.kv_heads;
        if (pos >= all) return it;
        if (pos < before) level = highest(p), before = upto = 0;
        if (pos >= upto) {
            int low = 0, high = level, from_high = upto, from_low = all;
            while (high - low > 1) {
                const int mid = (low + high) >> 1, n = items_from(p, per, mid, lane);
                if (n > pos) low = mid, from_low = n; else high = mid, from_high = n;
            }
            level = low, before = from_high, upto = from_low;
        }
        int rest = pos - before;
        for (int s0 = 0; s0 < p.sequences; s0 += 32) {
            const SequenceSpan sp = s0 + lane < p.sequences ? span_of(p, s0 + lane) : SequenceSpan{0, 0};
            const bool has = sp.len > level * per;
            const uint32_t mask = __ballot_sync(0xffffffffu, has);
            const int count = __popc(mask);
            if (rest >= count) {
                rest -= count;
                continue;
            }
            const int owner = __ffs(__ballot_sync(0xffffffffu, has && __popc(mask & ((1u << lane) - 1u)) == rest)) - 1;
            it.start = __shfl_sync(0xffffffffu, sp.start, owner);
            it.len = __shfl_sync(0xffffffffu, sp.len, owner);
            it.head = index % p.kv_heads;
            it.token0 = level * per;
            const int end0 = min(it.token0 + p.tile_tokens, it.len), end1 = min(it.token0 + per, it.len);
            it.tiles0 = ((p.causal ? end0 : it.len) + kPKeys - 1) / kPKeys;
            it.tiles1 = end1 <= it.token0 + p.tile_tokens ? 0 : ((p.causal ? end1 : it.len) + kPKeys - 1) / kPKeys;
            return it;
        }
        return it;
    }
};

template <bool BF16>
__device__ __forceinline__ float unpack(unsigned short bits) {
    return BF16 ? __uint_as_float(static_cast<uint32_t>(bits) << 16) : __half2float(__ushort_as_half(bits));
}

// Whether a 16-bit number is infinite or NaN.
template <bool BF16>
__device__ __forceinline__ bool non_finite(unsigned short bits) {
    constexpr unsigned short mask = BF16 ? 0x7F80 : 0x7C00;
    return (bits & mask) == mask;
}

// A value row (128 coordinates in two halves of 128 bytes) that some row of the tile may not see: `drop` clears it (a token
// behind the sequence), otherwise its infinities and NaN are cleared, because a weight of 0 does not silence them.  The 16-byte
// pieces are taken in an order that keeps the lanes on different banks.  Returns whether something non-finite was there.
template <bool BF16>
__device__ __forceinline__ bool tame_value_row(unsigned char* row, bool drop, int lane) {
    uint32_t seen = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            uint4* at = reinterpret_cast<uint4*>(row + h * kPKHalf + (((i + lane) & 7) << 4));
            if (drop) {
                *at = make_uint4(0, 0, 0, 0);
            } else {
                const uint4 v = *at;
                constexpr uint32_t mask = BF16 ? 0x7F807F80u : 0x7C007C00u, one = BF16 ? 0x00800080u : 0x04000400u;
                seen |= ((v.x & mask) + one) | ((v.y & mask) + one) | ((v.z & mask) + one) | ((v.w & mask) + one);
            }
        }
    if (drop || !(seen & 0x80008000u)) return false;
    for (int h = 0; h < 2; ++h)
        for (int i = 0; i < 64; ++i) {
            unsigned short* at = reinterpret_cast<unsigned short*>(row + h * kPKHalf) + i;
            if (non_finite<BF16>(*at)) *at = 0;
        }
    return true;
}

struct __align__(16) PromptShared {
    uint64_t kv_full[kPStages], kv_empty[kPStages];
    uint64_t q_full, q_empty, s_full[2], s_empty[2], p_full[2], p_empty[2], item_full[2], item_empty[2], cancel;
    uint4 cancel_reply;
    PromptItem item[2];
    int tamed[2];   // of an item: infinities or NaN were cleared in a tile of values
    uint32_t tmem;
};

__device__ __forceinline__ bool wait_once(bool& lost, uint64_t* bar, uint32_t parity) {
    if (!lost) lost = !mbar_wait(bar, parity);
    return !lost;
}

// The same for a warp whose lanes have to agree on it, because they go on by what it says.
__device__ __forceinline__ void wait_together(bool& lost, uint64_t* bar, uint32_t parity) {
    wait_once(lost, bar, parity);
    lost = __any_sync(0xffffffffu, lost);
}

// Whether the next item has been posted: every warp waits for that whether it has lost a wait before or not, and longer than for all
// else together, so that the warps leave together.
__device__ __forceinline__ bool item_posted(uint64_t* bar, uint32_t parity) {
    for (int i = 0; i < 16; ++i)
        if (mbar_wait(bar, parity)) return true;
    return false;
}

// 32 bytes, on a 32-byte boundary.
__device__ __forceinline__ void store32(void* to, const uint32_t (&v)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
                 "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

// A product takes its descriptors from uniform registers; what they depend on is kept uniform in the compiler's eyes too, or each
// costs moves that take longer than the product.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __reduce_or_sync(0xffffffffu, x); }

// The loop of a warp that issues products: items, key tiles, row tiles.  `first`: place of the first tile of keys (0) or of values
// (1) in the ring.  begin(n) before item n, product(i, j, stage, issues) for row tile i and key tile j, end(issues) behind an item;
// the commands themselves are for the one lane for which `issues` holds.  Returns the number of items.
template <class Begin, class Product, class End>
__device__ __forceinline__ int for_key_tiles(PromptShared& sh, bool& lost, int lane, uint32_t first, Begin begin, Product product, End end) {
    const bool issues = elect_one();
    uint32_t stage = first, parity = 0, last_stage = 0, last_parity = 0;
    int n = 0;
    for (;; ++n) {
        const int slot = n & 1;
        if (!item_posted(&sh.item_full[slot], (n >> 1) & 1)) lost = true;
        const int tiles0 = static_cast<int>(uniform(sh.item[slot].tiles0)), tiles1 = static_cast<int>(uniform(sh.item[slot].tiles1));
        if (lane == 0) mbar_arrive(&sh.item_empty[slot]);
        if (tiles0 == 0 || __any_sync(0xffffffffu, lost)) break;
        const int kv_tiles = max(tiles0, tiles1);
        begin(n);
        for (int j = 0; j < kv_tiles; ++j) {
            wait_once(lost, &sh.kv_full[stage], parity);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (j < (i ? tiles1 : tiles0)) product(i, j, stage, issues);
                __syncwarp();
            }
            if (issues) umma_commit(&sh.kv_empty[stage]);
            __syncwarp();
            last_stage = stage, last_parity = parity;
            stage += 2;
            if (stage >= kPStages) stage -= kPStages, parity ^= 1;
        }
        end(issues);
        __syncwarp();
    }
    // the last commits have arrived before the block ends, whether a wait has run out before or not
    if (n > 0) lost |= !mbar_wait(&sh.kv_empty[last_stage], last_parity);
    return n;
}

template <bool BF16>
__global__ void __launch_bounds__(kPThreads, 1)
prompt_attention_kernel(const PromptParams p, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                        const __grid_constant__ CUtensorMap v_map) {
    extern __shared__ unsigned char raw[];
    __shared__ PromptShared sh;
    unsigned char* smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    unsigned char* qs = smem;                 // two row tiles
    unsigned char* ring = smem + 2 * kPQTile;  // K0 V0 K1 V1 ...
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rows = p.tile_tokens * p.group;
    if (tid == 0) {
        for (int s = 0; s < kPStages; ++s) mbar_init(&sh.kv_full[s], 1), mbar_init(&sh.kv_empty[s], 1);
        mbar_init(&sh.q_full, 1), mbar_init(&sh.q_empty, 1), mbar_init(&sh.cancel, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.s_full[i], 1), mbar_init(&sh.p_empty[i], 1);    // products
            mbar_init(&sh.s_empty[i], 4), mbar_init(&sh.p_full[i], 4);    // softmax warps of a row tile
            mbar_init(&sh.item_full[i], 1), mbar_init(&sh.item_empty[i], 10);  // softmax warps, the warps of the products
        }
        mbar_fence_init();
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // Rows of the query tiles that no head has (128 is no multiple of the group): what an earlier kernel left there would be a row's
    // scores, never stored, but far from 0 or NaN its warp would take the long way at every tile (4000 tokens, 5 heads per KV head: 213
    // for 176 us behind a call with NaN).
    for (int at = rows * 128 + tid * 16; at < kPQHalf; at += kPThreads * 16)
#pragma unroll
        for (int half = 0; half < 4; ++half) *reinterpret_cast<uint4*>(qs + half * kPQHalf + at) = make_uint4(0, 0, 0, 0);
    proxy_fence();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    bool lost = false;

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPOtherRegs));
        if (warp == 9) {
            // ---- copies, and the next item: the grid has a CTA for every item that there may be, and a CTA that has finished takes
            // over one that has not started yet -------------------------------------------------------------------------------
            int index = blockIdx.x, tile = 0, queries = 0;  // queries: items whose rows have been asked for
            ItemSearch search(p, lane);
            for (int n = 0;; ++n) {
                const int slot = n & 1;
                const PromptItem it = search.find(p, index, lane);
                if (n >= 2) wait_together(lost, &sh.item_empty[slot], ((n >> 1) - 1) & 1);
                if (lane == 0) {
                    sh.item[slot] = it;
                    if (lost) sh.item[slot].tiles0 = 0;
                    sh.tamed[slot] = 0;
                    mbar_arrive(&sh.item_full[slot]);
                }
                if (it.tiles0 == 0 || lost) break;
                const int kv_tiles = max(it.tiles0, it.tiles1), row_tiles = it.tiles1 ? 2 : 1;
                if (lane == 0) {
                    mbar_arrive_expect_tx(&sh.cancel, 16);
                    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                                     smem_u32(&sh.cancel_reply)),
                                 "r"(smem_u32(&sh.cancel))
                                 : "memory");
                }
                for (int j = 0; j < 2 * kv_tiles; ++j, ++tile) {
                    const int stage = tile % kPStages;
                    if (tile >= kPStages) wait_together(lost, &sh.kv_empty[stage], (tile / kPStages - 1) & 1);
                    if (lost) break;
                    if (lane == 0) {
                        mbar_arrive_expect_tx(&sh.kv_full[stage], kPKTile);
                        for (int h = 0; h < 2; ++h)
                            tma_load_3d(ring + stage * kPKTile + h * kPKHalf, j & 1 ? &v_map : &k_map, 64 * h, it.head,
                                        it.start + (j >> 1) * kPKeys, &sh.kv_full[stage]);
                    }
                    __syncwarp();
                    if (j > 0) continue;
                    // the first keys are on their way before the query tiles of the item in front are given back
                    if (n > 0) wait_together(lost, &sh.q_empty, (n - 1) & 1);
                    if (lost) {
                        ++tile;
                        break;
                    }
                    ++queries;
                    if (lane == 0) {
                        mbar_arrive_expect_tx(&sh.q_full, row_tiles * rows * 256);
                        for (int i = 0; i < row_tiles; ++i)
                            for (int h = 0; h < 2; ++h)
                                tma_load_3d(qs + i * kPQTile + h * kPQHalf, &q_map, 64 * h, it.head * p.group,
                                            it.start + it.token0 + i * p.tile_tokens, &sh.q_full);
                    }
                    __syncwarp();
                }
                // the reply is a write to shared memory like the copies: it is awaited whether another wait has run out or not
                lost |= !__all_sync(0xffffffffu, mbar_wait(&sh.cancel, n & 1));
                uint32_t taken, first;
                asm volatile(
                    "{\n\t.reg .b128 reply;\n\t.reg .pred p;\n\t"
                    "ld.shared.b128 reply, [%2];\n\t"
                    "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, reply;\n\t"
                    "selp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
                    "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, reply;\n\t}"
                    : "=r"(taken), "=r"(first)
                    : "r"(smem_u32(&sh.cancel_reply))
                    : "memory");
                proxy_fence();  // the reply has been read before the next one is asked for
                __syncwarp();
                index = taken && !lost ? static_cast<int>(first) : 0x7fffffff;
            }
            if (lost) {  // no copy may land after the block's end
                for (int t = tile > kPStages ? tile - kPStages : 0; t < tile; ++t) mbar_wait(&sh.kv_full[t % kPStages], (t / kPStages) & 1);
                if (queries > 0) mbar_wait(&sh.q_full, (queries - 1) & 1);
            }
        } else if (warp == 8) {
            // ---- scores, for both row tiles, as soon as those in front have been read -------------------------------------------
            constexpr uint32_t idesc = umma_idesc(kPKeys, false, false, BF16);
            const UmmaDesc q0 = umma_desc_halves(smem_u32(qs), 16, 1024), k0 = umma_desc_halves(smem_u32(ring), 16, 1024);
            const uint32_t columns = uniform(tmem);
            uint32_t made[2] = {0, 0};
            const int items = for_key_tiles(
                sh, lost, lane, 0,
                [&](int n) { wait_once(lost, &sh.q_full, n & 1); },
                [&](int i, int, uint32_t stage, bool issues) {
                    if (made[i] > 0) wait_once(lost, &sh.s_empty[i], (made[i] - 1) & 1);
                    ++made[i];
                    tc_fence_after();
                    const uint32_t d = columns + score_column(i), q = q0.low + ((i * kPQTile) >> 4), k = k0.low + stage * (kPKTile >> 4);
                    if (issues) {
                        umma_f16<false>(d, q, k, k0.high, idesc);
#pragma unroll
                        for (int ks = 1; ks < 8; ++ks)
                            umma_f16<true>(d, q + (((ks >> 2) * kPQHalf + (ks & 3) * 32) >> 4), k + (((ks >> 2) * kPKHalf + (ks & 3) * 32) >> 4), k0.high, idesc);
                        umma_commit(&sh.s_full[i]);
                    }
                },
                [&](bool issues) {
                    if (issues) umma_commit(&sh.q_empty);
                });
            if (items > 0) lost |= !mbar_wait(&sh.q_empty, (items - 1) & 1);  // of the last item, which nobody else waits for
        } else if (warp == 10) {
            // ---- outputs, as soon as weights are there ----------------------------------------------------------------------------
            constexpr uint32_t idesc = umma_idesc(128, false, true, BF16);
            const UmmaDesc v0 = umma_desc_halves(smem_u32(ring), kPKHalf, 1024);
            const uint32_t columns = uniform(tmem);
            uint32_t made[2] = {0, 0};
            for_key_tiles(
                sh, lost, lane, 1, [](int) {},
                [&](int i, int j, uint32_t stage, bool issues) {
                    wait_once(lost, &sh.p_full[i], made[i] & 1);
                    ++made[i];
                    tc_fence_after();
                    const uint32_t d = columns + output_column(i), a = columns + weight_column(i), v = v0.low + stage * (kPKTile >> 4);
                    if (issues) {
                        umma_f16_ta(d, a, v, v0.high, idesc, j > 0);
#pragma unroll
                        for (int ks = 1; ks < kPChunks; ++ks) umma_f16_ta(d, a + ks * 8, v + ks * (2048 >> 4), v0.high, idesc, 1);
                        umma_commit(&sh.p_empty[i]);
                    }
                },
                [](bool) {});
        }
    } else {
        // ---- softmax and output: thread = row -----------------------------------------------------------------------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPSoftmaxRegs));
        const int i = warp >> 2, row = tid & 127;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t s_at = tmem + lanes + score_column(i), p_at = tmem + lanes + weight_column(i), o_at = tmem + lanes + output_column(i);
        const int row_token = row / p.group, row_head = row - row_token * p.group;
        const float scale = p.scale_log2, slack = kPSlack / scale;
        // Finite, and finite times `scale`: scores of -infinity less it have weights of 0, and what comes later finds a sum of 0, no NaN.
        const float lowest = scale > 1.f ? kPLowest / scale : kPLowest;
        const auto arrive = [&](uint64_t* bar) {  // of the warp, behind its reads and writes of tensor memory
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        uint32_t seen = 0;
        int tile = 0;
        for (int n = 0;; ++n) {
            const int slot = n & 1;
            const bool posted = item_posted(&sh.item_full[slot], (n >> 1) & 1);
            const PromptItem it = sh.item[slot];
            lost |= !posted;
            if (it.tiles0 == 0 || __any_sync(0xffffffffu, !posted)) break;
            const int tiles = i ? it.tiles1 : it.tiles0, other = i ? it.tiles0 : it.tiles1;
            const int first_token = it.token0 + i * p.tile_tokens, token = first_token + row_token;
            const int limit = p.causal ? token : it.len - 1;  // last key that the row sees
            float m = 0.f, l = 0.f;
            bool far = false;  // the maximum of one of the warp's rows is
            for (int j = 0; j < tiles; ++j) {
                wait_once(lost, &sh.s_full[i], seen & 1);
                tc_fence_after();
                float s[kPChunks][16];
#pragma unroll
                for (int c = 0; c < kPChunks; ++c) tmem_ld16(s_at + c * 16, s[c]);
#pragma unroll
                for (int c = 0; c < kPChunks; ++c) tmem_ld_wait(s[c]);
                arrive(&sh.s_empty[i]);  // the next scores may come
                const bool masked = j * kPKeys + kPKeys > it.len || (p.causal && j * kPKeys + kPKeys - 1 > first_token);
                if (masked) {
                    const int last = limit - j * kPKeys;
#pragma unroll
                    for (int c = 0; c < kPChunks; ++c)
#pragma unroll
                        for (int e = 0; e < 16; ++e) s[c][e] = c * 16 + e <= last ? s[c][e] : -INFINITY;
                }
                float top[kPChunks];
#pragma unroll
                for (int c = 0; c < kPChunks; ++c) {
                    top[c] = max_nan(s[c][0], s[c][1]);
#pragma unroll
                    for (int e = 2; e < 16; e += 2) top[c] = max3_nan(top[c], s[c][e], s[c][e + 1]);
                }
                const float most = max3_nan(max3_nan(top[0], top[1], top[2]), top[3], top[4]);
                if (j > 0) {  // the product in front has read its weights, and the output is at rest
                    wait_once(lost, &sh.p_empty[i], (seen - 1) & 1);
                    tc_fence_after();
                }
                ++seen;
                if (j == 0) {
                    m = max_nan(most, lowest);
                    far = __any_sync(0xffffffffu, fabsf(m * scale) > kPNear);
                } else {
                    const bool grows = !(most <= m + slack);
                    if (__any_sync(0xffffffffu, grows)) {
                        const float next = grows ? max_nan(m, most) : m, factor = grows ? fast_exp2((m - next) * scale) : 1.f;
                        m = next, l *= factor;
                        far = __any_sync(0xffffffffu, fabsf(m * scale) > kPNear);
#pragma unroll 1
                        for (int c = 0; c < 4; ++c) {
                            float o[32];
                            tmem_ld32(o_at + c * 32, o);
                            tmem_ld_wait(o);
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] *= factor;
                            tmem_st32(o_at + c * 32, o);
                        }
                    }
                }
                // an infinite maximum: inf - inf, NaN for the whole row as in the formula
                float shift = m == INFINITY ? __int_as_float(0x7fffffff) : -m * scale;
                if (far) {
                    const bool mine = fabsf(shift) > kPNear;
                    const float off = mine ? m : 0.f;
#pragma unroll
                    for (int c = 0; c < kPChunks; ++c)
#pragma unroll
                        for (int e = 0; e < 16; ++e) s[c][e] -= off;
                    if (mine) shift = 0.f;
                }
                const float2 scales = make_float2(scale, scale), shifts = make_float2(shift, shift);
                float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int c = 0; c < kPChunks; ++c) {
                    float packed[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float2 x = fma2(make_float2(s[c][2 * e], s[c][2 * e + 1]), scales, shifts);
                        const float2 y = make_float2(fast_exp2(x.x), fast_exp2(x.y));
                        sum[e & 1] = add2(sum[e & 1], y);
                        packed[e] = __uint_as_float(pack2<BF16>(y.x, y.y));
                    }
                    tmem_st8(p_at + c * 8, packed);
                }
                if (masked && (i == 0 || j >= other) && row < kPKeys) {
                    const int vt = tile + 2 * j + 1, stage = vt % kPStages;
                    wait_once(lost, &sh.kv_full[stage], (vt / kPStages) & 1);
                    const bool behind = j * kPKeys + row >= it.len;
                    if ((behind || p.causal) && tame_value_row<BF16>(ring + stage * kPKTile + row * 128, behind, lane)) sh.tamed[slot] = 1;
                    proxy_fence();
                }
                __syncwarp();
                tmem_st_wait();
                arrive(&sh.p_full[i]);
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            }
            if (tiles) {
                wait_once(lost, &sh.p_empty[i], (seen - 1) & 1);
                tc_fence_after();
                const bool live = row < rows && token < it.len && !lost;
                const bool tamed = *static_cast<volatile int*>(&sh.tamed[slot]) != 0;
                const int64_t at = (static_cast<int64_t>(it.start + token) * p.kv_heads + it.head) * p.group + row_head;
                const float inv = 1.f / l;
                const uint32_t alive = __ballot_sync(0xffffffffu, live);
                // 64 columns (128 bytes) at a time.  Four lanes exchange their rows' quarters, so that together they write a row's 128
                // bytes: a line per four lanes where every lane's own row would be 32 lines an instruction.
#pragma unroll 1
                for (int c = 0; c < 2; ++c) {
                    uint32_t v[4][8];
#pragma unroll
                    for (int d = 0; d < 2; ++d) {
                        float o[32];
                        tmem_ld32(o_at + c * 64 + d * 32, o);
                        tmem_ld_wait(o);
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] *= inv;
                        if (tamed && live) {  // what was cleared reaches the rows that see it
                            for (int key = it.token0 / kPKeys * kPKeys; key <= limit; ++key) {
                                const unsigned short* from = p.v + (it.start + key) * p.v_token + it.head * p.v_head + c * 64 + d * 32;
#pragma unroll
                                for (int e = 0; e < 32; ++e)
                                    if (non_finite<BF16>(from[e])) o[e] += unpack<BF16>(from[e]);
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 16; ++e) v[2 * d + (e >> 3)][e & 7] = pack2<BF16>(o[2 * e], o[2 * e + 1]);
                    }
#pragma unroll
                    for (int step = 1; step < 4; step <<= 1)
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            if (x & step) continue;
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const bool upper = lane & step;
                                const uint32_t got = __shfl_xor_sync(0xffffffffu, upper ? v[x][e] : v[x | step][e], step);
                                if (upper) v[x][e] = got; else v[x | step][e] = got;
                            }
                        }
#pragma unroll
                    for (int x = 0; x < 4; ++x) {  // row x of the four
                        const int64_t there = __shfl_sync(0xffffffffu, at, (lane & 28) + x);
                        if (alive >> ((lane & 28) + x) & 1) store32(static_cast<unsigned short*>(p.out) + there * 128 + c * 64 + (lane & 3) * 16, v[x]);
                    }
                }
                tc_fence_before();
                if (live && p.lse) p.lse[at] = m * scale * kLn2 + logf(l);
            }
            tile += 2 * max(it.tiles0, it.tiles1);
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.item_empty[slot]);
        }
    }
    if (lost) atomicOr(p.status ? p.status : &g_prompt_status, RESKV_STATUS_WAIT_TIMEOUT);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

int check_rows(const char* what, const void* x, int64_t token, int64_t head) {
    if (!aligned16(x) || token % 8 || head % 8 || token <= 0 || head <= 0)
        return fail(RESKV_ERR_INVALID, "prompt_attention: %s must start on a 16-byte boundary, its strides be positive multiples of 8 elements", what);
    return check_device_pointer(x, "prompt_attention", what);
}

int rows_map(CUtensorMap* map, const void* x, int heads, int total, int64_t token, int64_t head, int box_heads, int box_tokens) {
    const cuuint64_t dims[3] = {kHeadDim, static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(total)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(head) * 2, static_cast<cuuint64_t>(token) * 2};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_tokens)};
    return encode_tensor_map(map, x, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, "prompt_attention");
}

template <bool BF16>
int launch(const PromptParams& p, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, unsigned items, cudaStream_t stream) {
    static std::atomic<unsigned long long> done{0};
    static const int registers = [] {
        cudaFuncAttributes a{};
        return cudaFuncGetAttributes(&a, prompt_attention_kernel<BF16>) == cudaSuccess ? a.numRegs : 0;
    }();
    if (registers != kPLaunchRegs)  // the softmax warps would wait for registers that nobody hands back
        return fail(RESKV_ERR_CUDA, "prompt_attention: built with %d registers a thread, not %d", registers, kPLaunchRegs);
    if (int rc = allow_smem(prompt_attention_kernel<BF16>, kPSmem, done, "cudaFuncSetAttribute(prompt_attention)")) return rc;
    return check_cuda(launch_overlapped(prompt_attention_kernel<BF16>, dim3(items), kPThreads, kPSmem, stream, false, p, q, k, v),
                      "prompt_attention launch");
}

}  // namespace
}  // namespace reskv

using namespace reskv;

extern "C" int reskv_prompt_attention(const void* q, const void* k, const void* v, const int32_t* cu_seqlens, int sequences, int total,
                                      int kv_heads, int q_heads, int bf16, int64_t q_token, int64_t q_head, int64_t k_token,
                                      int64_t k_head, int64_t v_token, int64_t v_head, float scaling, int causal, void* out, float* lse,
                                      void* stream) {
    return reskv_prompt_attention_reporting(q, k, v, cu_seqlens, sequences, total, kv_heads, q_heads, bf16, q_token, q_head, k_token, k_head,
                                            v_token, v_head, scaling, causal, out, lse, nullptr, stream);
}

extern "C" int reskv_prompt_attention_reporting(const void* q, const void* k, const void* v, const int32_t* cu_seqlens, int sequences,
                                                int total, int kv_heads, int q_heads, int bf16, int64_t q_token, int64_t q_head,
                                                int64_t k_token, int64_t k_head, int64_t v_token, int64_t v_head, float scaling, int causal,
                                                void* out, float* lse, uint32_t* status, void* stream) {
    if (sequences < 0 || total < 0 || kv_heads < 1 || q_heads < 1 || q_heads % kv_heads)
        return fail(RESKV_ERR_INVALID, "prompt_attention: %d sequences, %d tokens, %d query and %d KV heads", sequences, total, q_heads, kv_heads);
    if (q_heads / kv_heads > 128) return fail(RESKV_ERR_LIMIT, "prompt_attention: more than 128 query heads per KV head");
    if (!(scaling > 0.f) || !(scaling < 3.0e38f)) return fail(RESKV_ERR_INVALID, "prompt_attention: scaling must be positive and finite");
    if (sequences == 0 || total == 0) return RESKV_OK;
    if (!q || !k || !v || !cu_seqlens || !out) return fail(RESKV_ERR_INVALID, "prompt_attention: null pointer");
    if (int rc = check_rows("q", q, q_token, q_head)) return rc;
    if (int rc = check_rows("k", k, k_token, k_head)) return rc;
    if (int rc = check_rows("v", v, v_token, v_head)) return rc;
    if (reinterpret_cast<uintptr_t>(out) & 31u) return fail(RESKV_ERR_INVALID, "prompt_attention: out must start on a 32-byte boundary");
    if (int rc = check_device_pointer(out, "prompt_attention", "out")) return rc;
    if (int rc = check_device_pointer(cu_seqlens, "prompt_attention", "cu_seqlens")) return rc;
    if (lse)
        if (int rc = check_device_pointer(lse, "prompt_attention", "lse")) return rc;
    if (status)
        if (int rc = check_device_pointer(status, "prompt_attention", "status")) return rc;
    PromptParams p{};
    p.cu = cu_seqlens, p.sequences = sequences, p.total = total, p.kv_heads = kv_heads, p.group = q_heads / kv_heads;
    p.tile_tokens = 128 / p.group;
    p.v = static_cast<const unsigned short*>(v), p.v_token = v_token, p.v_head = v_head;
    p.out = out, p.lse = lse, p.scale_log2 = scaling * kLog2e, p.causal = causal != 0, p.status = status;
    CUtensorMap qm, km, vm;
    if (int rc = rows_map(&qm, q, q_heads, total, q_token, q_head, p.group, p.tile_tokens)) return rc;
    if (int rc = rows_map(&km, k, kv_heads, total, k_token, k_head, 1, kPKeys)) return rc;
    if (int rc = rows_map(&vm, v, kv_heads, total, v_token, v_head, 1, kPKeys)) return rc;
    // One row tile per item where all of them find an SM of their own, which the device counts unless the tokens alone say no.  us with
    // one and with two: 1 x 300 tokens, 32 / 8 heads 12.0 and 13.3, 1 x 512 14.5 and 16.8, five short ones 12.9 and 13.7; five of 100
    // (160 items of one row tile, 12 of them behind others) 13.4 and 12.1.
    const int64_t parts = sequences < total ? sequences : total;
    p.most_single = total / p.tile_tokens * kv_heads <= sm_count() ? sm_count() : 0;
    // every sequence has at most one item that is not full
    const int64_t items = (total / (p.most_single ? p.tile_tokens : 2 * p.tile_tokens) + parts) * kv_heads;
    if (items > 0x7ffffffe) return fail(RESKV_ERR_LIMIT, "prompt_attention: too many tokens for one call");
    const auto st = static_cast<cudaStream_t>(stream);
    return bf16 ? launch<true>(p, qm, km, vm, static_cast<unsigned>(items), st) : launch<false>(p, qm, km, vm, static_cast<unsigned>(items), st);
}

extern "C" int reskv_prompt_attention_status(uint32_t* status, void* stream) {
    if (!status) return fail(RESKV_ERR_INVALID, "prompt_attention_status: null destination");
    if (int rc = check_cuda(cudaStreamSynchronize(static_cast<cudaStream_t>(stream)), "prompt_attention_status synchronize")) return rc;
    return check_cuda(cudaMemcpyFromSymbol(status, g_prompt_status, sizeof(uint32_t)), "prompt_attention_status copy");
}
