// Attention over packed prompts (attention_packed) and of a batch whose
// requests share a prefix (attention_prefix): y = softmax(scale q K^T) V per
// head, without writing the scores.
//
// Both run one tcgen05 kernel over a list of items. Query heads that share a
// kv head are rows of the same tile (row r of a tile: token r / G, head r % G
// of the G heads of the kv head), so grouped heads read K and V once.
//
// One CTA per SM at a time, one item per CTA of the grid; a running CTA takes
// the items of CTAs that are not launched yet (cluster launch control), so
// uneven items spread by themselves and a CTA's set-up is paid once. Two
// streams of work per CTA, each with a 128-row query tile, score accumulator
// and softmax warps of its own:
//   warps 0-3    stream 0: softmax and epilogue, a row to a thread
//   warps 4-7    stream 1: the same
//   warp 8       MMA issuer
//   warp 9       TMA producer (Q tiles; K and V tiles of 128 keys in a ring)
//   warp 10      scheduler: writes the items into a ring for the other warps
//   warp 11      idle (12 warps leave 168 registers to a thread)
// TMEM: two score tiles (128 f32 columns each; the tile's probabilities
// overwrite its first half as 16-bit pairs and are the A operand of P V) and
// two output accumulators (128 columns each). For one stream the issuer
// alternates P V of key tile j and Q K^T of tile j + 1; the streams interleave,
// so one's softmax runs under the other's products. An item's streams are
// either two query tiles over the same keys (`paired`) or one query tile over
// alternate key tiles, joined in the block.
//
// What bounds it (d 128, f16, a causal prompt of 8192 with 32 heads: 0.49 ms,
// 1.12 PFLOP/s at the 1.6-1.75 GHz that the chip holds then; 65 % of the
// measured matrix peak): a pair's step over 128 keys takes about 3800 cycles,
// 2048 of them matrix work. A stream's own chain is longer than half of the
// step: 1700-1900 cycles of softmax (768 of them the exponentials that stay on
// the special-function unit), then its two products, 1024 cycles alone and
// 1300 behind the other stream's, then the way through two barriers. TMEM is
// full, so a third tile in flight would have to be smaller, which was slower:
// 64-key score tiles, two of them to a stream (the products then read Q twice
// as often); two threads to a row (more exchange than it saved); P handed on
// in parts; a second issuing warp.
//
// Softmax: running row maximum m (of the raw scores) and sum in f32;
// p = 2^(c s - r), c = scale log2 e and r = c m rounded: one rounding to a p, and
// what r is off by is a factor that all of a row's p share. Where results over
// different keys meet they are scaled from r to r (in a block) or the factor is
// taken out first (partial results). From |r| = 2^22 on it grows past what the
// 16-bit formats hold: such a row is computed again from s - m (slowRow).
// The accumulator is rescaled only when a row's maximum has grown by more than
// 2^8 since the last rescale: until then p stays within 2^8 of 1, far inside the
// 16-bit formats' range, and the factor cancels in the final division. The commit
// that makes Q K^T of tile j + 1 visible also covers P V of tile j (one thread
// issues both), so a rescale finds the accumulator at rest without another barrier.
//
// p is rounded to the inputs' 16-bit type for the product with V (the tensor
// cores take equal operand types); its row sum is taken before that rounding.
// f16 has few bits below 2^-14 and none below 2^-25, where the many small p of a
// long row may lie, so there p is held 2^7 times its value: at most 2^15, and the
// smallest step is 2^-31 of the row's largest (2^18 keys at e^-17.5 of the largest
// came to nothing without it). The factor cancels like the others.
//
// Keys past an item's end are masked in the scores and zeroed in V's tile (a
// zero probability times a NaN would be NaN). Values that only some rows of a
// tile may see (the causal edge) cannot be zeroed: a row whose result has a
// NaN or an infinity is computed again from its own keys (slowRow), which costs
// about 7 us a key and warp where all rows of a tile need it (a prompt of 8192
// whose values are all NaN: 180 ms; one such value: 51 ms).
//
// Every mbarrier wait is bounded; on a timeout the CTA raises the device
// status word, drains its copies, frees TMEM and returns.
#include <cudaTypedefs.h>

#include <atomic>
#include <climits>
#include <type_traits>

#include "heads.cuh"
#include "tc_common.cuh"

namespace mlkb {
int makeTmap3d(CUtensorMap* map, CUtensorMapDataType type, int elem_bytes, const void* base,
               const int64_t (&dims)[3], const int64_t (&strides)[2], const int (&box)[3],
               CUtensorMapSwizzle swizzle);

namespace {

constexpr int kTile = 128;   // rows of a query tile, keys of a key tile
constexpr int kWalk = 256;   // about how many groups a block may look at to find its items (512 single tokens
                             // over 10^6 keys: 0.80-0.87 ms; with levels of one key tile always, 1.05 ms)
constexpr int kItems = 2;    // item ring: the one in work and the next
constexpr int kThreads = 12 * 32;
constexpr int kMma = 8, kTma = 9, kSched = 10;  // warps; 0 to 7 are softmax warps, 11 is idle
constexpr int kConsumers = 10;                  // warps that read an item
constexpr uint64_t kLimitNs = 2000000000ull;  // of a wait, and its share for each key an item may have:
constexpr uint64_t kKeyNs = 16000, kMostNs = 60000000000ull;  // 32 rows done again take up to 7 us a key
constexpr float kRescale = 8.0f;  // log2 of the growth of a row maximum that forces a rescale
constexpr float kFar = 0x1p22f;   // scaled row maxima up to which c m may be rounded
constexpr int kPoly = 2;          // of 8 pairs of exponentials, how many go to the FMA pipe (0, 1, 3, 4: slower)
constexpr int kMaxSlots = 128;    // partial results a row may have: 16 x 4 of the prefix, as many of its own keys
constexpr int kOwnItems = 2;      // items of own keys an SM should get (4: more epilogues than the even end gives)
constexpr int kOwnTiles = 32;     // and their most key tiles (16 to 64: within 3 %)
constexpr int64_t kMaxHeadTotal = int64_t(1) << 40;  // rows x heads of a call, so that workspace bytes fit 64 bits

// What one pass through the pipeline computes. Keys are counted from the
// item's first; row limits (how many keys token i of a stream sees) are
// clamp(vis0 + i, 0, nk) when causal, nk otherwise.
struct Item {
    int32_t live;      // 0: no more items
    int32_t paired;    // streams: two query tiles over all keys / one, over alternate key tiles
    int32_t causal;
    int32_t src;       // key source: 0 = rows of map 0, 1 = rows or pages of map 1
    int32_t kvh;
    int32_t nk;        // keys
    int32_t k_row;     // contiguous source: row of the first key
    int32_t page_row;  // paged source: first entry of the request's page table
    int32_t key0;      // paged source: first key's index in the request
    int32_t q_row[2];  // first token row of each stream
    int32_t tok[2];    // its tokens
    int32_t n[2];      // its key tiles
    int32_t vis0[2];
    int32_t slot;      // partial-result slot
    int32_t parts;     // packed: chunks the keys are cut into
    int32_t spread;    // at most 32 rows, four times in the tile: each 32 lanes take 32 of a tile's keys
};

struct KeySource {
    const void* k;
    const void* v;
    int64_t k_row, k_head, v_row, v_head;  // strides, elements
};

struct Params {
    int32_t heads, kv_heads, group, d, tt;  // tt: tokens of a query tile
    uint64_t pair_inv;                      // 2^64 / (2 tt), upwards: exact quotients below 2^31
    float c2, grow;                         // scale * log2 e; kRescale / c2
    uint64_t limit;                         // of a wait, ns
    int* status;
    const void* q;
    int64_t q_row, q_head;
    KeySource src[2];
    void* y;
    int64_t y_row, y_head;
    // packed
    const int32_t* q_starts;
    const int32_t* k_starts;
    int32_t seqs, q_rows, k_rows, causal;  // slots > 0: keys may be cut into as many chunks
    // prefix
    const int32_t* lens;
    const int32_t* pages;
    int32_t batch, steps, prefix;
    int32_t page, page_shift, wide, n_pages;  // page size; pages of a request; pages in all
    int32_t pre_items, pre_tiles, pre_splits, pre_mt, pre_pairs;  // prefix items
    int32_t suf_slots, suf_mt, tickets, sms;                      // request items
    int32_t pre_spread, suf_spread, spread_tt;  // which items are spread; tokens of a spread tile
    int32_t pre_parts, suf_parts;               // slots of an item: 4 when spread, else 1
    int32_t* chunk;                                               // keys of a chunk, for the join
    float* part;
    float2* lse;         // of each partial result: row maximum, log2 of the sum of 2^(c s - c m)
    int32_t slots;       // partial results of a row, side by side
    int32_t wide_store;  // they start at multiples of 32 bytes
};

template <int D>
struct Smem {
    static constexpr int kHalves = D / 64;
    static constexpr uint32_t kBox = kTile * 128;          // 16 KB: 128 rows x 64 elements
    static constexpr uint32_t kTileBytes = kHalves * kBox;
    static constexpr int kStages = D == 64 ? 11 : 5;       // K / V ring: what fits
    uint8_t q[2][kTileBytes];
    uint8_t kv[kStages][kTileBytes];
    Item item[kItems];
    alignas(16) uint4 cancel;
    uint64_t full[kStages], empty[kStages];
    uint64_t qfull[2], qempty[2];
    uint64_t sfull[2], pfull[2], ofull[2];  // [stream]
    uint64_t xbar[4];                   // [lane quarter]: the streams' warps meet
    uint64_t ifull[kItems], iempty[kItems], cfull, cnext;
    float2 xch[2][kTile];               // [stream][row]: maximum and sum
    uint32_t tmem_base;
    int abort;
};

static_assert(Smem<128>::kStages > 4 && Smem<64>::kStages > 4, "ring places move by up to 4");
static_assert(sizeof(Smem<128>) <= 227 * 1024 && sizeof(Smem<64>) <= 227 * 1024, "shared memory of a block");

__device__ __forceinline__ int ceilDiv(int a, int b) { return (a + b - 1) / b; }

__device__ __forceinline__ int rowLimit(const Item& it, int st, int token) {
    int v = it.causal ? (st == 0 ? it.vis0[0] : it.vis0[1]) + token : it.nk;
    v = v < 0 ? 0 : v;
    return v < it.nk ? v : it.nk;
}

// Key tiles of an item.
__device__ __forceinline__ int itemTiles(const Item& it) {
    return it.paired ? (it.n[0] > it.n[1] ? it.n[0] : it.n[1]) : it.n[0] + it.n[1];
}

// Key tiles of the two streams of one query tile whose rows see at most `keys` keys.
__device__ __forceinline__ void splitTiles(Item& it, int keys) {
    const int tiles = ceilDiv(keys, kTile);
    it.n[0] = (tiles + 1) / 2;
    it.n[1] = tiles / 2;
}

// ---- scheduling: packed prompts ------------------------------------------------------
// Items are (sequence, pair of query tiles, kv head), numbered in order of
// falling cost (key tiles of the pair), so that the long ones start first. No
// list is stored: the warp walks cost levels x groups of 32 sequences, each
// lane counting its sequence's pairs of that cost, and goes on to the
// next cost that any sequence has (level by level: 63 us instead of 32 for 4
// queries over 16380 uneven keys, most of it spent by blocks that find no item).
// Where there are few items the keys of the long ones are cut into chunks, items
// of their own.
struct Seq {
    int q0, nq, k0, nk;
};

struct Walker {
    int level, base;     // cost level; first sequence of the current group
    int next;            // highest level below that any group seen at this one has
    int chunk;           // packed: most key tiles of an item, 0: any
    int top, step;       // packed: the first level; key tiles of a level
    int64_t before;      // items before (level, group)
    // packed, what is known of (level, group): its items, those up to the lane's
    // sequence, and of that its items, pairs, pairs from the level on and chunks
    bool known;
    int64_t total, upto, mine;
    Seq seq;
    int np, ge, parts;
    bool falls;          // some starts fall; then the highest start before the next group
    int floor;
};

// Sequence `s` (its starts fall or leave the operands: without queries, and
// refused); `falls`: whether those of the queries fall.
__device__ __forceinline__ Seq loadSeq(const Params& p, int s, bool& falls) {
    Seq r = {0, 0, 0, 0};
    if (s < p.seqs) {
        const int a = p.q_starts[s], b = p.q_starts[s + 1];
        const int c = p.k_starts[s], e = p.k_starts[s + 1];
        falls = falls || b < a;
        if (a < 0 || b < a || b > p.q_rows || c < 0 || e < c || e > p.k_rows) {
            if (p.status != nullptr) atomicExch(p.status, MLKB_ERR_INVALID);
        } else {
            r = {a, b - a, c, e - c};
        }
    }
    return r;
}

// The start of sequence `s` where it lies inside the operands, else 0.
__device__ __forceinline__ int startOf(const Params& p, int s) {
    const int start = s < p.seqs ? p.q_starts[s] : 0;
    return start >= 0 && start <= p.q_rows ? start : 0;
}

// Where some starts fall: a sequence that begins below an earlier start is
// refused too, so that no row is claimed twice. `s`, `r`: the lane's sequence, of
// 32; floor: the highest start (inside the operands) before those, and then before
// the next 32.
__device__ __forceinline__ void keepOrder(const Params& p, int s, int lane, int& floor, Seq& r) {
    int high = startOf(p, s);
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, high, o);
        if (lane >= o) high = max(high, t);
    }
    high = max(high, floor);
    floor = __shfl_sync(0xffffffffu, high, 31);
    if (r.q0 < high) r.nq = 0;  // a start that falls was refused already
}

// Pair of query tiles that has token `t`.
__device__ __forceinline__ int pairOf(const Params& p, int t) {
    return static_cast<int>(__umul64hi(static_cast<uint64_t>(t), p.pair_inv));
}

// Of a sequence's `np` pairs, how many have at least level `c` (they are its last).
__device__ __forceinline__ int pairsFrom(const Params& p, const Seq& s, int np, int c, int step) {
    if (c <= 0) return np;
    const int64_t need = static_cast<int64_t>(c - 1) * step * kTile + 1;  // keys
    if (s.nk < need) return 0;
    if (!p.causal) return np;
    const int tokens = static_cast<int>(need) - (s.nk - s.nq);  // the pair's last token is at least this one
    return np - (tokens <= 0 ? 0 : pairOf(p, tokens - 1));
}

// Level of the pair that ends with the sequence's token `end` (from 1).
__device__ __forceinline__ int pairLevel(const Params& p, const Seq& s, int end, int step) {
    const int keys = p.causal ? s.nk - s.nq + min(end, s.nq) : s.nk;
    const int tiles = keys <= 0 ? 0 : ceilDiv(keys, kTile);
    return step == 1 ? tiles : ceilDiv(tiles, step);
}

__device__ bool nextPacked(const Params& p, Walker& w, int64_t idx, Item& it, int lane) {
    if (idx < w.before) {  // numbers usually rise
        w.level = w.top;
        w.base = 0;
        w.next = -1;
        w.before = 0;
        w.known = false;
        w.floor = 0;
    }
    for (;;) {
        if (w.level < 0) return false;
        if (!w.known) {
            w.known = true;
            if (p.seqs > 32) {
                bool falls = false;
                w.seq = loadSeq(p, w.base + lane, falls);
                if (w.falls) keepOrder(p, w.base + lane, lane, w.floor, w.seq);
            }
            const Seq& s = w.seq;
            w.np = s.nq > 0 ? pairOf(p, s.nq - 1) + 1 : 0;
            w.ge = pairsFrom(p, s, w.np, w.level, w.step);
            w.parts = w.chunk > 0 && w.level > w.chunk ? ceilDiv(w.level, w.chunk) : 1;
            w.mine = static_cast<int64_t>(w.ge - pairsFrom(p, s, w.np, w.level + 1, w.step)) * p.kv_heads * w.parts;
            if (__any_sync(0xffffffffu, w.mine > 1 << 25)) {
                w.upto = w.mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int64_t t = __shfl_up_sync(0xffffffffu, w.upto, o);
                    if (lane >= o) w.upto += t;
                }
            } else {  // the sums fit 32 bits
                int upto = static_cast<int>(w.mine);
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int t = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += t;
                }
                w.upto = upto;
            }
            w.total = __shfl_sync(0xffffffffu, w.upto, 31);
            const int below = w.np - w.ge;  // pairs of a lower level; the last one's:
            w.next = max(w.next, below > 0 ? pairLevel(p, s, below * 2 * p.tt, w.step) : -1);
        }
        if (idx < w.before + w.total) {
            const int64_t at = idx - w.before;
            const unsigned hit = __ballot_sync(0xffffffffu, at < w.upto);
            if (lane == __ffs(hit) - 1) {
                const Seq& s = w.seq;
                const int unit = p.kv_heads * w.parts;
                const int rem = static_cast<int>(at - (w.upto - w.mine));
                const int pair = w.np - w.ge + rem / unit;
                const int part = rem % unit / p.kv_heads;
                const int c0 = w.parts > 1 ? part * w.chunk * kTile : 0;
                it.live = 1;
                it.causal = p.causal;
                it.src = 0;
                it.kvh = rem % p.kv_heads;
                it.nk = w.parts > 1 ? min(s.nk - c0, w.chunk * kTile) : s.nk;
                it.k_row = s.k0 + c0;
                it.page_row = 0;
                it.key0 = 0;
                it.slot = part;
                it.parts = w.parts;
                it.spread = 0;
                for (int st = 0; st < 2; ++st) {
                    const int t0 = (2 * pair + st) * p.tt;
                    int n = s.nq - t0;
                    n = n < 0 ? 0 : n < p.tt ? n : p.tt;
                    it.q_row[st] = s.q0 + t0;
                    it.tok[st] = n;
                    it.vis0[st] = s.nk - s.nq + t0 + 1 - c0;
                    it.n[st] = n > 0 ? ceilDiv(rowLimit(it, st, n - 1), kTile) : 0;
                }
                it.paired = it.tok[1] > 0;
                if (!it.paired) {
                    it.q_row[1] = it.q_row[0];
                    it.tok[1] = it.tok[0];
                    it.vis0[1] = it.vis0[0];
                    splitTiles(it, rowLimit(it, 0, it.tok[0] - 1));
                }
            }
            return true;
        }
        w.known = false;
        w.before += w.total;
        w.base += 32;
        if (w.base >= p.seqs) {
            w.base = 0;
            w.level = __reduce_max_sync(0xffffffffu, w.next);
            w.next = -1;
            w.floor = 0;
        }
    }
}

// ---- scheduling: a shared prefix ------------------------------------------------------
// Items 0 .. pre_items-1: (query tile or pair, key split, kv head) over the
// prefix, all tokens of the batch as rows; then the requests' own keys, cut
// into chunks: (request and chunk, kv head, query tile). Pairs come first and a
// single tile last: side by side over the same keys, pairs took 4.2 us for a
// key tile and singles 1.9, apart 2.3 and 1.5 (80 requests over 32768 keys: 165
// us with the query tile counted fastest, 139 us so).
struct OwnKeys {
    int keys;       // of a chunk; 0: not planned yet
    int64_t items;  // chunks of all requests x kv heads x query tiles
};

__device__ __forceinline__ int ownLength(const Params& p, int b) {
    const int cap = p.wide * p.page;
    int len = p.lens[b];
    if (len < 0 || len > cap) {
        if (p.status != nullptr) atomicExch(p.status, MLKB_ERR_INVALID);
        len = len < 0 ? 0 : cap;
    }
    return len;
}

// The chunk length, from the lengths on the device (the same in every block):
// enough chunks for kOwnItems items on each SM, but none under 2 tiles or, where there
// is work enough, over kOwnTiles, and at most suf_slots to a request.
__device__ void planOwnKeys(const Params& p, OwnKeys& own, int lane) {
    if (own.keys > 0) return;
    int64_t tiles = 0;
    int most = 0;
    for (int b = lane; b < p.batch; b += 32) {
        const int n = ceilDiv(ownLength(p, b), kTile);
        tiles += n;
        most = n > most ? n : most;
    }
    most = __reduce_max_sync(0xffffffffu, most);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
    const int64_t unit = static_cast<int64_t>(p.kv_heads) * p.suf_mt;
    const int64_t want = (tiles * unit + kOwnItems * p.sms - 1) / (kOwnItems * p.sms);
    int per = want < 2 ? 2 : want < kOwnTiles ? static_cast<int>(want) : kOwnTiles;
    const int least = ceilDiv(most, p.suf_slots);
    per = per > least ? per : least;
    int64_t chunks = 0;
    for (int b = lane; b < p.batch; b += 32) {
        chunks += ceilDiv(ceilDiv(ownLength(p, b), kTile), per);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) chunks += __shfl_xor_sync(0xffffffffu, chunks, o);
    own.keys = per * kTile;
    own.items = chunks * unit;
}

__device__ bool nextPrefix(const Params& p, OwnKeys& own, Walker& w, int64_t idx, Item& it,
                           int lane) {
    if (idx < p.pre_items) {
        if (lane == 0) {
            const int per_mt = p.pre_items / p.pre_mt;
            const int mt = static_cast<int>(idx) / per_mt;
            const int r = static_cast<int>(idx) % per_mt;
            const int split = r / p.kv_heads;
            const int first = split * p.pre_tiles * kTile;
            const int last = min(first + p.pre_tiles * kTile, p.prefix);
            const int tokens = p.batch * p.steps;
            it.live = 1;
            it.page_row = 0;
            it.key0 = 0;
            it.kvh = r % p.kv_heads;
            it.paired = mt < p.pre_pairs;  // the last query tile may be alone
            it.causal = 0;
            it.src = 0;
            it.k_row = first;
            it.nk = last - first;
            it.slot = split * p.pre_parts;
            it.spread = p.pre_spread;
            for (int st = 0; st < 2; ++st) {
                const int t0 = (2 * mt + (it.paired ? st : 0)) * p.tt;
                const int n = max(0, min(tokens - t0, p.tt));
                it.q_row[st] = t0;
                it.tok[st] = n;
                it.vis0[st] = 0;
                it.n[st] = n > 0 ? ceilDiv(it.nk, kTile) : 0;
            }
            if (!it.paired) splitTiles(it, it.nk);
        }
        return true;
    }
    if (p.suf_slots == 0) return false;
    planOwnKeys(p, own, lane);
    idx -= p.pre_items;
    if (idx == 0 && lane == 0) *p.chunk = own.keys;  // one block meets this number
    if (idx >= own.items) return false;
    if (idx < w.before) w = {};  // a new number may stand for items before the last one's
    const int unit = p.kv_heads * p.suf_mt;
    for (;;) {  // groups of 32 requests, each lane counting its request's items
        const int b = w.base + lane;
        const int len = b < p.batch ? ownLength(p, b) : 0;
        const int64_t mine = static_cast<int64_t>(ceilDiv(len, own.keys)) * unit;
        int64_t upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t t = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += t;
        }
        const int64_t total = __shfl_sync(0xffffffffu, upto, 31);
        if (idx >= w.before + total) {
            w.before += total;
            w.base += 32;
            if (w.base >= p.batch) return false;
            continue;
        }
        const int64_t at = idx - w.before;
        const unsigned hit = __ballot_sync(0xffffffffu, at < upto);
        if (lane == __ffs(hit) - 1) {
            const int rem = static_cast<int>(at - (upto - mine));
            const int chunk = rem / unit, mt = rem % unit % p.suf_mt;
            const int c0 = chunk * own.keys;
            const int t0 = mt * p.tt, n = min(p.steps - t0, p.tt);
            it.live = 1;
            it.kvh = rem % unit / p.suf_mt;
            it.paired = 0;
            it.causal = 1;
            it.src = 1;
            it.nk = min(len - c0, own.keys);
            it.k_row = p.pages == nullptr ? b * p.page + c0 : 0;
            it.page_row = b * p.wide;
            it.key0 = c0;
            it.vis0[0] = it.vis0[1] = len - p.steps + t0 + 1 - c0;
            it.slot = p.pre_splits * p.pre_parts + chunk * p.suf_parts;
            it.spread = p.suf_spread;
            for (int st = 0; st < 2; ++st) {
                it.q_row[st] = b * p.steps + t0;
                it.tok[st] = n;
            }
            splitTiles(it, rowLimit(it, 0, n - 1));
        }
        return true;
    }
}

// ---- one row from its definition ----------------------------------------------------------
__device__ __forceinline__ int pageRow(const Params& p, const Item& it, int key) {
    const int at = it.key0 + key;
    const int pg = p.pages[it.page_row + (at >> p.page_shift)];
    // -1 for an index outside the pages: its keys and values are zeros
    return (pg < 0 || pg >= p.n_pages) ? -1 : (pg << p.page_shift) + (at & (p.page - 1));
}

// Row `row` of the query tile from the definition, over the item's keys that
// the row sees (of a spread item, those of `part`), by a warp: a lane scores
// one of 32 keys and then owns four columns of the result. o: those columns
// (normalised); returns the row's maximum and the log2 of its sum. All lanes
// have one row.
template <typename T>
__device__ __noinline__ float2 slowRow(const Params& p, const Item& it, int st, int row, int part,
                                      float (&o)[4]) {
    const int lane = threadIdx.x & 31;
    const int token = row / p.group, head = it.kvh * p.group + row % p.group;
    const T* q = static_cast<const T*>(p.q) + (it.q_row[st] + token) * p.q_row + head * p.q_head;
    const KeySource& src = p.src[it.src];
    const T* kbase = static_cast<const T*>(src.k) + it.kvh * src.k_head;
    const T* vbase = static_cast<const T*>(src.v) + it.kvh * src.v_head + 4 * lane;
    const bool column = 4 * lane < p.d;
    const int lim = rowLimit(it, st, token);
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = 0.0f;
    for (int first = 0; first < lim; first += 32) {
        if (it.spread && (first >> 5 & 3) != part) continue;
        const int key = first + lane;
        int64_t krow = -1;
        float s = -INFINITY;
        if (key < lim) {
            krow = it.src == 1 && p.pages != nullptr ? pageRow(p, it, key)
                                                     : it.k_row + static_cast<int64_t>(key);
            s = 0.0f;
            if (krow >= 0) {
                const T* k = kbase + krow * src.k_row;
                for (int c = 0; c < p.d; c += 8) {
                    float a[8], b[8];
                    unpack8<T>(*reinterpret_cast<const uint4*>(q + c), a);
                    unpack8<T>(*reinterpret_cast<const uint4*>(k + c), b);
#pragma unroll
                    for (int i = 0; i < 8; ++i) s = fmaf(a[i], b[i], s);
                }
            }
        }
        float top = s;
        for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        if (__any_sync(0xffffffffu, s != s)) top = NAN;
        if (top == -INFINITY) continue;
        top = m > top ? m : top;  // a NaN score stays
        const float f = m == -INFINITY ? 0.0f : tc::ex2((m - top) * p.c2);
        m = top;
        const float e = key < lim ? tc::ex2((s - m) * p.c2) : 0.0f;
        float sum = e;
        for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        // o stays a weighted mean: sums of the largest bf16 values would leave the f32 range
        const float all = fmaf(l, f, sum), inv = 1.0f / all, keep = l * f * inv, share = e * inv;
        l = all;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] *= keep;
        for (int j = 0; j < 32; j += 8) {  // eight loads at a time
            uint2 u[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                const int64_t r = __shfl_sync(0xffffffffu, krow, j + x);
                u[x] = make_uint2(0, 0);
                if (r >= 0 && column) u[x] = *reinterpret_cast<const uint2*>(vbase + r * src.v_row);
            }
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                const float w = __shfl_sync(0xffffffffu, share, j + x);
                const float2 a = unpack2<T>(u[x].x), b = unpack2<T>(u[x].y);
                o[0] = fmaf(w, a.x, o[0]);
                o[1] = fmaf(w, a.y, o[1]);
                o[2] = fmaf(w, b.x, o[2]);
                o[3] = fmaf(w, b.y, o[3]);
            }
        }
        if (m != m) break;
    }
    if (m == -INFINITY) return make_float2(-INFINITY, -INFINITY);  // nothing to see: zeros
    return make_float2(m, log2f(l));
}

// 8 floats, in one store where `wide` says that the address is a multiple of 32.
__device__ __forceinline__ void store32(float* to, const uint64_t (&f)[4], int wide) {
    if (wide) {
        asm volatile("st.global.v4.b64 [%0], {%1, %2, %3, %4};" ::"l"(to), "l"(f[0]), "l"(f[1]), "l"(f[2]),
                     "l"(f[3])
                     : "memory");
    } else {
        reinterpret_cast<ulonglong2*>(to)[0] = make_ulonglong2(f[0], f[1]);
        reinterpret_cast<ulonglong2*>(to)[1] = make_ulonglong2(f[2], f[3]);
    }
}

// Among each four lanes, lane q's v[i] becomes lane i's v[q].
__device__ __forceinline__ void swap4(uint4& a, uint4& b, bool upper, int mask) {
    uint4 x = upper ? a : b;
    x.x = __shfl_xor_sync(0xffffffffu, x.x, mask);
    x.y = __shfl_xor_sync(0xffffffffu, x.y, mask);
    x.z = __shfl_xor_sync(0xffffffffu, x.z, mask);
    x.w = __shfl_xor_sync(0xffffffffu, x.w, mask);
    if (upper) {
        a = x;
    } else {
        b = x;
    }
}
__device__ __forceinline__ void transpose4(uint4 (&v)[4], int lane) {
    swap4(v[0], v[1], (lane & 1) != 0, 1);
    swap4(v[2], v[3], (lane & 1) != 0, 1);
    swap4(v[0], v[2], (lane & 2) != 0, 2);
    swap4(v[1], v[3], (lane & 2) != 0, 2);
}

// ---- the kernel ---------------------------------------------------------------------------
// kPrefix: attention_prefix, else attention_packed. kPartial: results go to the
// slots of the workspace, for the join.
template <int D, typename T, bool kPrefix, bool kPartial>
__global__ void __launch_bounds__(kThreads, 1)
attention_tcgen05(const __grid_constant__ CUtensorMap map_q,
                  const __grid_constant__ CUtensorMap map_qs,
                  const __grid_constant__ CUtensorMap map_k0,
                  const __grid_constant__ CUtensorMap map_v0,
                  const __grid_constant__ CUtensorMap map_k1,
                  const __grid_constant__ CUtensorMap map_v1, const __grid_constant__ Params p) {
    using Sm = Smem<D>;
    constexpr int kStages = Sm::kStages;
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    Sm& sm = *reinterpret_cast<Sm*>(smem_raw);
    if ((tc::smem_u32(smem_raw) & 1023u) != 0) {  // uniform: the swizzled tiles need this base
        if (threadIdx.x == 0 && p.status != nullptr) atomicExch(p.status, MLKB_ERR_INVALID);
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) {
            tc::mbar_init(&sm.full[i], 1);
            tc::mbar_init(&sm.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&sm.qfull[i], 1);
            tc::mbar_init(&sm.qempty[i], 1);
            tc::mbar_init(&sm.sfull[i], 1);
            tc::mbar_init(&sm.ofull[i], 1);
            tc::mbar_init(&sm.pfull[i], 4);
            tc::mbar_init(&sm.xbar[2 * i], 2);
            tc::mbar_init(&sm.xbar[2 * i + 1], 2);
        }
        for (int i = 0; i < kItems; ++i) {
            tc::mbar_init(&sm.ifull[i], 1);
            tc::mbar_init(&sm.iempty[i], kConsumers);
        }
        tc::mbar_init(&sm.cfull, 1);
        tc::mbar_init(&sm.cnext, 1);
        sm.abort = 0;
        tc::fence_barrier_init();
        tc::fence_proxy_async();
    }
    if (warp == kMma) tc::tmem_alloc(&sm.tmem_base, 512);
    if (warp == kTma && lane == 0) {
        tc::prefetch_tmap(&map_q);
        tc::prefetch_tmap(&map_k0);
        tc::prefetch_tmap(&map_v0);
        if (kPrefix) {
            tc::prefetch_tmap(&map_qs);
            tc::prefetch_tmap(&map_k1);
            tc::prefetch_tmap(&map_v1);
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    // Set-up overlaps the tail of the preceding grid; everything global waits for it.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t tmem = sm.tmem_base;
    volatile int* abort = &sm.abort;

    // Item `i` of this CTA once the scheduler has written it; null: no more, or
    // aborted. It stays in the ring until drop(i).
    auto take = [&](uint32_t i) -> const Item* {
        const Item& it = sm.item[i % kItems];
        if (!tc::mbar_wait(&sm.ifull[i % kItems], (i / kItems) & 1u, abort, p.limit)) return nullptr;
        return it.live != 0 ? &it : nullptr;
    };
    auto drop = [&](uint32_t i) {
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&sm.iempty[i % kItems]);
    };

    if (warp == kSched) {
        // ---------------- scheduler ----------------
        Walker w = {};
        OwnKeys own = {};
        if constexpr (!kPrefix) {
            int most = 0;
            int64_t tiles = 0;  // of all pairs, about: a pair in the middle for each
            auto add = [&](const Seq& q) {
                w.seq = q;
                if (q.nq > 0 && q.nk > most) most = q.nk;
                const int middle = p.causal ? max(q.nk - q.nq / 2, 0) : q.nk;
                tiles += static_cast<int64_t>(ceilDiv(q.nq, 2 * p.tt)) * ceilDiv(middle, kTile);
            };
            bool falls = false;
            for (int s = lane; s - lane < p.seqs; s += 32) add(loadSeq(p, s, falls));
            w.falls = __any_sync(0xffffffffu, falls);
            if (w.falls) {
                most = 0;
                tiles = 0;
                for (int s = lane, floor = 0; s - lane < p.seqs; s += 32) {
                    Seq q = loadSeq(p, s, falls);
                    keepOrder(p, s, lane, floor, q);
                    add(q);
                }
            }
            most = __reduce_max_sync(0xffffffffu, most);
            w.top = ceilDiv(most, kTile);
            w.step = 1;
            if (kPartial) {
                // About kOwnItems items for each SM, of 4 tiles at least, in the slots there are.
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
                const int64_t want = (tiles * p.kv_heads + kOwnItems * p.sms - 1) / (kOwnItems * p.sms);
                w.chunk = max(static_cast<int>(min(want, static_cast<int64_t>(w.top) + 1)), 4);
                w.chunk = max(w.chunk, ceilDiv(w.top, p.slots));
            } else {
                // With many sequences a level is several key tiles: the walk has fewer than
                // 2 kWalk steps, and up to two more for each group of 32 sequences.
                const int64_t steps = static_cast<int64_t>(w.top) * ceilDiv(p.seqs, 32);
                w.step = steps <= kWalk ? 1 : static_cast<int>(min(steps / kWalk, static_cast<int64_t>(max(w.top, 1))));
                w.top = ceilDiv(w.top, w.step);
            }
            w.level = w.top;
            w.next = -1;
        }
        int64_t at = blockIdx.x;  // the block's own item first, then those of blocks not yet launched
        for (uint32_t n = 0, asked = 0;;) {
            Item& slot = sm.item[n % kItems];
            if (n >= kItems &&
                !tc::mbar_wait(&sm.iempty[n % kItems], ((n / kItems) - 1) & 1u, abort, p.limit)) {
                break;
            }
            bool live = false;
            if (at >= 0) {
                if constexpr (kPrefix) {
                    live = nextPrefix(p, own, w, at, slot, lane);
                } else {
                    live = nextPacked(p, w, at, slot, lane);
                }
            }
            if (live || at < 0) {
                if (!live && lane == 0) slot.live = 0;
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&sm.ifull[n % kItems]);
                if (!live) break;
                // The next number is asked for towards the end of this item's loads:
                // earlier would take work that another block is free for.
                if (!tc::mbar_wait(&sm.cnext, n++ & 1u, abort, p.limit)) break;
                if (kPrefix && at >= p.pre_items) {  // every `tickets`-th item of the requests
                    at += p.tickets;
                    continue;
                }
            }
            if (lane == 0) tc::cancel_ask(&sm.cancel, &sm.cfull);
            __syncwarp();
            int never = 0;  // the answer lands before the block may exit
            if (!tc::mbar_wait(&sm.cfull, asked++ & 1u, &never, kLimitNs)) {
                if (lane == 0) *abort = 1;
                break;
            }
            at = tc::cancel_answer(&sm.cancel);
        }
    } else if (warp == kTma) {
        // ---------------- TMA producer ----------------
        uint32_t ring = 0, qn[2] = {0, 0};
        Item it = {};  // a copy
        bool ok = true;
        auto load_q = [&](int st) -> bool {
            if (qn[st] > 0 && !tc::mbar_wait(&sm.qempty[st], (qn[st] - 1) & 1u, abort, p.limit)) {
                return false;
            }
            ++qn[st];
            if (lane == 0) {
                if (kPrefix && it.spread) {  // the same rows for each 32 lanes
                    tc::mbar_arrive_expect_tx(&sm.qfull[st], Sm::kHalves * 512u * p.group * p.spread_tt);
                    for (int h = 0; h < 4 * Sm::kHalves; ++h) {
                        tc::tma_load_3d(sm.q[st] + (h >> 2) * Sm::kBox + (h & 3) * 4096, &map_qs,
                                        &sm.qfull[st], (h >> 2) * 64, it.kvh * p.group, it.q_row[0]);
                    }
                } else {
                    tc::mbar_arrive_expect_tx(&sm.qfull[st], Sm::kHalves * 128u * p.group * p.tt);
                    for (int h = 0; h < Sm::kHalves; ++h) {
                        tc::tma_load_3d(sm.q[st] + h * Sm::kBox, &map_q, &sm.qfull[st], h * 64,
                                        it.kvh * p.group, st == 0 ? it.q_row[0] : it.q_row[1]);
                    }
                }
            }
            __syncwarp();
            return true;
        };
        auto load_kv = [&](const CUtensorMap* map, int tile) -> bool {
            const uint32_t st = ring % kStages;
            if (!tc::mbar_wait(&sm.empty[st], ((ring / kStages) & 1u) ^ 1u, abort, p.limit)) {
                return false;
            }
            ++ring;
            if (kPrefix && it.src == 1 && p.pages != nullptr) {
                // one box per page (or one tile of a larger page); pages past the last key stay out
                const int box = p.page < kTile ? p.page : kTile;
                int keys = it.nk - tile * kTile;
                keys = keys < kTile ? keys : kTile;
                const int boxes = ceilDiv(keys, box);
                if (lane == 0) {
                    tc::mbar_arrive_expect_tx(&sm.full[st], Sm::kHalves * 128u * box * boxes);
                }
                __syncwarp();
                if (lane < boxes) {
                    int row = pageRow(p, it, tile * kTile + lane * box);
                    if (row < 0) {
                        row = kMaxHeadRows;
                        if (p.status != nullptr) atomicExch(p.status, MLKB_ERR_INVALID);
                    }
                    for (int h = 0; h < Sm::kHalves; ++h) {
                        tc::tma_load_3d(sm.kv[st] + h * Sm::kBox + lane * box * 128, map,
                                        &sm.full[st], h * 64, it.kvh, row);
                    }
                }
                __syncwarp();
            } else if (lane == 0) {
                tc::mbar_arrive_expect_tx(&sm.full[st], Sm::kTileBytes);
                for (int h = 0; h < Sm::kHalves; ++h) {
                    tc::tma_load_3d(sm.kv[st] + h * Sm::kBox, map, &sm.full[st], h * 64, it.kvh,
                                    it.k_row + tile * kTile);
                }
            }
            __syncwarp();
            return true;
        };
        for (uint32_t i = 0; ok; ++i) {
            const Item* next = take(i);
            if (next == nullptr) break;
            it = *next;
            drop(i);
            const int tiles = itemTiles(it);
            const CUtensorMap* mk = kPrefix && it.src == 1 ? &map_k1 : &map_k0;
            const CUtensorMap* mv = kPrefix && it.src == 1 ? &map_v1 : &map_v0;
            if (it.n[0] > 0) ok = load_q(0);
            for (int t = 0; ok && t < tiles; ++t) {
                if (t == tiles - 1 && lane == 0) tc::mbar_arrive(&sm.cnext);
                ok = load_kv(mk, t);
                if (ok && t == 0 && it.paired && it.n[1] > 0) ok = load_q(1);
                ok = ok && load_kv(mv, t);
            }
            if (tiles == 0 && lane == 0) tc::mbar_arrive(&sm.cnext);
        }
        if (*abort) {  // copies in flight land before the CTA may exit
            int never = 0;
            for (uint32_t j = ring > kStages ? ring - kStages : 0; j < ring; ++j) {
                (void)tc::mbar_wait(&sm.full[j % kStages], (j / kStages) & 1u, &never, kLimitNs);
            }
            for (int st = 0; st < 2; ++st) {
                if (qn[st] > 0) {
                    (void)tc::mbar_wait(&sm.qfull[st], (qn[st] - 1) & 1u, &never, kLimitNs);
                }
            }
        }
    } else if (warp == kMma) {
        // ---------------- MMA issuer ----------------
        // Everything an issue needs is in registers before its wait ends: the
        // time between two issues is time the tensor core may stand idle.
        const int ksteps = ceilDiv(p.d, 16);
        const uint32_t idesc_s = tc::idesc_f16_f32(kTile, kTile, 0, 0, kBf16);
        const uint32_t idesc_o = tc::idesc_f16_f32(kTile, ksteps * 16, 0, 1, kBf16);
        const uint64_t kdesc = tc::smem_desc_sw128(tc::smem_u32(sm.kv[0]), 16, 1024);
        const uint64_t vdesc = tc::smem_desc_sw128(tc::smem_u32(sm.kv[0]), Sm::kBox, 1024);
        const uint64_t qdesc = tc::smem_desc_sw128(tc::smem_u32(sm.q[0]), 16, 1024);
        constexpr uint32_t kStep = Sm::kTileBytes >> 4;  // a tile in descriptor units
        uint32_t qphase[2] = {0, 0}, pphase[2] = {0, 0};
        // A place in the K / V ring: stage and parity.
        struct Place {
            uint32_t stage, parity;
            __device__ __forceinline__ void move(uint32_t by) {  // by < kStages
                stage += by;
                if (stage >= kStages) {
                    stage -= kStages;
                    parity ^= 1u;
                }
            }
        };
        auto wait = [&](const Place& x) {
            return tc::mbar_wait(&sm.full[x.stage], x.parity, abort, p.limit);
        };
        auto loaded = [&](const Place& x) { return tc::mbar_test(&sm.full[x.stage], x.parity); };
        // S[st] = Q[slot] K^T, by one thread.
        auto scores = [&](int st, uint32_t slot, const Place& k, bool release, bool q_done) {
            const uint64_t q0 = qdesc + slot * kStep, k0 = kdesc + k.stage * kStep;
            const uint32_t s0 = tmem + st * kTile;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                const uint32_t off = ((kk >> 2) * Sm::kBox + (kk & 3) * 32) >> 4;
                if (kk < ksteps) tc::mma_f16(s0, q0 + off, k0 + off, idesc_s, kk > 0);
            }
            tc::mma_commit(&sm.sfull[st]);
            if (release) tc::mma_commit(&sm.empty[k.stage]);
            if (q_done) tc::mma_commit(&sm.qempty[slot]);
        };
        Place at = {0, 0};
        bool ok = true;
        for (uint32_t i = 0; ok; ++i) {
            const Item* it = take(i);
            if (it == nullptr) break;
            const int n[2] = {it->n[0], it->n[1]}, nk = it->nk, tiles = itemTiles(*it);
            const bool paired = it->paired != 0;
            drop(i);
            const uint32_t step = paired ? 2 : 4;  // ring places a stream's next tile is ahead
            // Each stream's next K and V, and whether they are known to have landed.
            Place k[2] = {at, at}, v[2];
            if (!paired) k[1].move(2);
            bool known[2] = {false, false};
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                v[st] = k[st];
                v[st].move(1);
                if (!ok || n[st] == 0) continue;
                const uint32_t slot = paired ? st : 0;
                if (paired || st == 0) ok = tc::mbar_wait(&sm.qfull[slot], qphase[slot], abort, p.limit);
                ok = ok && wait(k[st]);
                tc::tc_fence_after();
                // In a pair the second stream, where it reads a tile, is the tile's
                // last reader; alternate tiles have one reader each. Q's last reader
                // is the stream that owns it, or the item's last tile.
                if (ok && tc::elect_one()) {
                    scores(st, slot, k[st], !paired || st == 1 || n[1] == 0,
                           n[st] == 1 && (paired || (st == 0 ? n[1] == 0 : n[0] == 1)));
                }
                __syncwarp();
            }
            int t = 0;
            // The steady state of a pair, without the cases of the loop below: both
            // streams have a tile t + 1, stream 1 reads each tile last, and what
            // stream 0 has waited for is there for stream 1.
            for (; ok && paired && t + 1 < n[0] && t + 1 < n[1]; ++t) {
                const Place vp = v[0];
                k[0].move(2);
                v[0].move(2);
                const Place kp = k[0];
                const uint64_t v0 = vdesc + vp.stage * kStep;
#pragma unroll
                for (int st = 0; st < 2; ++st) {
                    if (st == 0 && !known[0]) ok = wait(vp) && wait(kp);
                    ok = ok && tc::mbar_wait(&sm.pfull[st], pphase[st], abort, p.limit);
                    pphase[st] ^= 1u;
                    if (!ok) break;
                    if (st == 1) {  // look ahead: the answer comes while the products are issued
                        Place kn = kp;
                        kn.move(2);
                        known[0] = loaded(v[0]) && loaded(kn);
                    }
                    tc::tc_fence_after();
                    if (tc::elect_one()) {
                        const uint32_t o0 = tmem + 2 * kTile + st * kTile, p0 = tmem + st * kTile;
#pragma unroll
                        for (int q = 0; q < kTile / 16; ++q) {
                            tc::mma_f16_ts(o0, p0 + q * 8, v0 + q * 128, idesc_o, q > 0 || t > 0);
                        }
                        if (st == 1) tc::mma_commit(&sm.empty[vp.stage]);
                        scores(st, st, kp, st == 1, t + 2 == n[st]);
                    }
                    __syncwarp();
                }
            }
            if (paired && t > 0) {
                k[1] = k[0];
                v[1] = v[0];
                known[0] = known[1] = false;
            }
            for (; ok && (t < n[0] || t < n[1]); ++t) {
#pragma unroll
                for (int st = 0; st < 2; ++st) {
                    // O (+)= P V of the stream's tile t, then S of its tile t + 1.
                    if (!ok || t >= n[st]) continue;
                    const bool more = t + 1 < n[st];
                    const uint32_t slot = paired ? st : 0;
                    const Place vp = v[st];
                    k[st].move(step);
                    v[st].move(step);
                    const Place kp = k[st];
                    if (!known[st]) ok = wait(vp);
                    const int valid = nk - (paired ? t : 2 * t + st) * kTile;
                    if (valid < kTile && (!paired || st == 0 || t >= n[0])) {  // its first reader
                        for (int h = 0; h < Sm::kHalves; ++h) {
                            uint4* z = reinterpret_cast<uint4*>(sm.kv[vp.stage] + h * Sm::kBox);
                            for (int x = valid * 8 + lane; x < kTile * 8; x += 32) z[x] = make_uint4(0, 0, 0, 0);
                        }
                        tc::fence_proxy_async();
                        __syncwarp();
                    }
                    ok = ok && tc::mbar_wait(&sm.pfull[st], pphase[st], abort, p.limit);
                    pphase[st] ^= 1u;
                    if (!ok) continue;
                    const bool k_known = known[st];
                    // Look ahead for the other stream's next step: the answer comes
                    // while this step's products are issued. A pair shares its tiles.
                    if (paired && st == 0) {
                        known[1] = more || t + 1 >= n[1];
                    } else {
                        Place vn = v[st ^ 1], kn = k[st ^ 1];
                        kn.move(step);
                        known[st ^ 1] = loaded(vn) && loaded(kn);
                    }
                    const bool k_done = !paired || st == 1 || t + 1 >= n[1];
                    const bool q_done = t + 2 == n[st] && (paired || (st == 0 ? n[1] < n[0] : n[1] == n[0]));
                    tc::tc_fence_after();
                    if (tc::elect_one()) {
                        const uint32_t o0 = tmem + 2 * kTile + st * kTile, p0 = tmem + st * kTile;
                        const uint64_t v0 = vdesc + vp.stage * kStep;  // 16 keys: 2 KB of V
#pragma unroll
                        for (int q = 0; q < kTile / 16; ++q) {
                            tc::mma_f16_ts(o0, p0 + q * 8, v0 + q * 128, idesc_o, q > 0 || t > 0);
                        }
                        if (!more) tc::mma_commit(&sm.ofull[st]);
                        if (!paired || st == 1 || t >= n[1]) tc::mma_commit(&sm.empty[vp.stage]);
                        if (more && k_known) scores(st, slot, kp, k_done, q_done);
                    }
                    __syncwarp();
                    if (more && !k_known) {
                        ok = wait(kp);
                        tc::tc_fence_after();
                        if (ok && tc::elect_one()) scores(st, slot, kp, k_done, q_done);
                        __syncwarp();
                    }
                }
            }
            if (n[0] > 0) qphase[0] ^= 1u;
            if (paired && n[1] > 0) qphase[1] ^= 1u;
            const uint32_t next = at.stage + 2 * tiles;
            at.parity ^= (next / kStages) & 1u;
            at.stage = next % kStages;
        }
    } else if (warp < kMma) {
        // ---------------- softmax and epilogue ----------------
        const int st = warp >> 2, quarter = warp & 3;
        const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t s_addr = tmem + lanes + st * kTile;
        const uint32_t o_addr = tmem + lanes + 2 * kTile;  // stream 1's is kTile further
        uint32_t sn = 0, on[2] = {0, 0}, xn = 0;  // tiles; accumulators, by stream; meetings
        // Meets the other stream's warp of the same rows.
        auto meet = [&]() -> bool {
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&sm.xbar[quarter]);
            return tc::mbar_wait(&sm.xbar[quarter], xn++ & 1u, abort, p.limit);
        };
        bool ok = true;
        for (uint32_t i = 0; ok; ++i) {
            const Item* item = take(i);  // kept in the ring: a copy would not fit the registers
            if (item == nullptr) break;
            const Item& it = *item;
            const bool spread = kPrefix && it.spread != 0;
            const int row = (spread ? 0 : quarter * 32) + lane;
            const int token = row / p.group, head_in = row - token * p.group;
            const int lim = rowLimit(it, st, token);
            const int n = st == 0 ? it.n[0] : it.n[1], theirs = st == 0 ? it.n[1] : it.n[0];
            // keys the row sees from the stream's current tile on
            int left = lim - (it.paired ? 0 : st * kTile);
            const int stride = it.paired ? kTile : 2 * kTile;
            const bool mine = token < (st == 0 ? it.tok[0] : it.tok[1]) &&
                              token < (spread ? p.spread_tt : p.tt);
            const bool idle = !__any_sync(0xffffffffu, mine);  // no row of the warp is wanted
            float m = -INFINITY, l = 0.0f;
            // What the row's exponents are counted from (r above), and by how much p is
            // held larger.
            constexpr float kUp = kBf16 ? 0.0f : 7.0f;
            auto scaled = [&](float x) { return __fmul_rn(x, p.c2); };
            // Takes a tile's row maximum into m, the sum and the accumulator (`begun`).
            auto raise = [&](float top, bool begun) {
                const bool grow = top > m + p.grow;
                if (!__any_sync(0xffffffffu, grow)) return;
                const float f = grow ? tc::ex2(scaled(m) - scaled(top)) : 1.0f;
                m = grow ? top : m;
                l *= f;
                if (!begun) return;
                for (int x = 0; x < p.d; x += 16) {
                    uint32_t o[16];
                    tc::tmem_ld16(o_addr + st * kTile + x, o);
                    tc::tmem_ld_wait(o);
#pragma unroll
                    for (int y = 0; y < 16; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
                    tc::tmem_st16(o_addr + st * kTile + x, o);
                }
            };
            for (int jj = 0; jj < n; ++jj, ++sn, left -= stride) {
                if (!tc::mbar_wait(&sm.sfull[st], sn & 1u, abort, p.limit)) {
                    ok = false;
                    break;
                }
                if (idle) {
                    if (lane == 0) tc::mbar_arrive(&sm.pfull[st]);
                    continue;
                }
                tc::tc_fence_after();
                if (spread) {
                    // 32 of the tile's keys; the others' probabilities are zeros here
                    uint32_t v[32], w[16], zero[16] = {};
                    tc::tmem_ld32(s_addr + quarter * 32, v);
                    tc::tmem_ld_wait(v);
                    const int seen = left - quarter * 32;
                    float mx[2] = {-INFINITY, -INFINITY};
                    if (__any_sync(0xffffffffu, seen < 32)) {
#pragma unroll
                        for (int x = 0; x < 32; ++x) {
                            if (x >= seen) v[x] = __float_as_uint(-INFINITY);
                        }
                    }
#pragma unroll
                    for (int x = 0; x < 32; x += 2) {
                        mx[x / 2 % 2] = tc::max3(mx[x / 2 % 2], __uint_as_float(v[x]),
                                                 __uint_as_float(v[x + 1]));
                    }
                    raise(fmaxf(mx[0], mx[1]), jj > 0);
                    const float nm = m == -INFINITY ? 0.0f : kUp - scaled(m);
                    float sum[2] = {0.0f, 0.0f};
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        const float a = tc::ex2(fmaf(__uint_as_float(v[2 * x]), p.c2, nm));
                        const float b = tc::ex2(fmaf(__uint_as_float(v[2 * x + 1]), p.c2, nm));
                        sum[0] += a;
                        sum[1] += b;
                        w[x] = pack2<T>(a, b);
                    }
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        if (c == quarter) {
                            tc::tmem_st16(s_addr + c * 16, w);
                        } else {
                            tc::tmem_st16(s_addr + c * 16, zero);
                        }
                    }
                    tc::tmem_st_wait();
                    tc::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&sm.pfull[st]);
                    l += sum[0] + sum[1];
                    continue;
                }
                // The tile's scores are read twice, 32 at a time, for the row maximum
                // and for the probabilities: held whole they would spill.
                const bool masked = __any_sync(0xffffffffu, left < kTile);
                uint32_t s[2][32];
                auto hide = [&](uint32_t (&v)[32], int c) {
#pragma unroll
                    for (int x = 0; x < 32; ++x) {
                        if (c * 32 + x >= left) v[x] = __float_as_uint(-INFINITY);
                    }
                };
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                tc::tmem_ld32(s_addr, s[0]);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    tc::tmem_ld_wait(s[c & 1]);
                    tc::tmem_ld32(s_addr + ((c + 1) & 3) * 32, s[(c + 1) & 1]);  // last: the first again
                    if (masked) hide(s[c & 1], c);
#pragma unroll
                    for (int x = 0; x < 32; x += 2) {
                        mx[x / 2 % 4] = tc::max3_nan(mx[x / 2 % 4], __uint_as_float(s[c & 1][x]),
                                                     __uint_as_float(s[c & 1][x + 1]));
                    }
                }
                const float top = tc::max3_nan(tc::max3_nan(mx[0], mx[1], mx[2]), mx[3], mx[3]);
                raise(top, jj > 0);
                const float nm = m == -INFINITY ? 0.0f : kUp - scaled(m);
                const uint64_t c2 = tc::pair(p.c2, p.c2), nm2 = tc::pair(nm, nm);
                uint64_t sum[2] = {0, 0};
                auto probabilities = [&](auto plain) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t w[16];
                        tc::tmem_ld_wait(s[c & 1]);
                        if (c < 3) tc::tmem_ld32(s_addr + (c + 1) * 32, s[(c + 1) & 1]);
                        if (!plain.value) hide(s[c & 1], c);
#pragma unroll
                        for (int x = 0; x < 16; ++x) {
                            uint64_t v = tc::fma2(tc::pair(__uint_as_float(s[c & 1][2 * x]),
                                                           __uint_as_float(s[c & 1][2 * x + 1])),
                                                  c2, nm2);
                            if (plain.value && x % 8 < kPoly) {
                                v = tc::ex2_poly(v);
                            } else {
                                const float2 z = tc::unpair(v);
                                v = tc::pair(tc::ex2(z.x), tc::ex2(z.y));
                            }
                            sum[x & 1] = tc::add2(sum[x & 1], v);
                            const float2 z = tc::unpair(v);
                            w[x] = pack2<T>(z.x, z.y);
                        }
                        tc::tmem_st16(s_addr + c * 16, w);
                    }
                };
                // Masked scores are -inf, which only ex2 takes to an exact 0.
                if (masked) {
                    probabilities(std::false_type{});
                } else {
                    probabilities(std::true_type{});
                }
                tc::tmem_st_wait();
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&sm.pfull[st]);
                const float2 z = tc::unpair(tc::add2(sum[0], sum[1]));
                l = top == top ? l + (z.x + z.y) : top;  // a NaN score: ex2_poly may have passed over it
            }
            if (!ok) break;
            // Accumulators done with this item, of either stream.
            const uint32_t o_own = on[st], o_other = on[st ^ 1];
            on[st] += n > 0;
            on[st ^ 1] += theirs > 0;
            if (idle) {
                drop(i);
                continue;
            }
            // No score above -inf: nothing was seen. (A NaN score shows in l.)
            if (m == -INFINITY && l < 0x1p60f) l = 0.0f;
            // ---- the row's result ----
            // A pair's streams have rows of their own. Otherwise both have seen
            // half of the same rows' keys: each joins the two results for half
            // of the columns.
            if (n > 0 && !tc::mbar_wait(&sm.ofull[st], o_own & 1u, abort, p.limit)) break;
            float f0 = 1.0f, f1 = 0.0f;  // shares of this stream's and the other's accumulator
            int from = 0, to = D;
            if (!it.paired) {
                sm.xch[st][quarter * 32 + lane] = make_float2(m, l);
                if (!meet()) break;
                const float2 o = sm.xch[st ^ 1][quarter * 32 + lane];
                if (theirs > 0 && !tc::mbar_wait(&sm.ofull[st ^ 1], o_other & 1u, abort, p.limit)) break;
                const float both = fmaxf(m, o.x);
                f0 = l == 0.0f ? 0.0f : tc::ex2(scaled(m) - scaled(both));
                f1 = o.y == 0.0f ? 0.0f : tc::ex2(scaled(o.x) - scaled(both));
                l = l * f0 + o.y * f1;
                m = both;
                from = st * (D / 2);
                to = from + D / 2;
            }
            tc::tc_fence_after();
            const int64_t tok_row = (st == 0 ? it.q_row[0] : it.q_row[1]) + token;
            const int head = it.kvh * p.group + head_in;
            // 0 for a row that sees nothing; NaN stays
            const float inv = l > 0.0f ? 1.0f / l : l;
            f0 *= inv;
            f1 *= inv;
            using Out = typename std::conditional<kPartial, float, T>::type;
            constexpr int kVec = 16 / sizeof(Out);  // elements of a 16-byte store
            constexpr int kPass = 4 * kVec;         // columns at a time: 64 bytes of a row
            const int64_t slot = it.slot + (spread ? quarter : 0);
            Out* out = kPartial
                ? reinterpret_cast<Out*>(p.part) + ((tok_row * p.heads + head) * p.slots + slot) * p.d
                : static_cast<Out*>(p.y) + tok_row * p.y_row + head * p.y_head;
            // Four lanes store four rows together, 64 bytes of one row at a time. A
            // row that sees nothing is left to the end. (Every p of a row may
            // underflow where its maximum is far from 0.)
            const bool far = m != -INFINITY && !(fabsf(scaled(m)) < kFar);
            const bool store = mine && l != 0.0f;
            const int end = to < p.d ? to : p.d;
            const uint64_t f02 = tc::pair(f0, f0), f12 = tc::pair(f1, f1);
            uint64_t bad2 = 0;  // 0 times every value: NaN when one is infinite or NaN
            if (spread) {
                // Few rows, each for itself: all of both accumulators at once, stored 32
                // bytes at a time (16: 29.9 us instead of 27.4 for 24 requests of 5
                // tokens; whole tiles' rows are faster four lanes together, below).
                if constexpr (kPartial) {
                    uint32_t o[D / 32][16], u[D / 32][16];
#pragma unroll
                    for (int g = 0; g < D / 32; ++g) {
                        tc::tmem_ld16(o_addr + st * kTile + from + g * 16, o[g]);
                        tc::tmem_ld16(o_addr + (st ^ 1) * kTile + from + g * 16, u[g]);
                    }
#pragma unroll
                    for (int g = 0; g < D / 32; ++g) {
                        tc::tmem_ld_wait(o[g]);
                        tc::tmem_ld_wait(u[g]);
                        const bool done = from + g * 16 < p.d;  // columns that were computed
#pragma unroll
                        for (int y = 0; y < 16; y += 8) {
                            uint64_t f[4] = {0, 0, 0, 0};
#pragma unroll
                            for (int z = 0; z < 4; ++z) {
                                const int c = y + 2 * z;
                                if (n > 0 && done) {
                                    f[z] = tc::fma2(tc::pair(__uint_as_float(o[g][c]), __uint_as_float(o[g][c + 1])),
                                                    f02, 0);
                                }
                                if (theirs > 0 && done) {
                                    f[z] = tc::fma2(tc::pair(__uint_as_float(u[g][c]), __uint_as_float(u[g][c + 1])),
                                                    f12, f[z]);
                                }
                                bad2 = tc::fma2(f[z], 0, bad2);
                            }
                            if (store && from + g * 16 + y < end) store32(out + from + g * 16 + y, f, p.wide_store);
                        }
                    }
                }
            } else {
                Out* rows[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int src = (lane & ~3) + r;
                    const int64_t addr = __shfl_sync(0xffffffffu, reinterpret_cast<int64_t>(out), src);
                    rows[r] = __shfl_sync(0xffffffffu, static_cast<int>(store), src) != 0
                        ? reinterpret_cast<Out*>(addr) + (lane & 3) * kVec
                        : nullptr;
                }
#pragma unroll 1
                for (int x = from; x < end; x += kPass) {
                    uint4 v[4] = {};
#pragma unroll
                    for (int g = 0; g < kPass / 16; ++g) {
                        if (x + g * 16 >= end) break;  // columns there are not computed
                        uint32_t o[16];
                        uint64_t f[8] = {};
                        if (n > 0) {
                            tc::tmem_ld16(o_addr + st * kTile + x + g * 16, o);
                            tc::tmem_ld_wait(o);
#pragma unroll
                            for (int y = 0; y < 8; ++y) {
                                f[y] = tc::fma2(tc::pair(__uint_as_float(o[2 * y]), __uint_as_float(o[2 * y + 1])),
                                                f02, 0);
                            }
                        }
                        if (!it.paired && theirs > 0) {
                            tc::tmem_ld16(o_addr + (st ^ 1) * kTile + x + g * 16, o);
                            tc::tmem_ld_wait(o);
#pragma unroll
                            for (int y = 0; y < 8; ++y) {
                                f[y] = tc::fma2(tc::pair(__uint_as_float(o[2 * y]), __uint_as_float(o[2 * y + 1])),
                                                f12, f[y]);
                            }
                        }
                        uint32_t w[16];
#pragma unroll
                        for (int y = 0; y < 8; ++y) {
                            bad2 = tc::fma2(f[y], 0, bad2);
                            const float2 z = tc::unpair(f[y]);
                            if constexpr (kPartial) {
                                w[2 * y] = __float_as_uint(z.x);
                                w[2 * y + 1] = __float_as_uint(z.y);
                            } else {
                                w[y] = pack2<T>(z.x, z.y);
                            }
                        }
#pragma unroll
                        for (int y = 0; y < (kPartial ? 4 : 2); ++y) {
                            v[(kPartial ? 0 : 2 * g) + y] = make_uint4(w[4 * y], w[4 * y + 1], w[4 * y + 2], w[4 * y + 3]);
                        }
                    }
                    transpose4(v, lane);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        if (rows[r] != nullptr && x + (lane & 3) * kVec < end) {
                            *reinterpret_cast<uint4*>(rows[r] + x) = v[r];
                        }
                    }
                }
            }
            float2 lse = l > 0.0f ? make_float2(m, log2f(l) - kUp - fmaf(m, p.c2, -scaled(m)))
                                  : make_float2(-INFINITY, -INFINITY);
            // A NaN or an infinity among the scores or the values (beside a score of +inf
            // ex2_poly gives numbers), or a maximum too far from 0.
            const float2 bad = tc::unpair(bad2);
            const bool again = mine && (far || (l != 0.0f && (!(l < 0x1p60f) || bad.x != 0.0f || bad.y != 0.0f)));
            const bool zeros = !kPartial && mine && l == 0.0f && !far;
            const unsigned todo = __ballot_sync(0xffffffffu, again || zeros);
            if (todo != 0) {
                __syncwarp();  // after the other lanes' stores
                const unsigned slow = __ballot_sync(0xffffffffu, again);
                for (unsigned left_rows = todo; left_rows != 0; left_rows &= left_rows - 1) {
                    const int src = __ffs(left_rows) - 1;
                    Out* to_row = reinterpret_cast<Out*>(
                        __shfl_sync(0xffffffffu, reinterpret_cast<int64_t>(out), src));
                    float o[4] = {};
                    if (slow >> src & 1u) {
                        const float2 z = slowRow<T>(p, it, st, __shfl_sync(0xffffffffu, row, src), quarter, o);
                        if (lane == src) lse = z;
                    }
                    if (4 * lane >= from && 4 * lane < end) {
                        if constexpr (kPartial) {
                            *reinterpret_cast<float4*>(to_row + 4 * lane) = make_float4(o[0], o[1], o[2], o[3]);
                        } else {
                            *reinterpret_cast<uint2*>(to_row + 4 * lane) =
                                make_uint2(pack2<T>(o[0], o[1]), pack2<T>(o[2], o[3]));
                        }
                    }
                }
            }
            if (kPartial && mine && from == 0) {
                float2* out_lse = p.lse + (tok_row * p.heads + head) * p.slots;
                out_lse[slot] = lse;
                if (!kPrefix && it.slot == 0) {  // slots without a chunk
                    for (int x = it.parts; x < p.slots; ++x) out_lse[x] = make_float2(-INFINITY, -INFINITY);
                }
            }
            tc::tc_fence_before();  // the reads above come before the next item's products
            const bool together = !it.paired;
            drop(i);
            if (together && !meet()) break;
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    if (warp == kMma) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, 512);
    }
    if (threadIdx.x == 0 && sm.abort && p.status != nullptr) atomicExch(p.status, MLKB_ERR_TIMEOUT);
}

// ---- joining the partial results of attention_prefix ----------------------------------------
// Bound by latency at the sizes there are (13 slots of 2560 rows: 17 MB out of
// L2), so slots lie side by side and eight are loaded at a time (a slot's rows
// side by side, one load at a time: 171 us instead of 153 for a whole call over
// a prefix of 32768). One warp per result row: y = sum_i w_i o_i / sum_i w_i over
// the row's slots, w_i = 2^(c (m_i - top) + log2 of slot i's sum) with the largest
// of the maxima m_i as top; slots that saw no key have m = -inf and are not read.
struct JoinParams {
    const float* part;
    const float2* lse;
    float c2;
    int64_t rows, y_row, y_head;
    int32_t slots, heads, d;
    // prefix: slots of the prefix, of a chunk of own keys, and the chunk
    int32_t prefix_slots, parts, cap, per_request;
    const int32_t* chunk;
    const int32_t* lens;
};

template <typename T, bool kPrefix>
__global__ void __launch_bounds__(256)
attention_join(const __grid_constant__ JoinParams p, const __grid_constant__ Params seqs, T* y) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    if (row >= p.rows) return;
    int slots = p.slots;
    const int d = p.d;
    if constexpr (!kPrefix) {  // a row of no sequence was not computed
        const int token = static_cast<int>(row / p.heads);
        bool mine = false, falls = false;
#pragma unroll 1
        for (int s = lane, floor = 0; s - lane < seqs.seqs; s += 32) {
            Seq q = loadSeq(seqs, s, falls);
            const int high = __reduce_max_sync(0xffffffffu, startOf(seqs, s));
            int before = floor;
            if (__any_sync(0xffffffffu, falls)) keepOrder(seqs, s, lane, before, q);
            floor = max(floor, high);
            mine = mine || (token >= q.q0 && token < q.q0 + q.nq);
        }
        if (!__any_sync(0xffffffffu, mine)) return;
    }
    // The prefix' slots are all written; of its own keys those of chunks that exist.
    const float2* mine = p.lse + row * slots;
    const float* part = p.part + row * slots * d;
    const float2 none = make_float2(-INFINITY, -INFINITY);
    float2 z[kMaxSlots / 32];
#pragma unroll
    for (int i = 0; i < kMaxSlots / 32; ++i) {
        z[i] = lane + 32 * i < slots ? mine[lane + 32 * i] : none;
    }
    if (kPrefix && slots > p.prefix_slots) {
        const int keys = *p.chunk;
        int len = p.lens[row / p.per_request];
        len = len < 0 ? 0 : len < p.cap ? len : p.cap;
        slots = p.prefix_slots + (len + keys - 1) / keys * p.parts;
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kMaxSlots / 32; ++i) {
        if (lane + 32 * i >= slots) z[i] = none;
        top = fmaxf(top, z[i].x);
    }
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float sum = 0.0f, e[kMaxSlots / 32];
#pragma unroll
    for (int i = 0; i < kMaxSlots / 32; ++i) {
        e[i] = z[i].x == -INFINITY ? 0.0f : tc::ex2(fmaf(z[i].x - top, p.c2, z[i].y));
        sum += e[i];
    }
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < kMaxSlots / 32; ++i) e[i] *= inv;  // first: sums of large values may leave the f32 range
    const bool live = 4 * lane < d;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < kMaxSlots / 32; ++i) {
        for (int s = 0; s < 32 && 32 * i + s < slots; s += 8) {  // eight loads at a time
            float4 v[8];
            float w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                w[j] = __shfl_sync(0xffffffffu, e[i], s + j);
                v[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                // a weight of 0: no key seen there, or nothing beside the others
                if (live && w[j] != 0.0f) {
                    v[j] = *reinterpret_cast<const float4*>(part + (32 * i + s + j) * d + 4 * lane);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                acc.x = fmaf(w[j], v[j].x, acc.x);
                acc.y = fmaf(w[j], v[j].y, acc.y);
                acc.z = fmaf(w[j], v[j].z, acc.z);
                acc.w = fmaf(w[j], v[j].w, acc.w);
            }
        }
    }
    if (live) {
        T* out = y + (row / p.heads) * p.y_row + (row % p.heads) * p.y_head + 4 * lane;
        *reinterpret_cast<uint2*>(out) =
            make_uint2(pack2<T>(acc.x, acc.y), pack2<T>(acc.z, acc.w));
    }
}

// ---- host ---------------------------------------------------------------------------------
struct Maps {
    CUtensorMap q, qs, k0, v0, k1, v1;
};

// [rows, heads, d] view as a 3-D map, box [box_rows, box_heads, 64]. A view
// without rows is never loaded from: it gets a stand-in address.
int headsMap(CUtensorMap* map, const mlkb_heads& t, int64_t heads, int64_t d, int dtype,
             int box_heads, int box_rows, const void* standin) {
    const int64_t dims[3] = {d, heads, t.rows > 0 ? t.rows : 1};
    const int64_t strides[2] = {t.head_stride, t.row_stride};
    const int box[3] = {64, box_heads, box_rows};
    return makeTmap3d(map,
                      dtype == MLKB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                        : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                      2, t.rows > 0 ? t.data : standin, dims, strides, box,
                      CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int D, typename T, bool kPrefix, bool kPartial>
int launchKernel(const Maps& m, const Params& p, int grid, cudaStream_t s) {
    static std::atomic<bool> attr[64];
    int dev = 0;
    cudaGetDevice(&dev);
    auto kernel = attention_tcgen05<D, T, kPrefix, kPartial>;
    if (dev >= 0 && dev < 64 && !attr[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   static_cast<int>(sizeof(Smem<D>)));
        if (e != cudaSuccess) return setCudaError(MLKB_ERR_LAUNCH, e, "attention smem attribute");
        attr[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = sizeof(Smem<D>);
    cfg.stream = s;
    cudaLaunchAttribute pdl[1];
    pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = pdl;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, m.q, m.qs, m.k0, m.v0, m.k1, m.v1, p);
    return e == cudaSuccess ? okStatus() : setCudaError(MLKB_ERR_LAUNCH, e, "attention launch");
}

template <bool kPrefix, bool kPartial>
int launchAttention(const Maps& m, const Params& p, int dtype, int grid, cudaStream_t s) {
    if (dtype == MLKB_F16) {
        return p.d <= 64 ? launchKernel<64, __half, kPrefix, kPartial>(m, p, grid, s)
                         : launchKernel<128, __half, kPrefix, kPartial>(m, p, grid, s);
    }
    return p.d <= 64 ? launchKernel<64, __nv_bfloat16, kPrefix, kPartial>(m, p, grid, s)
                     : launchKernel<128, __nv_bfloat16, kPrefix, kPartial>(m, p, grid, s);
}

int64_t joinBlocks(int64_t rows) { return (rows + 7) / 8; }

template <bool kPrefix>
int launchJoin(const JoinParams& j, const Params& p, void* y, int dtype, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(joinBlocks(j.rows)));
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cudaLaunchAttribute pdl[1];
    pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = pdl;
    cfg.numAttrs = 1;
    const cudaError_t e =
        dtype == MLKB_F16
            ? cudaLaunchKernelEx(&cfg, attention_join<__half, kPrefix>, j, p, static_cast<__half*>(y))
            : cudaLaunchKernelEx(&cfg, attention_join<__nv_bfloat16, kPrefix>, j, p,
                                 static_cast<__nv_bfloat16*>(y));
    return e == cudaSuccess ? okStatus() : setCudaError(MLKB_ERR_LAUNCH, e, "attention join launch");
}

bool headsFit(int64_t heads, int64_t kv_heads) {
    return heads >= 1 && kv_heads >= 1 && kv_heads <= 65536 && heads % kv_heads == 0 &&
           heads / kv_heads <= kTile;
}
bool sizeFits(int64_t d) { return d >= 8 && d <= 128 && d % 8 == 0; }
bool shapeFits(int64_t heads, int64_t kv_heads, int64_t d) { return headsFit(heads, kv_heads) && sizeFits(d); }

// Checks what both entries share.
int checkShape(int64_t heads, int64_t kv_heads, int64_t d, double scale, int32_t dtype) {
    if (dtype != MLKB_F16 && dtype != MLKB_BF16) {
        return setError(MLKB_ERR_INVALID, "attention: dtype must be f16 or bf16");
    }
    if (!headsFit(heads, kv_heads)) {
        return setError(MLKB_ERR_INVALID,
                        "attention: heads must be a multiple of kv heads, at most 128 to each");
    }
    if (!sizeFits(d)) {
        return setError(MLKB_ERR_INVALID, "attention: d must be a multiple of 8, 8 to 128");
    }
    const float c2 = static_cast<float>(scale * 1.4426950408889634);
    if (!(scale > 0) || !std::isfinite(c2) || c2 < 1e-30f) {
        return setError(MLKB_ERR_INVALID, "attention: scale must be positive and finite");
    }
    return MLKB_OK;
}

void setShape(Params& p, int64_t heads, int64_t kv_heads, int64_t d, double scale, int64_t keys) {
    p.heads = static_cast<int32_t>(heads);
    p.kv_heads = static_cast<int32_t>(kv_heads);
    p.group = static_cast<int32_t>(heads / kv_heads);
    p.d = static_cast<int32_t>(d);
    p.tt = kTile / p.group;
    p.pair_inv = ~uint64_t(0) / static_cast<uint64_t>(2 * p.tt) + 1;
    p.c2 = static_cast<float>(scale * 1.4426950408889634);
    p.grow = kRescale / p.c2;
    p.limit = kLimitNs + kKeyNs * static_cast<uint64_t>(keys);
    if (p.limit > kMostNs) p.limit = kMostNs;
    p.status = deviceStatusPtr();
}

KeySource keySource(const mlkb_heads& k, const mlkb_heads& v) {
    return {k.data, v.data, k.row_stride, k.head_stride, v.row_stride, v.head_stride};
}

// How attention_packed cuts its work.
struct PackedPlan {
    int64_t items, slots, rows;
    int64_t bytes(int64_t d) const { return slots * rows * (d + 2) * 4; }
};

PackedPlan planPacked(int64_t rows, int64_t key_rows, int64_t seqs, int64_t heads, int64_t kv_heads,
                      int64_t d) {
    PackedPlan r = {};
    const int64_t sms = smCount(), pair = 2 * (kTile / (heads / kv_heads));
    // Most pairs of query tiles there can be: every sequence may end inside one.
    r.items = (rows / pair + (seqs < rows ? seqs : rows)) * kv_heads;
    r.rows = rows * heads;
    // Items for at most half the SMs, and sequences that may be long: keys are cut
    // into up to 64 chunks of 4 tiles at least, no more than one to an SM. With
    // about an item to an SM joining costs more than it gives (1030 queries of 5
    // sequences, 32 heads: 84 us cut, 63 us whole); one query over 16384 keys, 8
    // heads to a kv head: 131 us whole, 30 us in 8 chunks, 25 us in 32; twice as
    // many chunks, or chunks of 2 tiles, are no faster or slower there (28 us).
    const int64_t tiles = (key_rows + kTile - 1) / kTile;
    // Each block looks through the sequences, 32 at a time, for each key count among
    // the pairs, and each row's join once more: with very many empty sequences that
    // costs more than cutting gives (that query among 4096 sequences 86 us cut, 159
    // whole; among 16384 275 and 239; among 10^6 15.4 and 6.7 ms).
    const int64_t walk = (seqs + 31) / 32 * (r.items / kv_heads);
    if (r.items > 0 && 2 * r.items <= sms && tiles > 8 && walk <= kWalk) {
        r.slots = sms / r.items;
        if (r.slots > tiles / 4) r.slots = tiles / 4;
        if (r.slots > 64) r.slots = 64;
    }
    return r;
}

// How attention_prefix cuts its work, from shapes alone (the lengths are on
// the device).
struct PrefixPlan {
    int64_t tt, rows, pairs, mt, tiles, splits, pre_items;
    int64_t suf_mt, suf_slots, tickets, slots;
    int64_t spread_tt, pre_spread, suf_spread;

    // The partial results, their maxima and log-sums, and the chunk length.
    int64_t bytes(int64_t d) const { return slots * rows * (d + 2) * 4 + 32; }

    // Whether the kernels' 32-bit counts hold it: items, those of a request, and the
    // join's rows of a request and blocks.
    bool fits(int64_t steps, int64_t heads, int64_t kv_heads) const {
        return pre_items + tickets <= INT_MAX && slots <= kMaxSlots &&
               kv_heads * suf_mt * suf_slots <= INT_MAX && steps * heads <= INT_MAX &&
               joinBlocks(rows) <= INT_MAX;
    }
};

PrefixPlan planPrefix(int64_t batch, int64_t steps, int64_t heads, int64_t kv_heads,
                      int64_t prefix, int64_t cap) {
    PrefixPlan r = {};
    r.tt = kTile / (heads / kv_heads);
    r.rows = batch * steps * heads;
    const int64_t sms = smCount();
    const int64_t qt = (batch * steps + r.tt - 1) / r.tt;
    r.pairs = qt / 2;
    r.mt = (qt + 1) / 2;
    const int64_t tiles = (prefix + kTile - 1) / kTile;
    if (tiles > 0) {
        // At most 16 splits, none shorter than 2 tiles: the number for which the
        // items' rounds over the SMs are shortest (an item costs about 2 tiles more).
        const int64_t units = r.mt * kv_heads;
        int64_t best = INT64_MAX;
        for (int64_t s = 1; s <= 16 && s <= (tiles + 1) / 2; ++s) {
            const int64_t per = (tiles + s - 1) / s, n = (tiles + per - 1) / per;
            const int64_t cost = (units * n + sms - 1) / sms * (per + 2);
            if (cost < best) {
                best = cost;
                r.tiles = per;
                r.splits = n;
            }
        }
    }
    r.pre_items = r.splits * kv_heads * r.mt;
    r.suf_mt = (steps + r.tt - 1) / r.tt;
    const int64_t most = (cap + 2 * kTile - 1) / (2 * kTile);  // chunks of 2 tiles
    r.suf_slots = most < 16 ? most : 16;
    // The requests' items are numbered modulo the tickets: how many there are is
    // known on the device only, and a block that finds none costs its launch.
    const int64_t items = batch * kv_heads * r.suf_mt * r.suf_slots;
    r.tickets = items < 8 * sms ? items : 8 * sms;
    // Few rows: spread over the tile's lanes. That divides the softmax, the
    // longest link between two products, by four (128 requests of up to 4096
    // own keys: 203 us, 5.4 TB/s, 83 % of the measured copy rate).
    r.spread_tt = 32 / (heads / kv_heads);
    r.pre_spread = r.spread_tt >= batch * steps;
    r.suf_spread = r.spread_tt >= steps;
    r.slots = r.splits * (r.pre_spread ? 4 : 1) + r.suf_slots * (r.suf_spread ? 4 : 1);
    return r;
}

}  // namespace
}  // namespace mlkb

extern "C" int mlkb_attention_packed(const mlkb_heads* q, const mlkb_heads* k, const mlkb_heads* v,
                                     const mlkb_heads* y, int64_t heads, int64_t kv_heads,
                                     int64_t d, const int32_t* q_starts, const int32_t* k_starts,
                                     int64_t n_seqs, int32_t causal, double scale,
                                     int32_t elem_dtype, void* workspace, int64_t workspace_bytes,
                                     void* stream) {
    using namespace mlkb;
    if (int st = checkShape(heads, kv_heads, d, scale, elem_dtype)) return st;
    mlkb_heads hq = {}, hk = {}, hv = {}, hy = {};
    if (int st = checkHeads(q, heads, d, false, "attention q", &hq)) return st;
    if (int st = checkHeads(k, kv_heads, d, false, "attention k", &hk)) return st;
    if (int st = checkHeads(v, kv_heads, d, false, "attention v", &hv)) return st;
    if (int st = checkHeads(y, heads, d, true, "attention y", &hy)) return st;
    if (hq.rows * heads > kMaxHeadTotal) return setError(MLKB_ERR_INVALID, "attention: too many rows");
    if (hk.rows != hv.rows || hq.rows != hy.rows) {
        return setError(MLKB_ERR_INVALID, "attention: k and v, and q and y, must have equal rows");
    }
    if (n_seqs < 0 || n_seqs > kMaxHeadRows || workspace_bytes < 0) {
        return setError(MLKB_ERR_INVALID, "attention: bad number of sequences");
    }
    if (n_seqs == 0 || hq.rows == 0) return okStatus();
    if (q_starts == nullptr || k_starts == nullptr ||
        ((reinterpret_cast<uintptr_t>(q_starts) | reinterpret_cast<uintptr_t>(k_starts)) & 3u) != 0) {
        return setError(MLKB_ERR_INVALID, "attention: q_starts and k_starts needed");
    }
    if (sameStart(hy, hq) || sameStart(hy, hk) || sameStart(hy, hv)) {
        return setError(MLKB_ERR_INVALID, "attention: y may not overlap the inputs");
    }
    if (int st = needDevice()) return st;
    Params p = {};
    setShape(p, heads, kv_heads, d, scale, hk.rows + n_seqs);
    p.q = hq.data;
    p.q_row = hq.row_stride;
    p.q_head = hq.head_stride;
    p.src[0] = keySource(hk, hv);
    p.y = hy.data;
    p.y_row = hy.row_stride;
    p.y_head = hy.head_stride;
    p.q_starts = q_starts;
    p.k_starts = k_starts;
    p.seqs = static_cast<int32_t>(n_seqs);
    p.q_rows = static_cast<int32_t>(hq.rows);
    p.k_rows = static_cast<int32_t>(hk.rows);
    p.causal = causal != 0;
    Maps m;
    if (int st = headsMap(&m.q, hq, heads, d, elem_dtype, p.group, p.tt, nullptr)) return st;
    if (int st = headsMap(&m.k0, hk, kv_heads, d, elem_dtype, 1, kTile, hq.data)) return st;
    if (int st = headsMap(&m.v0, hv, kv_heads, d, elem_dtype, 1, kTile, hq.data)) return st;
    m.qs = m.q;
    m.k1 = m.k0;
    m.v1 = m.v0;
    const PackedPlan r = planPacked(hq.rows, hk.rows, n_seqs, heads, kv_heads, d);
    const bool cut = r.slots > 0 && workspace != nullptr && workspace_bytes >= r.bytes(d);
    const int64_t items = r.items * (cut ? r.slots : 1);
    if (items > INT_MAX) return setError(MLKB_ERR_INVALID, "attention: too much work for one call");
    const int grid = static_cast<int>(items);
    if (!cut) return launchAttention<false, false>(m, p, elem_dtype, grid, asStream(stream));
    if (!aligned16(workspace)) {
        return setError(MLKB_ERR_INVALID, "attention: workspace must be 16-byte aligned");
    }
    p.sms = smCount();
    p.slots = static_cast<int32_t>(r.slots);
    p.part = static_cast<float*>(workspace);
    p.lse = reinterpret_cast<float2*>(p.part + r.slots * r.rows * d);
    if (int st = launchAttention<false, true>(m, p, elem_dtype, grid, asStream(stream))) return st;
    JoinParams j = {};
    j.part = p.part;
    j.lse = p.lse;
    j.c2 = p.c2;
    j.rows = r.rows;
    j.y_row = hy.row_stride;
    j.y_head = hy.head_stride;
    j.slots = p.slots;
    j.heads = p.heads;
    j.d = p.d;
    return launchJoin<false>(j, p, hy.data, elem_dtype, asStream(stream));
}

extern "C" int64_t mlkb_attention_packed_workspace(int64_t rows, int64_t key_rows, int64_t n_seqs,
                                                   int64_t heads, int64_t kv_heads, int64_t d) {
    using namespace mlkb;
    if (!shapeFits(heads, kv_heads, d) || rows < 0 || key_rows < 0 || n_seqs < 0 || rows > kMaxHeadRows ||
        key_rows > kMaxHeadRows || n_seqs > kMaxHeadRows || rows * heads > kMaxHeadTotal) {
        return -1;
    }
    return planPacked(rows, key_rows, n_seqs, heads, kv_heads, d).bytes(d);
}

extern "C" int64_t mlkb_attention_prefix_workspace(int64_t batch, int64_t steps, int64_t heads,
                                                   int64_t kv_heads, int64_t d, int64_t prefix_rows,
                                                   int64_t page_size, int64_t pages_per_request) {
    using namespace mlkb;
    if (!shapeFits(heads, kv_heads, d) || batch < 0 || steps < 1 || prefix_rows < 0 || page_size < 0 ||
        pages_per_request < 0 || batch > kMaxHeadRows || steps > kMaxHeadRows ||
        prefix_rows > kMaxHeadRows || page_size > kMaxHeadRows || pages_per_request > kMaxHeadRows ||
        page_size * pages_per_request > kMaxHeadRows || batch * steps > kMaxHeadRows ||
        batch * steps * heads > kMaxHeadTotal) {
        return -1;
    }
    const PrefixPlan r =
        planPrefix(batch, steps, heads, kv_heads, prefix_rows, page_size * pages_per_request);
    return r.fits(steps, heads, kv_heads) ? r.bytes(d) : -1;
}

extern "C" int mlkb_attention_prefix(const mlkb_heads* q, const mlkb_heads* prefix_k,
                                     const mlkb_heads* prefix_v, const mlkb_heads* k_pages,
                                     const mlkb_heads* v_pages, const mlkb_heads* y, int64_t batch,
                                     int64_t steps, int64_t heads, int64_t kv_heads, int64_t d,
                                     int64_t page_size, int64_t pages_per_request,
                                     const int32_t* pages, const int32_t* lens, double scale,
                                     int32_t elem_dtype, void* workspace, int64_t workspace_bytes,
                                     void* stream) {
    using namespace mlkb;
    if (int st = checkShape(heads, kv_heads, d, scale, elem_dtype)) return st;
    mlkb_heads hq = {}, hpk = {}, hpv = {}, hk = {}, hv = {}, hy = {};
    if (int st = checkHeads(q, heads, d, false, "attention q", &hq)) return st;
    if (int st = checkHeads(prefix_k, kv_heads, d, false, "attention prefix_k", &hpk)) return st;
    if (int st = checkHeads(prefix_v, kv_heads, d, false, "attention prefix_v", &hpv)) return st;
    if (int st = checkHeads(k_pages, kv_heads, d, false, "attention k_pages", &hk)) return st;
    if (int st = checkHeads(v_pages, kv_heads, d, false, "attention v_pages", &hv)) return st;
    if (int st = checkHeads(y, heads, d, true, "attention y", &hy)) return st;
    if (batch < 0 || steps < 1 || batch > kMaxHeadRows || steps > kMaxHeadRows ||
        hq.rows != batch * steps || hy.rows != hq.rows) {
        return setError(MLKB_ERR_INVALID, "attention: q and y must have batch * steps rows");
    }
    if (hq.rows * heads > kMaxHeadTotal) return setError(MLKB_ERR_INVALID, "attention: too many rows");
    if (hpk.rows != hpv.rows || hk.rows != hv.rows) {
        return setError(MLKB_ERR_INVALID, "attention: k and v must have equal rows");
    }
    if (page_size < 0 || pages_per_request < 0 || page_size > kMaxHeadRows ||
        pages_per_request > kMaxHeadRows) {
        return setError(MLKB_ERR_INVALID, "attention: bad page size or page count");
    }
    const int64_t cap = page_size * pages_per_request;
    if (cap > kMaxHeadRows) return setError(MLKB_ERR_INVALID, "attention: a request may hold 2^30 keys");
    if (pages != nullptr) {
        if (page_size < 16 || (page_size & (page_size - 1)) != 0 || hk.rows % page_size != 0) {
            return setError(MLKB_ERR_INVALID,
                            "attention: page size must be a power of two from 16 on, and the pages "
                            "whole");
        }
        if (batch * pages_per_request > INT_MAX) {
            return setError(MLKB_ERR_INVALID, "attention: page table too large");
        }
    } else if (cap > 0 && (pages_per_request != 1 || hk.rows != batch * page_size)) {
        return setError(MLKB_ERR_INVALID,
                        "attention: without a page table each request has one page, in order");
    }
    if (hq.rows == 0) return okStatus();
    if (cap > 0 && (lens == nullptr || ((reinterpret_cast<uintptr_t>(lens) |
                                         reinterpret_cast<uintptr_t>(pages)) & 3u) != 0)) {
        return setError(MLKB_ERR_INVALID, "attention: lens needed");
    }
    const PrefixPlan r = planPrefix(batch, steps, heads, kv_heads, hpk.rows, cap);
    if (!r.fits(steps, heads, kv_heads)) {
        return setError(MLKB_ERR_INVALID, "attention: too much work for one call");
    }
    if (workspace_bytes < r.bytes(d) || workspace == nullptr || !aligned16(workspace)) {
        return setError(MLKB_ERR_INVALID,
                        "attention: workspace (16-byte aligned) smaller than "
                        "mlkb_attention_prefix_workspace says");
    }
    if (sameStart(hy, hq) || sameStart(hy, hpk) || sameStart(hy, hpv) || sameStart(hy, hk) ||
        sameStart(hy, hv)) {
        return setError(MLKB_ERR_INVALID, "attention: y may not overlap the inputs");
    }
    if (int st = needDevice()) return st;
    Params p = {};
    setShape(p, heads, kv_heads, d, scale, (hpk.rows > cap ? hpk.rows : cap) + batch);
    p.q = hq.data;
    p.q_row = hq.row_stride;
    p.q_head = hq.head_stride;
    p.src[0] = keySource(hpk, hpv);
    p.src[1] = keySource(hk, hv);
    p.lens = lens;
    p.pages = pages;
    p.batch = static_cast<int32_t>(batch);
    p.steps = static_cast<int32_t>(steps);
    p.prefix = static_cast<int32_t>(hpk.rows);
    p.page = static_cast<int32_t>(page_size);
    p.wide = static_cast<int32_t>(pages_per_request);
    if (pages != nullptr) {
        while ((int64_t(1) << p.page_shift) < page_size) ++p.page_shift;
        p.n_pages = static_cast<int32_t>(hk.rows / page_size);
    }
    p.pre_items = static_cast<int32_t>(r.pre_items);
    p.pre_tiles = static_cast<int32_t>(r.tiles);
    p.pre_splits = static_cast<int32_t>(r.splits);
    p.pre_mt = static_cast<int32_t>(r.mt);
    p.pre_pairs = static_cast<int32_t>(r.pairs);
    p.suf_slots = static_cast<int32_t>(r.suf_slots);
    p.suf_mt = static_cast<int32_t>(r.suf_mt);
    p.tickets = static_cast<int32_t>(r.tickets);
    p.pre_spread = static_cast<int32_t>(r.pre_spread);
    p.suf_spread = static_cast<int32_t>(r.suf_spread);
    p.spread_tt = static_cast<int32_t>(r.spread_tt);
    p.pre_parts = r.pre_spread ? 4 : 1;
    p.suf_parts = r.suf_spread ? 4 : 1;
    p.sms = smCount();
    p.slots = static_cast<int32_t>(r.slots);
    p.chunk = static_cast<int32_t*>(workspace);
    p.part = static_cast<float*>(workspace) + 8;
    p.wide_store = (reinterpret_cast<uintptr_t>(p.part) & 31u) == 0;
    p.lse = reinterpret_cast<float2*>(p.part + r.slots * r.rows * d);
    Maps m;
    const int box = pages != nullptr && page_size < kTile ? static_cast<int>(page_size) : kTile;
    if (int st = headsMap(&m.q, hq, heads, d, elem_dtype, p.group, p.tt, nullptr)) return st;
    m.qs = m.q;
    if (p.pre_spread || p.suf_spread) {
        if (int st = headsMap(&m.qs, hq, heads, d, elem_dtype, p.group, p.spread_tt, nullptr)) return st;
    }
    if (int st = headsMap(&m.k0, hpk, kv_heads, d, elem_dtype, 1, kTile, hq.data)) return st;
    if (int st = headsMap(&m.v0, hpv, kv_heads, d, elem_dtype, 1, kTile, hq.data)) return st;
    if (int st = headsMap(&m.k1, hk, kv_heads, d, elem_dtype, 1, box, hq.data)) return st;
    if (int st = headsMap(&m.v1, hv, kv_heads, d, elem_dtype, 1, box, hq.data)) return st;
    const int64_t items = r.pre_items + r.tickets;
    cudaStream_t s = asStream(stream);
    if (items > 0) {
        if (int st = launchAttention<true, true>(m, p, elem_dtype, static_cast<int>(items), s)) return st;
    }
    JoinParams j = {};
    j.part = p.part;
    j.lse = p.lse;
    j.c2 = p.c2;
    j.rows = r.rows;
    j.y_row = hy.row_stride;
    j.y_head = hy.head_stride;
    j.slots = p.slots;
    j.heads = p.heads;
    j.d = p.d;
    j.prefix_slots = p.pre_splits * p.pre_parts;
    j.parts = p.suf_parts;
    j.cap = static_cast<int32_t>(cap);
    j.per_request = p.steps * p.heads;
    j.chunk = p.chunk;
    j.lens = lens;
    return launchJoin<true>(j, p, hy.data, elem_dtype, s);
}
