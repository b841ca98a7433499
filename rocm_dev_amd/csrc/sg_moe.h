// A mixture-of-experts layer for a few tokens: what its translation units share (include/sgemm.h says what it computes).
//
// Launches: the router's logits (moe_route, moe_layer); the choice of experts, for more than kMoeFused tokens one of its own; gate and
// up projections of every reached expert, whose workgroups each make the plan - who goes where - and, for few tokens, the choice for
// themselves; down projections, added up over a token's experts.  Each hands over through the caller's workspace and the
// end of a launch: nothing waits on the device, so calls that overlap cannot wait for each other.
#pragma once

#include "sg_device.h"
#include "sg_host.h"

namespace sg {

constexpr int kMoeTokens = 64;      // a token is a bit of 64 in the plan
constexpr int kMoeExperts = 512;
constexpr int kMoeTopK = 16;

constexpr int kMoeSide = 1 << 20;   // hidden, inner: rows of a tile, of all activations and of W1's count within 32 bits
constexpr int kMoeFused = 8;        // tokens whose experts every workgroup chooses for itself

// The plan: dwords [number of parts][part: expert | entries << 16][its first entry][entry: token << 16 | row of h = token * top_k + the
// choice that names the expert first][its weight].  An entry is a token and an expert that it names; a part is up to COLS entries of one
// expert, the columns of one product: an expert with more is read once for each part.  Gate and up keep it in LDS up to the weights.
struct MoePlanLayout {
    int parts_at, first_at, rows_at, weights_at, dwords, most;
};
__host__ __device__ inline MoePlanLayout moe_plan_layout(int m, int experts, int top_k, int cols) {
    const int pairs = m * top_k;
    MoePlanLayout l;
    l.most = (experts < pairs ? experts : pairs) + pairs / cols;      // parts
    l.parts_at = 4;
    l.first_at = l.parts_at + l.most;
    l.rows_at = l.first_at + l.most;
    l.weights_at = l.rows_at + pairs;
    l.weights_at = (l.weights_at + 3) / 4 * 4;
    l.dwords = (l.weights_at + pairs + 3) / 4 * 4;
    return l;
}

// A tile's workgroups in the down projections: at most kMoeSplits of them, and kMoeSplitRows rows of partial sums in all.
constexpr int kMoeSplits = 8, kMoeSplitRows = 16384;
inline int moe_most_splits(int hidden) { return kMoeSplits * hidden <= kMoeSplitRows ? kMoeSplits : hidden < kMoeSplitRows ? kMoeSplitRows / hidden : 1; }

struct MoeLayout {
    size_t plan_at, h_at, sums_at, bytes;     // logits first
};
inline bool moe_takes(int m, int hidden, int inner, int experts, int top_k) {
    return m > 0 && m <= kMoeTokens && hidden > 0 && hidden % 16 == 0 && hidden <= kMoeSide && inner > 0 && inner % 16 == 0 &&
           inner <= kMoeSide && experts > 0 && experts <= kMoeExperts && top_k > 0 && top_k <= kMoeTopK && top_k <= experts;
}
inline MoeLayout moe_layout(int m, int hidden, int inner, int experts, int top_k) {
    MoeLayout l;
    l.plan_at = ((size_t)m * experts * 4 + 255) / 256 * 256;
    l.h_at = l.plan_at + ((size_t)moe_plan_layout(m, experts, top_k, 4).dwords * 4 + 255) / 256 * 256;
    l.sums_at = l.h_at + ((size_t)m * top_k * inner * 2 + 255) / 256 * 256;
    const int splits = moe_most_splits(hidden);
    l.bytes = l.sums_at + (splits > 1 ? (size_t)splits * m * hidden * 4 : 0);
    return l;
}

struct MoeArgs {
    const uint8_t* X;                // [m][hidden] bf16
    const uint8_t* R;                // [experts][hidden] bf16
    const uint8_t* W1;               // [experts][2 * inner][hidden] E4M3
    const float* S1;                 // [experts][2 * inner], or NULL
    const uint8_t* W2;               // [experts][hidden][inner] E4M3
    const float* S2;                 // [experts][hidden], or NULL
    uint16_t* D;                     // [m][hidden] bf16
    int32_t* ids;                    // [m][top_k]
    float* weights;                  // [m][top_k]
    float* logits;                   // [m][experts]
    int32_t* plan;
    uint8_t* H;                      // [m * top_k][inner] bf16
    int m, hidden, inner, experts, top_k, renormalize;
    float* sums;                     // [splits][m][hidden]
    int splits;                      // down projections: workgroups that share a tile's steps
    int share_log;                   // gate and up: 1 << this of four waves share an item's columns
    int stride_parts, stride_tiles;  // ... and from a wave's item to its next one, as parts and tiles
    uint32_t turn;                   // ... 2^32 / steps of a wave: the next tile begins a step later
    uint32_t inv_tiles, inv_steps, inv_sharers;      // div_reciprocal: gate and up's tiles, the down projections' steps and sharers
};

}  // namespace sg
