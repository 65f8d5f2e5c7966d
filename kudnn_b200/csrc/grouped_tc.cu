// Host side of the tensor-core kernel for grouped and block-scaled products (grouped_tc.cuh).
#include "grouped_tc.cuh"

#include <algorithm>
#include <atomic>
#include <cmath>

namespace kb {

using namespace grp;

namespace {

// Row pitch and group distance as the tensor maps want them: a single row or group has none of its own.
long long pitch_of(long long extent, long long stride, long long inner, int es)
{
    return extent > 1 ? stride : (inner * es + 15) / 16 * 16 / es;
}

bool pitch_fits(long long pitch, long long inner, int es)
{
    return pitch >= inner && pitch * es % 16 == 0 && pitch * es < (1ll << 40);
}

template <int kMode, int kTN, bool kRows = false>
cudaError_t launch_shape(const GroupedParams &g, TcParams &p, long long item_bound, int sm_count, const CUtensorMap &tb, cudaStream_t stream)
{
    using S = Shape<kMode, kTN, kRows>;
    constexpr int es = S::kScaled ? 1 : 2;
    auto kernel = grouped_tc_kernel<kMode, kTN, kRows>;
    static std::atomic<unsigned long long> prepared{0};  // devices, a bit each
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) {
        return e;
    }
    if (dev >= 64 || (prepared.load() >> dev & 1ull) == 0) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
        if (e != cudaSuccess) {
            return e;
        }
        if (dev < 64) {
            prepared.fetch_or(1ull << dev);
        }
    }
    CUtensorMap ta;
    e = tc_encode_groups(&ta, g.a, g.ab_dtype, 1, g.rows, g.k, pitch_of(1, 0, g.k, es), pitch_of(g.rows, g.a_sm, g.k, es), S::kBoxRows);
    if (e != cudaSuccess) {
        return e;
    }
    // Where the items leave SMs idle, two or four CTAs of a cluster cut K, if that fills the SMs better: 86 items of one row, 32 blocks of K,
    // all of it in L2: 11.8 us uncut, 12.2 at two (172 CTAs on 148 SMs), 10.4 at four (13.0 from HBM).  Clusters of 8 and odd ones find no room
    // next to one another.
    // The CTAs that then share an SM share its memory for their rings.
    auto filled = [&](long long ctas) { return static_cast<double>(ctas) / sm_count / ((ctas + sm_count - 1) / sm_count); };
    p.splits = 1;
    if (S::kSplits) {
        for (int s = 2; s <= 4; s *= 2) {
            if (item_bound * s <= static_cast<long long>(sm_count) * S::kCtas && p.num_kb >= 4 * s &&
                (s - 1) * ((p.num_kb + s - 1) / s) < p.num_kb && filled(item_bound * s) > 1.05 * filled(item_bound * p.splits)) {
                p.splits = s;
            }
        }
    }
    const int sharing = static_cast<int>(std::clamp<long long>((item_bound * p.splits + sm_count - 1) / sm_count, 1, S::kCtas));
    const int fixed = S::kFixedBytes + (g.groups + 1) * 8;
    const int budget = sharing == 1 ? kSmemLimit : kSmemPerSm / sharing - 1024;  // 1 KiB per CTA is the system's
    p.stages = std::min(kMaxStages, std::max(S::kLeastStages, (budget - fixed) / S::kStageBytes));
    const long long slots = static_cast<long long>(sm_count) * sharing;
    p.kb_per_split = (p.num_kb + p.splits - 1) / p.splits;
    const size_t smem = static_cast<size_t>(fixed + p.stages * S::kStageBytes);
    long long ctas = p.splits > 1 ? item_bound * p.splits : std::min<long long>(std::max<long long>(item_bound, 1), slots);
    if (S::kPair) {
        // as many pairs as the GPU's partitions hold
        const int pairs = tc_pair_clusters(KUDNN_B200_F16, kSmemLimit);
        ctas = 2 * std::min<long long>(std::max<long long>(item_bound, 1), pairs > 0 ? pairs : sm_count / 2);
    }
    return launch_chained(kernel, dim3(static_cast<unsigned>(ctas)), dim3(S::kThreads), smem, stream, static_cast<unsigned>(S::kPair ? 2 : p.splits), ta, tb, p);
}

// The width of the tiles: the one with the least time by what a block of K was measured to take an SM (cycles, at 1.9 GHz; a pair of SMs
// for tiles of 256), times the rounds that the items make.  Short tiles share an SM, so that their rounds need not be whole ones.
// 333 x 11008 x 4096 in 8 bits: 31.9 / 29.4 / 35.4 us on tiles of 64 / 128 / 256 rows, 512 x 2048 x 4096 14.1 / 16.9 / 19.7,
// 1024 x 4096 x 4096 32.0 / 29.8 / 21.0.
struct TileCost {
    int rows;
    double alone, shared, finish;  // one CTA on an SM, as many as fit; results of a tile
};
constexpr TileCost kScaledCost[4] = {{32, 450, 330, 1000}, {64, 564, 470, 1500}, {128, 757, 757, 2500}, {256, 850, 850, 2500}};
constexpr TileCost kPlainCost[4] = {{32, 450, 330, 1000}, {64, 500, 400, 1500}, {128, 560, 560, 1000}, {256, 540, 540, 1000}};

int choose_tile(const GroupedParams &g, const TcParams &p, bool scaled, bool tall_on_m, int sm_count)
{
    const double busy = std::min(g.groups, g.rows);
    int best = 256;
    double least = 0.0;
    for (int i = 0; i < 4; ++i) {
        const TileCost &c = scaled ? kScaledCost[i] : kPlainCost[i];
        const int wide = c.rows == 256 ? 256 : 128;
        // groups are uneven: half of a group's last tile is empty, on average
        const double tiles = g.offsets == nullptr ? (g.rows + c.rows - 1) / c.rows : std::max(busy, g.rows / static_cast<double>(c.rows) + 0.5 * busy);
        const double items = tiles * ((g.n + wide - 1) / wide), fill = std::min(1.0, g.rows / (tiles * c.rows));
        double cycles;
        if (c.rows <= 64) {
            cycles = std::max(c.alone * p.num_kb, c.shared * p.num_kb * items / sm_count) + c.finish;
        } else {
            // weights on the M side: a block of K takes less where the tile has fewer rows
            const double each = c.rows == 128 || tall_on_m ? c.alone : (scaled ? 1170.0 : c.alone) * std::max(0.55, fill);
            const double rounds = std::ceil(items / (c.rows == 256 ? sm_count / 2 : sm_count));
            cycles = rounds * (each * p.num_kb + c.finish);
        }
        if (i == 0 || cycles < least) {
            least = cycles;
            best = c.rows;
        }
    }
    return best;
}

template <int kMode>
cudaError_t launch_kind(const GroupedParams &g, TcParams &p, int sm_count, const CUtensorMap &tb, GroupedTile *tile, cudaStream_t stream)
{
    constexpr bool kScaled = kMode == kWithScales;
    // Tall tiles of scaled products: rows on the M side, unless the groups' last tiles, which that pads to 256 rows, would take more than the
    // faster sums save (850 against 1170 cycles per block of K).
    if (tile->rows == 0) {
        const bool tall_on_m = kScaled && (g.offsets == nullptr || g.rows >= 192ll * g.groups);
        tile->rows = choose_tile(g, p, kScaled, tall_on_m, sm_count);
        tile->on_m = tall_on_m && tile->rows == 256 ? 1 : 0;
    }
    const int tn = tile->rows;
    // offsets may leave out rows and make up to min(groups, rows) short tiles
    const long long tiles = g.offsets == nullptr ? (g.rows + tn - 1) / tn : std::min(g.groups, g.rows) + g.rows / tn;
    p.tiles_n = tn == 256 ? (g.n + 2 * kTileN - 1) / (2 * kTileN) : (g.n + kTileN - 1) / kTileN;
    p.idesc = make_idesc(g.ab_dtype == KUDNN_B200_BF16 ? KUDNN_B200_BF16 : KUDNN_B200_F16, 0, tn == 256 ? 2 * kTileN : kTileN);  // e4m3 and fp16: code 0
    const long long bound = tiles * p.tiles_n;
    if constexpr (kScaled) {
        if (tile->on_m != 0) {
            p.idesc |= 256u >> 3 << 17;
            if (p.vec != 0 && g.c_sm * dtype_size(g.c_dtype) % 32 == 0 && reinterpret_cast<uintptr_t>(g.c) % 32 == 0) {
                p.vec = 2;
            }
            return launch_shape<kWithScales, 256, true>(g, p, bound, sm_count, tb, stream);
        }
    }
    switch (tn) {
        case 32: return launch_shape<kMode, 32>(g, p, bound, sm_count, tb, stream);
        case 64: return launch_shape<kMode, 64>(g, p, bound, sm_count, tb, stream);
        case 128: return launch_shape<kMode, 128>(g, p, bound, sm_count, tb, stream);
        default: return launch_shape<kMode, 256>(g, p, bound, sm_count, tb, stream);
    }
}

}  // namespace

bool grouped_tc_takes(const GroupedParams &p)
{
    const int es = p.ab_dtype == KUDNN_B200_E4M3 ? 1 : 2;
    const long long ld_a = pitch_of(p.rows, p.a_sm, p.k, es), ld_b = pitch_of(p.n, p.b_sn, p.k, es);
    return tc_available() && (p.a_sk == 1 || p.k == 1) && (p.b_sk == 1 || p.k == 1) &&
           ((reinterpret_cast<uintptr_t>(p.a) | reinterpret_cast<uintptr_t>(p.b)) & 15u) == 0 && pitch_fits(ld_a, p.k, es) &&
           pitch_fits(ld_b, p.k, es) && (p.groups == 1 || pitch_fits(p.b_sg, p.k, es));
}

cudaError_t launch_grouped_tc(const GroupedParams &g, int sm_count, DeviceStatus *status, long long wait_limit_cycles, int skip_kblock,
                              GroupedTile *tile, cudaStream_t stream)
{
    const bool scaled = g.ab_dtype == KUDNN_B200_E4M3;
    const int es = scaled ? 1 : 2, c_size = dtype_size(g.c_dtype);
    const long long ld_b = pitch_of(g.n, g.b_sn, g.k, es);
    CUtensorMap tb;
    const cudaError_t e = tc_encode_groups(&tb, g.b, g.ab_dtype, g.groups, g.n, g.k, g.groups > 1 ? g.b_sg : pitch_of(1, 0, g.k, es), ld_b, kTileN);
    if (e != cudaSuccess) {
        return e;
    }
    TcParams p;
    p.g = g;
    p.kb_elems = 128 / es;
    p.num_kb = (g.k + p.kb_elems - 1) / p.kb_elems;
    p.band = 16;
    const bool short_act = g.act == KUDNN_B200_ACT_NONE || g.act == KUDNN_B200_ACT_RELU || g.act == KUDNN_B200_ACT_SWISH ||
                           (g.act == KUDNN_B200_ACT_GELU_TANH && g.c_dtype != KUDNN_B200_F32);
    p.vec = short_act && (g.c_sn == 1 || g.n == 1) && (g.rows == 1 || g.c_sm % 4 == 0) && reinterpret_cast<uintptr_t>(g.c) % (4 * c_size) == 0 ? 1 : 0;
    p.load_kb = skip_kblock >= 0 ? std::min(skip_kblock, p.num_kb) : p.num_kb;
    p.status = status;
    p.wait_limit = wait_limit_cycles > 0 ? wait_limit_cycles : kDefaultWaitLimitCycles;
    p.drain = 4;
    p.splits = 1;
    const cudaError_t launched = scaled ? launch_kind<kWithScales>(g, p, sm_count, tb, tile, stream)
                                 : g.c_dtype == KUDNN_B200_F32 && p.num_kb > p.drain ? launch_kind<kDrained>(g, p, sm_count, tb, tile, stream)
                                                                                     : launch_kind<kPlain>(g, p, sm_count, tb, tile, stream);
    tile->splits = p.splits;
    return launched;
}

}  // namespace kb
