// Which form of the group norm's kernels a call takes, and its launches.
#pragma once
#include "group_norm_rows.h"
#include "group_norm_span.h"

namespace {

enum class Form { kRows, kTiles, kParts };

struct Plan {
  Form form;
  int ev, n;   // elements of a chunk; rows: chunks a lane
  bool part;   // rows: a group's last chunk is not whole; tiles: whole chunks over groups (group_norm_span.h)
  RowsPlan rows;
  TilePlan tile;
  int64_t parts;   // rows of partial sums by channel
  int coded;       // rows: lanes of a code block where the forward pass makes the codes; 0: a kernel of their own does
};

inline int power_of_two(int64_t n) {
  int p = 1;
  while (p < n) p *= 2;
  return p;
}

// A team for samples of so many positions of chunks: its lanes along a position and in all, and the chunks of a lane (0: too
// large).  Of teams that divide the positions differently the one with the fewest idle lanes, then the largest.  (1,024
// samples of 256 x 64 FP32 channels, each its own group, by teams of a wave, each load 64 lines: 168 us forward.)
struct RowsChoice {
  int across, team, n;
};

inline RowsChoice rows_choice(int64_t positions, int chunks, int groups, int bytes, int most_chunks) {
  const int across = std::min(64, power_of_two(chunks));
  if (positions == 1) {
    if (chunks <= 256) return {across, across, (chunks + 63) / 64};
    const int n = (chunks + 255) / 256;   // the block is the team
    return n <= 8 ? RowsChoice{256, 256, n <= 2 ? 2 : n <= 4 ? 4 : 8} : RowsChoice{};
  }
  RowsChoice best = {};
  if (chunks > 64) return best;
  double most = 0.0;
  for (int strips = 64 / across; strips >= 1; strips /= 2) {
    const int64_t n = (positions + strips - 1) / strips;
    const double used = (double)positions / (double)(strips * n);
    if (n > most_chunks || (strips > 1 && strips / 2 >= positions)) continue;
    // a wave's groups side by side: 64 bytes of a position, or all there are
    if (std::min(64 / (across * strips), groups) * bytes < std::min(64, groups * bytes)) continue;
    if (used > most + 0.01) most = used, best = {across, across * strips, (int)n};
  }
  return best;
}

// second: of the gradients of the gradients
inline Plan plan_of(int element, int64_t samples, int64_t positions, int channels, int groups, bool second) {
  Plan p = {};
  const int per = channels / groups;
  p.ev = 16 / element;
  while (per % p.ev) p.ev /= 2;
  // Groups of no whole number of 16-byte chunks: of them all the same, the last in part, where the chunks that divide a group
  // have one or two channels.  (Fours of eight: there are one fewer of these than twice the others.)
  const int whole = 16 / element;
  const bool part = p.ev < 4 && p.ev < whole && per >= whole;
  RowsChoice choice = rows_choice(positions, part ? (per + whole - 1) / whole : per / p.ev, groups, per * element, 4);
  // (the second derivative keeps too much of three and four chunks of eight: 131,072 samples of 9 x 64 bfloat16 655 us, by two 542)
  if (second && positions > 1 && choice.n > 2 && (part ? whole : p.ev) == 8) {
    const RowsChoice two = rows_choice(positions, part ? (per + whole - 1) / whole : per / p.ev, groups, per * element, 2);
    if (two.n > 0) choice = two;
  }
  if (choice.team == 256 && (part || p.ev != whole || choice.n * p.ev > 32)) choice = {};   // (kernels there are none of)
  if (choice.n > 0) {
    p.form = Form::kRows;
    p.part = part;
    if (part) p.ev = whole;
    const int chunks = (per + p.ev - 1) / p.ev, across = choice.across;
    p.n = choice.n;
    RowsPlan& r = p.rows;
    r.team = choice.team;
    while ((1 << r.shift) < r.team) ++r.shift;
    r.across = across;
    r.rows = positions == 1 ? 0 : choice.team / across;
    r.columns = positions == 1 ? across : 0;
    const int teams = 256 / r.team;
    r.groups = std::min(groups, teams);
    r.slots = teams / r.groups;
    r.blocks_y = (groups + r.groups - 1) / r.groups;
    const int64_t want = (samples + r.slots - 1) / r.slots;
    // (the gradients' blocks each leave sums of all channels)
    const int most = r.team == 256 ? 256 : r.team == 64 && p.n > 1 ? 512 : 1024;
    r.blocks_x = (int)std::max<int64_t>(1, std::min<int64_t>(want, std::max(1, most / r.blocks_y)));
    r.blocks_fwd = (int)std::max<int64_t>(1, std::min<int64_t>(want, std::max(1, 1024 / r.blocks_y)));
    p.parts = r.blocks_x;
    // every lane has a chunk, and a block of codes is an aligned power of two of lanes side by side
    const bool full = positions == 1 && !p.part && p.ev == whole && (chunks <= 64 ? chunks == across : per % kCodeBlock == 0);
    const int lanes = std::min(channels, kCodeBlock) / p.ev;
    if (full && (channels <= kCodeBlock ? power_of_two(lanes) == lanes : channels % kCodeBlock == 0) &&
        r.groups * r.team % lanes == 0)
      p.coded = lanes;
    return p;
  }
  TilePlan& t = p.tile;
  // whole groups of 128 bytes a position or more, where there are; of samples that a block takes whole down to 64 while there
  // are few blocks; and of whole chunks over groups 768.  These where a chunk that divides a group is a quarter of 16 bytes or
  // less, and from eight million elements: chunks of a group / over groups in us, forward and gradients: 1,024 samples of 256
  // x 64 FP32, each channel its group, 110 / 95, bfloat16 121 / 78; 500 of 1,000 x 30 bfloat16 in five 120 / 75; 300 of 3,000
  // x 35 in seven 230 / 172; one of 131,072 x 65 in thirteen 110 / 97; the other way 300 of 300 x 35 in seven 41 / 46, three
  // of 40,000 x 21 49 / 56; FP32 by twos, 5,000 of 100 x 30 in three 101 / 110.
  const int want = std::max(1, 128 / (per * element)), span = std::max(1, std::min(64, 768 / (per * element)));
  p.part = !second && p.ev * 4 <= whole && samples * positions * channels >= 1 << 23 &&
           (span * per + whole - 1) / whole <= kThreads;
  if (p.part) p.ev = whole;
  const int chunks = (per + p.ev - 1) / p.ev;   // (of a group alone)
  const int at_once = p.ev >= 8 || p.part ? 2 : 4, few = 10 * at_once;   // positions of a thread that are few
  t.chunks = chunks;
  t.tiles_per = p.part ? 1 : (chunks + kThreads - 1) / kThreads;
  if (t.tiles_per == 1) {
    t.groups = std::min(groups, p.part ? span : std::min(want, kThreads / chunks));
    while (positions <= few * (kThreads / chunks) && t.groups > 1 && t.groups * per * element > 64 &&
           samples * ((groups + t.groups - 1) / t.groups) < 512)
      t.groups = (t.groups + 1) / 2;
    t.lanes = p.part ? (t.groups * per + whole - 1) / whole : t.groups * chunks;
    t.tiles = (groups + t.groups - 1) / t.groups;
  } else {
    t.groups = 1;
    t.lanes = kThreads;
    t.tiles = groups * t.tiles_per;
  }
  t.rows = (int)std::min<int64_t>(kThreads / t.lanes, positions);
  t.splits = 1;
  t.per_split = positions;
  const int64_t blocks = samples * t.tiles, steps = (positions + t.rows - 1) / t.rows;
  if (t.tiles_per == 1 && (blocks >= 512 || steps <= few)) {
    p.form = Form::kTiles;
  } else {
    p.form = Form::kParts;
    const int64_t most = (steps + at_once - 1) / at_once;
    const int64_t splits = std::max<int64_t>(1, std::min<int64_t>(most, (1024 + blocks) / (blocks + 1)));
    t.per_split = (steps + splits - 1) / splits * t.rows;
    t.splits = (int)((positions + t.per_split - 1) / t.per_split);
  }
  t.powers = t.lanes <= 64 && power_of_two(t.lanes) == t.lanes && (p.part || power_of_two(chunks) == chunks);
  t.slots = (int)std::max<int64_t>(1, std::min<int64_t>(samples, 2048 / (t.tiles * t.splits)));
  p.parts = (int64_t)t.slots * t.splits;
  return p;
}

// Blocks of a wave for each sample's group.
inline dim3 unit_blocks(int64_t units) { return dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>(1 << 20, (units + 3) / 4))); }

// Few parts of a group, for tiles of few whole groups: the blocks that need their sums add them.
inline bool own_parts(const Plan& p) {
  const TilePlan& t = p.tile;
  return t.tiles_per == 1 && t.splits <= kOwnParts && (p.part || t.groups <= kOwnGroups);
}

#define GN_LAUNCH(kernel, ...) hipLaunchKernelGGL((kernel), grid, dim3(256), 0, a.stream, __VA_ARGS__)
#define GN_TEAM(N_, WIDE_, PART_, kernel, ...)                        \
  {                                                                   \
    constexpr int N = N_;                                             \
    constexpr bool WIDE = WIDE_, PART = PART_;                        \
    GN_LAUNCH(kernel, __VA_ARGS__);                                   \
  }
// Teams of a block and parts of chunks: where a chunk is 16 bytes.
#define GN_ROWS(kernel, ...)                                          \
  if (p.part) {                                                       \
    if constexpr (EV == kChunk<T>) {                                  \
      if (p.n == 1) GN_TEAM(1, false, true, kernel, __VA_ARGS__)      \
      else if (p.n == 2) GN_TEAM(2, false, true, kernel, __VA_ARGS__) \
      else if (p.rows.team < 256) GN_TEAM(4, false, true, kernel, __VA_ARGS__) \
    }                                                                 \
  } else if (p.rows.team == 256) {                                    \
    if constexpr (EV == kChunk<T>) {                                  \
      if (p.n == 2) GN_TEAM(2, true, false, kernel, __VA_ARGS__)      \
      else if (p.n == 4) GN_TEAM(4, true, false, kernel, __VA_ARGS__) \
      else if constexpr (EV == 4) GN_TEAM(8, true, false, kernel, __VA_ARGS__) \
    }                                                                 \
  } else {                                                            \
    if (p.n == 1) GN_TEAM(1, false, false, kernel, __VA_ARGS__)       \
    else if (p.n == 2) GN_TEAM(2, false, false, kernel, __VA_ARGS__)  \
    else if (p.n == 3) GN_TEAM(3, false, false, kernel, __VA_ARGS__)  \
    else GN_TEAM(4, false, false, kernel, __VA_ARGS__)                \
  }

template <typename T, int EV, bool SILU>
void launch_fwd(ictc::GroupNormCall a, const Plan& p) {
  const int per = a.channels / a.groups;
  if (p.form == Form::kRows) {
    const dim3 grid(p.rows.blocks_fwd, p.rows.blocks_y);
    if constexpr (EV == kChunk<T>) {
      if (a.codes_out && p.coded) {
        GN_ROWS((gn_rows_fwd_kernel<T, EV, N, WIDE, PART, SILU, !PART>), a, p.rows, per, p.coded)
        return;
      }
    }
    GN_ROWS((gn_rows_fwd_kernel<T, EV, N, WIDE, PART, SILU, false>), a, p.rows, per, 0)
    return;
  }
  const dim3 grid((unsigned)p.tile.slots * p.tile.splits * p.tile.tiles);
  if (p.form == Form::kTiles && p.part) {
    if constexpr (EV == kChunk<T>) GN_LAUNCH((gn_span_fwd_kernel<T, EV, SILU>), a, p.tile, per, (double*)nullptr);
    return;
  }
  if (p.form == Form::kTiles) {
    hipLaunchKernelGGL((gn_tile_fwd_kernel<T, EV, SILU>), grid, dim3(kThreads), 0, a.stream, a, p.tile, per);
    return;
  }
  const int64_t units = a.samples * a.groups;
  const int parts = p.tile.splits * p.tile.tiles_per;
  double* part = (double*)a.ws;
  if (p.part) {
    if constexpr (EV == kChunk<T>) GN_LAUNCH((gn_span_fwd_kernel<T, EV, SILU>), a, p.tile, per, part);
  } else {
    GN_LAUNCH((gn_part_stats_kernel<T, EV>), a, p.tile, per, part);
  }
  const bool own = own_parts(p);
  const double* parts_of = own ? part : nullptr;
  if (!own) {   // means that nobody wants, or in one value each, go behind the parts
    float* kept = (float*)(part + units * parts * 2);
    if (!a.rest) a.rest = kept;
    if (!a.mean) a.mean = kept + units, a.rstd = kept + 2 * units;
    hipLaunchKernelGGL(gn_part_moments_kernel<T>, unit_blocks(units), dim3(256), 0, a.stream, a, part, units, parts, per);
  }
  if (p.part) {
    if constexpr (EV == kChunk<T>) GN_LAUNCH((gn_span_part_fwd_kernel<T, EV, SILU>), a, p.tile, per, parts_of);
  } else {
    GN_LAUNCH((gn_part_fwd_kernel<T, EV, SILU>), a, p.tile, per, parts_of);
  }
}

template <typename T>
void launch_channels(const ictc::GroupNormCall& a, const Plan& p, const float* part_w, const float* part_b) {
  if (a.out_w || a.out_b)
    hipLaunchKernelGGL(gn_channels_kernel<T>, dim3((unsigned)((a.channels + 15) / 16), 2), dim3(256), 0, a.stream, part_w,
                       (T*)a.out_w, part_b, (T*)a.out_b, p.parts, a.channels);
}

// Where the second and first derivatives' workspace begins: sums by channel; then, of parts, K sums of each part and of
// each sample's group.
struct Workspace {
  float *w, *b, *part, *sums;
  Workspace(const ictc::GroupNormCall& a, const Plan& p, int K) {
    const int64_t size = p.parts * a.channels;
    w = (float*)a.ws;
    b = w + size;
    part = b + size;
    sums = part + a.samples * a.groups * (p.tile.splits * p.tile.tiles_per) * K;
  }
};

// The parts' sums of every sample's group, or the parts themselves for blocks that add them.
template <int K>
const float* launch_sums(const ictc::GroupNormCall& a, const Plan& p, const Workspace& ws, bool own) {
  if (own) return ws.part;
  const int64_t units = a.samples * a.groups;
  hipLaunchKernelGGL(gn_part_sums_kernel<K>, unit_blocks(units), dim3(256), 0, a.stream, ws.part, units,
                     p.tile.splits * p.tile.tiles_per, ws.sums);
  return ws.sums;
}

template <typename T, int EV, bool SILU, bool EIGHT>
void launch_bwd(const ictc::GroupNormCall& a, const Plan& p) {
  const int per = a.channels / a.groups;
  const Workspace ws(a, p, 2);
  float *pw = a.out_w ? ws.w : nullptr, *pb = a.out_b ? ws.b : nullptr;
  if (p.form == Form::kRows) {
    const dim3 grid(p.rows.blocks_x, p.rows.blocks_y);
    GN_ROWS((gn_rows_bwd_kernel<T, EV, N, WIDE, PART, SILU, EIGHT>), a, p.rows, per, pw, pb)
  } else {
    const bool parts = p.form == Form::kParts, own = own_parts(p);
    const dim3 grid((unsigned)p.tile.slots * p.tile.splits * p.tile.tiles);
    float* none = nullptr;
    if (p.part) {
      if constexpr (EV == kChunk<T>) {
        if (parts)
          GN_LAUNCH((gn_span_bwd_kernel<T, EV, SILU, EIGHT, false>), a, p.tile, per, ws.part, pw, pb);
        else
          GN_LAUNCH((gn_span_bwd_kernel<T, EV, SILU, EIGHT, true>), a, p.tile, per, none, pw, pb);
      }
    } else if (parts) {
      GN_LAUNCH((gn_tile_bwd_kernel<T, EV, SILU, EIGHT, false>), a, p.tile, per, ws.part, pw, pb);
    } else {
      GN_LAUNCH((gn_tile_bwd_kernel<T, EV, SILU, EIGHT, true>), a, p.tile, per, none, pw, pb);
    }
    if (parts && a.out) {
      const float* sums = launch_sums<2>(a, p, ws, own);
      if (p.part) {
        if constexpr (EV == kChunk<T>) GN_LAUNCH((gn_span_part_bwd_kernel<T, EV, SILU, EIGHT>), a, p.tile, per, sums, own);
      } else {
        GN_LAUNCH((gn_part_bwd_kernel<T, EV, SILU, EIGHT>), a, p.tile, per, sums, own);
      }
    }
  }
  launch_channels<T>(a, p, pw, pb);
}

template <typename T, int EV, bool SILU, bool EIGHT>
void launch_bwd2(const ictc::GroupNormCall& a, const Plan& p) {
  const int per = a.channels / a.groups;
  const Workspace ws(a, p, kSums);
  float *pw = a.out_w ? ws.w : nullptr, *pb = a.out_b ? ws.b : nullptr;
  if (p.form == Form::kRows) {
    const dim3 grid(p.rows.blocks_x, p.rows.blocks_y);
    GN_ROWS((gn_rows_bwd2_kernel<T, EV, N, WIDE, PART, SILU, EIGHT>), a, p.rows, per, pw, pb)
  } else {
    const bool own = own_parts(p);
    const dim3 grid((unsigned)p.tile.slots * p.tile.splits * p.tile.tiles);
    float* none = nullptr;
    const float* sums = nullptr;
    if (p.form == Form::kParts) {
      hipLaunchKernelGGL((gn_tile_bwd2_kernel<T, EV, SILU, EIGHT, Phase::kSums>), grid, dim3(kThreads), 0, a.stream, a,
                         p.tile, per, ws.part, sums, false, none, none);
      sums = launch_sums<kSums>(a, p, ws, own);
      hipLaunchKernelGGL((gn_tile_bwd2_kernel<T, EV, SILU, EIGHT, Phase::kResults>), grid, dim3(kThreads), 0, a.stream, a,
                         p.tile, per, none, sums, own, pw, pb);
    } else {
      hipLaunchKernelGGL((gn_tile_bwd2_kernel<T, EV, SILU, EIGHT, Phase::kAll>), grid, dim3(kThreads), 0, a.stream, a,
                         p.tile, per, none, sums, false, pw, pb);
    }
  }
  launch_channels<T>(a, p, pw, pb);
}

}  // namespace

namespace ictc {

#define GN_CHUNKS(launch, second)                              \
  const Plan p = plan_of((int)sizeof(T), a.samples, a.positions, a.channels, a.groups, second); \
  if constexpr (sizeof(T) == 2) {                              \
    if (p.ev == 8) { constexpr int EV = 8; return launch; }    \
  }                                                            \
  if (p.ev == 4) { constexpr int EV = 4; return launch; }      \
  if (p.ev == 2) { constexpr int EV = 2; return launch; }      \
  constexpr int EV = 1;                                        \
  return launch;

template <typename T>
void group_norm_fwd(const GroupNormCall& a) {
  GN_CHUNKS((a.silu ? launch_fwd<T, EV, true>(a, p) : launch_fwd<T, EV, false>(a, p)), false)
}

#define GN_KIND(f) \
  (a.codes ? a.silu ? f<T, EV, true, true>(a, p) : f<T, EV, false, true>(a, p) \
           : a.silu ? f<T, EV, true, false>(a, p) : f<T, EV, false, false>(a, p))

template <typename T>
void group_norm_bwd(const GroupNormCall& a) {
  GN_CHUNKS(GN_KIND(launch_bwd), false)
}
template <typename T>
void group_norm_bwd2(const GroupNormCall& a) {
  GN_CHUNKS(GN_KIND(launch_bwd2), true)
}

}  // namespace ictc
