// Tensor-core path of attention: scores and outputs as 3xFP16 products on tcgen05, the probabilities between them in registers and TMEM.
//
// One kernel, four kinds.  A CTA holds 128 rows and streams tiles of 128 columns of the other side past them:
//
//   kind  rows     scores                      weights                          product           results
//   fwd   queries  S = Q K^T                   P = 2^(z - running max)          P V               o, row maxima and sums
//   dq    queries  S = Q K^T, Y = dO' V^T      E (Y - D') (cap's derivative)    dS K              dq
//   dk    keys     S = K Q^T, Y = V dO'^T      the same, transposed             dS^T Q            dk
//   dv    keys     S = K Q^T                   E = 2^(z - max of the column)    E^T dO'           dv
//
// with dO' and D' the output gradient and its product with the output, divided by the row's sum: P is E over that sum.  Gradients form the scores
// again, twice as often as one kernel of all three would (8 products of the tile's size instead of 5), but nothing is added across CTAs: no
// atomics, the same bits every run.
//
// Operands.  A packing kernel writes every tile of 128 tokens x one head as fp16 halves hi and lo of x times a power of two that the tile's largest finite
// element chooses (queries also times the mantissa of what scores are scaled by, so that a score is a product times a power of two), in the 128-byte swizzle of the shared-memory descriptors, so a tile part is one bulk copy and no tensor map is needed.  The same image is read
// with the head along K (scores) and with the tokens along K (products), by descriptors of the other major.  Products are hi*lo + lo*hi + hi*hi, the small ones first.
// Weights are split in registers and go back to TMEM as the A operand, over the scores they came from; each is scaled by a power of two so that their largest
// (bounded for gradients by the norms of dO' rows and V) is just below 2^15.  Scales of a tile are undone where its product is added up: the tensor core
// truncates as it accumulates, so every tile's product is added to fp32 registers (round to nearest) by the warps that make the weights.
//
// Tokens of different sizes.  What a row does not see (padding, other documents, tokens behind it) may be of any size, and must not cost it bits.  Where a tile's tokens are further
// apart than a scale serves (kOrders), each is packed with a scale of its own.  The warps undo those in the scores, put those of the product's operand into the weights, and scale a row's
// weights by the largest that it sees, found first: a second pass over such tiles, in code of its own beside the loop that all others take.  With every tile of the values like that
// 2 x 4096 tokens, 16 over 4 heads of 128, causal, take 475 us forward instead of 393 and 1607 back instead of 1534; 8 heads of 64, every key seen, 710 instead of 426 and 2129 of 1720.
//
// Bound by the tensor rate: 3 products of 16-bit halves for each product.  The tile of the next scores is issued ahead of the product of the present weights,
// so the tensor cores work while 8 warps (two a TMEM lane quarter) make weights.  4 x 4096 tokens, 8 heads of 128, every key seen: forward 750 us (366 TFLOP/s of the formula,
// three times that in halves), gradients 3096; heads of 64: 419 and 1690.  There the power limit holds the clock at 1.45 to 1.6 GHz of 1.97, which differs by a tenth from box to box.
// A CTA's start and end take 8 us, so rows that see few tiles are bound by those.
//
// A token that holds a value which is not finite is packed as if that value were zero and marked; weights that see it become NaN.  So it reaches what depends on it and nothing
// else, while a zero weight times it would reach every row of the tile.
#include "attention.h"
#include <cuda_fp16.h>
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>
#include "tcgen05.h"

namespace tf {
namespace {

enum { kFwd, kDq, kDk, kDv };
constexpr int kTile = 128;
// Warps: 0 copies, 1 issues MMAs and owns TMEM, 2 and 3 idle, 4-7 and 8-11 make weights.  With one score product the two groups take every other tile, each thread a whole
// row, so that one computes while the other waits; with two, whose second scores have one buffer, both take half the columns of every tile.
constexpr int kThreads = 384;
// Registers a thread: 168 at the launch (64,512 of the block); the first four warps give 96 of theirs, the others take 48 each, the same sum.
constexpr int kFewRegisters = 72, kManyRegisters = 216;
constexpr int kWeightExp = 14;                   // weights are scaled to below 2^15
constexpr float kWeightScale = 1 << kWeightExp;
constexpr int kFar = 1 << 26;                    // beyond every position

// Of one tile of one head
struct __align__(16) TileInfo {
  float inv, top;                                // 1 / scale; negative where every token has one of its own; largest finite magnitude
  float norm, delta;                             // dO': largest row norm and |D'|
  uint32_t bad[4];                               // tokens with values that are not finite
  float low, peak, unused[2];                    // dO': smallest row norm that is not zero; largest magnitude of the rows' maxima
};
struct Packed { const char* image; const TileInfo* info; const float* scale; };           // 1 / scale of every token; 0 for tokens of zeros among others with scales of their own
struct TcArgs {
  AttentionArgs a;
  Packed q, k, v, d;
  const float *row_max, *row_delta, *row_norm;   // of every sequence, head and query, tiles padded with zeros
  const float4* documents;                       // of every sequence and key tile: smallest, largest, whether there is padding
  float *dk_part, *dv_part;                      // where the query heads of a key-value head are dealt to several CTAs: their sums, one after another
  int q_tiles, k_tiles, D16, shares;
  float by, dk_factor;                           // power of two of scores (0: all are 0); what dk's sums are multiplied by, their queries being so already
  int* err;
};

// ---- packing ----------------------------------------------------------------------------------------------------------------
struct PackJob {
  const float* x;
  char* image;
  TileInfo* info;
  float* scale;
  int heads, length, tiles;
  int gradient;                                  // dout: times 1 / sum, with its row's D' and norm
  float times;                                   // 1; queries: what scores are scaled by, but for its power of two, so that scores are products times a power of two and not rounded again
};
struct PackArgs {
  AttentionArgs a;
  PackJob job[4];
  int first[5];                                  // blocks of the jobs
  int jobs;
  float *row_max, *row_delta, *row_norm;
  float4* documents;
  int document_job;
};

__device__ __forceinline__ uint32_t halves(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// 2^e as a float
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }
__device__ __forceinline__ int exponent_of(float positive) { return (int)((__float_as_uint(positive) >> 23) & 255u) - 127; }

// Joins four numbers over kAcross lanes; lane l is left with that of number l / (kAcross / 4)
template <int kAcross, class F> __device__ __forceinline__ float joined(const float* v, F&& join) {
  const bool upper = threadIdx.x & (kAcross / 2), odd = threadIdx.x & (kAcross / 4);
  float w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) w[i] = join(upper ? v[i + 2] : v[i], __shfl_xor_sync(0xffffffffu, upper ? v[i] : v[i + 2], kAcross / 2));
  float x = join(odd ? w[1] : w[0], __shfl_xor_sync(0xffffffffu, odd ? w[0] : w[1], kAcross / 4));
#pragma unroll
  for (int o = kAcross / 8; o > 0; o >>= 1) x = join(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}
// The largest of each, of numbers that are not negative: where a row has all lanes, a reduction instruction each is less than the exchange
template <int kAcross> __device__ __forceinline__ float largest(const float* v) {
  if (kAcross < 32) return joined<kAcross>(v, [](float x, float y) { return fmaxf(x, y); });
  uint32_t x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = __reduce_max_sync(0xffffffffu, __float_as_uint(v[i]));
  const int mine = threadIdx.x / (kAcross / 4) % 4;
  return __uint_as_float(mine & 2 ? (mine & 1 ? x[3] : x[2]) : (mine & 1 ? x[1] : x[0]));
}
// Binary orders between the largest magnitudes of two tokens of a tile up to which they share a scale.  A value is held to 2^-39 of the tile's largest, so 8 orders leave 2^-31 of the
// token's own, and the scale of the gradients' weights, which goes by the largest value, 8 bits of 25 to spare.  Output gradients over their row's sum, which differ by as much as the
// sums do, up to the number of keys: 14 orders leave 2^-25.
constexpr int kOrders = 8, kOrdersOfGradient = 14;
// Of the weights of dk below the bound that scales them: a weight is held to 2^-39 of that, and what scales it is about 2^4 above the largest of them.
constexpr int kOrdersOfBound = 7, kOrdersOfSeen = 10;
// Largest maximum, in units of log 2, of rows whose weights are taken as they come in the gradients.  Above it a forward call of other kernels may have rounded scores by so much that a
// weight is 2 and more, not 1: the way of tokens that are apart takes at most 1.
constexpr float kPeak = 65536.f;
// max * scale in [2^below, 2^(below + 1)): 14, or 13 where a factor of less than 2 follows; subnormal maxima, and those from 2^126, as far as the scale and its reciprocal are normal numbers
__device__ __forceinline__ int scale_exponent(float most, int below) { return most > 0.f ? min(126, max(-126, below - exponent_of(most))) : 0; }

// A block packs one tile of one head, 16 G threads a row, 4 columns each.  HBM-bound: 4 bytes an element read and written, for dout 8 read.  Half the rows' loads in flight a
// thread where there are few tiles (2 x 777 tokens, 6 over 2 heads of 72: 27.0 us forward and 54.5 back with twice the threads, 29.0 and 56.4 without; 8 x 1024 tokens, 16
// heads of 64: 138.5 and 367, 125.7 and 359).
constexpr int pack_threads(int G, bool few) { return (few ? 512 : 256) * G; }
template <int G, bool WIDE, bool FEW>
__global__ void __launch_bounds__(pack_threads(G, FEW), 1024 / pack_threads(G, FEW)) attention_pack_kernel(const __grid_constant__ PackArgs p) {
  constexpr int kPackWarps = pack_threads(G, FEW) / 32;
  constexpr int kAcross = 16 * G, kRowsAtOnce = 32 / kAcross, kRowsOfWarp = kTile / kPackWarps, kSteps = kRowsOfWarp / kRowsAtOnce;
  constexpr int kShare = kAcross / 4, kGroups = kSteps / 4;            // of four steps' rows a lane looks after one, with kShare - 1 others
  __shared__ float red[kPackWarps], red_least[kPackWarps], red_norm[kPackWarps], red_delta[kPackWarps], red_low[kPackWarps], red_peak[kPackWarps], token_scale[kTile];
  __shared__ uint32_t bad_words[4];
  grid_dep_sync();
  int j = 0;
  while (j + 1 < p.jobs && (int)blockIdx.x >= p.first[j + 1]) ++j;
  const PackJob& job = p.job[j];
  const int index = (int)blockIdx.x - p.first[j], tile = index % job.tiles, bh = index / job.tiles, h = bh % job.heads, b = bh / job.heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = (lane % kAcross) * 4, sub = lane / kAcross;
  const int D = p.a.D;
  if (threadIdx.x < 4) bad_words[threadIdx.x] = 0u;
  float v[kSteps][4];
  float most_norm = 0.f, most_delta = 0.f, low = INFINITY, peak = 0.f;
  const auto load4 = [&](const float* from, int t, float* w) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = 0.f;
    if (t < job.length && col < D) {
      from += (((int64_t)b * job.length + t) * job.heads + h) * D + col;
      if (WIDE) { const float4 x = __ldg(reinterpret_cast<const float4*>(from)); w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w; }
      else
#pragma unroll
        for (int i = 0; i < 4; ++i) if (col + i < D) w[i] = __ldg(from + i);
    }
  };
  const auto row_of = [&](int s) { return warp * kRowsOfWarp + s * kRowsAtOnce + sub; };
#pragma unroll
  for (int s = 0; s < kSteps; ++s) load4(job.x, tile * kTile + row_of(s), v[s]);
  __syncthreads();
  const auto own_row = [&](int g) { return row_of(4 * g + lane % kAcross / kShare); };
  const auto add = [](float x, float y) { return x + y; };
  float own_max[kGroups], own_delta[kGroups], own_norm[kGroups], own_top[kGroups];
  if (job.gradient) {
    const float* const stats = p.a.stats + 2 * (((int64_t)b * job.heads + h) * job.length + tile * kTile);
    const int rows = job.length - tile * kTile;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      float o[4][4], stat_inv[4], delta[4], norm[4];
      own_max[g] = own_row(g) < rows ? __ldg(stats + 2 * own_row(g)) : 0.f;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        load4(p.a.out, tile * kTile + row_of(4 * g + s), o[s]);
        stat_inv[s] = row_of(4 * g + s) < rows ? __ldg(stats + 2 * row_of(4 * g + s) + 1) : 0.f;
      }
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        delta[s] = norm[s] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float& w = v[4 * g + s][i];
          w *= stat_inv[s];
          delta[s] = fmaf(w, o[s][i], delta[s]);
          norm[s] = fmaf(w, w, norm[s]);
        }
      }
      own_delta[g] = joined<kAcross>(delta, add);
      own_norm[g] = joined<kAcross>(norm, add);
    }
  }
  float most = 0.f, least = INFINITY;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    float top[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      bool fine = true;
      top[s] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float& w = v[4 * g + s][i];
        if (!(fabsf(w) < INFINITY)) { w = 0.f; fine = false; }
        top[s] = fmaxf(top[s], fabsf(w));
      }
      if (!fine) atomicOr(&bad_words[row_of(4 * g + s) >> 5], 1u << (row_of(4 * g + s) & 31));
    }
    own_top[g] = largest<kAcross>(top);
    most = fmaxf(most, own_top[g]);
    if (own_top[g] > 0.f) least = fminf(least, own_top[g]);
    if (job.gradient) {
      const int r = own_row(g);
      // where squares leave the numbers' range, a bound
      float norm = own_norm[g] > 1e-30f && own_norm[g] < 1e37f ? sqrtf(own_norm[g]) : fminf(own_top[g] * sqrtf((float)D), 3e38f);
      if (!(fabsf(own_delta[g]) < INFINITY && fabsf(own_max[g]) < INFINITY)) {
        atomicOr(&bad_words[r >> 5], 1u << (r & 31));
        own_max[g] = own_delta[g] = norm = 0.f;
      }
      if (lane % kShare == 0) {
        const int64_t at = ((int64_t)bh * job.tiles + tile) * kTile + r;
        p.row_max[at] = own_max[g]; p.row_delta[at] = own_delta[g]; p.row_norm[at] = norm;
      }
      most_norm = fmaxf(most_norm, norm); most_delta = fmaxf(most_delta, fabsf(own_delta[g]));
      if (norm > 0.f) low = fminf(low, norm);
      peak = fmaxf(peak, fabsf(own_max[g]));
    }
  }
#pragma unroll
  for (int o = 16; o >= kShare; o >>= 1) {
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
  }
  if (job.gradient) {
#pragma unroll
    for (int o = 16; o >= kShare; o >>= 1) {
      most_norm = fmaxf(most_norm, __shfl_xor_sync(0xffffffffu, most_norm, o));
      most_delta = fmaxf(most_delta, __shfl_xor_sync(0xffffffffu, most_delta, o));
      low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
      peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, o));
    }
  }
  if (lane == 0) { red[warp] = most; red_least[warp] = least; red_norm[warp] = most_norm; red_delta[warp] = most_delta; red_low[warp] = low; red_peak[warp] = peak; }
  __syncthreads();
  most = red[lane & (kPackWarps - 1)]; least = red_least[lane & (kPackWarps - 1)];
#pragma unroll
  for (int o = kPackWarps / 2; o > 0; o >>= 1) {
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
  }
  if (job.gradient && warp == 0) {
    most_norm = red_norm[lane & (kPackWarps - 1)]; most_delta = red_delta[lane & (kPackWarps - 1)]; low = red_low[lane & (kPackWarps - 1)]; peak = red_peak[lane & (kPackWarps - 1)];
#pragma unroll
    for (int o = kPackWarps / 2; o > 0; o >>= 1) {
      most_norm = fmaxf(most_norm, __shfl_xor_sync(0xffffffffu, most_norm, o));
      most_delta = fmaxf(most_delta, __shfl_xor_sync(0xffffffffu, most_delta, o));
      low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
      peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, o));
    }
  }
  const bool apart = most > 0.f && exponent_of(most) - exponent_of(least) > (job.gradient ? kOrdersOfGradient : kOrders);
  const int below = job.times == 1.f ? 14 : 13, e = scale_exponent(most, below);
  const int64_t at_tile = (int64_t)bh * job.tiles + tile;
  if (lane % kShare == 0) {
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const int of_token = apart ? scale_exponent(own_top[g], below) : e;
      if (apart) token_scale[own_row(g)] = power_of_two(of_token) * job.times;    // its warp's rows
      job.scale[at_tile * kTile + own_row(g)] = apart && own_top[g] == 0.f ? 0.f : power_of_two(-of_token);
    }
  }
  if (threadIdx.x == 0) {
    TileInfo& info = job.info[at_tile];
    info.inv = apart ? -1.f : power_of_two(-e); info.top = most; info.norm = most_norm; info.delta = most_delta; info.low = low; info.peak = peak;
#pragma unroll
    for (int i = 0; i < 4; ++i) info.bad[i] = bad_words[i];
  }
  if (apart) __syncwarp();
  char* const image = job.image + at_tile * (2 * G * 16384);
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int r = row_of(s);
    const float scale = apart ? token_scale[r] : power_of_two(e) * job.times;
    float hi[4], x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[i] = v[s][i] * scale; hi[i] = __half2float(__float2half_rn(x[i])); }
    const int at = (col >> 6) * 16384 + r * 128 + ((((col & 63) >> 3) ^ (r & 7)) << 4) + (col & 4) * 2;
    *reinterpret_cast<uint2*>(image + at) = make_uint2(halves(hi[0], hi[1]), halves(hi[2], hi[3]));
    *reinterpret_cast<uint2*>(image + G * 16384 + at) = make_uint2(halves(x[0] - hi[0], x[1] - hi[1]), halves(x[2] - hi[2], x[3] - hi[3]));
  }
  if (p.documents && j == p.document_job && h == 0 && warp == 0) {       // what the tile's documents are
    float low = INFINITY, high = -INFINITY;
    int padding = 0;
    for (int r = lane; r < kTile; r += 32) {
      const float d = document_of(p.a, b, tile * kTile + r);
      if (d >= 0.f) { low = fminf(low, d); high = fmaxf(high, d); } else padding = 1;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o)); high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o)); }
    padding = __any_sync(0xffffffffu, padding);
    if (lane == 0) p.documents[(int64_t)b * job.tiles + tile] = make_float4(low, high, padding ? 1.f : 0.f, 0.f);
  }
}

// ---- which tiles of the other side a CTA's rows see ------------------------------------------------------------------------------
// A warp looks at 32 tiles at a time.  Every role walks the same list.
template <int KIND> struct Walk {
  static constexpr bool kRowsAreKeys = KIND == kDk || KIND == kDv;
  const TcArgs& p;
  int b, head, heads_end, tiles, base, prefix;
  int from, to;                                  // rows: positions of queries, or keys
  float low, high;                               // their documents
  bool padding;
  uint32_t any, whole;
  __device__ __forceinline__ Walk(const TcArgs& args, int b_, int row_head, int share, int tile) : p(args), b(b_) {
    const AttentionArgs& a = p.a;
    const int off = a.Tk - a.Tq;
    prefix = prefix_of(a, b);
    tiles = kRowsAreKeys ? p.q_tiles : p.k_tiles;
    if (kRowsAreKeys) { heads_end = a.group / p.shares; head = row_head * a.group + share * heads_end; heads_end += head; from = tile * kTile; to = min(from + kTile, a.Tk) - 1; }
    else { head = row_head; heads_end = head + 1; from = tile * kTile + off; to = min(from + kTile - 1, a.Tk - 1); }
    low = high = 0.f; padding = false;
    if (p.documents) documents(from, to, low, high, padding);
    base = -32; any = whole = 0u;
  }
  __device__ __forceinline__ void documents(int first, int last, float& lo, float& hi, bool& pad) const {
    const float4 u = p.documents[(int64_t)b * p.k_tiles + first / kTile], w = p.documents[(int64_t)b * p.k_tiles + last / kTile];
    lo = fminf(u.x, w.x); hi = fmaxf(u.y, w.y); pad = u.z + w.z > 0.f;
  }
  __device__ __forceinline__ void look(int lane) {
    const AttentionArgs& a = p.a;
    const int t = base + lane;
    bool sees_any = false, sees_whole = false;
    if (t < tiles) {
      const int off = a.Tk - a.Tq;
      // first and last query position, first and last key
      const int p0 = kRowsAreKeys ? t * kTile + off : from, p1 = kRowsAreKeys ? min(p0 + kTile - 1, a.Tk - 1) : to;
      const int j0 = kRowsAreKeys ? from : t * kTile, j1 = kRowsAreKeys ? to : j0 + kTile - 1;
      const Sight first = sight_of(a, p0), last = sight_of(a, p1);
      sees_any = j0 < prefix || (j0 <= last.hi && j1 >= first.lo);
      const bool full_tile = (kRowsAreKeys ? t * kTile + kTile <= a.Tq : j1 < a.Tk);            // columns behind the end are hidden one by one
      sees_whole = full_tile && (j1 < prefix || (j1 <= first.hi && j0 >= last.lo));
      if (sees_any && p.documents) {
        float lo, hi;
        bool pad;
        if (kRowsAreKeys) documents(p0, p1, lo, hi, pad); else documents(j0, min(j1, a.Tk - 1), lo, hi, pad);
        sees_any = lo <= high && low <= hi;
        sees_whole = sees_whole && !pad && !padding && lo == hi && low == high && lo == low;
      }
    }
    any = __ballot_sync(0xffffffffu, sees_any);
    whole = __ballot_sync(0xffffffffu, sees_whole);
  }
  // The next tile: its head and number, and whether every row sees all of it
  __device__ __forceinline__ bool next(int lane, int& at_head, int& t, bool& all) {
    while (!any) {
      base += 32;
      if (base >= tiles) {
        if (++head >= heads_end) return false;
        base = 0;
      }
      look(lane);
    }
    const int bit = __ffs(any) - 1;
    any &= any - 1;
    at_head = head; t = base + bit; all = (whole >> bit) & 1u;
    return true;
  }
};

// ---- the kernel ----------------------------------------------------------------------------------------------------------------
template <int KIND, int G> struct Shape {
  static constexpr bool kTwo = KIND == kDq || KIND == kDk;           // two score products
  static constexpr bool kRowsAreKeys = KIND == kDk || KIND == kDv;
  static constexpr bool kTurns = !kTwo;                              // groups of warps take turns
  static constexpr int kWeightWarps = kTurns ? 4 : 8;                // of a tile
  static constexpr int kChunks = kTurns ? 4 : 2;                     // of 32 columns, a thread
  static constexpr int kSums = kTurns ? 64 * G : 32 * G;             // columns of the product that a thread adds up
  // The rows' first operand lies in TMEM where there is room beside scores and products: an MMA of 128 columns takes 73 cycles then, 102 with both operands in shared memory.
  static constexpr bool kRowsInTmem = !kTwo || G == 1;
  static constexpr int kPart = G * 16384;                            // one half (hi or lo) of a tile
  static constexpr int kResident = (kTwo ? 2 : 0) * kPart + (kRowsInTmem ? 0 : 2) * kPart;
  static constexpr int kControl = 768 + (KIND == kFwd ? 1024 : 0) + (kRowsAreKeys ? 2048 : 0) + (kTwo ? 256 : 0);
  static constexpr int kFits = (232448 - kControl - kResident) / kPart, kStages = kFits < 8 ? kFits : 8;
  static constexpr int kSmem = kResident + kStages * kPart + kControl;
  // TMEM columns: scores 0 and 128, then
  static constexpr int kYAt = 256;                                   // second scores
  static constexpr int kOuts = !kTwo && G == 1 ? 2 : 1;
  static constexpr int kRowsAt = kTwo ? 448 : 256;                   // hi, then lo
  static constexpr int kOutAt = kTwo ? 384 : 256 + 64 * G;
  static_assert(kStages >= 3 && kOutAt + kOuts * 64 * G <= (kTwo && G == 1 ? 448 : 512), "fits");
  static_assert(!kTurns || kStages * kPart >= kSums * kTile * 4, "the sums of a group fit the ring");
};
// Of one tile of columns, for the warps: written by the copying warp, which walks the list.  Eight of them in turn: by the time a copy for tile n + 8 can be issued,
// the weights of tile n + 4 have been made.
struct __align__(16) Entry {
  int flags, head, col, at;                      // 1: there is a tile, 2: every row sees all of it, and all of it is finite, 4: its tokens or the rows have scales of their own; position of its first column; its number, or behind the last how many there were
  float inv1, inv2, x, y;                        // 1 / scale of both operands; dq: largest magnitude of V, dk: largest norm and |D'| of dO'
};

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
// Descriptors in two words each
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_low, uint32_t a_high, uint32_t b_low, uint32_t b_high, uint32_t idesc, uint32_t keep) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"((uint64_t)a_low | (uint64_t)a_high << 32), "l"((uint64_t)b_low | (uint64_t)b_high << 32), "r"(idesc), "r"(keep) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_low, uint32_t b_high, uint32_t idesc, uint32_t keep) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
               ::"r"(d), "r"(a), "l"((uint64_t)b_low | (uint64_t)b_high << 32), "r"(idesc), "r"(keep) : "memory");
}

// tanh of 32 numbers.  Up to 0.35 by the series of odd powers (x^13 behind it is 1.2e-8 of x there), whose error is relative; above by 1 - 2 / (e^2x + 1), whose error
// is a rounding of 1.  Scores far below the cap, most of all, take the series alone, and below 0.15 only its first terms (x^9 behind them is 6e-9 of x).
__device__ __forceinline__ void tanh32(float* t) {
  float most = 0.f;
#pragma unroll
  for (int k = 0; k < 32; ++k) most = fmaxf(most, fabsf(t[k]));
  const bool small = __all_sync(0xffffffffu, most < 0.15f), large = __any_sync(0xffffffffu, !(most < 0.35f));
#pragma unroll
  for (int k = 0; k < 32; k += 2) {
    const float2 x = at2(t, k), s = mul2(x, x);
    float2 y = both(-17.f / 315.f);
    if (!small) y = fma2(fma2(both(-1382.f / 155925.f), s, both(62.f / 2835.f)), s, y);
    y = fma2(fma2(y, s, both(2.f / 15.f)), s, both(-1.f / 3.f));
    y = fma2(mul2(y, s), x, x);
    if (__builtin_expect(large, 0)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float v = i ? x.y : x.x, far = 1.f - 2.f * reciprocal(exp2_fast(2.f * kLog2e * fabsf(v)) + 1.f);
        if (!(fabsf(v) < 0.35f)) (i ? y.y : y.x) = copysignf(far, v);
      }
    }
    put2(t, k, y);
  }
}
// 32 numbers times `by` and a scale each, powers of two or zero
__device__ __forceinline__ void times32(float* z, const float* __restrict__ scale, float by) {
#pragma unroll
  for (int k = 0; k < 32; k += 4) {
    const float4 f = __ldg(reinterpret_cast<const float4*>(scale + k));
    z[k] *= f.x * by; z[k + 1] *= f.y * by; z[k + 2] *= f.z * by; z[k + 3] *= f.w * by;
  }
}
// hi and lo halves of 32 weights, as the A operand has them: 16 weights are 8 words of hi and 8 of lo
__device__ __forceinline__ void split32(const float* w, uint32_t* words) {
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    // the upper 11 bits, which fp16 holds exactly down to 2^-14; below, the rounding is 2^-25 of weights that reach 2^14
    const float a = __uint_as_float(__float_as_uint(w[2 * k]) & 0xffffe000u), b = __uint_as_float(__float_as_uint(w[2 * k + 1]) & 0xffffe000u);
    const float2 rest = add2(at2(w, 2 * k), make_float2(-a, -b));
    words[(k >> 3) * 16 + (k & 7)] = halves(a, b);
    words[(k >> 3) * 16 + 8 + (k & 7)] = halves(rest.x, rest.y);
  }
}
__device__ __forceinline__ uint32_t bits_between(int lo, int hi) {               // bits lo .. hi of a word, as far as it has them
  const uint32_t below = hi >= 31 ? 0xffffffffu : hi < 0 ? 0u : (2u << hi) - 1u;
  return lo <= 0 ? below : lo > 31 ? 0u : below & (0xffffffffu << lo);
}

// mbar_wait_mark in few instructions: eight warps and the issuer share the instruction cache
__device__ __forceinline__ void await(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int& bad) {
  if (bad || mbar_try_wait(bar, parity)) return;
  const long long t0 = clock64();
#pragma unroll 1
  while (!mbar_try_wait(bar, parity)) {
    if (*abort_flag) { bad = 1; break; }
    if (clock64() - t0 > kWaitCycles) { *abort_flag = 1; bad = 1; break; }
  }
}

template <int KIND, int G, bool SHAPED>
__device__ __forceinline__ void attention_rows(const TcArgs& p, int block) {
  using S = Shape<KIND, G>;
  constexpr bool kTwo = S::kTwo, kRowsAreKeys = S::kRowsAreKeys;
  constexpr int kPart = S::kPart, kStages = S::kStages, kOuts = S::kOuts;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* const resident = smem;
  uint8_t* const ring = smem + S::kResident;
  uint64_t* const full = reinterpret_cast<uint64_t*>(ring + kStages * kPart);
  uint64_t* const empty = full + 8;
  uint64_t* const entry_full = empty + 8;        // [8] an entry is written
  uint64_t* const resident_full = entry_full + 8;
  uint64_t* const s_full = resident_full + 1;    // [2] scores are in TMEM
  uint64_t* const w_full = s_full + 2;           // [2] weights are
  uint64_t* const y_full = w_full + 2;           // [2] second scores are in TMEM
  uint64_t* const y_empty = y_full + 2;          // [2] and have been read
  uint64_t* const o_full = y_empty + 2;          // [2] the product is
  uint64_t* const o_empty = o_full + 2;          // [2] and has been added up
  uint64_t* const columns_full = o_empty + 2;    // [2] maxima and D' of a tile of queries
  uint64_t* const merge = columns_full + 2;      // the second group's sums are in shared memory
  uint64_t* const rows_full = merge + 1;         // the rows are in TMEM
  uint64_t* const swap_full = rows_full + 1;     // both groups' largest weights of every row are in shared memory
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(swap_full + 1);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  Entry* const entries = reinterpret_cast<Entry*>(full + 64);        // [8]
  float* const statistics = reinterpret_cast<float*>(entries + 8);   // fwd: [2][128] of the second group
  float* const columns = statistics;                                 // dk, dv: [2][2][128]
  uint8_t* const swapped = reinterpret_cast<uint8_t*>(columns + (S::kRowsAreKeys ? 512 : 0));            // dq, dk: [2][128] exponents of the groups' largest weights
  static_assert(8 + 8 + 8 + 1 + 7 * 2 + 3 + 2 <= 64, "barriers fit");
  const AttentionArgs& a = p.a;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (warp == 0) {
    if (lane == 0) {
      for (int i = 0; i < kStages; ++i) { mbar_init(full + i, 1); mbar_init(empty + i, 1); }
      for (int i = 0; i < 8; ++i) mbar_init(entry_full + i, 1);
      mbar_init(resident_full, 1);
      for (int i = 0; i < 2; ++i) {              // tiles take turns, also where one buffer serves both
        mbar_init(s_full + i, 1); mbar_init(w_full + i, S::kWeightWarps);
        mbar_init(y_full + i, 1); mbar_init(y_empty + i, S::kWeightWarps);
        mbar_init(o_full + i, 1); mbar_init(o_empty + i, S::kWeightWarps);
        mbar_init(columns_full + i, 1);
      }
      mbar_init(merge, 4); mbar_init(rows_full, 8); mbar_init(swap_full, 8);
      *abort_flag = (smem_u32(smem) & 1023u) ? 1 : 0;                // nothing is issued then
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncwarp();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  grid_dep_sync();

  // rows that see most go first
  const int row_heads = kRowsAreKeys ? a.G : a.H, col_tiles = kRowsAreKeys ? p.q_tiles : p.k_tiles, row_tiles = kRowsAreKeys ? p.k_tiles : p.q_tiles;
  const int shares = kRowsAreKeys ? p.shares : 1, across = a.B * row_heads * shares, order = block / across, place = block - order * across;
  const int b = place / (row_heads * shares), row_head = place / shares - b * row_heads, share = place % shares;
  const int tile = kRowsAreKeys ? order : row_tiles - 1 - order;
  const int64_t row_at = ((int64_t)b * row_heads + row_head) * row_tiles + tile;
  const Packed &r1 = kRowsAreKeys ? p.k : p.q, &r2 = kRowsAreKeys ? p.v : p.d;                 // rows
  const Packed &c1 = kRowsAreKeys ? p.q : p.k, &c2 = kRowsAreKeys ? p.d : p.v;                 // columns
  const auto col_at = [&](int head, int t) { return kRowsAreKeys ? ((int64_t)b * a.H + head) * col_tiles + t : ((int64_t)b * a.G + head / a.group) * col_tiles + t; };
  int bad = *abort_flag;

  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegisters));
  if (warp == 0) {
    // ---- copies: the rows once, then tiles in the order in which the MMAs take them, the lo half first
    int stage = 0;
    uint32_t phase = 0, armed = 0, phases = 0, columns_armed = 0;
    bool rows_armed = false;
    if (S::kResident && !bad) {
      if (elect_one()) {
        mbar_expect_tx(resident_full, S::kResident);
        bulk_load(resident, r2.image + row_at * 2 * kPart, 2 * kPart, resident_full);
        if (!S::kRowsInTmem) bulk_load(resident + 2 * kPart, r1.image + row_at * 2 * kPart, 2 * kPart, resident_full);
      }
      rows_armed = true;
    }
    Walk<KIND> walk(p, b, row_head, share, tile);
    const TileInfo& rows2 = kTwo ? r2.info[row_at] : r1.info[row_at];
    const float rows_inv1 = r1.info[row_at].inv, rows_inv2 = rows2.inv, rows_top = rows2.top, rows_peak = rows2.peak;
    // What an entry says is asked for a tile ahead, and looked at behind the tile's first copies
    struct Next { bool there, all; int head, t; int64_t at; float inv1, inv2, x, y, low, peak; uint4 bad1, bad2; };
    const auto look_ahead = [&] {
      Next x;
      x.there = walk.next(lane, x.head, x.t, x.all);
      x.at = x.there ? col_at(x.head, x.t) : 0;
      const TileInfo &i1 = c1.info[x.at], &i2 = c2.info[x.at];
      x.inv1 = i1.inv; x.inv2 = i2.inv; x.x = KIND == kDq ? i2.top : i2.norm; x.y = i2.delta; x.low = i2.low; x.peak = i2.peak;
      x.bad1 = *reinterpret_cast<const uint4*>(i1.bad); x.bad2 = *reinterpret_cast<const uint4*>(i2.bad);
      return x;
    };
    const auto flags_of = [&](const Next& x) {
      const bool spoils = (x.bad1.x | x.bad1.y | x.bad1.z | x.bad1.w | x.bad2.x | x.bad2.y | x.bad2.z | x.bad2.w) != 0u, whole = x.all && !spoils;
      bool apart = fminf(fminf(rows_inv1, rows_inv2), fminf(x.inv1, x.inv2)) < 0.f || (KIND != kFwd && (kRowsAreKeys ? x.peak : rows_peak) > kPeak);
      // dk: one bound of the tile's queries scales the weights of all keys.  Where a key may see the smallest of them alone, and that is kOrdersOfBound below it, or where all see all,
      // kOrdersOfSeen, the tile goes the way of tokens that are apart.
      const float top = rows_top * sqrtf((float)a.D);
      if (KIND == kDk && fmaf(x.x, top, x.y) > (float)(1 << (whole ? kOrdersOfSeen : kOrdersOfBound)) * (x.low * top)) apart = true;
      return 1 | (int)whole << 1 | (int)apart << 2;
    };
    const auto load = [&](const Packed& from, int64_t at) {
#pragma unroll
      for (int lo = 1; lo >= 0; --lo) {
        await(&empty[stage], phase ^ 1, abort_flag, bad);
        bad = __any_sync(0xffffffffu, bad);
        if (!bad) {
          if (elect_one()) {
            mbar_expect_tx(&full[stage], kPart);
            bulk_load(ring + stage * kPart, from.image + (at * 2 + lo) * kPart, kPart, &full[stage]);
          }
          armed |= 1u << stage;
          phases = (phases & ~(1u << stage)) | phase << stage;
        }
        if (++stage == kStages) { stage = 0; phase ^= 1; }
      }
    };
    int64_t before = -1;
    Next next = look_ahead();
    for (int n = 0;; ++n) {
      const Next now = next;
      if (now.there) load(c1, now.at);           // before the entry, which waits for what it says; it waits for no tile but those in front of it
      if (lane == 0) {
        entries[n & 7] = Entry{now.there ? flags_of(now) : 0, now.head, now.t * kTile + (kRowsAreKeys ? a.Tk - a.Tq : 0), now.there ? (int)now.at : n, now.inv1, now.inv2, now.x, now.y};
        mbar_arrive(entry_full + (n & 7));
      }
      __syncwarp();
      if (!now.there) {                          // and for the other group, whose tile would be the next
        if (lane == 0) { entries[(n + 1) & 7].flags = 0; entries[(n + 1) & 7].at = n; mbar_arrive(entry_full + ((n + 1) & 7)); }
        break;
      }
      next = look_ahead();
      if (kTwo) load(c2, now.at);
      if (kRowsAreKeys) {                        // maxima and D' of the tile's queries, when the weights of the tile before the last are made
        if (n >= 2) await(&w_full[n & 1], ((n - 2) >> 1) & 1, abort_flag, bad);
        bad = __any_sync(0xffffffffu, bad);
        if (!bad) {
          if (elect_one()) {
            mbar_expect_tx(columns_full + (n & 1), kTwo ? 1024 : 512);
            bulk_load(columns + (n & 1) * 256, p.row_max + now.at * kTile, 512, columns_full + (n & 1));
            if (kTwo) bulk_load(columns + (n & 1) * 256 + 128, p.row_delta + now.at * kTile, 512, columns_full + (n & 1));
          }
          columns_armed = n + 1;
        }
      }
      if (before >= 0) load(kTwo ? c1 : c2, before);
      before = now.at;
    }
    if (before >= 0) load(kTwo ? c1 : c2, before);
    __syncwarp();
    if (*abort_flag) {                           // copies in flight land before the CTA gives its shared memory back
      for (int i = -1; i < kStages; ++i) {
        if (i < 0 ? !rows_armed : !((armed >> i) & 1u)) continue;
        const long long t0 = clock64();
        while (!mbar_try_wait(i < 0 ? resident_full : &full[i], i < 0 ? 0 : (phases >> i) & 1u) && clock64() - t0 < 100000000ll) {}
      }
      for (uint32_t n = columns_armed > 2 ? columns_armed - 2 : 0; n < columns_armed; ++n) {
        const long long t0 = clock64();
        while (!mbar_try_wait(columns_full + (n & 1), (n >> 1) & 1) && clock64() - t0 < 100000000ll) {}
      }
    } else if (rows_armed) {
      await(resident_full, 0, abort_flag, bad);             // rows that see nothing: nobody else waits for them
    }
  } else if (warp == 1) {
    // ---- MMAs
    constexpr uint32_t kIdesc = (1u << 4) | ((uint32_t)(kTile >> 4) << 24), kScores = kIdesc | ((uint32_t)(kTile >> 3) << 17);
    const uint32_t products = kIdesc | (1u << 16) | ((uint32_t)(p.D16 >> 3) << 17);            // the B operand has its columns (the head) along the rows of memory
    const int steps = p.D16 / 16;
    int stage = 0;
    uint32_t phase = 0;
    // Descriptors differ in their low word alone, by constants from one MMA to the next
    constexpr uint32_t kHigh = (1024u >> 4) | 1u << 14 | 2u << 29;
    const auto k_major = [](uint32_t at) { return (at & 0x3FFFFu) >> 4 | 1u << 16; };
    const auto mn_major = [](uint32_t at) { return (at & 0x3FFFFu) >> 4 | (16384u >> 4) << 16; };
    // both halves of a tile are there; the lo half is in the present stage
    const auto wait_tile = [&] {
      const bool wraps = stage + 1 == kStages;
      await(&full[stage], phase, abort_flag, bad);
      await(&full[wraps ? 0 : stage + 1], wraps ? phase ^ 1 : phase, abort_flag, bad);
      __syncwarp();
      tcgen05_fence_after();
    };
    const auto next_stage = [&] { if (++stage == kStages) { stage = 0; phase ^= 1; } };
    // rows: the low word of their descriptor, or where they lie in TMEM
    const auto score_steps = [&](uint32_t d, uint32_t rows, bool in_tmem, uint32_t cols_low, uint32_t keep) {
#pragma unroll
      for (int ks = 0; ks < 4 * G; ++ks) {
        const uint32_t step = (ks >> 2) * 1024 + (ks & 3) * 2;
        if (ks >= steps) continue;
        if (in_tmem) mma_ts(d, rows + 8 * ks, cols_low + step, kHigh, kScores, ks ? 1u : keep);
        else mma_ss(d, rows + step, kHigh, cols_low + step, kHigh, kScores, ks ? 1u : keep);
      }
    };
    const auto product_steps = [&](uint32_t d, uint32_t w, uint32_t cols_low, uint32_t idesc, uint32_t keep) {
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) mma_ts(d, w + 16 * ks, cols_low + ks * 128, kHigh, idesc, ks ? 1u : keep);
    };
    // Scores add up the queries' lo halves times the keys' hi halves, then the other way around, then both hi halves, whichever are the rows, so that both directions truncate alike
    // and form the same scores.  `lo_pass` reads the columns' lo half, whose stage is given back behind it.
    const auto scores = [&](uint32_t d, uint32_t rows_hi, auto in_tmem, int lo_pass, uint64_t* done) {
      wait_tile();
      const int lo = stage;
      next_stage();
      if (!bad && elect_one()) {
        const uint32_t at_lo = k_major(smem_u32(ring + lo * kPart)), at_hi = k_major(smem_u32(ring + stage * kPart));
#pragma unroll 1
        for (int pass = 0; pass < 3; ++pass) {
          score_steps(d, rows_hi + (pass != 1 - lo_pass ? 0 : decltype(in_tmem)::value ? 32 * G : kPart >> 4), decltype(in_tmem)::value, pass == lo_pass ? at_lo : at_hi, pass);
          if (pass == lo_pass) tcgen05_commit(&empty[lo]);
        }
        tcgen05_commit(&empty[stage]);
        tcgen05_commit(done);
      }
      __syncwarp();
      next_stage();
    };
    const auto product = [&](int n) {
      const int out = kOuts == 2 ? n & 1 : 0;
      const uint32_t w = tmem + (n & 1) * 128, d = tmem + S::kOutAt + out * 64 * G;
      await(&w_full[n & 1], (n >> 1) & 1, abort_flag, bad);
      if (n >= kOuts) await(&o_empty[(n - kOuts) & 1], ((n - kOuts) >> 1) & 1, abort_flag, bad);
      wait_tile();
      const int lo = stage;
      next_stage();
      if (!bad && elect_one()) {
        const uint32_t at_lo = mn_major(smem_u32(ring + lo * kPart)), at_hi = mn_major(smem_u32(ring + stage * kPart));
#pragma unroll 1
        for (int pass = 0; pass < 3; ++pass) {
          product_steps(d, w + (pass == 1 ? 8 : 0), pass ? at_hi : at_lo, products, pass);
          if (pass == 0) tcgen05_commit(&empty[lo]);
        }
        tcgen05_commit(&empty[stage]);
        tcgen05_commit(&o_full[n & 1]);
      }
      __syncwarp();
      next_stage();
    };
    if (S::kResident) await(resident_full, 0, abort_flag, bad);
    if (S::kRowsInTmem) { await(rows_full, 0, abort_flag, bad); __syncwarp(); tcgen05_fence_after(); }
    const uint32_t rows2 = k_major(smem_u32(resident)), rows1 = S::kRowsInTmem ? tmem + S::kRowsAt : rows2 + (2 * kPart >> 4);
    int n = 0;
    for (;; ++n) {
      await(entry_full + (n & 7), (n >> 3) & 1, abort_flag, bad);
      bad = __any_sync(0xffffffffu, bad);
      if (bad || !(entries[n & 7].flags & 1)) break;
      scores(tmem + (n & 1) * 128, rows1, std::integral_constant<bool, S::kRowsInTmem>(), kRowsAreKeys ? 0 : 1, &s_full[n & 1]);
      if (kTwo) {
        if (n >= 1) await(&y_empty[(n - 1) & 1], ((n - 1) >> 1) & 1, abort_flag, bad);
        scores(tmem + S::kYAt, rows2, std::false_type(), 0, &y_full[n & 1]);
      }
      if (n > 0) product(n - 1);
    }
    if (n > 0) product(n - 1);
  }
  } else {
    // ---- weights
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegisters));
    const int quarter = warp & 3, group = (warp - 4) >> 2, row = quarter * 32 + lane;
    const uint32_t mine = tmem + ((uint32_t)(quarter * 32) << 16);
    if (S::kRowsInTmem) {                        // one group moves the hi halves of the rows, the other the lo halves
      const char* const image = r1.image + (row_at * 2 + group) * kPart + row * 128;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        uint4 words[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) words[c] = *reinterpret_cast<const uint4*>(image + g * 16384 + ((c ^ (row & 7)) << 4));
        tmem_st32(mine + S::kRowsAt + group * 32 * G + g * 32, reinterpret_cast<const uint32_t*>(words));
      }
      tmem_st_wait();
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(rows_full);
    }
    const int off = a.Tk - a.Tq, self = tile * kTile + row;            // query or key
    const bool there = self < (kRowsAreKeys ? a.Tk : a.Tq);
    // columns that the row sees: positions [lo, hi] and those before `extra`
    int lo, hi, extra;
    if (kRowsAreKeys) {
      lo = a.causal ? self : a.window ? self - a.window + 1 : -kFar;
      hi = min(a.window ? self + a.window - 1 : kFar, a.Tk - 1);       // no query is behind the last key
      extra = self < prefix_of(a, b) ? a.Tk : -kFar;
    } else {
      const Sight s = sight_of(a, self + off);
      lo = s.lo; hi = min(s.hi, a.Tk - 1); extra = prefix_of(a, b);
    }
    const float document = p.documents ? document_of(a, b, kRowsAreKeys ? self : self + off) : 0.f;
    const TileInfo& info1 = r1.info[row_at];
    bool spoiled = (info1.bad[quarter] >> lane) & 1u;
    if (kTwo) spoiled = spoiled || ((r2.info[row_at].bad[quarter] >> lane) & 1u);
    const bool careful = __any_sync(0xffffffffu, spoiled);
    const bool cap = SHAPED && a.cap > 0.f;
    const float inv2 = kTwo ? r2.info[row_at].inv : 0.f;
    // The unit of rows that share a scale.  Powers of two: a score less its maximum is rounded once, in both directions alike, and the largest is 0, however large it is.
    const float unit = info1.inv * p.by, wide = cap ? a.cap * kLog2e : 1.f;
    float row_max = 0.f, row_delta = 0.f, row_norm = 0.f;
    if (KIND == kDq) { row_max = p.row_max[row_at * kTile + row]; row_delta = p.row_delta[row_at * kTile + row]; row_norm = p.row_norm[row_at * kTile + row] * sqrtf((float)a.D); }
    const float norm_top = KIND == kDk ? r2.info[row_at].top * sqrtf((float)a.D) : 0.f;
    constexpr bool kTurns = S::kTurns;
    constexpr int kSums = S::kSums;
    const int col_part = kTurns ? 0 : group * 64, sum_part = kTurns ? 0 : group * kSums;       // of the tile and of the product
    float acc[kSums];
#pragma unroll
    for (int i = 0; i < kSums; ++i) acc[i] = 0.f;
    float most = -INFINITY, sum = 0.f;                                 // fwd
    float alpha = 1.f, out_factor = 0.f;                               // of the product in flight
    float slope = 0.f;
    int slope_head = -1;
    uint32_t swaps = 0;                                                // dq, dk

    const auto arrive = [&](uint64_t* bar) { tcgen05_fence_before(); __syncwarp(); if (lane == 0) mbar_arrive(bar); };
    const auto wait_for = [&](uint64_t* bar, uint32_t parity) { await(bar, parity, abort_flag, bad); __syncwarp(); tcgen05_fence_after(); };
    const auto add_up = [&](int n) {
      wait_for(&o_full[n & 1], (n >> 1) & 1);
      const uint32_t from = mine + S::kOutAt + (kOuts == 2 ? (n & 1) * 64 * G : 0) + sum_part;
#pragma unroll
      for (int c = 0; c < kSums / 32; ++c) {
        float o[32];
        tmem_ld32(from + 32 * c, o);
        tmem_ld_wait();
        if (c == kSums / 32 - 1) arrive(&o_empty[n & 1]);
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          float2 x = at2(acc, 32 * c + k);
          if (KIND == kFwd) x = mul2(x, both(alpha));
          put2(acc, 32 * c + k, fma2(at2(o, k), both(out_factor), x));
        }
      }
    };

    int n = kTurns ? group : 0;
    constexpr int kStep = kTurns ? 2 : 1;
    const int at_row = kRowsAreKeys ? self : self + off;
    // of the tile at hand
    Entry now = {};
    int col0 = 0;                                // position of the first column
    bool masked = false;
    uint32_t from = 0;
    float theirs[S::kChunks] = {};               // a column's document in every lane
    // scores of a chunk of 32 columns, capped and biased, in units of log 2; turned: 1 - the cap's tanh squared
    const auto shape32 = [&](float* z, float* turned, int c, float by) {
#pragma unroll
      for (int k = 0; k < 32; k += 2) put2(z, k, mul2(at2(z, k), both(by)));
      if (cap) {
        tanh32(z);
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          const float2 t = at2(z, k);
          if (turned) put2(turned, k, fma2(mul2(t, both(-1.f)), t, both(1.f)));
          put2(z, k, mul2(t, both(wide)));
        }
      } else if (turned) {
#pragma unroll
        for (int k = 0; k < 32; ++k) turned[k] = 1.f;
      }
      if (a.slopes) {
        const float away = (float)(at_row - (col0 + 32 * c));
#pragma unroll
        for (int k = 0; k < 32; ++k) z[k] = fmaf(-slope, fabsf(away - (float)k), z[k]);
      }
    };
    // hides the columns of a chunk that the row does not see, and makes NaN of those that are not finite
    const auto mask32 = [&](float* z, int c, float hidden) {
      const int first = col0 + 32 * c;
      uint32_t seen = bits_between(lo - first, hi - first) | bits_between(-1, extra - 1 - first);
      if (p.documents) {
        uint32_t same = 0u;
        float of = theirs[0];
#pragma unroll
        for (int i = 1; i < S::kChunks; ++i) of = c == i ? theirs[i] : of;
#pragma unroll
        for (int k = 0; k < 32; ++k) same |= __shfl_sync(0xffffffffu, of, k) == document ? 1u << k : 0u;
        seen &= document >= 0.f ? same : 0u;
      }
      const uint32_t spoils = seen & (spoiled ? 0xffffffffu : c1.info[now.at].bad[col_part / 32 + c] | c2.info[now.at].bad[col_part / 32 + c]);
#pragma unroll
      for (int k = 0; k < 32; ++k) z[k] = (seen >> k) & 1u ? z[k] : hidden;
      if (__builtin_expect(spoils != 0u, 0)) {
#pragma unroll
        for (int k = 0; k < 32; ++k) if ((spoils >> k) & 1u) z[k] = NAN;
      }
    };

    for (;;) {
      bool apart = false;
      // Tiles whose tokens share a scale: nothing else in this loop, which the instruction cache is small for
      for (;; n += kStep) {
        await(entry_full + (n & 7), (n >> 3) & 1, abort_flag, bad);
        bad = __any_sync(0xffffffffu, bad);
        now = entries[n & 7];
        if (bad || !(now.flags & 1)) break;
        if (kTurns && n >= 2) add_up(n - 2);     // while the scores are being made
        if (SHAPED && a.slopes && slope_head != (kRowsAreKeys ? now.head : row_head)) {
          slope_head = kRowsAreKeys ? now.head : row_head;
          slope = __ldg(a.slopes + slope_head) * kLog2e;
        }
        col0 = now.col + col_part;
        masked = !(now.flags & 2) || careful;
        from = mine + (n & 1) * 128 + col_part;
        if (p.documents && masked) {             // asked for while the scores are being made
#pragma unroll
          for (int c = 0; c < S::kChunks; ++c) theirs[c] = document_of(a, b, col0 + 32 * c + lane);
        }
        wait_for(&s_full[n & 1], (n >> 1) & 1);
        if (now.flags & 4) { apart = true; break; }
        const float f = now.inv1 * unit;
        if (KIND == kFwd) {
          // Scores that are not plain products are written back, so that both passes read them
          const bool rewritten = SHAPED || masked;
          float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
          for (int c = 0; c < S::kChunks; ++c) {
            float z[32];
            tmem_ld32(from + 32 * c, z);
            tmem_ld_wait();
            if (__builtin_expect(rewritten, SHAPED)) {
              if (SHAPED) shape32(z, nullptr, c, f);
              else
#pragma unroll
                for (int k = 0; k < 32; ++k) z[k] *= f;
              if (masked) mask32(z, c, -INFINITY);
              tmem_st32(from + 32 * c, reinterpret_cast<const uint32_t*>(z));
            }
#pragma unroll
            for (int k = 0; k < 32; ++k) m[k & 3] = fmaxf(m[k & 3], z[k]);
          }
          if (rewritten) tmem_st_wait();
          const float g = rewritten ? 1.f : f;
          // of -infinity: NaN if g is 0, which the maximum leaves out
          const float at_most = fmaxf(most, fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])) * g), base = max_of_finite_or(at_most);
          const float faded = exp2_fast(most - base);
          most = at_most;
          float2 s[2] = {both(0.f), both(0.f)};
#pragma unroll 1
          for (int c = 0; c < S::kChunks; ++c) {
            float z[32];
            uint32_t words[32];
            tmem_ld32(from + 32 * c, z);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 32; k += 2) {
              const float2 e = fma2(at2(z, k), both(g), both(-base)), w = make_float2(exp2_fast(e.x), exp2_fast(e.y));
              s[(k >> 1) & 1] = add2(s[(k >> 1) & 1], w);
              put2(z, k, mul2(w, both(kWeightScale)));
            }
            split32(z, words);
            tmem_st32(from + 32 * c, words);
          }
          tmem_st_wait();
          arrive(&w_full[n & 1]);
          sum = fmaf(sum, faded, (s[0].x + s[0].y) + (s[1].x + s[1].y));
          alpha = faded;
          out_factor = now.inv2 * (1.f / kWeightScale);
        } else {
          // The weights' power of two is a factor: added to the exponential's argument it would cost bits of that, the more the smaller the output gradient (dq 6e-7 off at 1e-7 of it
          // instead of 1e-7)
          float factor, lift = kWeightScale;
          if (KIND == kDv) {
            factor = now.inv2 * (1.f / kWeightScale);
          } else {
            const float bound = KIND == kDq ? fmaf(row_norm, now.x, fabsf(row_delta)) : fmaf(now.x, norm_top, now.y);
            const int shift = min(100, max(-100, kWeightExp - exponent_of(bound)));
            lift = power_of_two(shift);
            factor = now.inv1 * power_of_two(-shift);
          }
          const float fy = KIND == kDq ? inv2 * lift * now.inv2 : inv2 * now.inv2;         // dq: the row's numbers have it, the others' weights
          const float *const col_max = columns + (n & 1) * 256 + col_part, *const col_delta = col_max + 128;
          if (kRowsAreKeys) await(&columns_full[n & 1], (n >> 1) & 1, abort_flag, bad);
          if (kTwo) wait_for(&y_full[n & 1], (n >> 1) & 1);
#pragma unroll 1
          for (int c = 0; c < S::kChunks; ++c) {
            float z[32], y[32], turned[SHAPED && kTwo ? 32 : 1];
            tmem_ld32(from + 32 * c, z);
            if (kTwo) tmem_ld32(mine + S::kYAt + col_part + 32 * c, y);
            tmem_ld_wait();
            if (kTwo && c == S::kChunks - 1) arrive(&y_empty[n & 1]);
            if (SHAPED) shape32(z, kTwo ? turned : nullptr, c, f);
            const float g = SHAPED ? 1.f : f;
            if (kRowsAreKeys) {
#pragma unroll
              for (int k = 0; k < 32; k += 4) {
                const float4 m4 = *reinterpret_cast<const float4*>(col_max + 32 * c + k);
                put2(z, k, fma2(at2(z, k), both(g), make_float2(-m4.x, -m4.y)));
                put2(z, k + 2, fma2(at2(z, k + 2), both(g), make_float2(-m4.z, -m4.w)));
                if (KIND == kDk) {
                  const float4 d4 = *reinterpret_cast<const float4*>(col_delta + 32 * c + k);
                  put2(y, k, fma2(at2(y, k), both(fy), make_float2(-d4.x, -d4.y)));
                  put2(y, k + 2, fma2(at2(y, k + 2), both(fy), make_float2(-d4.z, -d4.w)));
                }
              }
            } else {
              const float delta = row_delta * lift;
#pragma unroll
              for (int k = 0; k < 32; k += 2) { put2(z, k, fma2(at2(z, k), both(g), both(-row_max))); put2(y, k, fma2(at2(y, k), both(fy), both(-delta))); }
            }
#pragma unroll
            for (int k = 0; k < 32; k += 2) {
              float2 w = make_float2(exp2_fast(z[k]), exp2_fast(z[k + 1]));
              if (kRowsAreKeys) w = mul2(w, both(lift));
              if (kTwo) w = mul2(w, SHAPED ? mul2(at2(y, k), at2(turned, k)) : at2(y, k));
              put2(z, k, w);
            }
            if (__builtin_expect(masked, 0)) mask32(z, c, 0.f);
            uint32_t words[32];
            split32(z, words);
            tmem_st32(from + 32 * c, words);
          }
          tmem_st_wait();
          arrive(&w_full[n & 1]);
          if (!kTurns && n >= 1) add_up(n - 1);
          out_factor = factor;
        }
      }
      if (!apart) break;
      // Tokens of different sizes, among the columns or the rows.  Their scales go into the scores and, those of the product's operand, into the weights, which are held in TMEM until
      // the largest of their row is known and scales them: so no token costs a bit of what does not depend on it.
      const float row_unit = r1.scale[row_at * kTile + row] * p.by, row_inv2 = kTwo ? r2.scale[row_at * kTile + row] : 0.f;
      const float *const scale1 = c1.scale + (int64_t)now.at * kTile + col_part, *const scale2 = c2.scale + (int64_t)now.at * kTile + col_part;
      const float *const col_max = columns + (n & 1) * 256 + col_part, *const col_delta = col_max + 128;
      if (kRowsAreKeys) await(&columns_full[n & 1], (n >> 1) & 1, abort_flag, bad);
      if (kTwo) wait_for(&y_full[n & 1], (n >> 1) & 1);
      float at_most = most;
#pragma unroll 1
      for (int c = 0; c < (KIND == kFwd ? S::kChunks : 0); ++c) {      // the maximum first
        float z[32];
        tmem_ld32(from + 32 * c, z);
        tmem_ld_wait();
        times32(z, scale1 + 32 * c, row_unit);
        if (SHAPED) shape32(z, nullptr, c, 1.f);
        if (masked) mask32(z, c, -INFINITY);
#pragma unroll
        for (int k = 0; k < 32; ++k) at_most = fmaxf(at_most, z[k]);
        tmem_st32(from + 32 * c, reinterpret_cast<const uint32_t*>(z));
      }
      if (KIND == kFwd) tmem_st_wait();
      const float base = max_of_finite_or(at_most);
      float s = 0.f, heaviest = 0.f;
#pragma unroll 1
      for (int c = 0; c < S::kChunks; ++c) {
        float z[32], other[kTwo ? 32 : 1];       // the cap's derivatives, then the second scores
        tmem_ld32(from + 32 * c, z);
        tmem_ld_wait();
        if (KIND != kFwd) {
          times32(z, scale1 + 32 * c, row_unit);
          if (SHAPED) shape32(z, kTwo ? other : nullptr, c, 1.f);
        }
#pragma unroll
        for (int k = 0; k < 32; ++k) {           // scores above the row's statistics: another kernel's forward call rounded them otherwise
          z[k] = exp2_fast(KIND == kFwd ? z[k] - base : fminf(z[k] - (kRowsAreKeys ? col_max[32 * c + k] : row_max), 0.f));
          if (KIND == kFwd) s += z[k];
        }
        if (kTwo) {
          if (SHAPED)
#pragma unroll
            for (int k = 0; k < 32; ++k) z[k] *= other[k];
          tmem_ld32(mine + S::kYAt + col_part + 32 * c, other);
          tmem_ld_wait();
          times32(other, scale2 + 32 * c, row_inv2);
#pragma unroll
          for (int k = 0; k < 32; ++k) z[k] *= other[k] - (kRowsAreKeys ? col_delta[32 * c + k] : row_delta);
        }
        times32(z, (kTwo ? scale1 : scale2) + 32 * c, 1.f);
        if (KIND != kFwd && masked) mask32(z, c, 0.f);
#pragma unroll
        for (int k = 0; k < 32; ++k) heaviest = fmaxf(heaviest, fabsf(z[k]));
        tmem_st32(from + 32 * c, reinterpret_cast<const uint32_t*>(z));
      }
      tmem_st_wait();
      int e = (int)(__float_as_uint(heaviest) >> 23);
      if (kTwo) {                                // the groups have half of the row's weights each
        swapped[group * kTile + row] = (uint8_t)e;
        __syncwarp();
        if (lane == 0) mbar_arrive(swap_full);
        await(swap_full, swaps++ & 1, abort_flag, bad);
        __syncwarp();
        e = max(e, (int)swapped[(group ^ 1) * kTile + row]);
        arrive(&y_empty[n & 1]);                 // behind it, so that nobody is at the next tile's exchange before
      }
      const int shift = min(126, max(-126, kWeightExp + 127 - e));
#pragma unroll 1
      for (int c = 0; c < S::kChunks; ++c) {
        float z[32];
        uint32_t words[32];
        tmem_ld32(from + 32 * c, z);
        tmem_ld_wait();
#pragma unroll
        for (int k = 0; k < 32; ++k) z[k] *= power_of_two(shift);
        split32(z, words);
        tmem_st32(from + 32 * c, words);
      }
      tmem_st_wait();
      arrive(&w_full[n & 1]);
      if (KIND == kFwd) {
        alpha = exp2_fast(most - base);
        most = at_most;
        sum = fmaf(sum, alpha, s);
      }
      if (!kTurns && n >= 1) add_up(n - 1);
      out_factor = power_of_two(-shift);
      n += kStep;
    }
    if (n >= (kTurns ? 2 : 1)) add_up(n - (kTurns ? 2 : 1));           // n: where the list ends for this warp

    float last = KIND == kDv ? 1.f : KIND == kDk ? p.dk_factor : a.scale;
    if (kTurns) {
      // The second group's sums go through the ring, once the last product has read it.  Columns by rows, so that a warp's words lie side by side.
      float* const handed = reinterpret_cast<float*>(ring);
      volatile int* const any_handed = abort_flag + 1;
      if (group == 1) {
        const int tiles = entries[n & 7].at;
        if (n >= 3 && !bad) await(&o_full[(tiles - 1) & 1], ((tiles - 1) >> 1) & 1, abort_flag, bad);
        if (n >= 3 && !bad) {
#pragma unroll
          for (int k = 0; k < kSums; ++k) handed[k * kTile + row] = acc[k];
        }
        if (KIND == kFwd) { statistics[row] = most; statistics[kTile + row] = sum; }
        if (lane == 0) *any_handed = n >= 3 && !bad;
        __syncwarp();
        if (lane == 0) mbar_arrive(merge);
      } else {
        await(merge, 0, abort_flag, bad);
        float other = last;
        if (KIND == kFwd) {
          const float base = max_of_finite_or(fmaxf(most, statistics[row])), here = exp2_fast(most - base), over_there = exp2_fast(statistics[row] - base);
          sum = sum * here + statistics[kTile + row] * over_there;
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          last = inv * here; other = inv * over_there;
          if (a.stats && there) {
            float* const to = a.stats + 2 * (((int64_t)b * a.H + row_head) * a.Tq + self);
            to[0] = base; to[1] = inv;
          }
        }
        if (*any_handed) {
#pragma unroll
          for (int k = 0; k < kSums; ++k) acc[k] = fmaf(handed[k * kTile + row], other, acc[k] * last);
        } else {
#pragma unroll
          for (int k = 0; k < kSums; ++k) acc[k] *= last;
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < kSums; ++k) acc[k] *= last;
    }
    if (!(kTurns && group == 1) && !*abort_flag) {
      // A warp turns its rows around in the ring, which nothing else uses any more, so that it stores whole lines: rows are 4 floats apart from each other's banks.
      constexpr int kPitch = 64 * G + 4;
      static_assert((kTurns ? kSums * kTile * 4 : 0) + kTile * kPitch * 4 <= kStages * kPart, "rows fit the ring");
      float* const turned = reinterpret_cast<float*>(ring) + (kTurns ? kSums * kTile : 0) + quarter * 32 * kPitch + sum_part;
#pragma unroll
      for (int k = 0; k < kSums; k += 4) *reinterpret_cast<float4*>(turned + lane * kPitch + k) = make_float4(acc[k], acc[k + 1], acc[k + 2], acc[k + 3]);
      __syncwarp();
      float* result = KIND == kFwd ? a.o : KIND == kDq ? a.dq : KIND == kDk ? a.dk : a.dv;
      if (shares > 1) result = (KIND == kDk ? p.dk_part : p.dv_part) + share * ((int64_t)a.B * a.Tk * a.G * a.D);
      const int length = kRowsAreKeys ? a.Tk : a.Tq, first = tile * kTile + quarter * 32, cols = a.D - sum_part;
      const int64_t stride = (int64_t)row_heads * a.D;
      result += ((int64_t)b * length + first) * stride + row_head * a.D + sum_part;
      const bool wide_rows = a.D % 4 == 0 && (reinterpret_cast<uintptr_t>(result) & 15) == 0;
      constexpr int kAcross = kSums / 4;         // lanes of a row
      constexpr int kRowsAtOnce = 32 / kAcross > 0 ? 32 / kAcross : 1;         // rows of a store
      const int k = lane % kAcross * 4, r0 = lane / kAcross;
      if (wide_rows && k < cols) {
#pragma unroll 8
        for (int r = r0; r < 32; r += kRowsAtOnce)
          if (first + r < length) *reinterpret_cast<float4*>(result + r * stride + k) = *reinterpret_cast<const float4*>(turned + r * kPitch + k);
      } else if (k < cols) {
        for (int r = r0; r < 32 && first + r < length; r += kRowsAtOnce)
#pragma unroll
          for (int i = 0; i < 4; ++i) if (k + i < cols) result[r * stride + k + i] = turned[r * kPitch + k + i];
      }
    }
  }

  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
  if (threadIdx.x == 0 && *abort_flag && p.err) atomicExch(p.err, 1);
}

template <int G, bool SHAPED> __global__ void __launch_bounds__(kThreads, 1) attention_tc_fwd_kernel(const __grid_constant__ TcArgs p) { attention_rows<kFwd, G, SHAPED>(p, blockIdx.x); }
// All gradients in one launch, the longest first: dk and dv of the first keys see all queries of all heads that share them.
template <int G, bool SHAPED> __global__ void __launch_bounds__(kThreads, 1) attention_tc_bwd_kernel(const __grid_constant__ TcArgs p, int dk_blocks, int dv_blocks) {
  const int block = blockIdx.x;
  if (block < dk_blocks) attention_rows<kDk, G, SHAPED>(p, block);
  else if (block < dk_blocks + dv_blocks) attention_rows<kDv, G, SHAPED>(p, block - dk_blocks);
  else attention_rows<kDq, G, SHAPED>(p, block - dk_blocks - dv_blocks);
}

// The sums of the shares, in their order; dk (y 0) and dv (y 1).
__global__ void __launch_bounds__(256) attention_add_kernel(const float* __restrict__ dk_part, const float* __restrict__ dv_part, float* dk, float* dv, int64_t n, int shares) {
  grid_dep_sync();
  const float* const part = blockIdx.y ? dv_part : dk_part;
  float* const to = blockIdx.y ? dv : dk;
  if (!to) return;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    float s = 0.f;
#pragma unroll 4
    for (int k = 0; k < shares; ++k) s += __ldg(part + k * n + i);
    to[i] = s;
  }
}

// ---- host side ------------------------------------------------------------------------------------------------------------
template <int G, bool SHAPED> cudaError_t launch_fwd(const TcArgs& p, cudaStream_t s) {
  static std::atomic<uint64_t> ready{0};
  const auto kernel = attention_tc_fwd_kernel<G, SHAPED>;
  const int bytes = Shape<kFwd, G>::kSmem;
  const cudaError_t e = once_per_device(ready, [kernel, bytes] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); });
  return e != cudaSuccess ? e : launch_dep(kernel, dim3((unsigned)(p.a.B * p.a.H * p.q_tiles)), dim3(kThreads), (size_t)bytes, s, p);
}
template <int G, bool SHAPED> cudaError_t launch_bwd(const TcArgs& p, cudaStream_t s) {
  static std::atomic<uint64_t> ready{0};
  const auto kernel = attention_tc_bwd_kernel<G, SHAPED>;
  const int bytes = std::max(std::max(Shape<kDq, G>::kSmem, Shape<kDk, G>::kSmem), Shape<kDv, G>::kSmem);
  const cudaError_t e = once_per_device(ready, [kernel, bytes] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); });
  const int keys = p.a.B * p.a.G * p.shares * p.k_tiles, dk = p.a.dk ? keys : 0, dv = p.a.dv ? keys : 0, dq = p.a.dq ? p.a.B * p.a.H * p.q_tiles : 0;
  return e != cudaSuccess ? e : launch_dep(kernel, dim3((unsigned)(dk + dv + dq)), dim3(kThreads), (size_t)bytes, s, p, dk, dv);
}
template <class F> cudaError_t with_form(const AttentionArgs& a, F&& f) {
  const bool shaped = a.cap > 0.f || a.slopes;
  if (a.D <= 64) return shaped ? f(std::integral_constant<int, 1>(), std::true_type()) : f(std::integral_constant<int, 1>(), std::false_type());
  return shaped ? f(std::integral_constant<int, 2>(), std::true_type()) : f(std::integral_constant<int, 2>(), std::false_type());
}

}  // namespace

// Whether the path takes the call: heads of up to 128 elements, grids that the launch can have
bool attention_tc_takes(const AttentionArgs& a) {
  const int64_t q_tiles = (a.Tq + kTile - 1) / kTile, k_tiles = (a.Tk + kTile - 1) / kTile;
  return a.D <= 128 && a.Tk > 0 && (int64_t)a.B * (2 * a.H * q_tiles + 2 * a.H * k_tiles) < (1ll << 31);
}
// CTAs that the query heads of a key-value head are dealt to in dk and dv.  One, unless the longest CTA would outlast the others: then as few as end that, if what they save (2.5 us a
// tile) is more than adding up their sums takes.  2 x 6 heads over 2, 777 queries: 105 us with one, 49 with three.
static int shares_of(const AttentionArgs& a) {
  const double qt = (a.Tq + kTile - 1) / kTile, kt = (a.Tk + kTile - 1) / kTile, sms = device_sm_count();
  const double total = (double)a.B * a.H * qt * kt * 8 * (a.causal && !a.prefix ? 0.5 : 1.0), nk = (double)a.B * a.Tk * a.G * a.D;
  for (int s = 1; s <= a.group; ++s) {
    if (a.group % s) continue;
    const double longest = 3.0 * (a.group / s) * qt;
    if (longest <= 0.6 * total / sms || s == a.group)
      return (a.group - a.group / s) * qt * 2.5 > 3.0 + nk * 16 * s / 5e6 ? s : 1;
  }
  return 1;
}
// Scratch, in bytes, of a forward or a backward call; with `base`, where its parts lie
static size_t lay_out(const AttentionArgs& a, bool backward, char* base, PackArgs* pack, TcArgs* tc) {
  const int q_tiles = (a.Tq + kTile - 1) / kTile, k_tiles = (a.Tk + kTile - 1) / kTile, g = a.D <= 64 ? 1 : 2;
  const size_t nq = (size_t)a.B * a.H * q_tiles, nk = (size_t)a.B * a.G * k_tiles, image = (size_t)2 * g * 16384;
  size_t at = 0;
  const auto take = [&](size_t bytes) { const size_t from = at; at += (bytes + 255) / 256 * 256; return base ? base + from : nullptr; };
  const int jobs = backward ? 4 : 3;
  // What products are multiplied by to make scores in units of log 2, or of the cap: mantissa (with its sign) and power of two
  const double by = a.cap > 0.f ? (double)a.scale / a.cap : a.scale * 1.4426950408889634;
  int exponent = 0;
  const float mantissa = by == 0.0 ? 1.f : (float)(2.0 * std::frexp(by, &exponent));
  const float* const from[4] = {a.q, a.k, a.v, a.dout};
  Packed* const to[4] = {tc ? &tc->q : nullptr, tc ? &tc->k : nullptr, tc ? &tc->v : nullptr, tc ? &tc->d : nullptr};
  int blocks = 0;
  for (int j = 0; j < jobs; ++j) {
    const bool queries = j == 0 || j == 3;
    const size_t n = queries ? nq : nk;
    char* const img = take(n * image);
    char* const info = take(n * sizeof(TileInfo));
    char* const scale = take(n * kTile * sizeof(float));
    if (base) {
      pack->job[j] = PackJob{from[j], img, (TileInfo*)info, (float*)scale, queries ? a.H : a.G, queries ? a.Tq : a.Tk, queries ? q_tiles : k_tiles, j == 3, j == 0 ? mantissa : 1.f};
      pack->first[j] = blocks;
      *to[j] = Packed{img, (const TileInfo*)info, (const float*)scale};
    }
    blocks += (int)n;
  }
  char* rows[3] = {nullptr, nullptr, nullptr};
  if (backward) for (char*& r : rows) r = take(nq * kTile * sizeof(float));
  const int shares = backward ? shares_of(a) : 1;
  const size_t part = shares > 1 ? (size_t)shares * a.B * a.Tk * a.G * a.D * sizeof(float) : 0;
  char *const dk_part = a.dk && part ? take(part) : nullptr, *const dv_part = a.dv && part ? take(part) : nullptr;
  char* const docs = a.documents ? take((size_t)a.B * k_tiles * sizeof(float4)) : nullptr;
  if (base) {
    pack->a = a; pack->jobs = jobs; pack->first[jobs] = blocks; pack->document_job = 1;
    pack->row_max = (float*)rows[0]; pack->row_delta = (float*)rows[1]; pack->row_norm = (float*)rows[2]; pack->documents = (float4*)docs;
    tc->a = a; tc->row_max = pack->row_max; tc->row_delta = pack->row_delta; tc->row_norm = pack->row_norm; tc->documents = pack->documents;
    tc->q_tiles = q_tiles; tc->k_tiles = k_tiles; tc->D16 = (a.D + 15) / 16 * 16; tc->err = tensor_error_word(); tc->by = by == 0.0 ? 0.f : (float)std::ldexp(1.0, std::min(127, std::max(-126, exponent - 1))); tc->dk_factor = (float)(a.scale / (double)mantissa);
    tc->shares = shares; tc->dk_part = (float*)dk_part; tc->dv_part = (float*)dv_part;
  }
  return at;
}
// 0: launched; -1: error; 1: short of *bytes
int attention_tc(const AttentionArgs& a, bool backward, size_t* bytes, cudaStream_t s, const char* what) {
  TF_REQUIRE(tensor_path_error() == 0, "%s: an earlier tensor-core kernel timed out on a barrier; refusing to launch", what);
  StreamLease lease(s);
  *bytes = lay_out(a, backward, nullptr, nullptr, nullptr);
  char* const base = (char*)lease.scratch(kScratchAttention, *bytes);
  if (!base) return 1;
  PackArgs pack;
  TcArgs tc;
  memset(&pack, 0, sizeof(pack));
  memset(&tc, 0, sizeof(tc));
  lay_out(a, backward, base, &pack, &tc);
  uintptr_t bits = (uintptr_t)a.D * sizeof(float);
  for (const void* x : {(const void*)a.q, (const void*)a.k, (const void*)a.v, (const void*)a.dout, (const void*)a.out}) bits |= reinterpret_cast<uintptr_t>(x);
  const bool wide = bits % 16 == 0;
  const dim3 blocks((unsigned)pack.first[pack.jobs]);
  const auto run_pack = [&](auto g, auto w, auto few) {
    constexpr int G = decltype(g)::value;
    constexpr bool kFew = decltype(few)::value;
    return launch_dep(attention_pack_kernel<G, decltype(w)::value, kFew>, blocks, dim3(pack_threads(G, kFew)), 0, s, pack);
  };
  const auto with_width = [&](auto g, auto few) { return wide ? run_pack(g, std::true_type(), few) : run_pack(g, std::false_type(), few); };
  const auto with_few = [&](auto g) { return (int)blocks.x <= 2 * device_sm_count() ? with_width(g, std::true_type()) : with_width(g, std::false_type()); };
  TF_CUDA(a.D <= 64 ? with_few(std::integral_constant<int, 1>()) : with_few(std::integral_constant<int, 2>()));
  TF_AFTER(s, what);
  TF_CUDA(with_form(a, [&](auto g, auto shaped) { return backward ? launch_bwd<decltype(g)::value, decltype(shaped)::value>(tc, s) : launch_fwd<decltype(g)::value, decltype(shaped)::value>(tc, s); }));
  TF_AFTER(s, what);
  if (tc.shares > 1) {
    const int64_t n = (int64_t)a.B * a.Tk * a.G * a.D;
    TF_CUDA(launch_dep(attention_add_kernel, dim3((unsigned)grid_for(n, 256, 4), 2), dim3(256), 0, s, (const float*)tc.dk_part, (const float*)tc.dv_part, a.dk, a.dv, n, tc.shares));
    TF_AFTER(s, what);
  }
  return 0;
}

}  // namespace tf
