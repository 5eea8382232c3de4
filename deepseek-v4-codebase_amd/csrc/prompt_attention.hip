// Causal attention over whole prompts: packed sequences of different lengths, grouped heads.
//
// Sequence b has queries cu_q[b] .. cu_q[b + 1] and keys cu_k[b] .. cu_k[b + 1]; its i-th query sees its keys
// j <= i + (keys - queries), so that the last query sees every key (a chunk of a prompt comes with the keys before it).
//   out_i = sum_j p_ij v_j,  p_ij = exp(scale q_i . k_j) / (sum exp(scale q_i . k) + exp(sink)),  lse_i = log of that sum.
// A query that sees nothing gives 0 and a log sum of the sink's, or -inf.
//
// Work split.  The G heads of a KV head's group share its keys: the rows of a sequence and KV head are (query, head),
// query-major, and a workgroup takes 32 WR consecutive ones, 32 per wave.  Tiles of 64 keys and values stream through
// two LDS buffers, loaded one tile ahead straight into LDS; with KS = 2 two waves share a row group and take half of every
// tile each, merged at the end.  One pass: running maximum and sum, the output rescaled only where a maximum moved by more
// than kMargin.  The weights are rounded once to the input's 16 bits for their product with V (the sums of weights and of
// products are fp32): bf16 has fp32's range, so every weight keeps its 8 bits; fp16 ends at 2^-24, so its weights are held
// 2^kLift higher, the largest between 2^7 and 2^15, and all down to 2^-21 of the largest are normal numbers (the part of 16384
// keys 17 nats below a dominant one was off by 4 to 44 %, by at most 0.1 % with it).  Few row tiles over many keys take the keys
// in pieces, merged by a second kernel.
//
// Bound by the matrix instructions and the exponentials between them, which two waves of a SIMD (three at dim 64) overlap:
// 16384 tokens, 12 heads of 4, dim 128: 787 to 845 us by box, 980 to 1050 TFLOP/s, where a large bf16 product reaches 1228.  Two
// row groups to a wave read a key for twice the rows but leave one wave to a SIMD, and went through accumulation registers:
// 1494 us.  Short sequences are bound by what comes around the loop (offsets, queries, first tile, output: some 10 us of a
// workgroup that its neighbour on the CU covers in part): 16 of up to 2048, 120 to 126 us, 710 to 740 TFLOP/s.
//
// Matrix layout (v_mfma_f32_32x32x16: A lane l holds A[l % 32][8 (l / 32) + j], B lane l holds B[8 (l / 32) + j][l % 32],
// D lane l register v holds D[8 (v / 4) + 4 (l / 32) + v % 4][l % 32]), h = l / 32:
//   S^T = K Q^T: m = key, n = row; a lane reads 16-byte chunks of its key's row.
//   O^T += V^T P^T: m = dim, n = row, k = key; lane h holds keys 16 c + 4 h + j and 16 c + 8 + 4 h + j of a 16-key chunk c,
//   its own scores, and V^T comes from the row-major tile through the transposing LDS load.
// LDS rows keep their 16-byte chunks XOR-swizzled by their key, so that both reads touch all banks once.
#include "attn_tile.h"

namespace aekv {
namespace {

constexpr int kTile = 64;              // keys of a tile
constexpr int kPieceTiles = 8;         // least tiles of a piece of the keys

struct PromptArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;  // strides in elements
  const int32_t* cu_q;  // [B + 1]
  const int32_t* cu_k;  // [B + 1]
  const float* sink;    // [H] or null
  uint16_t* out;        // [n_q, H, D]
  float* lse;           // [n_q, H] or null
  float* part;          // [n_q, H, n_split, D + 4] where the keys are split: reference, sum (log2 units), 2 pad, output
  int32_t n_split, tiles;
  int32_t n_q, n_k, B, H, heads, G;
  int32_t clear;        // rows in no sequence: 0 to leave out as it is, 1 to write zeros
  int32_t by_work;      // the tiles' order: 0 the sequences', -1 that without gaps, else by work (half of a power of two above
                        // every level)
  uint32_t fold;        // tiles of the launch's second round of workgroups, which are taken from its end; 0: none
  float scale2;         // |softmax scale| * log2(e), not 0 (times a masked product of -inf it stays -inf); where the
  int32_t flip;         // scale is negative the queries' signs are flipped: a row's largest product is its largest logit.  Where
  uint32_t nan;         // it is NaN, 1 stands for it and the queries become NaN (0x7fff is one in both types; else 0): only
                        // what a row sees meets them
};

template <int D>
struct PromptGeom {
  static constexpr int kRow = 2 * D;             // bytes of a tile row
  static constexpr int kChunks = kRow / 16;      // 16-byte chunks of a row
  static constexpr int kTileBytes = kTile * kRow;
};

struct TileAt {
  int32_t q0, lq, k0, lk;  // the sequence's queries and keys
  int32_t row;             // the tile's first row
};

// The workgroup's `t`-th tile (tiles of `rows` rows of G per query, in the sequences' order; a sequence's last rows, which
// see the most keys, come first).  Sequence b, whose rows start at r, has the places from floor(r / rows) + b on: at least
// as many as tiles, and rows / tiles + B in all.  64 sequences are looked at in a memory round, so that up to 64 are searched
// in one round, up to 4096 in two.  False where the place has no tile.
__device__ __forceinline__ bool find_tile(const PromptArgs& a, int32_t t, int rows, int lane, TileAt* at) {
  int32_t lo = 0, hi = a.B;
  for (;;) {
    const int32_t step = (hi - lo + 63) / 64, b = lo + min(step * lane, hi - 1 - lo);
    const int32_t c0 = a.cu_q[b], c1 = a.cu_q[b + 1], d0 = a.cu_k[b], d1 = a.cu_k[b + 1];
    const int32_t q0 = min(max(c0, 0), a.n_q);  // (n_q H, with a tile's rows, fits 31 bits)
    const int32_t place = q0 * a.G / rows;
    const uint64_t from = __builtin_amdgcn_ballot_w64(t - place >= b && step * lane < hi - lo);
    if (!from) return false;  // before the first sequence
    const int l = 63 - __builtin_clzll(from);
    if (step == 1) {
      const int32_t lq = min(max(c1, q0), a.n_q) - q0;
      const int32_t k0 = min(max(d0, 0), a.n_k), lk = min(max(d1, k0), a.n_k) - k0;
      const int32_t tiles = (lq * a.G + rows - 1) / rows, left = tiles - 1 - (t - place - b);
      at->q0 = __builtin_amdgcn_readlane(q0, l);
      at->lq = __builtin_amdgcn_readlane(lq, l);
      at->k0 = __builtin_amdgcn_readlane(k0, l);
      at->lk = __builtin_amdgcn_readlane(lk, l);
      at->row = __builtin_amdgcn_readlane(left, l) * rows;
      return at->row >= 0;
    }
    lo += l * step;
    hi = min(lo + step, hi);
  }
}

// The same of up to 64 sequences with every place before the last tile's taken: where the workgroups about fill the chip,
// places without a tile among them leave some parts of it with more than fits, and a second round.
__device__ __forceinline__ bool find_tile_dense(const PromptArgs& a, int32_t t, int rows, int lane, TileAt* at) {
  const int32_t b = min(lane, a.B - 1);
  const int32_t c0 = a.cu_q[b], c1 = a.cu_q[b + 1], d0 = a.cu_k[b], d1 = a.cu_k[b + 1];
  const int32_t q0 = min(max(c0, 0), a.n_q), lq = min(max(c1, q0), a.n_q) - q0;
  const int32_t k0 = min(max(d0, 0), a.n_k), lk = min(max(d1, k0), a.n_k) - k0;
  const int32_t tiles = lane < a.B ? (lq * a.G + rows - 1) / rows : 0;
  int32_t s = tiles;  // inclusive sum over the lanes
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int32_t o = __shfl_up(s, d);
    if (lane >= d) s += o;
  }
  const uint64_t mine = __builtin_amdgcn_ballot_w64(s > t && s - tiles <= t);
  if (!mine) return false;
  const int l = __builtin_ctzll(mine);
  at->q0 = __builtin_amdgcn_readlane(q0, l);
  at->lq = __builtin_amdgcn_readlane(lq, l);
  at->k0 = __builtin_amdgcn_readlane(k0, l);
  at->lk = __builtin_amdgcn_readlane(lk, l);
  at->row = (__builtin_amdgcn_readlane(s, l) - 1 - t) * rows;
  return true;
}

__device__ __forceinline__ int32_t lane_sum(int32_t v) {
  auto step = [&](auto hl) { v += __builtin_bit_cast(int32_t, xor_lane<decltype(hl)::value>(__builtin_bit_cast(float, v))); };
  step(std::integral_constant<int, 1>{}), step(std::integral_constant<int, 2>{}), step(std::integral_constant<int, 4>{});
  step(std::integral_constant<int, 8>{}), step(std::integral_constant<int, 16>{}), step(std::integral_constant<int, 32>{});
  return v;
}

// The same of up to 64 sequences by the tiles' work, the most keys first: a sequence's tiles have the levels `from` ..
// from + its tiles, a level being the keys that one tile of rows adds, and the t-th of all is found by halving over levels.
// It shortens the launch's end, where the longest tiles of the last sequence would run alone, and costs the keys' locality:
// all sequences' keys are in use at once.
__device__ __forceinline__ bool find_tile_by_work(const PromptArgs& a, int32_t t, int rows, int lane, TileAt* at) {
  const int32_t b = min(lane, a.B - 1);
  const int32_t c0 = a.cu_q[b], c1 = a.cu_q[b + 1], d0 = a.cu_k[b], d1 = a.cu_k[b + 1];
  const int32_t q0 = min(max(c0, 0), a.n_q), lq = min(max(c1, q0), a.n_q) - q0;
  const int32_t k0 = min(max(d0, 0), a.n_k), lk = min(max(d1, k0), a.n_k) - k0;
  const int32_t tiles = lane < a.B ? (lq * a.G + rows - 1) / rows : 0;
  const int64_t ahead = static_cast<int64_t>(max(lk - lq, 0)) * a.G / rows;
  const int32_t from = static_cast<int32_t>(ahead < (1 << 25) ? ahead : 1 << 25);
  auto at_least = [&](int32_t level) { return min(max(from + tiles - level, 0), tiles); };  // own tiles of that level or more
  if (lane_sum(tiles) <= t) return false;
  int32_t level = 0;  // the highest with more than t tiles at or above it
#pragma unroll 1
  for (int32_t bit = a.by_work; bit > 0; bit >>= 1)
    if (lane_sum(at_least(level + bit)) > t) level += bit;
  const int32_t above = lane_sum(at_least(level + 1));
  uint64_t with = __builtin_amdgcn_ballot_w64(at_least(level) > at_least(level + 1));  // sequences with a tile of it
  for (int32_t i = above; i < t && with; ++i) with &= with - 1;
  if (!with) return false;  // (offsets that are no prefix sums)
  const int l = __builtin_ctzll(with);
  at->q0 = __builtin_amdgcn_readlane(q0, l);
  at->lq = __builtin_amdgcn_readlane(lq, l);
  at->k0 = __builtin_amdgcn_readlane(k0, l);
  at->lk = __builtin_amdgcn_readlane(lk, l);
  at->row = (level - __builtin_amdgcn_readlane(from, l)) * rows;
  return true;
}

template <int DT, int D, int WR, int KS>
__global__ __launch_bounds__(64 * WR * KS) __attribute__((amdgpu_waves_per_eu(D == 64 ? 3 : 2))) void prompt_attention_kernel(PromptArgs a) {
  using E = Elem<DT>;
  using Gm = PromptGeom<D>;
  using v8 = typename E::v8;
  constexpr int kWaves = WR * KS, kRows = 32 * WR, kRow = Gm::kRow;
  constexpr int kKB = 2 / KS;                              // 32-key blocks of a tile per wave
  constexpr int kPass = 1024 * kWaves;                     // bytes that the workgroup stages at a time
  constexpr int kPasses = Gm::kTileBytes / kPass;
  constexpr int kMB = D / 32, kKSteps = D / 16;
  static_assert(KS == 1 || KS == 2, "a tile is two 32-key blocks");
  static_assert(Gm::kTileBytes % kPass == 0 && kPass % kRow == 0, "whole rows per pass");
  // [buffer][K, V][key][swizzled chunks]: separate arrays, so that the compiler sees that loads into one buffer do not
  // write what is read from the other
  __shared__ __align__(16) uint8_t L0[2 * Gm::kTileBytes];
  __shared__ __align__(16) uint8_t L1[2 * Gm::kTileBytes];
  __shared__ uint16_t s_p[kWaves][32][32];  // a block's weights by key and row (values that are no numbers)

  const int lane = threadIdx.x & 63, rl = lane & 31, hh = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wv % WR, kh = wv / WR;
  // workgroups: KV heads innermost, then row tiles, then pieces of the keys
  const int32_t head = static_cast<int32_t>(blockIdx.x % a.heads);
  uint32_t index = blockIdx.x / a.heads;
  int32_t split = 0;
  if (a.n_split > 1) {
    split = static_cast<int32_t>(index / a.tiles);
    index -= split * a.tiles;
  } else if (index >= a.fold && index < 2 * a.fold) {  // (tiles >= 2 fold)
    index = 3 * a.fold - 1 - index;
  }
  TileAt at;
  const bool found = a.by_work > 0   ? find_tile_by_work(a, static_cast<int32_t>(index), kRows, lane, &at)
                     : a.by_work < 0 ? find_tile_dense(a, static_cast<int32_t>(index), kRows, lane, &at)
                                     : find_tile(a, static_cast<int32_t>(index), kRows, lane, &at);
  if (a.clear || a.lse) {  // rows in no sequence: shared out over the workgroups
    const int32_t s0 = min(max(a.cu_q[0], 0), a.n_q), s1 = min(max(a.cu_q[a.B], s0), a.n_q);
    const int64_t words = static_cast<int64_t>(s0 + a.n_q - s1) * a.H * (D / 2);
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * (64 * kWaves) + threadIdx.x; i < words; i += static_cast<int64_t>(gridDim.x) * (64 * kWaves)) {
      const int64_t r = i / (D / 2), row = r < static_cast<int64_t>(s0) * a.H ? r : r + static_cast<int64_t>(s1 - s0) * a.H;
      if (a.clear) reinterpret_cast<uint32_t*>(a.out)[row * (D / 2) + i % (D / 2)] = 0;
      if (a.lse && i % (D / 2) == 0) a.lse[row] = kNegInf;
    }
  }
  if (!found) return;  // (the whole workgroup)
  const int32_t q0 = at.q0, lq = at.lq, k0 = at.k0, lk = at.lk, row0 = at.row;
  const int32_t n_rows = lq * a.G;
  auto sees_of = [&](int32_t row) {  // keys that a row sees
    const int64_t s = static_cast<int64_t>(row / a.G) + 1 + lk - lq;
    return static_cast<int32_t>(s < 0 ? 0 : s > lk ? lk : s);
  };
  const int32_t last_row = (row0 + kRows < n_rows ? row0 + kRows : n_rows) - 1;
  const int32_t n_keys = __builtin_amdgcn_readfirstlane(sees_of(last_row));
  const int all_tiles = (n_keys + kTile - 1) / kTile;
  int first_tile = 0, n_tiles = all_tiles;
  if (a.n_split > 1) {
    const int per_piece = max((all_tiles + a.n_split - 1) / a.n_split, kPieceTiles);
    first_tile = min(split * per_piece, all_tiles), n_tiles = min(first_tile + per_piece, all_tiles);
  }

  // rows past the last are computed as copies of it
  const int32_t w0 = row0 + 32 * wr;  // the wave's first row
  v8 qb[kKSteps];
  const int32_t row = w0 + rl, own = row < n_rows ? row : n_rows - 1;
  const int32_t sees = sees_of(own), qi = own / a.G, h = head * a.G + (own - qi * a.G);
  const uint16_t* qp = a.q + static_cast<int64_t>(q0 + qi) * a.q_token + h * a.q_head + 8 * hh;
#pragma unroll
  for (int ks = 0; ks < kKSteps; ++ks) {
    uint4 w = *reinterpret_cast<const uint4*>(qp + 16 * ks);
    if (a.flip) w.x ^= 0x80008000u, w.y ^= 0x80008000u, w.z ^= 0x80008000u, w.w ^= 0x80008000u;
    if (a.nan) w.x |= a.nan, w.y |= a.nan, w.z |= a.nan, w.w |= a.nan;
    qb[ks] = __builtin_bit_cast(v8, w);
  }
  const int32_t wave_least = __builtin_amdgcn_readfirstlane(sees_of(w0 < n_rows ? w0 : n_rows - 1));
  const int32_t wl = w0 + 31;
  const int32_t wave_most = __builtin_amdgcn_readfirstlane(sees_of(wl < n_rows ? wl : n_rows - 1));

  // staging: pass c of wave wv writes bytes [kPass c + 1024 wv, + 1024) of a tile, lane l at + 16 l, so lane l loads the
  // chunk that the swizzle puts there.  A pass is a multiple of 16 rows or half of one, so the swizzle repeats.
  const int lin = 1024 * wv + 16 * lane;
  const int key_in = lin / kRow, place = (lin % kRow) / 16;
  static_assert(kPass / kRow % 8 == 0, "the swizzle repeats after two passes");
  int koff[2], voff[2];
  const int k_stride = static_cast<int>(a.k_token) * 2, v_stride = static_cast<int>(a.v_token) * 2;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int c = place ^ swizzle<D>((kPass / kRow * p + key_in) & 15);
    koff[p] = key_in * k_stride + 16 * c;
    voff[p] = key_in * v_stride + 16 * c;
  }
  const uint8_t* kbase = reinterpret_cast<const uint8_t*>(a.k + k0 * a.k_token + head * a.k_head);
  const uint8_t* vbase = reinterpret_cast<const uint8_t*>(a.v + k0 * a.v_token + head * a.v_head);
  // Tile `it`, read through buffer resources whose range ends at the sequence's last key that the workgroup sees: rows
  // past it are zero and touch no memory; past the last tile the range is empty.
  auto load_tile = [&, n_keys, k_stride, v_stride, kbase, vbase](int it, auto buf_c) __attribute__((always_inline)) {
    uint8_t* const dst = decltype(buf_c)::value ? L1 : L0;
    const int left = n_keys - it * kTile, n = left < 0 ? 0 : left < kTile ? left : kTile;
    const int64_t base = n > 0 ? static_cast<int64_t>(it) * kTile : 0;
    const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(kbase + base * k_stride), 0, n > 0 ? (n - 1) * k_stride + kRow : 0, kBufWord3);
    const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(vbase + base * v_stride), 0, n > 0 ? (n - 1) * v_stride + kRow : 0, kBufWord3);
#pragma unroll
    for (int c = 0; c < kPasses; ++c)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(kr, (lds_void_t*)(dst + kPass * c + 1024 * wv), 16, koff[c & 1], kPass / kRow * c * k_stride, 0, 0);
#pragma unroll
    for (int c = 0; c < kPasses; ++c)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(vr, (lds_void_t*)(dst + Gm::kTileBytes + kPass * c + 1024 * wv), 16, voff[c & 1], kPass / kRow * c * v_stride, 0, 0);
  };

  // LDS byte offsets.  Row-chunk reads (K): key 32 kb + rl, chunk (2 ks + hh) ^ swizzle(rl): sA ^ 32 ks.  Transposing reads
  // (V, 16-lane group G = lane / 16, s = lane % 16): key 16 c + 8 e + 4 hh + s / 4, dims 32 mb + 16 (G % 2) + 4 (s % 4) ..,
  // i.e. chunk 4 mb + x with x = 2 (G % 2) + (s % 4) / 2, xor the swizzle of the key.
  const int sA = (32 * kKB * kh + rl) * kRow + ((hh ^ swizzle<D>(rl & 15)) << 4);
  int tA[2];
  {
    const int s16 = lane & 15, x = 2 * ((lane >> 4) & 1) + ((s16 & 3) >> 1);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int key = 8 * e + 4 * hh + (s16 >> 2);
      tA[e] = (32 * kKB * kh + key) * kRow + ((x ^ swizzle<D>(key)) << 4) + ((s16 & 1) << 3);
    }
  }

  float m = kNegInf, l = 0.0f;  // the reference that weights are relative to (a maximum less kLift), their sum
  f32x16_t O[kMB];
#pragma unroll
  for (int mb = 0; mb < kMB; ++mb) O[mb] = f32x16_t{};

  // one tile; `masked`: some row of the wave does not see all of it
  auto tile = [&](int it, const uint8_t* kt, auto masked_c) __attribute__((always_inline)) {
    constexpr bool masked = decltype(masked_c)::value;
    const uint8_t* vt = kt + Gm::kTileBytes;
    const int base = it * kTile + 32 * kKB * kh;
    f32x16_t s[kKB];
    float top = kNegInf;
#pragma unroll
    for (int kb = 0; kb < kKB; ++kb) {
      s[kb] = f32x16_t{};
#pragma unroll
      for (int ks = 0; ks < kKSteps; ++ks) {
        const v8 ka = __builtin_bit_cast(v8, *reinterpret_cast<const uint4*>(kt + 32 * kRow * kb + (sA ^ (ks << 5))));
        s[kb] = E::mma(ka, qb[ks], s[kb]);
      }
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        if constexpr (masked) {
          const int key = base + 32 * kb + 8 * (v >> 2) + 4 * hh + (v & 3);
          s[kb][v] = key < sees ? s[kb][v] : kNegInf;
        }
        top = fmaxf(top, s[kb][v]);
      }
    }
    top = fmaxf(top, xor_lane<32>(top)) * a.scale2;
    // (each row by itself: a row's bits do not depend on the others'; the difference, as m and a constant may round up)
    const bool moved = top - m > kMargin + E::kLift;
    if (__builtin_amdgcn_ballot_w64(moved)) {
      const float to = top - E::kLift, r = moved ? __builtin_amdgcn_exp2f(m - to) : 1.0f;
      l *= r;
#pragma unroll
      for (int mb = 0; mb < kMB; ++mb) O[mb] *= r;
      m = moved ? to : m;
    }
    float nm = m == kNegInf ? 0.0f : -m, by = a.scale2;
    // beyond kFar the reference, which is a rounded logit, may lie further from the exact product than the exponentials reach:
    // there a row's logits are all rounded as the reference was
    const bool far = fabsf(m) > kFar && m > kNegInf;
    if (__builtin_amdgcn_ballot_w64(far)) {
#pragma unroll
      for (int kb = 0; kb < kKB; ++kb)
#pragma unroll
        for (int v = 0; v < 16; ++v) s[kb][v] = far ? s[kb][v] * a.scale2 + nm : s[kb][v];
      by = far ? 1.0f : by, nm = far ? 0.0f : nm;
    }
#pragma unroll
    for (int kb = 0; kb < kKB; ++kb) {
      float p[16];
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        p[v] = __builtin_amdgcn_exp2f(fmaf(s[kb][v], by, nm));
        l += p[v];
      }
      v8 pb[2];
#pragma unroll
      for (int c = 0; c < 2; ++c)
        pb[c] = __builtin_bit_cast(v8, make_uint4(E::pack(p[8 * c], p[8 * c + 1]), E::pack(p[8 * c + 2], p[8 * c + 3]),
                                                  E::pack(p[8 * c + 4], p[8 * c + 5]), E::pack(p[8 * c + 6], p[8 * c + 7])));
      u32x4_t w[2][kMB];
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int mb = 0; mb < kMB; ++mb) {
          const uint8_t* vc = vt + (32 * kb + 16 * c) * kRow;
          const i16x4_t lo = read_tr16(vc + (tA[0] ^ (mb << 6))), hi = read_tr16(vc + (tA[1] ^ (mb << 6)));
          w[c][mb] = __builtin_bit_cast(u32x4_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
      bool odd = false;
      if constexpr (masked) {
        // a value that is no finite number must not reach rows that do not see it (0 times it is no 0): it goes in as 0,
        // and is added below to the rows that do
        u16x2_t most = {0, 0};
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int mb = 0; mb < kMB; ++mb)
#pragma unroll
            for (int i = 0; i < 4; ++i) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2_t, w[c][mb][i] & 0x7FFF7FFFu));
        odd = __builtin_amdgcn_ballot_w64(most[0] >= E::kExp || most[1] >= E::kExp);
        if (odd) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int mb = 0; mb < kMB; ++mb)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint32_t u = w[c][mb][i];
                w[c][mb][i] = ((u & 0x7FFFu) >= E::kExp ? 0u : u & 0xFFFFu) | (((u >> 16) & 0x7FFFu) >= E::kExp ? 0u : u & 0xFFFF0000u);
              }
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int mb = 0; mb < kMB; ++mb) O[mb] = E::mma(__builtin_bit_cast(v8, w[c][mb]), pb[c], O[mb]);
      if constexpr (masked) {
        if (odd) {
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int c = 0; c < 2; ++c) {  // element j of lane half h is key 16 c + 4 h + j, or 16 c + 8 + 4 h + j - 4
            const u32x4_t u = __builtin_bit_cast(u32x4_t, pb[c]);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              s_p[wv][16 * c + 8 * (j >> 2) + 4 * hh + (j & 3)][rl] = static_cast<uint16_t>(u[j >> 1] >> (16 * (j & 1)));
          }
          __builtin_amdgcn_wave_barrier();
#pragma unroll 1
          for (int key = 0; key < 32; ++key) {
            const float pk = E::value(s_p[wv][key][rl]);
            const bool in = base + 32 * kb + key < sees;
            const int kr = 32 * kKB * kh + 32 * kb + key;
#pragma unroll
            for (int mb = 0; mb < kMB; ++mb)
#pragma unroll
              for (int v = 0; v < 16; ++v) {
                const int d = 32 * mb + 8 * (v >> 2) + 4 * hh + (v & 3);
                const uint32_t x = *reinterpret_cast<const uint16_t*>(vt + kr * kRow + (((d >> 3) ^ swizzle<D>(kr & 15)) << 4) + 2 * (d & 7));
                if (in && (x & 0x7FFFu) >= E::kExp) O[mb][v] += pk * E::value(x);
              }
          }
        }
      }
    }
  };
  auto step = [&](int it, auto buf_c) __attribute__((always_inline)) {
    constexpr int buf = decltype(buf_c)::value;
    __builtin_amdgcn_s_waitcnt(0);  // this wave's part of tile `it` has landed (the compiler does not track these loads)
    __syncthreads();                // every wave's, and the other buffer's readers are done
    if (it + 1 < n_tiles) load_tile(it + 1, std::integral_constant<int, buf ^ 1>{});
    const uint8_t* kt = buf ? L1 : L0;
    const int end = (it + 1) * kTile;
    if (end <= wave_least) tile(it, kt, std::false_type{});
    else if (it * kTile < wave_most) tile(it, kt, std::true_type{});
  };
  if (first_tile < n_tiles) load_tile(first_tile, std::integral_constant<int, 0>{});
#pragma unroll 1
  for (int it = first_tile; it < n_tiles; it += 2) {
    step(it, std::integral_constant<int, 0>{});
    if (it + 1 < n_tiles) step(it + 1, std::integral_constant<int, 1>{});
  }
  l += xor_lane<32>(l);  // both halves' keys

  if constexpr (KS == 2) {  // the second key half's states into the first's, through the tile buffers
    static_assert(WR * kMB * 16 * 64 * 4 + WR * 2 * 64 * 4 <= 4 * Gm::kTileBytes, "the states fit both buffers");
    __syncthreads();
    constexpr int kPer = kMB * 16 * 64, kFit = 2 * Gm::kTileBytes / 4;  // floats
    auto slot = [&](int i) -> float* { return i < kFit ? reinterpret_cast<float*>(L0) + i : reinterpret_cast<float*>(L1) + (i - kFit); };
    static_assert(kFit % 64 == 0, "a run of 64 floats lies in one buffer");
    const int at = wr * (kPer + 128);
    if (kh == 1) {
#pragma unroll
      for (int mb = 0; mb < kMB; ++mb)
#pragma unroll
        for (int v = 0; v < 16; ++v) slot(at + (mb * 16 + v) * 64)[lane] = O[mb][v];
      slot(at + kPer)[lane] = m;
      slot(at + kPer + 64)[lane] = l;
    }
    __syncthreads();
    if (kh == 1) return;
    const float m1 = slot(at + kPer)[lane], l1 = slot(at + kPer + 64)[lane];
    const float up = fmaxf(m, m1);
    // (a state of nothing has a sum of 0; NaN alone leaves a maximum of -inf, and a sum that says so)
    const float f0 = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - up), f1 = l1 == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m1 - up);
    l = (l == 0.0f ? 0.0f : l * f0) + (l1 == 0.0f ? 0.0f : l1 * f1);
    m = up;
#pragma unroll
    for (int mb = 0; mb < kMB; ++mb)
#pragma unroll
      for (int v = 0; v < 16; ++v) O[mb][v] = O[mb][v] * f0 + slot(at + (mb * 16 + v) * 64)[lane] * f1;
  }
  const int64_t orow = static_cast<int64_t>(q0 + qi) * a.H + h;
  if (a.n_split > 1) {
    if (row >= n_rows) return;
    float* p = a.part + (orow * a.n_split + split) * (D + 4);
    if (hh == 0) *reinterpret_cast<float2*>(p) = make_float2(m, l);
    if (first_tile < n_tiles) {  // (an empty piece's sum of 0 says that it has no output)
#pragma unroll
      for (int mb = 0; mb < kMB; ++mb)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<float4*>(p + 4 + 32 * mb + 8 * i + 4 * hh) = make_float4(O[mb][4 * i], O[mb][4 * i + 1], O[mb][4 * i + 2], O[mb][4 * i + 3]);
    }
    return;
  }
  const float sk = a.sink ? a.sink[h] * kLog2e : kNegInf;
  const float up = fmaxf(m, sk);
  const float f = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - up);
  const float sum = (l == 0.0f ? 0.0f : l * f) + (sk == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(sk - up));
  const float r = sum == 0.0f ? 0.0f : f / sum;
  if (a.lse && hh == 0 && row < n_rows) a.lse[orow] = sum == 0.0f ? kNegInf : (up + __builtin_amdgcn_logf(sum)) * kLn2;
  if constexpr (KS == 1) {
    // a lane holds 8-byte pieces of its row: the wave's rows go through LDS, their 16-byte chunks swizzled, so that a store
    // writes whole rows and passes by the caches, which keep the keys (64 prompts of 1024, 12 heads of 4: 354 -> 346 us)
    constexpr int kLanes = kRow / 16;  // of a row
    static_assert(kWaves * 32 * kRow <= 2 * Gm::kTileBytes, "the rows fit a buffer");
    uint8_t* const w = L0 + wv * 32 * kRow;
    __syncthreads();  // the last tile's readers are done
#pragma unroll
    for (int mb = 0; mb < kMB; ++mb)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<uint2*>(w + rl * kRow + (((4 * mb + i) ^ (rl % kLanes)) << 4) + 8 * hh) =
            make_uint2(E::pack(O[mb][4 * i] * r, O[mb][4 * i + 1] * r), E::pack(O[mb][4 * i + 2] * r, O[mb][4 * i + 3] * r));
    __builtin_amdgcn_wave_barrier();
    const int c = lane % kLanes;
#pragma unroll
    for (int i = 0; i < 32; i += 64 / kLanes) {
      const int wr_row = i + lane / kLanes, at_row = w0 + wr_row;
      if (at_row >= n_rows) continue;
      const int32_t qn = at_row / a.G, hn = head * a.G + (at_row - qn * a.G);
      __builtin_nontemporal_store(*reinterpret_cast<const u32x4_t*>(w + wr_row * kRow + ((c ^ (wr_row % kLanes)) << 4)),
                                  reinterpret_cast<u32x4_t*>(a.out + (static_cast<int64_t>(q0 + qn) * a.H + hn) * D + 8 * c));
    }
  } else {
    if (row >= n_rows) return;
    uint16_t* op = a.out + orow * D + 4 * hh;
#pragma unroll
    for (int mb = 0; mb < kMB; ++mb)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<uint2*>(op + 32 * mb + 8 * i) = make_uint2(E::pack(O[mb][4 * i] * r, O[mb][4 * i + 1] * r),
                                                                     E::pack(O[mb][4 * i + 2] * r, O[mb][4 * i + 3] * r));
  }
}

// Merges the pieces of the rows: D / 4 lanes hold a row, 4 dims each.  Bound by the chain of its loads, so that they go out
// together: 64 queries over 8192 keys, 16 heads of 2, dim 64, 16 pieces: the call 17.2 us, one piece after another 23.4; 11744
// rows of 2 pieces, 6 MB, 4 us.
template <int DT, int D>
__global__ __launch_bounds__(256) void prompt_merge_kernel(PromptArgs a) {
  using E = Elem<DT>;
  constexpr int PER = D / 4;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / PER) + threadIdx.x / PER;
  if (row >= static_cast<int64_t>(a.n_q) * a.H) return;
  const int32_t n = static_cast<int32_t>(row / a.H), h = static_cast<int32_t>(row - static_cast<int64_t>(n) * a.H);
  const int j = threadIdx.x % PER;
  const float* p = a.part + row * a.n_split * (D + 4);
  const int32_t c0 = a.cu_q[0], c1 = a.cu_q[a.B];
  const float sk = a.sink ? a.sink[h] * kLog2e : kNegInf;
  float top = sk, sum = sk == kNegInf ? 0.0f : 1.0f;
  float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  // CH pieces at a time, all their loads issued together (a piece past the last reads the last, and counts as empty)
  auto merge = [&](auto ch) __attribute__((always_inline)) {
    constexpr int CH = decltype(ch)::value;
    for (int s0 = 0; s0 < a.n_split; s0 += CH) {
      float2 ml[CH];
      float4 o[CH];
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const float* ps = p + min(s0 + c, a.n_split - 1) * (D + 4);
        ml[c] = *reinterpret_cast<const float2*>(ps);
        o[c] = *reinterpret_cast<const float4*>(ps + 4 + 4 * j);
      }
      float up = top;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        if (s0 + c >= a.n_split || ml[c].y == 0.0f) ml[c] = make_float2(kNegInf, 0.0f), o[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);  // (nothing seen)
        up = fmaxf(up, ml[c].x);
      }
      const float r = sum == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(top - up);
      sum = sum == 0.0f ? 0.0f : sum * r;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] *= r;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const float f = ml[c].y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml[c].x - up);
        sum += ml[c].y == 0.0f ? 0.0f : ml[c].y * f;
        x[0] = fmaf(o[c].x, f, x[0]), x[1] = fmaf(o[c].y, f, x[1]), x[2] = fmaf(o[c].z, f, x[2]), x[3] = fmaf(o[c].w, f, x[3]);
      }
      top = up;
    }
  };
  if (a.n_split <= 2) merge(std::integral_constant<int, 2>{});
  else merge(std::integral_constant<int, 4>{});
  if (n < c0 || n >= c1) return;  // in no sequence
  const float r = sum == 0.0f ? 0.0f : 1.0f / sum;
  *reinterpret_cast<uint2*>(a.out + row * D + 4 * j) = make_uint2(E::pack(x[0] * r, x[1] * r), E::pack(x[2] * r, x[3] * r));
  if (a.lse && j == 0) a.lse[row] = sum == 0.0f ? kNegInf : (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

using prompt_fn = void (*)(PromptArgs);
template <int WR, int KS>
prompt_fn pick_prompt(int32_t dtype, int32_t d) {
  if (dtype == AEKV_F16) return d == 64 ? prompt_attention_kernel<AEKV_F16, 64, WR, KS> : prompt_attention_kernel<AEKV_F16, 128, WR, KS>;
  return d == 64 ? prompt_attention_kernel<AEKV_BF16, 64, WR, KS> : prompt_attention_kernel<AEKV_BF16, 128, WR, KS>;
}

// How a launch is cut: rows of a workgroup, and pieces of the keys where the row tiles alone leave CUs without a workgroup
// (as many as are resident together: three of a CU at head dim 64, two at 128).
//
// 128 rows to a workgroup read a tile of keys once for twice the rows; 64 give twice the workgroups.  128 where they fill the
// chip; of several sequences with tiles of like work also where they about fill it and (as if all were as long) run together;
// and in at least two pieces of enough work to pay for the pieces' merge.  64 / 128 rows, dim 128:
// 8 x 512 queries over 4096 keys, 16 heads of 2, 512 tiles 194 / 142 us; 10 x 512 over their own, 12 heads of 4, 480 27.7 /
// 20.6; 5 x 512 over 4096, 16 of 2, 320 131 / 122; below: 7 x 384 over 1024, 12 of 4, 252 27.3 / 27.6; above: 15 x 320 over
// 2112, 12 of 12, 540 98 / 110; tiles of different work: 2 x 2048 over their own, 12 of 4, 384 46 / 51, one of 4096 71 / 74.
// In pieces, 12 heads of 4: 1024 queries over 8192 keys (the least) 81 / 69, over 32768 287 / 225, 512 over 8192 46 / 48; 16
// heads of 16, 2048 over 8192 (one piece of 128) 149 / 160.
//
// Pieces have to save a row the time of some kPieceTiles tiles, which is what their merge costs: 16 heads of 2, dim 64, whole / in
// pieces: 1024 queries over their own keys 14.0 / 18.6 us, 1500 18.7 / 23.6, 64 queries over 2048 keys 22.3 / 11.6, 16 over
// 1024 13.6 / 10.9.
struct PromptPlan {
  int64_t rows, tiles, split;
};
constexpr int64_t kWideWork = int64_t(3) << 25;  // rows x keys of a sequence
PromptPlan plan_prompt(int64_t B, int64_t n_q, int64_t n_k, int64_t H, int64_t heads, int32_t d) {
  PromptPlan p;
  const int64_t rows = n_q * (H / heads), resident = d == 64 ? 768 : 512;
  const int64_t groups = heads * (rows / 128);
  const bool alike = B > 1 && (2 * n_q <= n_k || n_q / B <= 1024);  // tiles of like work
  const int64_t each = rows / B, tiles = heads * B * ceil_div(each - each / 64, static_cast<int64_t>(128));  // (a buffer's end may be unused)
  const bool wide = groups >= 512 || (alike && groups >= (d == 64 ? 400 : 300) && tiles <= resident) || (n_q * H * (n_k / B) >= kWideWork && 2 * heads * (rows / 128 + B) <= resident);
  p.rows = wide ? 128 : 64;
  p.tiles = rows / p.rows + B;  // at least every sequence's, whatever their lengths
  const int64_t sees = (n_q < n_k ? n_k - n_q / 2 : n_k / 2) / B, piece = kTile * kPieceTiles;  // keys of a row, on average
  const int64_t room = resident / (p.tiles * heads), most = ceil_div(sees, piece);
  p.split = room < most ? room : most;
  if (p.split < 1 || 8 * sees * (p.split - 1) < 7 * piece * p.split) p.split = 1;
  return p;
}

}  // namespace
}  // namespace aekv

using namespace aekv;

extern "C" size_t aekv_prompt_attention_workspace_size(int64_t B, int64_t n_q, int64_t n_k, int64_t H, int64_t heads,
                                                       int32_t d) {
  if (B <= 0 || n_q <= 0 || n_k <= 0 || H <= 0 || heads <= 0 || d <= 0 || H % heads) return 0;
  if (n_q > 0x7fffffff || n_k > 0x7fffffff || B > 0x7ffffffe || H > 65535 || n_q * H > 0x7fff0000) return 0;  // (the call refuses it)
  const PromptPlan p = plan_prompt(B, n_q, n_k, H, heads, d);
  return p.split > 1 ? static_cast<size_t>(n_q * H) * static_cast<size_t>(p.split) * (d + 4) * 4 : 0;
}

extern "C" int aekv_prompt_attention(const void* q, const void* k, const void* v, int32_t dtype, int64_t q_token_stride,
                                     int64_t q_head_stride, int64_t k_token_stride, int64_t k_head_stride,
                                     int64_t v_token_stride, int64_t v_head_stride, const int32_t* cu_seqlens_q,
                                     const int32_t* cu_seqlens_k, int64_t B, int64_t n_q, int64_t n_k, int64_t H,
                                     int64_t heads, int32_t d, const float* sink, float softmax_scale, void* out,
                                     float* lse, int32_t clear_rest, void* ws, size_t ws_bytes, void* stream) {
  const char* who = "aekv_prompt_attention";
  if (dtype != AEKV_F16 && dtype != AEKV_BF16) return fail(AEKV_ERR_DTYPE, "%s: q, k and v must be F16 or BF16", who);
  if (d != 64 && d != 128) return fail(AEKV_ERR_UNSUPPORTED, "%s: head dim %d (64 or 128 supported)", who, d);
  if (B < 0 || n_q < 0 || n_k < 0 || heads < 1 || H < 1 || H % heads)
    return fail(AEKV_ERR_SHAPE, "%s: B=%lld n_q=%lld n_k=%lld, and %lld query heads are no multiple of %lld KV heads", who,
                (long long)B, (long long)n_q, (long long)n_k, (long long)H, (long long)heads);
  if (n_q == 0) return AEKV_OK;
  if (!q || !out || (B > 0 && (!cu_seqlens_q || !cu_seqlens_k)) || (n_k > 0 && (!k || !v)))
    return fail(AEKV_ERR_VALUE, "%s: null pointer", who);
  if (B == 0) return fail(AEKV_ERR_SHAPE, "%s: %lld queries in no sequence", who, (long long)n_q);
  if (!is_aligned(q, 16) || !is_aligned(k, 16) || !is_aligned(v, 16) || !is_aligned(out, 16) || (q_token_stride % 8) ||
      (q_head_stride % 8) || (k_token_stride % 8) || (k_head_stride % 8) || (v_token_stride % 8) || (v_head_stride % 8))
    return fail(AEKV_ERR_ALIGN, "%s: q, k and v rows and out must be 16-byte aligned", who);
  if (n_q > 0x7fffffff || n_k > 0x7fffffff || B > 0x7ffffffe || H > 65535 || n_q * H > 0x7fff0000)
    return fail(AEKV_ERR_UNSUPPORTED, "%s: B=%lld n_q=%lld n_k=%lld H=%lld exceed the grid", who, (long long)B,
                (long long)n_q, (long long)n_k, (long long)H);
  if (k_token_stride * 2 * kTile > 0x3fffffff || v_token_stride * 2 * kTile > 0x3fffffff || k_token_stride < 0 || v_token_stride < 0)
    return fail(AEKV_ERR_UNSUPPORTED, "%s: token strides of %lld and %lld elements", who, (long long)k_token_stride,
                (long long)v_token_stride);
  const PromptPlan plan = plan_prompt(B, n_q, n_k, H, heads, d);
  const size_t want = aekv_prompt_attention_workspace_size(B, n_q, n_k, H, heads, d);
  if (want && (!ws || ws_bytes < want)) return fail(AEKV_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, got %zu", who, want, ws_bytes);
  if (!is_aligned(ws, 16)) return fail(AEKV_ERR_ALIGN, "%s: workspace must be 16-byte aligned", who);
  if (plan.tiles * heads * plan.split > kMaxGridThreads / 256 || ceil_div(n_q * H, 256 / (d / 4)) > kMaxGridThreads / 256)
    return fail(AEKV_ERR_UNSUPPORTED, "%s: B=%lld n_q=%lld H=%lld exceed the grid", who, (long long)B, (long long)n_q, (long long)H);
  // By work where the keys and values that an XCD reads are at most three times its 4 MB L2 (a KV head's workgroups lie on
  // 8 / heads XCDs, or an XCD has heads / 8): 16 prompts of up to 2048, 12 heads of 4, 9.7 MB: 132 against 142 us; 8 of 2048,
  // 8.4 MB: 128 against 144; 64 of 1024, 34 MB: 360 against 340; 32 of 2048, 16 heads of 16, 67 MB: 1007 against 712.
  int32_t by_work = 0;
  if (B > 1 && B <= 64 && plan.tiles * heads > (d == 64 ? 768 : 512) && n_k * ceil_div(heads, static_cast<int64_t>(8)) * 4 * d <= (12 << 20)) {
    const int64_t levels = n_k * (H / heads) / plan.rows + plan.tiles;
    for (by_work = 1; by_work < (1 << 25) && 2 * by_work <= levels;) by_work *= 2;
  } else if (B > 1 && B <= 64 && plan.tiles * heads * plan.split > 256) {
    by_work = -1;
  }
  // Tiles come with the most keys first; the second workgroup of each CU is taken from the short end of its round, so that the
  // pairs have like work (one prompt of 11000, 12 heads of 4: 400 -> 381 us; 8192, 16 heads of 16: 300 -> 288; else 0 to 3 %).
  const uint32_t fold = static_cast<uint32_t>(plan.tiles * heads >= 512 ? 256 / heads : 0);
  const bool none = softmax_scale != softmax_scale;
  PromptArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v), q_token_stride,
               q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride, cu_seqlens_q, cu_seqlens_k, sink,
               static_cast<uint16_t*>(out), lse, static_cast<float*>(ws), static_cast<int32_t>(plan.split), static_cast<int32_t>(plan.tiles),
               static_cast<int32_t>(n_q), static_cast<int32_t>(n_k), static_cast<int32_t>(B), static_cast<int32_t>(H),
               static_cast<int32_t>(heads), static_cast<int32_t>(H / heads), clear_rest,
               by_work, fold, none ? 1.0f : fmaxf(fabsf(softmax_scale) * kLog2e, 0x1p-126f), softmax_scale < 0.0f, none ? 0x7fff7fffu : 0u};
  const hipStream_t st = as_stream(stream);
  auto fn = plan.rows == 128 ? pick_prompt<4, 1>(dtype, d) : pick_prompt<2, 2>(dtype, d);
  hipLaunchKernelGGL(fn, dim3(static_cast<uint32_t>(plan.tiles * heads * plan.split)), dim3(256), 0, st, a);
  if (const int rc = check_launch(who)) return rc;
  if (plan.split == 1) return AEKV_OK;
  auto mg = dtype == AEKV_F16 ? (d == 64 ? prompt_merge_kernel<AEKV_F16, 64> : prompt_merge_kernel<AEKV_F16, 128>)
                              : (d == 64 ? prompt_merge_kernel<AEKV_BF16, 64> : prompt_merge_kernel<AEKV_BF16, 128>);
  hipLaunchKernelGGL(mg, dim3(static_cast<uint32_t>(ceil_div(n_q * H, 256 / (d / 4)))), dim3(256), 0, st, a);
  return check_launch(who);
}
