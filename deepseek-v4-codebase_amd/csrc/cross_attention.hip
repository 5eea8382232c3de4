// Attention of packed queries over all states of an encoder, whose length is another: no query waits for a state.
//
// Sequence b has queries cu_q[b] .. cu_q[b + 1] (one query each where there is no cu_q) and reads the states e = states[b]
// (b without a list): keys and values cu_k[e] .. cu_k[e + 1], heads grouped over KV heads.
//   out_i = sum_j p_ij v_j,  p_ij = exp(scale q_i . k_j) / (sum exp(scale q_i . k) + exp(sink)),  lse_i = log of that sum.
// A query over no states gives 0 and a log sum of the sink's, or -inf.
//
// Rows.  The G heads of a KV head's group share its keys, and so do neighbouring sequences that read the same states (the answers
// to one input): a run's rows are (query, head), query-major, over all its sequences.  Runs end at multiples of 64 sequences.
// One pass: running maximum and sum, the output rescaled only where a maximum moved by more than kMargin.  The weights are rounded
// to the input's 16 bits for their product with V, the sums of weights and of products are fp32: bf16 has fp32's range; fp16
// ends at 2^-24, so its weights are held 2^kLift higher, and all down to 2^-21 of the largest are normal numbers.  With few rows,
// where the matrix units wait for memory, what the rounding leaves off is multiplied as well, so that a weight is off by 2^-16 (fp16
// 2^-22) of itself; with many rows, which they bound, that would be half as many products again, and a weight is off by 2^-8 (2^-11).
#include "attn_tile.h"

namespace aekv {
namespace {

constexpr int kFewShift = 7;   // log2 of a unit's keys: with few rows, all heads that a workgroup takes at a time together
constexpr int kManyShift = 6;  // with many rows
// Units that a tile costs beside its own.  Few rows, with 0, 1, 2, 3 of them: 64 sequences of up to 4096 states 63.4, 63.2, 63.8, 63.0
// us, 64 beams over 8 x up to 2999 18.8, 18.3, 17.5, 17.6; 24 other calls of 10 to 55 us take from 6 % less to 9 % more with 2 or 3 than
// with 1, in the mean 0.3 and 0.9 % more.  Many rows, with 1, 2, 3, 4: 16 packed prompts 54.3, 52.3, 51.7, 51.8 us, 8192 queries over
// 16384 states 842, 830, 839, 834.
constexpr int kFewStart = 1;
constexpr int kManyStart = 2;
constexpr int kTable = 256;    // sequences of a launch

struct alignas(16) LineTile {  // the tile that a part starts within (whole 16 bytes: the partial rows lie behind any number of them)
  int64_t start, chunk;        // its first place, -1: none; places of a part
  int32_t units, q0, n_rows, row0, head;
};

struct CrossArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;  // strides in elements
  const int32_t* cu_q;    // [B + 1] or null
  const int32_t* cu_k;    // [E + 1]
  const int32_t* states;  // [B] or null
  const float* sink;      // [H] or null
  uint16_t* out;          // [n_q, H, D]
  float* lse;             // [n_q, H] or null
  float* part;            // partial rows: reference, sum (log2 units), 2 pad, output
  LineTile* desc;         // [workgroups]
  int32_t n_q, n_k, B, E, H, heads, G;
  int32_t clear;          // rows in no sequence: 0 to leave out as it is, 1 to write zeros
  int32_t b0, nb;         // the launch's sequences
  int32_t least;          // units of a workgroup's part at least
  int32_t share;          // log2 of the KV heads that a workgroup takes at a time
  float scale2;           // |softmax scale| * log2(e), not 0 (times a masked product of -inf it stays -inf); where the
  int32_t flip;           // scale is negative the queries' signs are flipped: a row's largest product is its largest logit.  Where
  uint32_t nan;           // it is NaN, 1 stands for it and the queries become NaN (0x7fff is one in both types; else 0)
};

__device__ __forceinline__ int64_t uniform(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v)), hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
  return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}

struct Run {
  int32_t q0, lq, k0, lk;  // the run's queries and keys
};

__device__ __forceinline__ int32_t query_start(const CrossArgs& a, int32_t b) {
  const int32_t c = load_or(a.cu_q, b, a.q, b);
  return min(max(c, 0), a.n_q);  // (n_q H, with a tile's rows, fits 31 bits)
}

// Lane l's view of sequence b0 + l, l < n (b0 a multiple of 64): whether a run starts there, and that run.
__device__ __forceinline__ bool find_run(const CrossArgs& a, int32_t b0, int32_t n, int lane, Run* r) {
  const int32_t b = b0 + min(lane, n - 1);
  int32_t state = b;
  if (a.states) state = a.states[b];  // (without them all loads here go out together)
  const int32_t c0 = query_start(a, b), c1 = query_start(a, b + 1);
  const int32_t before = __shfl_up(state, 1);
  const bool head = lane < n && (lane == 0 || state != before);
  const uint64_t later = __builtin_amdgcn_ballot_w64(head) & ~((2ull << lane) - 1);
  const int last = (later ? __builtin_ctzll(later) : n) - 1;
  const int32_t end = __shfl(c1, last);
  const bool there = state >= 0 && state < a.E;
  const int32_t e = there ? state : 0;
  const int32_t d0 = a.E > 0 ? a.cu_k[e] : 0, d1 = a.E > 0 ? a.cu_k[e + 1] : 0;
  r->q0 = c0, r->lq = max(end - c0, 0);
  r->k0 = min(max(d0, 0), a.n_k), r->lk = there ? min(max(d1, r->k0), a.n_k) - r->k0 : 0;
  return head;
}

// Rows in no sequence (before the first, from the last's end on): shared out over the workgroups.
__device__ __forceinline__ void clear_rest(const CrossArgs& a, int32_t s0, int32_t s1, int words_of_row) {
  const int64_t words = static_cast<int64_t>(s0 + a.n_q - s1) * a.H * words_of_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < words; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t r = i / words_of_row, row = r < static_cast<int64_t>(s0) * a.H ? r : r + static_cast<int64_t>(s1 - s0) * a.H;
    if (a.clear) reinterpret_cast<uint32_t*>(a.out)[row * words_of_row + i % words_of_row] = 0;
    if (a.lse && i % words_of_row == 0) a.lse[row] = kNegInf;
  }
}

// Queries as matrix operands, with signs and NaN as the scale asks for (rarely: else nothing waits here for them).
template <int N>
__device__ __forceinline__ void take_queries(const CrossArgs& a, uint4 (&q)[N]) {
  if (!(a.flip | a.nan)) return;
#pragma unroll
  for (int i = 0; i < N; ++i) q[i] = make_uint4((q[i].x ^ a.flip) | a.nan, (q[i].y ^ a.flip) | a.nan, (q[i].z ^ a.flip) | a.nan, (q[i].w ^ a.flip) | a.nan);
}

// Four dims (4 c ..) of one finished row, whose sum is relative to m.
template <int DT, int D>
__device__ __forceinline__ void finish(const CrossArgs& a, int64_t orow, int32_t h, int c, float m, float l, float4 o) {
  using E = Elem<DT>;
  const float sk = a.sink ? a.sink[h] * kLog2e : kNegInf;
  const float up = fmaxf(m, sk);
  const float f = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - up);
  const float sum = (l == 0.0f ? 0.0f : l * f) + (sk == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(sk - up));
  const float r = sum == 0.0f ? 0.0f : f / sum;
  *reinterpret_cast<uint2*>(a.out + orow * D + 4 * c) = make_uint2(E::pack(o.x * r, o.y * r), E::pack(o.z * r, o.w * r));
  if (a.lse && c == 0) a.lse[orow] = sum == 0.0f ? kNegInf : (up + __builtin_amdgcn_logf(sum)) * kLn2;
}

// The line.  All tiles' units (2^kShift keys of a KV head or of a few, for a tile of kRows rows) lie in one line: run by run, its KV
// heads, their tiles, their units.  Every workgroup takes an equal part, so that the chip is loaded evenly whatever the lengths; a tile that lies
// in several parts is merged by a second kernel.  A tile's units come behind kStart places without any, for what it costs
// to begin and end one; a border among those is one before the tile.
//
// A die takes neighbouring parts, which read the same keys.  With neighbours on different dies and a tile's heads next to each other:
// 16 x up to 512 queries over up to 2048 states, 12 heads of 4 (dim 128) 76 us for 73, 16 of 2 (dim 64) 56.7 for 55.5; 8192 queries
// over 16384 states 853 for 860.
struct LineTable {
  int64_t end[kTable];  // a run is at its first sequence, the others' work is 0
  int32_t q0[kTable], lq[kTable], k0[kTable], lk[kTable];
  int64_t sum[4];
};
// Units of lk keys: one at least, which ends the tile of rows that see none.
template <int kShift>
__device__ __forceinline__ int32_t units_of(const CrossArgs& a, int32_t lk) {
  const int shift = kShift == kFewShift ? kShift - a.share : kShift;
  return max((lk + (1 << shift) - 1) >> shift, 1);
}
struct LinePart {
  int64_t start, stop, chunk;
  int32_t index;
};
template <int D, int kRows, int kShift, int kStart>
__device__ __forceinline__ LinePart line_part(const CrossArgs& a, LineTable& s, int wv, int lane) {
  const int32_t s0 = query_start(a, 0), s1 = max(query_start(a, a.B), s0);
  Run r{};
  int64_t x = 0;
  const int32_t n = min(a.nb - 64 * wv, 64);
  if (n > 0 && find_run(a, a.b0 + 64 * wv, n, lane, &r))
    x = static_cast<int64_t>((r.lq * a.G + kRows - 1) / kRows) * (a.heads >> a.share) * (kStart + units_of<kShift>(a, r.lk));
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t o = __shfl_up(x, d);
    if (lane >= d) x += o;
  }
  if (lane == 63) s.sum[wv] = x;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 3; ++w) x += w < wv ? s.sum[w] : 0;
  const int at = 64 * wv + lane;
  s.end[at] = x, s.q0[at] = r.q0, s.lq[at] = r.lq, s.k0[at] = r.k0, s.lk[at] = r.lk;
  __syncthreads();
  const int64_t total = uniform(s.end[kTable - 1]);
  if ((a.clear || a.lse) && s0 + a.n_q - s1 > 0) clear_rest(a, s0, s1, D / 2);
  LinePart p;
  p.chunk = total >> 31 ? (total + gridDim.x - 1) / gridDim.x : (static_cast<uint32_t>(total) + gridDim.x - 1) / gridDim.x;
  p.chunk = p.chunk > a.least ? p.chunk : a.least;
  // every die takes a stretch of the line (workgroups go to the eight of them in turn)
  const uint32_t parts = total >> 31 ? gridDim.x : (static_cast<uint32_t>(total + p.chunk) - 1) / static_cast<uint32_t>(p.chunk);  // (a long line fills them all)
  const uint32_t die = blockIdx.x % 8, rest = parts % 8;
  p.index = blockIdx.x < parts ? die * (parts / 8) + (die < rest ? die : rest) + blockIdx.x / 8 : blockIdx.x;
  p.start = p.index * p.chunk, p.stop = p.start + p.chunk;
  p.start = p.start < total ? p.start : total, p.stop = p.stop < total ? p.stop : total;
  if (p.start >= p.stop && threadIdx.x == 0) a.desc[p.index].start = -1;
  return p;
}

// The tile at place `pos` of the line.
struct Place {
  int32_t q0, n_rows, k0, lk, units, head, row0, u0, u1;  // its rows, (first) KV head and units; the part's units of it, if u0 < u1
  int64_t next;                                           // where the part goes on
};
template <int kRows, int kShift, int kStart>
__device__ __forceinline__ Place line_place(const CrossArgs& a, const LineTable& s, const LinePart& p, int64_t pos) {
  int32_t lo = kTable;  // the first run that ends behind pos
#pragma unroll
  for (int i = kTable / 64 - 1; i >= 0; --i) {
    const uint64_t behind = __builtin_amdgcn_ballot_w64(s.end[64 * i + (threadIdx.x & 63)] > pos);
    lo = behind ? 64 * i + __builtin_ctzll(behind) : lo;
  }
  Place at;
  const int64_t local = pos - uniform(lo ? s.end[lo - 1] : 0);
  at.q0 = __builtin_amdgcn_readfirstlane(s.q0[lo]), at.n_rows = __builtin_amdgcn_readfirstlane(s.lq[lo]) * a.G;
  at.k0 = __builtin_amdgcn_readfirstlane(s.k0[lo]), at.lk = __builtin_amdgcn_readfirstlane(s.lk[lo]);
  at.units = units_of<kShift>(a, at.lk);
  const uint32_t places = static_cast<uint32_t>(at.units) + kStart;
  const uint32_t th = static_cast<uint32_t>(local >> 31 ? static_cast<uint64_t>(local) / places : static_cast<uint32_t>(local) / places);  // (tiles x heads fit 32 bits)
  const int64_t from = pos - (local - static_cast<int64_t>(th) * places), end = from + places;  // the tile's
  at.next = end < p.stop ? end : p.stop;
  at.u0 = max(static_cast<int32_t>(pos - from) - kStart, 0), at.u1 = max(static_cast<int32_t>(at.next - from) - kStart, 0);
  const uint32_t tiles = static_cast<uint32_t>(at.n_rows + kRows - 1) / kRows;
  at.head = static_cast<int32_t>(th / tiles) << a.share, at.row0 = static_cast<int32_t>(th % tiles * kRows);
  if (pos == p.start && threadIdx.x == 0)
    a.desc[p.index] = LineTile{at.u0 > 0 ? from : -1, p.chunk, at.units, at.q0, at.n_rows, at.row0, at.head};
  return at;
}

// The head that row `at` belongs to, where up to four heads have `rows` each.
__device__ __forceinline__ int head_of_row(int at, int rows) { return (at >= rows) + (at >= 2 * rows) + (at >= 3 * rows); }

// Merges the tiles that lie in several parts: workgroup i has the tile across the border to part i + 1, if that is the tile's first.
// Bound by the chain of its loads, so that several parts' go out together and a workgroup has one row to D / 4 threads.
template <int DT, int D, int kRows, int kStart>
__global__ __launch_bounds__(256) void cross_merge_kernel(CrossArgs a) {
  const LineTile d = a.desc[blockIdx.x + 1];
  if (d.start < 0 || (d.start + kStart) / d.chunk != blockIdx.x) return;
  const int32_t q0 = d.q0, n_rows = d.n_rows, row0 = d.row0;
  const int32_t last = static_cast<int32_t>((d.start + kStart + d.units - 1) / d.chunk);  // part of the tile's last unit
  const int first_slot = blockIdx.x * d.chunk >= d.start ? 0 : 1;
  const int c = threadIdx.x % (D / 4), at = blockIdx.y * (256 / (D / 4)) + threadIdx.x / (D / 4), rows = min(kRows, n_rows - row0);
  if (at < rows << a.share) {
    const int sub = head_of_row(at, rows), r = at - sub * rows, own = d.head + sub;
    float m = kNegInf, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    constexpr int CH = kRows <= 32 ? 8 : 4;
    for (int32_t w0 = blockIdx.x; w0 <= last; w0 += CH) {
      float2 ml[CH];
      float4 x[CH];
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int32_t w = min(w0 + i, last);
        const int slot = w == static_cast<int32_t>(blockIdx.x) ? first_slot : 0;
        const float* p = a.part + (((2 * static_cast<int64_t>(w) + slot) << a.share) * kRows + sub * kRows + r) * (D + 4);
        ml[i] = *reinterpret_cast<const float2*>(p);
        x[i] = *reinterpret_cast<const float4*>(p + 4 + 4 * c);
      }
      float up = m;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        if (w0 + i > last || ml[i].y == 0.0f) ml[i] = make_float2(kNegInf, 0.0f), x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);  // (nothing seen)
        up = fmaxf(up, ml[i].x);
      }
      const float f0 = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - up);
      l = l == 0.0f ? 0.0f : l * f0;
      o.x *= f0, o.y *= f0, o.z *= f0, o.w *= f0;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const float f = ml[i].y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml[i].x - up);
        l += ml[i].y == 0.0f ? 0.0f : ml[i].y * f;
        o.x = fmaf(x[i].x, f, o.x), o.y = fmaf(x[i].y, f, o.y), o.z = fmaf(x[i].z, f, o.z), o.w = fmaf(x[i].w, f, o.w);
      }
      m = up;
    }
    const int32_t row = row0 + r, qi = row / a.G, h = own * a.G + (row - qi * a.G);
    finish<DT, D>(a, static_cast<int64_t>(q0 + qi) * a.H + h, h, c, m, l, o);
  }
}

// ---- few rows ------------------------------------------------------------------------------------------------------
//
// Tiles of 16 NT rows to each of the workgroup's heads, bound by reading the keys and values: 64 sequences of up to 4096 states, 12
// heads of 4, dim 128, 305 MB in 50 us, 6.1 TB/s where 256 MB of them can be in the last-level cache, 4.8 TB/s with the merge where
// nothing is.  A wave takes 32 keys of a unit and head by itself: keys go straight to registers, values to its own part of LDS, both
// one unit ahead, across tiles too, and no wave waits for another before the tile's end.  Heads that are neighbours in memory are read
// by one workgroup at the same time: by workgroups of their own the same bytes take 11 % longer.
//
// Matrix layout (v_mfma_f32_16x16x32: A lane l holds A[l % 16][8 (l / 16) + j], B lane l holds B[8 (l / 16) + j][l % 16], D lane
// l register v holds D[4 (l / 16) + v][l % 16]), g = l / 16:
//   S^T = K Q^T: m = key, n = row; two blocks of 16 keys.
//   O^T += V^T P^T: m = dim, n = row; lane group g holds keys 4 g + j and 16 + 4 g + j, its own scores.
template <int DT, int D, int NT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1))) void cross_few_kernel(CrossArgs a) {
  using E = Elem<DT>;
  using v8 = typename E::v8;
  constexpr int kRow = 2 * D, kKS = D / 32, kMB = D / 16, kRT = 16 * NT;
  constexpr int kPer = 1024 / kRow, kLoads = 32 / kPer;  // rows of a staging load, loads of 32 rows
  __shared__ __align__(16) uint8_t V0[4][32 * kRow];
  __shared__ __align__(16) uint8_t V1[4][32 * kRow];
  __shared__ __align__(16) uint8_t s_more[NT == 1 ? 1 : 4][NT == 1 ? 16 : 32 * kRow];  // the second 16 rows' states
  __shared__ LineTable s_line;
  __shared__ float2 s_ml[4][kRT];
  const int tid = threadIdx.x, lane = tid & 63, n16 = lane & 15, g = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const LinePart line = line_part<D, kRT, kFewShift, kFewStart>(a, s_line, wv, lane);
  if (line.start >= line.stop) return;
  const int shift = kFewShift - a.share, sub = wv & ((1 << a.share) - 1), block = wv >> a.share;  // the wave's head and keys of a unit

  // staging: load i of 32 rows writes 1024 bytes, lane l at + 16 l, so lane l loads the chunk that the swizzle puts there
  const int key_in = 16 * lane / kRow, placed = (16 * lane % kRow) / 16;
  int voff[4];
  const int k_stride = static_cast<int>(a.k_token) * 2, v_stride = static_cast<int>(a.v_token) * 2;
#pragma unroll
  for (int i = 0; i < 4; ++i) voff[i] = key_in * v_stride + 16 * (placed ^ swizzle<D>((kPer * i + key_in) & 15));
  const int koff = n16 * k_stride + 16 * g;
  int tA[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int key = 16 * e + 4 * g + (n16 >> 2), x = (n16 & 3) >> 1;
    tA[e] = key * kRow + ((x ^ swizzle<D>(key & 15)) << 4) + ((n16 & 1) << 3);
  }

  struct Tile {
    Place at;
    const uint8_t *k, *v;
  };
  auto find = [&](int64_t pos, Tile* t) __attribute__((always_inline)) {  // the part's first tile with units from pos on
    for (; pos < line.stop; pos = t->at.next) {
      t->at = line_place<kRT, kFewShift, kFewStart>(a, s_line, line, pos);
      if (t->at.u0 >= t->at.u1) continue;
      t->k = reinterpret_cast<const uint8_t*>(a.k + t->at.k0 * a.k_token + (t->at.head + sub) * a.k_head);
      t->v = reinterpret_cast<const uint8_t*>(a.v + t->at.k0 * a.v_token + (t->at.head + sub) * a.v_head);
      return true;
    }
    return false;
  };
  uint4 qb[NT][kKS];
  auto load_queries = [&](const Place& p) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int32_t row = min(p.row0 + 16 * t + n16, p.n_rows - 1), qi = row / a.G, h = (p.head + sub) * a.G + (row - qi * a.G);
      const uint16_t* qp = a.q + static_cast<int64_t>(p.q0 + qi) * a.q_token + h * a.q_head + 8 * g;
#pragma unroll
      for (int ks = 0; ks < kKS; ++ks) qb[t][ks] = *reinterpret_cast<const uint4*>(qp + 32 * ks);
    }
  };
  u32x4_t kr[2][2][kKS];
  // the wave's 32 keys of unit u, read through buffer resources whose range ends at the last key: rows past it are zero, as
  // is all of the unit past the part's last (every step has as many loads under way)
  auto load = [&](const uint8_t* k, const uint8_t* v, int32_t lk, int32_t u, int32_t u1, auto buf_c) __attribute__((always_inline)) {
    constexpr int buf = decltype(buf_c)::value;
    const int32_t at = (u << shift) + 32 * block, left = u < u1 ? lk - at : 0;
    const int32_t m = __builtin_amdgcn_readfirstlane(left < 0 ? 0 : left < 32 ? left : 32);  // (the clamp is a vector instruction)
    const int64_t base = m > 0 ? at : 0;
    const __amdgpu_buffer_rsrc_t krs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(k + base * k_stride), 0, m > 0 ? (m - 1) * k_stride + kRow : 0, kBufWord3);
    const __amdgpu_buffer_rsrc_t vrs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(v + base * v_stride), 0, m > 0 ? (m - 1) * v_stride + kRow : 0, kBufWord3);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int ks = 0; ks < kKS; ++ks) kr[buf][t][ks] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(krs, koff + 64 * ks, 16 * t * k_stride, 0));
    uint8_t* const dst = buf ? V1[wv] : V0[wv];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) __builtin_amdgcn_raw_ptr_buffer_load_lds(vrs, (lds_void_t*)(dst + 1024 * i), 16, voff[i & 3], kPer * i * v_stride, 0, 0);
  };

  // all waves, with their LDS accesses done (and their loads under way)
  auto meet = [&]() __attribute__((always_inline)) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // A tile begins with its first unit under way in the first buffer, and its queries: the tile before asks for them
  int slot = 0;  // of the next partial tile
  Tile cur;
  if (!find(line.start, &cur)) return;
  load_queries(cur.at);
  load(cur.k, cur.v, cur.at.lk, cur.at.u0, cur.at.u1, std::integral_constant<int, 0>{});
  for (bool more = true; more;) {
    Tile next = cur;
    more = find(cur.at.next, &next);
    if (!more) next.at.u0 = next.at.u1;  // (nothing to load)
#pragma unroll
    for (int t = 0; t < NT; ++t) take_queries(a, qb[t]);
    const int32_t q0 = cur.at.q0, n_rows = cur.at.n_rows, lk = cur.at.lk, row0 = cur.at.row0, u0 = cur.at.u0, u1 = cur.at.u1;
    float m[NT], l[NT];
    f32x4_t O[NT][kMB], R[NT][kMB];  // R: by the weights' rests
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t] = kNegInf, l[t] = 0.0f;
#pragma unroll
      for (int mb = 0; mb < kMB; ++mb) O[t][mb] = R[t][mb] = f32x4_t{};
    }
    auto step = [&](int32_t u, auto buf_c) __attribute__((always_inline)) {
      constexpr int buf = decltype(buf_c)::value;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the other buffer's values have been read
      const bool over = buf && u + 1 >= u1;
      load(over ? next.k : cur.k, over ? next.v : cur.v, over ? next.at.lk : lk, over ? next.at.u0 : u + 1, over ? next.at.u1 : u1, std::integral_constant<int, buf ^ 1>{});
      if constexpr (D == 128) asm volatile("s_waitcnt vmcnt(16)" ::: "memory");  // (8 loads of keys, 8 of values under way)
      else asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
      const int32_t at = (u << shift) + 32 * block;
      if (at >= lk || u >= u1) return;
      const uint8_t* vt = buf ? V1[wv] : V0[wv];
      v8 pb[NT], pr[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        f32x4_t s[2];
        float top = kNegInf;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          s[kb] = f32x4_t{};
#pragma unroll
          for (int ks = 0; ks < kKS; ++ks) s[kb] = E::mma16(__builtin_bit_cast(v8, kr[buf][kb][ks]), __builtin_bit_cast(v8, qb[t][ks]), s[kb]);
        }
        if (at + 32 > lk) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[kb][i] = at + 16 * kb + 4 * g + i < lk ? s[kb][i] : kNegInf;
        }
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int i = 0; i < 4; ++i) top = fmaxf(top, s[kb][i]);
        top = fmaxf(top, xor_lane<16>(top));
        top = fmaxf(top, xor_lane<32>(top)) * a.scale2;
        const bool moved = top - m[t] > kMargin + E::kLift;
        if (__builtin_amdgcn_ballot_w64(moved)) {
          const float to = top - E::kLift, r = moved ? __builtin_amdgcn_exp2f(m[t] - to) : 1.0f;
          l[t] *= r;
#pragma unroll
          for (int mb = 0; mb < kMB; ++mb) O[t][mb] *= r, R[t][mb] *= r;
          m[t] = moved ? to : m[t];
        }
        float nm = m[t] == kNegInf ? 0.0f : -m[t], by = a.scale2;
        // beyond kFar the reference, which is a rounded logit, may lie further from the exact product than the exponentials
        // reach: there a row's logits are all rounded as the reference was
        const bool far = fabsf(m[t]) > kFar && m[t] > kNegInf;
        if (__builtin_amdgcn_ballot_w64(far)) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[kb][i] = far ? s[kb][i] * a.scale2 + nm : s[kb][i];
          by = far ? 1.0f : by, nm = far ? 0.0f : nm;
        }
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          p[i] = __builtin_amdgcn_exp2f(fmaf(s[i >> 2][i & 3], by, nm));
          l[t] += p[i];
        }
        uint32_t w[4], rest[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[i] = E::pack(p[2 * i], p[2 * i + 1]);
          rest[i] = E::pack(p[2 * i] - E::value(w[i] & 0xFFFFu), p[2 * i + 1] - E::value(w[i] >> 16));
        }
        pb[t] = __builtin_bit_cast(v8, make_uint4(w[0], w[1], w[2], w[3])), pr[t] = __builtin_bit_cast(v8, make_uint4(rest[0], rest[1], rest[2], rest[3]));
      }
#pragma unroll
      for (int mb = 0; mb < kMB; ++mb) {
        const i16x4_t x = read_tr16(vt + (tA[0] ^ (mb << 5))), y = read_tr16(vt + (tA[1] ^ (mb << 5)));
        const v8 w = __builtin_bit_cast(v8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int t = 0; t < NT; ++t) O[t][mb] = E::mma16(w, pb[t], O[t][mb]), R[t][mb] = E::mma16(w, pr[t], R[t][mb]);
      }
    };
    int32_t u = u0;
    do {
      step(u, std::integral_constant<int, 0>{});
      step(u + 1, std::integral_constant<int, 1>{});
      u += 2;
    } while (u < u1);

    load_queries(next.at);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int mb = 0; mb < kMB; ++mb)
#pragma unroll
        for (int i = 0; i < 4; ++i) O[t][mb][i] += fabsf(R[t][mb][i]) < __builtin_inff() ? R[t][mb][i] : 0.0f;  // (an infinite value by a rest of 0 or less is none)
    // the waves' states through their own second buffers: row n16's four dims at 16 mb + 4 g, chunks swizzled by the row
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      l[t] += xor_lane<16>(l[t]);
      l[t] += xor_lane<32>(l[t]);
      if (g == 0) s_ml[wv][16 * t + n16] = make_float2(m[t], l[t]);
      float* const w = reinterpret_cast<float*>(t ? s_more[NT == 1 ? 0 : wv] : V1[wv]) + n16 * D;
#pragma unroll
      for (int mb = 0; mb < kMB; ++mb) *reinterpret_cast<f32x4_t*>(w + 4 * ((4 * mb + g) ^ n16)) = O[t][mb];
    }
    meet();
    const bool whole = u1 - u0 == cur.at.units;
    float* const part = a.part + ((2 * static_cast<int64_t>(line.index) + slot) << a.share) * kRT * (D + 4);
    const int rows = min(kRT, n_rows - row0);
    for (int at = tid / (D / 4); at < rows << a.share; at += 256 / (D / 4)) {
      const int c = tid % (D / 4), of = head_of_row(at, rows), r = at - of * rows, row = row0 + r;
      float2 ml[4];  // of the head's waves
      float up = kNegInf;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ml[i] = make_float2(kNegInf, 0.0f);
        if (of + (i << a.share) < 4) ml[i] = s_ml[of + (i << a.share)][r];
        up = fmaxf(up, ml[i].x);
      }
      float sum = 0.0f;
      float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // (a state of nothing has a sum of 0; NaN alone leaves a maximum of -inf, and a sum that says so)
        if (ml[i].y == 0.0f) continue;
        const float f = __builtin_amdgcn_exp2f(ml[i].x - up);
        const int w = of + (i << a.share);
        const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(NT == 1 || r < 16 ? V1[w] : s_more[NT == 1 ? 0 : w]) + (r & 15) * D + 4 * (c ^ (r & 15)));
        sum += ml[i].y * f;
        o.x = fmaf(x.x, f, o.x), o.y = fmaf(x.y, f, o.y), o.z = fmaf(x.z, f, o.z), o.w = fmaf(x.w, f, o.w);
      }
      if (whole) {
        const int32_t qi = row / a.G, h = (cur.at.head + of) * a.G + (row - qi * a.G);
        finish<DT, D>(a, static_cast<int64_t>(q0 + qi) * a.H + h, h, c, up, sum, o);
      } else {
        float* p = part + (of * kRT + r) * (D + 4);
        if (c == 0) *reinterpret_cast<float2*>(p) = make_float2(up, sum);
        *reinterpret_cast<float4*>(p + 4 + 4 * c) = o;
      }
    }
    meet();
    slot = 1;
    cur = next;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the loads past the last tile write zeros to LDS)
}

// ---- many rows -----------------------------------------------------------------------------------------------------
//
// Tiles of 128 rows, 32 to a wave; units of 64 keys in two blocks.  8192 queries over 16384 states, 12 heads of 4, dim 128: 790 to 850
// us by card, 970 to 1050 TFLOP/s, at 1.8 GHz, as power allows (663 us on zeros); 256 rows to a tile took 924 for 894 then.  Bound by
// the matrix instructions and the exponentials, which one
// wave's instructions interleave: while the keys of a block are multiplied with the queries, the weights of the block before are made
// and those of the block before that are multiplied with their values, three parts that do not wait for each other.  Keys and values go
// straight to LDS, two buffers each: keys one unit ahead, values at the step that multiplies their keys.
//
// Matrix layout (v_mfma_f32_32x32x16: A lane l holds A[l % 32][8 (l / 32) + j], B lane l holds B[8 (l / 32) + j][l % 32],
// D lane l register v holds D[8 (v / 4) + 4 (l / 32) + v % 4][l % 32]), h = l / 32:
//   S^T = K Q^T: m = key, n = row; a lane reads 16-byte chunks of its key's row.
//   O^T += V^T P^T: m = dim, n = row, k = key; lane h holds keys 16 c + 4 h + j and 16 c + 8 + 4 h + j of a 16-key chunk c,
//   its own scores, and V^T comes from the row-major unit through the transposing LDS load.
// LDS rows keep their 16-byte chunks XOR-swizzled by their key, so that both reads touch all banks once.
template <int DT, int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D == 64 ? 3 : 2))) void cross_many_kernel(CrossArgs a) {
  using E = Elem<DT>;
  using v8 = typename E::v8;
  constexpr int kRows = 128, kManyKeys = 1 << kManyShift, kRow = 2 * D, kBytes = kManyKeys * kRow;
  constexpr int kMB = D / 32, kKS = D / 16;  // (kKS: products of a block's keys, and of its values)
  constexpr int kAhead = 2;                  // products ahead that their operands are read
  __shared__ __align__(16) uint8_t K0[kBytes], K1[kBytes], V0[kBytes], V1[kBytes];
  __shared__ LineTable s_line;

  const int lane = threadIdx.x & 63, rl = lane & 31, hh = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const LinePart line = line_part<D, kRows, kManyShift, kManyStart>(a, s_line, wv, lane);
  if (line.start >= line.stop) return;

  // staging: load c of wave wv writes bytes [4096 c + 1024 wv, + 1024) of a unit, lane l at + 16 l, so lane l loads the chunk that
  // the swizzle puts there (a load is 16 or 32 rows after the other, and the swizzle repeats after 16)
  const int lin = 1024 * wv + 16 * lane, key_in = lin / kRow, placed = ((lin % kRow) / 16) ^ swizzle<D>(key_in & 15);
  const int k_stride = static_cast<int>(a.k_token) * 2, v_stride = static_cast<int>(a.v_token) * 2;
  const int koff = key_in * k_stride + 16 * placed, voff = key_in * v_stride + 16 * placed;
  // LDS byte offsets.  Row-chunk reads (K): key rl, chunk (2 ks + hh) ^ swizzle(rl).  Transposing reads (V, 16-lane group
  // G = lane / 16, s = lane % 16): key 16 c + 8 e + 4 hh + s / 4, dims 32 mb + 16 (G % 2) + 4 (s % 4) .., i.e. chunk 4 mb + x with
  // x = 2 (G % 2) + (s % 4) / 2, xor the swizzle of the key.
  int xk[kKS], xv[2][kMB];
#pragma unroll
  for (int ks = 0; ks < kKS; ++ks) xk[ks] = rl * kRow + (((2 * ks + hh) ^ swizzle<D>(rl & 15)) << 4);
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int s16 = lane & 15, x = 2 * ((lane >> 4) & 1) + ((s16 & 3) >> 1), key = 8 * e + 4 * hh + (s16 >> 2);
#pragma unroll
    for (int mb = 0; mb < kMB; ++mb) xv[e][mb] = key * kRow + (((4 * mb + x) ^ swizzle<D>(key)) << 4) + ((s16 & 1) << 3);
  }
  // (made anew for the compiler at every block: it would keep the sums with each buffer's address, not the offsets alone)
  auto offsets = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int ks = 0; ks < kKS; ++ks) asm volatile("" : "+v"(xk[ks]));
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int mb = 0; mb < kMB; ++mb) asm volatile("" : "+v"(xv[e][mb]));
  };

  int slot = 0;  // of the next partial tile
  for (int64_t pos = line.start, next; pos < line.stop; pos = next) {
    const Place at = line_place<kRows, kManyShift, kManyStart>(a, s_line, line, pos);
    const int32_t q0 = at.q0, n_rows = at.n_rows, head = at.head, u0 = at.u0, u1 = at.u1;
    next = at.next;
    if (u0 >= u1) continue;
    const int32_t limit = min(at.lk, u1 * kManyKeys);  // of the part's keys
    // the next unit's rows of K (of V), read through a buffer resource whose range ends at the limit: rows past it are zero and
    // touch no memory
    const int64_t first_key = static_cast<int64_t>(at.k0) + static_cast<int64_t>(u0) * kManyKeys;
    const uint8_t* knext = reinterpret_cast<const uint8_t*>(a.k + first_key * a.k_token + head * a.k_head);
    const uint8_t* vnext = reinterpret_cast<const uint8_t*>(a.v + first_key * a.v_token + head * a.v_head);
    int32_t kleft = limit - u0 * kManyKeys, vleft = kleft;
    auto load = [&](const uint8_t*& from, int32_t& left, int stride, int off, uint8_t* to) __attribute__((always_inline)) {
      int32_t range = (kManyKeys - 1) * stride + kRow;
      if (left < kManyKeys) range = left > 0 ? (left - 1) * stride + kRow : 0;
      const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(from), 0, range, kBufWord3);
#pragma unroll
      for (int c = 0; c < kBytes / 4096; ++c)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void_t*)(to + 4096 * c + 1024 * wv), 16, off, 4096 / kRow * c * stride, 0, 0);
      left -= kManyKeys;
      from += left > 0 ? static_cast<int64_t>(kManyKeys) * stride : 0;
    };
    load(knext, kleft, k_stride, koff, K0);

    // rows past the last are computed as copies of it
    uint4 qb[kKS];
    const int32_t row = at.row0 + 32 * wv + rl;
    {
      const int32_t own = row < n_rows ? row : n_rows - 1, qi = own / a.G, h = head * a.G + (own - qi * a.G);
      const uint16_t* qp = a.q + static_cast<int64_t>(q0 + qi) * a.q_token + h * a.q_head + 8 * hh;
#pragma unroll
      for (int ks = 0; ks < kKS; ++ks) qb[ks] = *reinterpret_cast<const uint4*>(qp + 16 * ks);
      take_queries(a, qb);
    }

    // m: the reference that weights are relative to (a maximum less kLift); nm: -m, or 0 where nothing was seen; l: the weights' sum
    float m = kNegInf, nm = 0.0f, l = 0.0f, r = 1.0f;
    bool far = false;    // some row's reference lies beyond kFar
    f32x16_t O[kMB], S;  // S: the products of the block whose weights come next
    v8 pb[2];            // the weights whose values come next
#pragma unroll
    for (int mb = 0; mb < kMB; ++mb) O[mb] = f32x16_t{};

    auto key = [&](const uint8_t* kt, int ks) __attribute__((always_inline)) { return __builtin_bit_cast(v8, *reinterpret_cast<const uint4*>(kt + xk[ks])); };
    auto value = [&](const uint8_t* vt, int i) __attribute__((always_inline)) {  // keys 16 (i / kMB) .., dims 32 (i % kMB) ..
      const i16x4_t lo = read_tr16(vt + 16 * kRow * (i / kMB) + xv[0][i % kMB]), hi = read_tr16(vt + 16 * kRow * (i / kMB) + xv[1][i % kMB]);
      return __builtin_bit_cast(v8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    // The reference for the weights of S, whose first key is `first`; true where some row's moved, by the factor r
    auto reference = [&](int32_t first) __attribute__((always_inline)) -> bool {
      if (first + 32 > limit) {
        int32_t k = first + 4 * hh;
        asm volatile("" : "+v"(k));  // (else the comparisons are made for every block)
#pragma unroll
        for (int v = 0; v < 16; ++v) S[v] = k + 8 * (v >> 2) + (v & 3) < limit ? S[v] : kNegInf;
      }
      float top = kNegInf;  // of this lane's half of the row
#pragma unroll
      for (int v = 0; v < 16; ++v) top = fmaxf(top, S[v]);
      const bool any = __builtin_amdgcn_ballot_w64(fmaf(top, a.scale2, -m) > kMargin + E::kLift) != 0;
      if (any) {
        // (each row by itself, by the measure that brought the wave here: a row's bits do not depend on the others')
        top = fmaxf(top, xor_lane<32>(top));
        const bool moved = fmaf(top, a.scale2, -m) > kMargin + E::kLift;
        const float to = top * a.scale2 - E::kLift;
        r = moved ? __builtin_amdgcn_exp2f(m - to) : 1.0f;
        l *= r;
        m = moved ? to : m;
        nm = m == kNegInf ? 0.0f : -m;
        far = __builtin_amdgcn_ballot_w64(fabsf(m) > kFar && m > kNegInf) != 0;
      }
      return any;
    };
    // The weights of S's values from .. to, as pairs.  Beyond kFar the reference, which is a rounded logit, may lie further from
    // the exact product than the exponentials reach: there a row's logits are all rounded as the reference was
    auto weigh = [&](uint32_t (&w)[8], float by, float add, int from, int to) __attribute__((always_inline)) {
#pragma unroll
      for (int v = from; v < to; v += 2) {
        const float x = __builtin_amdgcn_exp2f(fmaf(S[v], by, add)), y = __builtin_amdgcn_exp2f(fmaf(S[v + 1], by, add));
        l += x;
        l += y;
        w[v / 2] = E::pack(x, y);
        asm volatile("" : "+v"(w[v / 2]), "+v"(l));  // (here, between the products: nothing else in the block needs them)
      }
    };
    // One block's three parts: products with the keys at kt (if any), the weights of S, products of pb's with the values at vt (if
    // any).  Then S and pb are the next ones.
    auto block = [&](auto with_keys, const uint8_t* kt, auto with_values, const uint8_t* vt, int32_t first) __attribute__((always_inline)) {
      constexpr bool keys = decltype(with_keys)::value, values = decltype(with_values)::value;
      offsets();
      v8 kf[kKS], vf[kKS];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if constexpr (keys) kf[i] = key(kt, i);
        if constexpr (values) vf[i] = value(vt, i);
      }
      const bool any = reference(first);
      float by = a.scale2, add = nm;
      if (far) {
        const bool here = fabsf(m) > kFar && m > kNegInf;
#pragma unroll
        for (int v = 0; v < 16; ++v) S[v] = here ? S[v] * a.scale2 + nm : S[v];
        by = here ? 1.0f : by, add = here ? 0.0f : add;
      }
      uint32_t w[8];
      f32x16_t sn = f32x16_t{};
#pragma unroll
      for (int i = 0; i < kKS; ++i) {  // a product of each kind, and the weights that the vector unit makes meanwhile
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (keys) {
          if (i + kAhead < kKS) kf[i + kAhead] = key(kt, i + kAhead);
          sn = E::mma(kf[i], __builtin_bit_cast(v8, qb[i]), sn);
        }
        if constexpr (values) {
          if (i + kAhead < kKS) vf[i + kAhead] = value(vt, i + kAhead);
          O[i % kMB] = E::mma(vf[i], pb[i / kMB], O[i % kMB]);
        }
        weigh(w, by, add, 16 / kKS * i, 16 / kKS * (i + 1));
      }
      __builtin_amdgcn_sched_barrier(0);
      if (any) {
        asm volatile("" : "+v"(r));  // (else the products are made for every block, and dropped)
#pragma unroll
        for (int mb = 0; mb < kMB; ++mb) O[mb] *= r;
      }
      S = sn;
#pragma unroll
      for (int c = 0; c < 2; ++c) pb[c] = __builtin_bit_cast(v8, make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]));
    };
    // before a step: this wave's loads have landed and its reads are done; then every wave's
    auto meet = [&]() __attribute__((always_inline)) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };
    constexpr std::true_type yes{};
    constexpr std::false_type no{};
    constexpr int kSecond = 32 * kRow;  // a unit's second block

    meet();
    load(knext, kleft, k_stride, koff, K1);
    load(vnext, vleft, v_stride, voff, V0);
    offsets();
    S = f32x16_t{};
#pragma unroll
    for (int ks = 0; ks < kKS; ++ks) S = E::mma(key(K0, ks), __builtin_bit_cast(v8, qb[ks]), S);
    block(yes, K0 + kSecond, no, V0, u0 * kManyKeys);
    auto step = [&](int32_t s, auto odd) __attribute__((always_inline)) {  // unit s's keys, unit s - 1's values
      constexpr bool p = decltype(odd)::value;
      const uint8_t *kt = p ? K1 : K0, *vt = p ? V0 : V1;
      meet();
      // first in every second unit: else the older of a CU's workgroups always are, the last one ends alone (53.4 for 52.7 us behind 16
      // prompts, 844 for 832 for a long one)
      __builtin_amdgcn_s_setprio(p ? 1 : 0);
      load(knext, kleft, k_stride, koff, p ? K0 : K1);
      load(vnext, vleft, v_stride, voff, p ? V1 : V0);
      block(yes, kt, yes, vt, s * kManyKeys - 32);
      block(yes, kt + kSecond, yes, vt + kSecond, s * kManyKeys);
    };
    int32_t s = u0 + 1;
    while (s < u1) {
      step(s++, yes);
      if (s == u1) break;
      step(s++, no);
    }
    meet();
    {
      const uint8_t* vt = (u1 - u0) & 1 ? V0 : V1;
      block(no, nullptr, yes, vt, u1 * kManyKeys - 32);
      vt += kSecond;
#pragma unroll
      for (int i = 0; i < kKS; ++i) O[i % kMB] = E::mma(value(vt, i), pb[i / kMB], O[i % kMB]);
    }
    l += xor_lane<32>(l);  // both halves' keys

    if (row < n_rows) {
      if (u1 - u0 == at.units) {
        int32_t own = row;
        asm volatile("" : "+v"(own));  // (the row's query and head are found again: kept through the loop they cost registers)
        const int32_t qi = own / a.G, h = head * a.G + (own - qi * a.G);
#pragma unroll
        for (int mb = 0; mb < kMB; ++mb)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            finish<DT, D>(a, static_cast<int64_t>(q0 + qi) * a.H + h, h, 8 * mb + 2 * i + hh, m, l, make_float4(O[mb][4 * i], O[mb][4 * i + 1], O[mb][4 * i + 2], O[mb][4 * i + 3]));
      } else {
        float* p = a.part + ((2 * static_cast<int64_t>(line.index) + slot) * kRows + 32 * wv + rl) * (D + 4);
        if (hh == 0) *reinterpret_cast<float2*>(p) = make_float2(m, l);
#pragma unroll
        for (int mb = 0; mb < kMB; ++mb)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<float4*>(p + 4 + 32 * mb + 8 * i + 4 * hh) = make_float4(O[mb][4 * i], O[mb][4 * i + 1], O[mb][4 * i + 2], O[mb][4 * i + 3]);
      }
    }
    meet();  // the buffers' readers are done
    slot = 1;
  }
}

using cross_fn = void (*)(CrossArgs);
template <int DT, int D>
cross_fn pick_rows(int64_t rows, bool merge) {
  if (rows == 16) return merge ? cross_merge_kernel<DT, D, 16, kFewStart> : cross_few_kernel<DT, D, 1>;
  if constexpr (D == 64) {
    if (rows == 32) return merge ? cross_merge_kernel<DT, D, 32, kFewStart> : cross_few_kernel<DT, D, 2>;
  }
  return merge ? cross_merge_kernel<DT, D, 128, kManyStart> : cross_many_kernel<DT, D>;
}
cross_fn pick_cross(int32_t dtype, int32_t d, int64_t rows, bool merge) {
  if (dtype == AEKV_F16) return d == 64 ? pick_rows<AEKV_F16, 64>(rows, merge) : pick_rows<AEKV_F16, 128>(rows, merge);
  return d == 64 ? pick_rows<AEKV_BF16, 64>(rows, merge) : pick_rows<AEKV_BF16, 128>(rows, merge);
}

struct CrossPlan {
  int64_t rows, groups;  // of a tile and head; workgroups of a launch
  int32_t least, share;  // units of a part at least; log2 of a tile's heads
};
CrossPlan plan_cross(int64_t B, int64_t E, int64_t n_q, int64_t n_k, int64_t H, int64_t heads, int32_t d) {
  CrossPlan p{};
  const int64_t rows = n_q * (H / heads), runs = E > 0 && E < B ? E : B, each = ceil_div(rows, runs);
  const int64_t resident = d == 64 ? 768 : 512;  // of the many rows' workgroups, by their registers
  // Few rows by the average run.  Over 64 x up to 4096 states, few / many: dim 128, 12 rows 68.8 / 72.4 us, 18 rows 75.2 / 74.7 (two
  // blocks of 16; with tiles of 16 93), 30 rows 81.3 / 75.7; dim 64, 24 rows 23.7 / 25.0, 32 rows 24.9 / 26.1, 48 rows 35.6 / 29.0
  const bool few = each <= (d == 64 ? 32 : 16);
  if (few) {
    // (a workgroup per CU: 60 us for 64 sequences of up to 4096 states, 20.6 for one of 16384; with two 60 and 24, with four 64 and 36)
    p.rows = each <= 16 ? 16 : 32, p.groups = 256, p.least = 1;
    // Heads that lie next to each other in a token are read together as long as that leaves tiles for a quarter of the workgroups.  64
    // sequences of up to 4096 states, 12 heads of 4, dim 128: 67.8 us with one head at a time, 64.9 with two, 63.1 with four (50 of them
    // the kernel's, 55 with one); dim 64: 39.2, 37.0, 36.6.  With fewer tiles, whose parts are merged: 8 sequences 17.1, 18.8, 23.0
    while (p.share < 2 && heads % (2 << p.share) == 0 && runs * (heads >> (p.share + 1)) >= 64) ++p.share;
  } else {
    // (a part begins, ends and is merged at some cost: 16 queries over 16 x 500 states 16.2 us with 3 units at least, 22.5 with 8)
    p.rows = 128, p.groups = resident, p.least = 3;
  }
  const int64_t keys = few ? (1 << kFewShift) >> p.share : 1 << kManyShift, start = few ? kFewStart : kManyStart;
  const double most = (static_cast<double>(rows / p.rows) + B) * (heads >> p.share) * (n_k / keys + 1 + start) / p.least + 1.0;  // parts of the longest line
  if (p.groups > most) p.groups = static_cast<int64_t>(most);
  return p;
}

}  // namespace
}  // namespace aekv

using namespace aekv;

static bool cross_fits(int64_t B, int64_t E, int64_t n_q, int64_t n_k, int64_t H) {
  return n_q <= 0x7fffffff && n_k <= 0x7fff0000 && B <= 0x7ffffffe && E <= 0x7ffffffe && H <= 65535 && n_q * H <= 0x7fff0000;
}

extern "C" size_t aekv_cross_attention_workspace_size(int64_t B, int64_t E, int64_t n_q, int64_t n_k, int64_t H, int64_t heads, int32_t d) {
  if (B <= 0 || E < 0 || n_q <= 0 || n_k < 0 || H <= 0 || heads <= 0 || (d != 64 && d != 128) || H % heads) return 0;
  if (!cross_fits(B, E, n_q, n_k, H)) return 0;  // (the call refuses it)
  const CrossPlan p = plan_cross(B, E, n_q, n_k, H, heads, d);
  return static_cast<size_t>(p.groups) * sizeof(LineTile) + static_cast<size_t>(p.groups) * 2 * (p.rows << p.share) * (d + 4) * 4;
}

extern "C" int aekv_cross_attention(const void* q, const void* k, const void* v, int32_t dtype, int64_t q_token_stride,
                                    int64_t q_head_stride, int64_t k_token_stride, int64_t k_head_stride,
                                    int64_t v_token_stride, int64_t v_head_stride, const int32_t* cu_seqlens_q,
                                    const int32_t* cu_seqlens_k, const int32_t* states, int64_t B, int64_t E, int64_t n_q,
                                    int64_t n_k, int64_t H, int64_t heads, int32_t d, const float* sink,
                                    float softmax_scale, void* out, float* lse, int32_t clear_rest, void* ws,
                                    size_t ws_bytes, void* stream) {
  const char* who = "aekv_cross_attention";
  if (dtype != AEKV_F16 && dtype != AEKV_BF16) return fail(AEKV_ERR_DTYPE, "%s: q, k and v must be F16 or BF16", who);
  if (d != 64 && d != 128) return fail(AEKV_ERR_UNSUPPORTED, "%s: head dim %d (64 or 128 supported)", who, d);
  if (B < 0 || E < 0 || n_q < 0 || n_k < 0 || heads < 1 || H < 1 || H % heads)
    return fail(AEKV_ERR_SHAPE, "%s: B=%lld E=%lld n_q=%lld n_k=%lld, and %lld query heads are no multiple of %lld KV heads", who,
                (long long)B, (long long)E, (long long)n_q, (long long)n_k, (long long)H, (long long)heads);
  if (n_q == 0) return AEKV_OK;
  if (!q || !out || (E > 0 && !cu_seqlens_k) || (n_k > 0 && (!k || !v))) return fail(AEKV_ERR_VALUE, "%s: null pointer", who);
  if (B == 0) return fail(AEKV_ERR_SHAPE, "%s: %lld queries in no sequence", who, (long long)n_q);
  if (!cu_seqlens_q && n_q != B) return fail(AEKV_ERR_SHAPE, "%s: without offsets every sequence has one query, got %lld for %lld", who, (long long)n_q, (long long)B);
  if (!states && E != B) return fail(AEKV_ERR_SHAPE, "%s: %lld sequences and %lld states need a list", who, (long long)B, (long long)E);
  if (!is_aligned(q, 16) || !is_aligned(k, 16) || !is_aligned(v, 16) || !is_aligned(out, 16) || (q_token_stride % 8) ||
      (q_head_stride % 8) || (k_token_stride % 8) || (k_head_stride % 8) || (v_token_stride % 8) || (v_head_stride % 8))
    return fail(AEKV_ERR_ALIGN, "%s: q, k and v rows and out must be 16-byte aligned", who);
  if (!cross_fits(B, E, n_q, n_k, H))
    return fail(AEKV_ERR_UNSUPPORTED, "%s: B=%lld E=%lld n_q=%lld n_k=%lld H=%lld exceed the grid", who, (long long)B, (long long)E,
                (long long)n_q, (long long)n_k, (long long)H);
  if (n_k < 2) k_token_stride = v_token_stride = d;  // (what no second row needs may be anything)
  // (rows that overlap: the range that ends a sequence's last row would let parts of further ones through, by a weight of 0)
  if (k_token_stride * 2 * 64 > 0x3fffffff || v_token_stride * 2 * 64 > 0x3fffffff || k_token_stride < d || v_token_stride < d)
    return fail(AEKV_ERR_UNSUPPORTED, "%s: token strides of %lld and %lld elements", who, (long long)k_token_stride, (long long)v_token_stride);
  const CrossPlan plan = plan_cross(B, E, n_q, n_k, H, heads, d);
  const size_t want = aekv_cross_attention_workspace_size(B, E, n_q, n_k, H, heads, d);
  if (want && (!ws || ws_bytes < want)) return fail(AEKV_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, got %zu", who, want, ws_bytes);
  if (!is_aligned(ws, 16)) return fail(AEKV_ERR_ALIGN, "%s: workspace must be 16-byte aligned", who);
  const bool none = softmax_scale != softmax_scale;
  CrossArgs a{};
  a.q = static_cast<const uint16_t*>(q), a.k = static_cast<const uint16_t*>(k), a.v = static_cast<const uint16_t*>(v);
  a.q_token = q_token_stride, a.q_head = q_head_stride, a.k_token = k_token_stride, a.k_head = k_head_stride, a.v_token = v_token_stride, a.v_head = v_head_stride;
  a.cu_q = cu_seqlens_q, a.cu_k = cu_seqlens_k, a.states = states, a.sink = sink, a.out = static_cast<uint16_t*>(out), a.lse = lse;
  a.n_q = static_cast<int32_t>(n_q), a.n_k = static_cast<int32_t>(n_k), a.B = static_cast<int32_t>(B), a.E = static_cast<int32_t>(E);
  a.H = static_cast<int32_t>(H), a.heads = static_cast<int32_t>(heads), a.G = static_cast<int32_t>(H / heads), a.clear = clear_rest;
  a.scale2 = none ? 1.0f : fmaxf(fabsf(softmax_scale) * kLog2e, 0x1p-126f), a.flip = softmax_scale < 0.0f ? 0x80008000u : 0u, a.nan = none ? 0x7fff7fffu : 0u;
  const hipStream_t st = as_stream(stream);
  a.desc = static_cast<LineTile*>(ws);
  a.part = reinterpret_cast<float*>(static_cast<char*>(ws) + plan.groups * sizeof(LineTile));
  a.least = plan.least, a.share = plan.share;
  const uint32_t groups = static_cast<uint32_t>(plan.groups);
  for (int64_t b0 = 0; b0 < B; b0 += kTable) {
    a.b0 = static_cast<int32_t>(b0), a.nb = static_cast<int32_t>(B - b0 < kTable ? B - b0 : kTable);
    hipLaunchKernelGGL(pick_cross(dtype, d, plan.rows, false), dim3(groups), dim3(256), 0, st, a);
    if (const int rc = check_launch(who)) return rc;
    if (groups == 1) continue;
    hipLaunchKernelGGL(pick_cross(dtype, d, plan.rows, true), dim3(groups - 1, static_cast<uint32_t>(ceil_div((plan.rows << plan.share) * d / 4, 256))), dim3(256), 0, st, a);
    if (const int rc = check_launch(who)) return rc;
  }
  return AEKV_OK;
}
