// The gated feed-forward block on fp16 parts: the products of large calls at a
// third of the fp16 MFMA rate, which is 16 times the fp32 one, with fp32's accuracy.
//
// A value x is kept as x 2^e = h + l / 2^11, two fp16 values rounded to nearest, and
// h h + (h l + l h) / 2^11 stands for a product.  The exponent e of a product's operand is one
// for each row (a token's values, an output's weights), or for each block of a row, such that
// the largest value lies in [2^14, 2^15): a value is then off by 2^-23 of itself, or by 2^-36,
// 2^-50 of the largest; values down to 2^-27 of that keep 24 bits (with exponents of blocks
// 2^-33, 2^-47 and 2^-24).  As factors of the product's rows and columns the exponents cost its
// loop nothing.  A matrix that is summed over its rows in one product and over its columns in
// another is split twice, with exponents each way.
//
// Smaller values still may be all that counts, where the other operand is zero at the large
// ones.  So a product looks at its results (`doubt`), and rows of a forward, or gradients, that
// parts may not hold are worked out again on fp32, by the launch that adds up the splits' sums.
//
// For x, dy and the weights a pass finds the maxima and another makes the parts; for Wg and Wu
// of a forward with few rows the second does both, tile by tile.  What a
// product leaves for the next one (m forward; dg, du, m backward) is split by its
// epilogue, which knows the largest value of its own tile's rows and columns only: the
// parts get that exponent, kept in a byte per row and tile, and the next product's loop takes
// them to that of the row's largest value by a power of two.  h of such parts is a multiple of
// 2^(kDown - 24), so that this rounds nothing; where more than 2^-kDown is asked for, the sums so
// far go to the block's exponent instead.
//
// The steps, forward:  maxima -> parts of x, Wg, Wu, Wd -> g, u and m's parts (one
// product over Wg and Wu, whose columns lie in turn, 32 by 32, so that a wave has g and
// u of one place) -> y.
// Backward:  maxima -> parts of dy, Wd, x, W -> dm, and from it parts of dg, du, m ->
// dx, dWg, dWu, dWd.
#include "dce_mlp.h"

namespace dce {

namespace {

constexpr int kT = 256;
constexpr int kTile = 128, kStep = 32;

using h8 = _Float16 __attribute__((ext_vector_type(8)));
using f16v = float __attribute__((ext_vector_type(16)));

inline uint32_t cdiv(uint64_t a, uint64_t b) { return uint32_t((a + b - 1) / b); }
inline uint32_t pad(uint32_t v, uint32_t to) { return (v + to - 1) / to * to; }

// The exponent for values of which the largest has this exponent field: it goes to
// [2^14, 2^15), unless it is below 2^-112 (2^127 is the largest factor).
__device__ __forceinline__ int exp_of(int field) { return min(141 - field, 127); }
__device__ __forceinline__ float pow2(int e) { return __int_as_float((127 + e) << 23); }
__device__ __forceinline__ int field_of(uint32_t bits) { return int(bits >> 23); }
// For a block: 0 is a block of zeros; values below 2^-126 have the exponent of those above.
__device__ __forceinline__ uint8_t block_field(uint32_t bits) { return uint8_t(bits ? max(field_of(bits), 1) : 0); }

// Parts in memory: 32 consecutive values of a row are 32 h, then 32 l (128 bytes).  x: 8
// values of the row at `to`, from value c on, times `by`.  DOWN: h is a multiple of 2^(DOWN - 24).
constexpr int kDown = 4;
template <int DOWN>
__device__ __forceinline__ void split8(const float* x, float by, h8& h, h8& l) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = x[i] * by;
    h[i] = _Float16(float(_Float16(v * (1.f / (1 << DOWN)))) * float(1 << DOWN));
    l[i] = _Float16((v - float(h[i])) * 2048.f);
  }
}
template <int DOWN = 0>
__device__ __forceinline__ void put8(float* to, uint32_t c, const float (&x)[8], float by) {
  h8 h, l;
  split8<DOWN>(x, by, h, l);
  h8* p = reinterpret_cast<h8*>(to + (c & ~31u)) + (c & 31u) / 8;
  p[0] = h;
  p[4] = l;
}
// |v| for a maximum: fmaxf drops NaN, which then counts as infinity.
__device__ __forceinline__ float size_of(float v) { return v == v ? fabsf(v) : INFINITY; }
// One operand of a product: [rows][depth] as parts.
struct Side {
  float* p;
  uint32_t* top;   // bits of the largest value of each row
  uint8_t* field;  // exponent field of the largest value of each row's block (block_field), [block][rows]; null: that of its row
  uint32_t rows, depth;
};

// A tile of 128 rows of COLS values in LDS, its octets of columns XORed by the octet of
// rows, so that neither a row's octets nor a column's meet in a bank often.  Rows of 128
// are in two arrays of 64 rows (a product's two stages), those of 64 in the first.
template <int COLS>
__device__ __forceinline__ float* tile_at(float* S0, float* S1, int r, int c) {
  float* S = COLS == 64 || r < 64 ? S0 : S1;
  return S + (COLS == 64 ? r : r & 63) * COLS + ((((c >> 3) ^ (r >> 3)) & (COLS / 8 - 1)) << 3) + (c & 7);
}
// Parts of its rows, with the exponents that they have in this tile, at row r0 and value c0 of t.
template <int COLS>
__device__ __forceinline__ void put_rows(float* S0, float* S1, const Side& t, uint32_t r0, uint32_t c0) {
  constexpr int OCT = COLS / 8;
  for (int u = threadIdx.x; u < 128 * OCT; u += kT) {
    const int r = u / OCT, o = u % OCT;
    const f4* p = reinterpret_cast<const f4*>(tile_at<COLS>(S0, S1, r, 8 * o));
    const f4 a = p[0], b = p[1];
    const float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, size_of(v[e]));
    m = group8_reduce(m, OpMaxR());
    if constexpr (OCT == 16) m = fmaxf(m, xl::dpp<xl::kRowMirror>(m));
    const uint32_t bits = __float_as_uint(m);
    put8<kDown>(t.p + size_t(r0 + r) * t.depth, c0 + 8 * o, v, pow2(exp_of(field_of(bits))));
    if (o == 0) {
      t.field[size_t(c0 / COLS) * t.rows + r0 + r] = block_field(bits);
      if (bits) atomicMax(t.top + r0 + r, bits);
    }
  }
}
// A column's place in a side where it lies in turn with those of another matrix.
__device__ __forceinline__ uint32_t in_turn(uint32_t c, int turn) {
  return turn < 0 ? c : (c >> 5) * 64 + uint32_t(turn) * 32 + (c & 31);
}
// Parts of a 128 x 128 tile's columns, likewise, at row c0 (in turn) and value r0 of t.
__device__ __forceinline__ void put_columns(float* S0, float* S1, const Side& t, uint32_t r0, uint32_t c0, int turn = -1) {
  for (int u = threadIdx.x; u < 128 * 16; u += kT) {
    const int c = u / 16, o = u % 16;
    const float* p = tile_at<128>(S0, S1, 8 * o, c);
    float v[8], m = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = p[e * 128];
      m = fmaxf(m, size_of(v[e]));
    }
    m = group8_reduce(m, OpMaxR());
    const uint32_t bits = __float_as_uint(fmaxf(m, xl::dpp<xl::kRowMirror>(m))), row = in_turn(c0 + c, turn);
    put8<kDown>(t.p + size_t(row) * t.depth, r0 + 8 * o, v, pow2(exp_of(field_of(bits))));
    if (o == 0) {
      t.field[size_t(r0 / 128) * t.rows + row] = block_field(bits);
      if (bits) atomicMax(t.top + row, bits);
    }
  }
}

// ---------------------------------------------------------------------------
// Maxima and parts of up to five matrices, [rows][cols].
// ---------------------------------------------------------------------------
struct Job {
  const float* src;
  uint32_t rows, cols;
  Side straight, across;  // of its rows, of its columns; p null: not wanted
  uint32_t c0;            // straight: the place of its columns
  int turn;               // across: 0, 1: its columns are those of Wg, Wu in turn; -1: no
  // (None where `across` has exponents of its blocks.)
  // Bits of the largest values of the rows in each workgroup's columns, [..][rows], and of
  // the columns in each one's rows, [..][cols]: `rowFrom` with those of the job that shares
  // the exponents (Wg and Wu have one for each row).
  uint32_t *rowPart, *colPart;
  const uint32_t* rowFrom;
  uint32_t rowCount, colCount;
};
constexpr int kJobs = 5;
struct Jobs {
  Job j[kJobs];
  uint32_t start[kJobs + 1];
  uint32_t count;
  uint32_t* clear;  // maxima that products will raise, `clears` of them
  uint32_t clears;
};
__device__ __forceinline__ int find_job(const Jobs& t, uint32_t blk) {
  int i = 0;
  while (i + 1 < int(t.count) && t.start[i + 1] <= blk) ++i;
  return i;
}
// 64 rows and 256 columns for each workgroup, 16 rows for each wave.  A width that is
// no multiple of 4 has its last quad end with the row.  Several such blocks for each, one
// after the other: of columns where rows alone are wanted (a row's values are brought
// together once), of rows where columns are and there are many.  The workgroups' largest values go
// side by side into memory and are brought together by k_mlp_split, for the 128 of its tile.
// (Atomics on one place take some 0.4 us after the other: 8192 x 128, 128 blocks of rows,
// 53 us.)  Bound by memory: of 8192 x 1024 x 4096 84 MB (x and three weights) 19 us, 117 MB backward 30.
constexpr uint32_t kMaxRows = 64, kMaxBlocks = 32;
struct Reach {
  uint32_t rows, cols;  // of a workgroup
};
__host__ __device__ inline Reach reach(uint32_t rows, bool across) {
  const uint32_t blocks = (rows + kMaxRows - 1) / kMaxRows;
  return across ? Reach{(blocks + kMaxBlocks - 1) / kMaxBlocks * kMaxRows, kT} : Reach{kMaxRows, 2 * kT};
}
__global__ void __launch_bounds__(kT) k_mlp_max(const Jobs t) {
  __shared__ uint32_t tops[4][kT];
  const int k = find_job(t, blockIdx.x);
  const Job J = t.j[k];
  for (uint32_t i = blockIdx.x * kT + threadIdx.x; i < t.clears; i += gridDim.x * kT) t.clear[i] = 0;
  const Reach by = reach(J.rows, J.across.p);
  const uint32_t wide = (J.cols + by.cols - 1) / by.cols, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const uint32_t id = blockIdx.x - t.start[k], first = id / wide * by.rows, c0 = id % wide * by.cols;
  float top[4] = {0.f, 0.f, 0.f, 0.f};
  for (uint32_t r0 = first + w * 16; r0 < min(first + by.rows, J.rows); r0 += kMaxRows) {
    float row[16];
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) row[i] = 0.f;
    for (uint32_t c1 = c0; c1 < min(c0 + by.cols, J.cols); c1 += kT) {
      const float* p = J.src + min(c1 + lane * 4, J.cols - 4);
      f4u v[16];
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i) v[i] = ldus<false, f4u>(p + size_t(min(r0 + i, J.rows - 1)) * J.cols);
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = size_of(v[i][e]);
          row[i] = fmaxf(row[i], x);
          top[e] = fmaxf(top[e], x);
        }
    }
    if (!J.straight.p) continue;
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) {
      const float m = wave_reduce(row[i], OpMaxR());
      if (lane == 0 && r0 + i < J.rows) J.rowPart[size_t(c0 / by.cols) * J.rows + r0 + i] = __float_as_uint(m);
    }
  }
  if (!J.across.p) return;
#pragma unroll
  for (int e = 0; e < 4; ++e) tops[w][lane * 4 + e] = __float_as_uint(top[e]);
  __syncthreads();
  // column threadIdx.x of the lanes' quads (two may be the same one)
  const uint32_t m = max(max(tops[0][threadIdx.x], tops[1][threadIdx.x]), max(tops[2][threadIdx.x], tops[3][threadIdx.x]));
  const uint32_t at = min(c0 + (threadIdx.x & ~3u), J.cols - 4) + (threadIdx.x & 3);
  J.colPart[size_t(first / by.rows) * J.cols + at] = m;
}

// A 128 x 128 tile through LDS, for the matrix' rows, its columns, or both at once, with
// the exponents of the rows and columns, or for the columns with those of the tile; a value is 4 bytes as it was.  Bound by memory: of 8192 x 1024 x 4096 84 MB in and 84 out
// forward, 34 us, 117 and 151 backward, 51 us, 5 TB/s.
__global__ void __launch_bounds__(kT) k_mlp_split(const Jobs t) {
  __shared__ __attribute__((aligned(16))) float S0[64 * 128];
  __shared__ __attribute__((aligned(16))) float S1[64 * 128];
  const int k = find_job(t, blockIdx.x);
  const Job J = t.j[k];
  const uint32_t tc = (J.cols + 127) / 128, id = blockIdx.x - t.start[k], i0 = id / tc * 128, j0 = id % tc * 128;
  // The rows' and columns' largest values; tiles at the edge leave them for the products.
  __shared__ uint32_t tops[256];
  const bool own = J.across.field;
  if (!own) {
    const uint32_t l = threadIdx.x & 127, r = i0 + l, c = j0 + l;
    uint32_t m = 0;
    if (threadIdx.x < 128) {
      if (J.straight.p && r < J.rows) {
#pragma unroll 4
        for (uint32_t i = 0; i < J.rowCount; ++i) m = max(m, J.rowFrom[size_t(i) * J.rows + r]);
      }
      if (J.straight.p && j0 == 0 && r < J.straight.rows) J.straight.top[r] = m;
    } else {
      if (J.across.p && c < J.cols) {
#pragma unroll 4
        for (uint32_t i = 0; i < J.colCount; ++i) m = max(m, J.colPart[size_t(i) * J.cols + c]);
      }
      if (J.across.p && i0 == 0 && in_turn(c, J.turn) < J.across.rows) J.across.top[in_turn(c, J.turn)] = m;
    }
    tops[threadIdx.x] = m;
  }
  {
    // a quad of 16 rows for each thread; the last one ends with the row, as above
    const uint32_t q = threadIdx.x & 31, c = j0 + q * 4, at = min(c, J.cols - 4), off = min(c - at, 4u);
    f4u v[16];
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i)
      v[i] = ldus<false, f4u>(J.src + size_t(min(i0 + (threadIdx.x >> 5) + 8 * i, J.rows - 1)) * J.cols + at);
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) {
      const uint32_t r = (threadIdx.x >> 5) + 8 * i;
      f4 x = {v[i][0], v[i][1], v[i][2], v[i][3]};
      if (off == 1) x = f4{x[1], x[2], x[3], 0.f};
      if (off == 2) x = f4{x[2], x[3], 0.f, 0.f};
      if (off == 3) x = f4{x[3], 0.f, 0.f, 0.f};
      if (off == 4 || i0 + r >= J.rows) x = f4{0.f, 0.f, 0.f, 0.f};
      *reinterpret_cast<f4*>(tile_at<128>(S0, S1, r, q * 4)) = x;
    }
  }
  __syncthreads();
  if (own) {
    put_columns(S0, S1, J.across, i0, j0, J.turn);
    return;
  }
  if (J.straight.p) {
    for (int u = threadIdx.x; u < 128 * 16; u += kT) {
      const int rl = u / 16, cl = u % 16 * 8;
      const uint32_t r = i0 + rl;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = tile_at<128>(S0, S1, rl, cl)[e];
      if (r < J.straight.rows && j0 + cl < J.straight.depth)
        put8(J.straight.p + size_t(r) * J.straight.depth, J.c0 + j0 + cl, v, pow2(exp_of(field_of(tops[rl]))));
    }
  }
  if (J.across.p) {
    for (int u = threadIdx.x; u < 128 * 16; u += kT) {
      const int cl = u / 16, rl = u % 16 * 8;
      const uint32_t c = in_turn(j0 + cl, J.turn), r = i0 + rl;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = tile_at<128>(S0, S1, rl, cl)[128 * e];
      if (c < J.across.rows && r < J.across.depth)
        put8(J.across.p + size_t(c) * J.across.depth, r, v, pow2(exp_of(field_of(tops[128 + cl]))));
    }
  }
}

// ---------------------------------------------------------------------------
// Products C = P Q^T of parts, both along their rows, in 128 x 128 tiles of four
// waves, 64 x 64 each (2 x 2 blocks of 32 x 32).  The depth goes in steps of 32 through
// two LDS stages, the next one's direct loads in flight while one is read and multiplied.  A
// stage's rows are eight 16-byte slots, four of h and four of l, XORed by the row
// so that a read of one slot of 16 rows covers the 64 banks once.  The two small
// products have an accumulator of their own: an MFMA cuts what it adds off at the
// scale of the largest addend, always downwards.
//
// An operand with exponents of its blocks is q, whose rows are the lanes' columns: sums that go
// to another exponent are multiplied by one power of two for each.  (Done for every block, instead of
// its fragments, that took the four products from 960 to 1150 us.)
//
// Bound by the MFMAs, for which power holds the clock to 1.7 GHz.  8192 x 1024 x 4096, in us
// and TFLOP/s of fp32 products (a large fp16 library product, divided by three: 374): g and u 421,
// 326; y 216, 318; dx, dWd, dWg and dWu 1000, 344; dm 390, 176, of which its epilogue, which reads
// 8 bytes a hidden value and writes 20, takes more than half.  The look at the results is 1 to 2 us of
// a tile's.  Two workgroups a CU, of 64 KB and some 200 to 220 registers a lane.  With one array for both stages every read waited for the loads
// (2.19 ms for 2.14 of a training pass).
// ---------------------------------------------------------------------------
enum Op { STORE, GATE, BLOCK_GATE, GRAD };  // STORE, BLOCK_GATE: q's parts have exponents of its blocks
struct Prod {
  Side p, q;
  uint32_t flip;           // STORE: the result's rows are q's, else p's
  uint32_t tm, tn, depth;  // tiles; values of a row that are multiplied
  uint32_t block;          // values of a block of q (a power of two)
  uint32_t rows, cols;     // of the result
  uint32_t *any, *again;   // set where fp32 is to work it out: something, and the results' rows (null: all of it)
  float* out;              // STORE
  float* part;             // splits > 1: their shares of out, one after the other
  uint32_t splits;         // of the depth
  float *g, *u;            // GATE: kept (null: not); GRAD: read
  uint32_t hidden;         // their pitch
  uint32_t start;          // STORE: the first workgroup
  Side m, mc, dr, dgc, duc;  // GATE: m; GRAD: m's columns (p null: not wanted), rows of dg and du, their columns
};

// Up to four products of one launch.
template <int N>
struct Prods {
  Prod a[N];
  uint32_t count;
};

constexpr int kStageBytes = kTile * kStep * 4;
__device__ __forceinline__ int swz(int row) { return (row >> 1) & 7; }
__device__ __forceinline__ void load_stage(const BRes& b, uint32_t pitchBytes, uint32_t k, char* S) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
  for (int i = 0; i < kStageBytes / 16 / kT; ++i) {
    const uint32_t slot = threadIdx.x + kT * i, row = slot / 8, c = (slot % 8) ^ swz(row);
    b.ld16_lds(row * pitchBytes + k * 4 + c * 16, S + (wave * 64 + i * kT) * 16);
  }
}
__device__ __forceinline__ h8 frag(const char* S, int row, int c) {
  return *reinterpret_cast<const h8*>(S + (row * 8 + (c ^ swz(row))) * 16);
}
// Blocks that much smaller than their row are left out: 2^37 2^-60 of a block of 128 terms at most, for
// which there is room wherever results are kept.
constexpr int kApart = 60;
// What a common exponent may add to the error of a product's result: max(4, sqrt(K) / 4) times 2^-24 of S, the
// sum of its K terms' absolute values, less than fp32's own roundings make of them.  With the scaled operands
// a, b, a value of which is off by 2^-36 (2^-33 of blocks) beside fp32's own rounding, it adds 2^-36 (sum |b| +
// sum |a|), or 8 sum |a|.  Values are below 2^15: that is 4 times 2^-24 of S, or less, where S is K kLeast.
template <bool SCALED>
constexpr float kLeast = (SCALED ? 8 + 1 : 1 + 1) * 8 / 4.f;  // 2^15 2^-36 / 2^-24 = 8
// S is at least |result|, and about a quarter of the small products' sum (|l| <= |h| but for values below
// 2^(kDown - 14), which leave no more than 2^(kDown + 1) + 2 < 2 kLeast of a term in it): half of what `size` adds
// up.  Each has a sign of its own, so this is enough for all but one result in 2^24 of normal operands (|result|
// alone: the four products take 50 us more of 960).
// For result (i, j) of the product, by one wave: is S, added up from the parts?
template <bool SCALED>
__device__ __forceinline__ bool held(const Prod& a, uint32_t i, uint32_t j, int top, uint32_t k0, uint32_t k1) {
  const _Float16* p = reinterpret_cast<const _Float16*>(a.p.p + size_t(i) * a.p.depth);
  const _Float16* q = reinterpret_cast<const _Float16*>(a.q.p + size_t(j) * a.q.depth);
  float S = 0.f, L = 0.f;
#pragma unroll 4
  for (uint32_t k = k0 + (threadIdx.x & 63) * 8; k < k1; k += 512) {
    const uint32_t at = (k & ~31u) * 2 + (k & 31);  // h, l 32 halves on
    const h8 ph = *reinterpret_cast<const h8*>(p + at), pl = *reinterpret_cast<const h8*>(p + at + 32);
    const h8 qh = *reinterpret_cast<const h8*>(q + at), ql = *reinterpret_cast<const h8*>(q + at + 32);
    float f = 1.f, drop = 0.f;
    if constexpr (SCALED) {
      const uint8_t field = a.q.field[size_t(k / a.block) * a.q.rows + j];
      if (!field) continue;
      f = ldexpf(1.f, top - exp_of(field));
      if (exp_of(field) > top + kApart) drop = 0x1p36f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = fabsf(float(ph[e]) + float(pl[e]) / 2048.f), y = fabsf(float(qh[e]) + float(ql[e]) / 2048.f) * f;
      S += drop ? 0.f : x * y;
      L += (SCALED ? 8.f : 1.f) * x * f + y + drop * (x * y);
    }
  }
  return wave_reduce(S) * (4096.f * fmaxf(4.f, 0.25f * sqrtf(float(k1 - k0)))) >= wave_reduce(L);
}

template <Op OP, MlpAct ACT, int N, bool NT>
__global__ void __launch_bounds__(kT) __attribute__((amdgpu_waves_per_eu(2))) k_mlp_product(const Prods<N> all) {
  constexpr bool SCALED = OP == STORE || OP == BLOCK_GATE;
  int which = 0;
  if constexpr (N > 1)
    while (which + 1 < int(all.count) && all.a[which + 1].start <= blockIdx.x) ++which;
  const Prod& a = all.a[which];
  // An array for each stage: the compiler then knows that a direct load into one is
  // nothing that a read of the other has to wait for.
  __shared__ __attribute__((aligned(16))) char S0[2 * kStageBytes];
  __shared__ __attribute__((aligned(16))) char S1[2 * kStageBytes];
  // bands of 8 rows of tiles: what an XCD runs at once reads few rows of either side
  uint32_t id = xcd_place(blockIdx.x - a.start, a.tm * a.tn * a.splits), sp = 0, k0 = 0, k1 = a.depth;
  if constexpr (OP == STORE) {
    const uint32_t blocks = a.depth / kTile;
    sp = id / (a.tm * a.tn);
    id -= sp * a.tm * a.tn;
    k0 = blocks * sp / a.splits * kTile;
    k1 = blocks * (sp + 1) / a.splits * kTile;
  }
  const uint32_t band = id / (8 * a.tn), in = id - band * 8 * a.tn, high = min(8u, a.tm - band * 8);
  const uint32_t tj = in / high, ti = band * 8 + (in - tj * high);
  BRes bp, bq;
  bp.init(a.p.p + size_t(ti) * kTile * a.p.depth, kTile * a.p.depth);
  bq.init(a.q.p + size_t(tj) * kTile * a.q.depth, kTile * a.q.depth);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
  const int col = lane & 31, half = lane >> 5;
  f16v big[2][2], small[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) big[i][j][e] = small[i][j][e] = 0.f;
  // This lane's columns: the exponents of their largest values, those that the sums are in, and the
  // block's factors towards them.
  const uint32_t qrow = tj * kTile + wn + col;
  uint32_t qtop[2];
  int own[2], now[2];
  uint8_t next[2] = {};
  _Float16 by[2] = {};
  auto fetch_next = [&](uint32_t k) {
#pragma unroll
    for (int j = 0; j < 2; ++j) next[j] = a.q.field[size_t(min(k, k1 - 1) / a.block) * a.q.rows + qrow + 32 * j];
  };
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    qtop[j] = a.q.top[qrow + 32 * j];
    own[j] = now[j] = exp_of(field_of(qtop[j]));
  }
  if constexpr (SCALED) fetch_next(k0);
  load_stage(bp, a.p.depth * 4, k0, S0);
  load_stage(bq, a.q.depth * 4, k0, S0 + kStageBytes);
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  // To the block at k.
  auto enter = [&](uint32_t k) __attribute__((always_inline)) {
    int d[2];
    bool out[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int e = exp_of(next[j]);
      out[j] = e > own[j] + kApart;
      d[j] = next[j] && !out[j] ? e - now[j] : 0;
    }
    if (__any(uint32_t(d[0]) > uint32_t(kDown) || uint32_t(d[1]) > uint32_t(kDown))) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int by = uint32_t(d[j]) > uint32_t(kDown) ? d[j] : 0;
        const float f = pow2(by);
        now[j] += by;
        d[j] -= by;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int t = 0; t < 16; ++t) {
            big[i][j][t] *= f;
            small[i][j][t] *= f;
          }
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) by[j] = out[j] ? _Float16(0.f) : _Float16(pow2(-d[j]));
    fetch_next(k + a.block);
  };
  auto step = [&](uint32_t k, const char* St, char* Sn) {
    if (k + kStep < k1) {
      load_stage(bp, a.p.depth * 4, k + kStep, Sn);
      load_stage(bq, a.q.depth * 4, k + kStep, Sn + kStageBytes);
    }
    h8 p[2][2][2], q[2][2][2];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          p[kk][i][e] = frag(St, wm + 32 * i + col, 4 * e + 2 * kk + half);
          q[kk][i][e] = frag(St + kStageBytes, wn + 32 * i + col, 4 * e + 2 * kk + half);
        }
    if constexpr (SCALED) {
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) q[kk][j][e] *= by[j];
    }
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          big[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[kk][i][0], q[kk][j][0], big[i][j], 0, 0, 0);
          small[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[kk][i][0], q[kk][j][1], small[i][j], 0, 0, 0);
          small[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[kk][i][1], q[kk][j][0], small[i][j], 0, 0, 0);
        }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
  };
  for (uint32_t k = k0; k < k1; k += 2 * kStep) {  // the depth is a multiple of 128
    if constexpr (SCALED)
      if ((k & (a.block - 1)) == 0) enter(k);
    step(k, S0, S1);
    step(k + kStep, S1, S0);
  }
  // Row 8 (e / 4) + 4 half + e % 4 of a block, column `col`.
  const uint32_t r0 = ti * kTile, c0 = tj * kTile;
  float *T0 = reinterpret_cast<float*>(S0), *T1 = reinterpret_cast<float*>(S1);
  auto row_of = [&](int i, int e) { return r0 + wm + 32 * i + 8 * (e >> 2) + 4 * half + (e & 3); };
  float low[2] = {INFINITY, INFINITY}, least[2];
  uint32_t top[2][16], least_top = ~0u, none = 0;  // none: a bit for each row of p that is zeros
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) top[i][e] = a.p.top[row_of(i, e)];
  auto size = [&](int i, int j, int e) { return fmaf(0.25f, fabsf(small[i][j][e]), fabsf(big[i][j][e])); };
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      least_top = min(least_top, top[i][e]);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        big[i][j][e] += small[i][j][e] * (1.f / 2048.f);
        low[j] = fminf(low[j], size(i, j, e));
      }
    }
  if (__any(least_top == 0)) {
    low[0] = low[1] = INFINITY;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        none |= uint32_t(top[i][e] == 0) << (16 * i + e);
#pragma unroll
        for (int j = 0; j < 2; ++j) low[j] = fminf(low[j], top[i][e] ? size(i, j, e) : INFINITY);
      }
  }
  bool sure = true;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    least[j] = float(k1 - k0) * (2.f * kLeast<SCALED>) * (SCALED ? pow2(now[j] - own[j]) : 1.f);
    sure = sure && (qtop[j] == 0 || low[j] >= least[j]);
  }
  // Which of a wave's results parts may not hold: not those of rows of zeros, and rows that are not finite are left at that.
  auto doubt = [&]() __attribute__((always_inline)) {
    uint32_t pend[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        if (top[i][e] == 0 || top[i][e] >= 0x7f800000u) continue;
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (!(size(i, j, e) >= least[j])) pend[j] |= 1u << (16 * i + e);
      }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      bool zeros = qtop[j] == 0;
      if constexpr (SCALED) {
        zeros = true;  // in this split of the depth
        for (uint32_t b = k0 / a.block; b < k1 / a.block; ++b) zeros = zeros && a.q.field[size_t(b) * a.q.rows + qrow + 32 * j] == 0;
      }
      if (zeros || qtop[j] >= 0x7f800000u) pend[j] = 0;
    }
    const bool flip = OP == STORE && a.flip;
    uint32_t looks = 128;
#pragma unroll
    for (int j = 0; j < 2; ++j)
      for (uint64_t m = __ballot(pend[j] != 0); m; m = __ballot(pend[j] != 0)) {
        if (!looks--) {  // many: all of them
          *a.any = 1;
          if (a.again) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int e = 0; e < 16; ++e)
#pragma unroll
                for (int t = 0; t < 2; ++t)
                  if (t >= j && (pend[t] >> (16 * i + e) & 1)) a.again[flip ? qrow + 32 * t : row_of(i, e)] = 1;
          }
          return;
        }
        const int l = __builtin_ctzll(m);
        const uint32_t bit = __builtin_ctz(xl::rdl32(pend[j], l));
        if (lane == l) pend[j] &= pend[j] - 1;
        const uint32_t pr = r0 + wm + 32 * (bit >> 4) + 8 * ((bit >> 2) & 3) + 4 * (l >> 5) + (bit & 3), qr = tj * kTile + wn + 32 * j + (l & 31);
        if (held<SCALED>(a, pr, qr, int(xl::rdl32(uint32_t(own[j]), l)), k0, k1)) continue;
        *a.any = 1;
        if (!a.again) return;
        a.again[flip ? qr : pr] = 1;  // the row's others need no look
        if (flip) {
          if (col == (l & 31)) pend[j] = 0;
        } else if (half == l >> 5) {
          pend[0] &= ~(1u << bit);
          pend[1] &= ~(1u << bit);
        }
      }
  };
  if (!__all(sure)) doubt();
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int ep = exp_of(field_of(top[i][e]));
#pragma unroll
      for (int j = 0; j < 2; ++j) big[i][j][e] = ldexpf(big[i][j][e], -(ep + now[j]));
    }
  if constexpr (OP == STORE) {
    float* out = a.splits > 1 ? a.part + size_t(sp) * a.rows * a.cols : a.out;
    if (a.flip) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            const uint32_t r = qrow + 32 * j, n = row_of(i, e);
            float* to = out + size_t(r) * a.cols + n;
            if (r < a.rows && n + 3 < a.cols) {
              stus<false>(to, f4u{big[i][j][e], big[i][j][e + 1], big[i][j][e + 2], big[i][j][e + 3]});
            } else if (r < a.rows) {
#pragma unroll
              for (int t = 0; t < 3; ++t)
                if (n + t < a.cols) to[t] = big[i][j][e + t];
            }
          }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint32_t r = row_of(i, e);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t n = qrow + 32 * j;
            if (r < a.rows && n < a.cols) out[size_t(r) * a.cols + n] = big[i][j][e];
          }
        }
    }
  }
  if constexpr (OP == GATE || OP == BLOCK_GATE) {
    const uint32_t f = ((c0 + wn) >> 1) + col;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint32_t r = r0 + wm + 32 * i + 8 * (e >> 2) + 4 * half + (e & 3);
        if (a.g && r < a.rows && f < a.hidden) {
          stus<NT>(a.g + size_t(r) * a.hidden + f, float(big[i][0][e]));
          stus<NT>(a.u + size_t(r) * a.hidden + f, float(big[i][1][e]));
        }
        *tile_at<64>(T0, T1, wm + 32 * i + 8 * (e >> 2) + 4 * half + (e & 3), (wn >> 1) + col) = act<ACT>(big[i][0][e]) * big[i][1][e];
      }
    __syncthreads();
    put_rows<64>(T0, T1, a.m, r0, c0 / 2);
  }
  if constexpr (OP == GRAD) {
    // g and u, zeros outside, where dm is zeros too (or its row has no value that counts).
    f16v u[2][2];
    const uint32_t at[2] = {c0 + wn + col < a.hidden ? (wm + 4 * half) * a.hidden + c0 + wn + col : kOob,
                            c0 + wn + 32 + col < a.hidden ? (wm + 4 * half) * a.hidden + c0 + wn + 32 + col : kOob};
    BRes bg, bu;
    bg.init(a.g + size_t(r0) * a.hidden, min(a.rows - r0, 128u) * a.hidden);
    bu.init(a.u + size_t(r0) * a.hidden, min(a.rows - r0, 128u) * a.hidden);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e)
#pragma unroll
        for (int j = 0; j < 2; ++j) {  // small: g
          const uint32_t off = at[j] + (32 * i + 8 * (e >> 2) + (e & 3)) * a.hidden;
          small[i][j][e] = NT ? bg.ld1nt(off) : bg.ld1(off);
          u[i][j][e] = NT ? bu.ld1nt(off) : bu.ld1(off);
        }
    // big: dm, then dg; small: g, then du; u, then m
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float d;
          const float y = act_grad<ACT>(small[i][j][e], d), dm = big[i][j][e], v = u[i][j][e];
          float dg = dm * v * d, du = dm * y, m = y * v;
          // Here and now: put off to where they are stored, they keep more alive than there are registers.
          asm volatile("" : "+v"(dg), "+v"(du), "+v"(m));
          big[i][j][e] = dg;
          small[i][j][e] = du;
          u[i][j][e] = m;
        }
    if (__any(none != 0)) {  // a token without a gradient has no part in dWd: its m, however large, is none (not finite: NaN)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            if (none >> (16 * i + e) & 1) u[i][j][e] *= 0.f;
    }
    auto tile = [&](const f16v (&v)[2][2]) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e)
#pragma unroll
          for (int j = 0; j < 2; ++j) *tile_at<128>(T0, T1, wm + 32 * i + 8 * (e >> 2) + 4 * half + (e & 3), wn + 32 * j + col) = v[i][j][e];
      __syncthreads();
    };
    tile(big);
    if (a.dr.p) put_rows<128>(T0, T1, a.dr, r0, c0);
    if (a.dgc.p) put_columns(T0, T1, a.dgc, r0, c0);
    tile(small);
    if (a.dr.p) put_rows<128>(T0, T1, a.dr, r0, a.dr.depth / 2 + c0);
    if (a.duc.p) put_columns(T0, T1, a.duc, r0, c0);
    if (!a.mc.p) return;
    tile(u);
    put_columns(T0, T1, a.mc, r0, c0);
  }
}

// Places in the workspace.
struct Places {
  size_t next = 0;
  size_t take(size_t floats) {
    const size_t p = next;
    next += (floats + 63) & ~size_t(63);
    return p;
  }
};

// The sides of a call's products, of whole tiles, and the passes that make the first ones.
struct Plan {
  Places at;
  size_t tops = 0, raised = 0;  // maxima, of which so many that products raise come first
  struct Made {
    Side* s;
    size_t p, top, field;
  };
  Made all[16];
  int count = 0;
  Jobs jobs{};
  size_t parts = 0;  // floats of the jobs' partial maxima
  // Of a product's result (with blocks of so many values, which come first), or of a matrix.
  void side(Side& s, uint32_t rows, uint32_t depth, uint32_t block = 0) {
    s.rows = rows;
    s.depth = depth;
    all[count++] = {&s, at.take(size_t(rows) * depth), tops, block ? at.take((size_t(rows) * (depth / block) + 3) / 4) : ~size_t(0)};
    tops += rows;
    if (block) raised = tops;
  }
  // Words that products set (after the sides of blocks, which come first).
  size_t words = 0;
  void flags(uint32_t n) {
    words = tops;
    tops += n;
    raised = tops;
  }
  // A matrix whose parts are to be made, of its rows or columns; both sides may still lack their places.
  struct Source {
    const float* src;
    uint32_t rows, cols;
    const Side *straight, *across;
    uint32_t c0;
    int turn;
  };
  Source sources[kJobs];
  uint32_t maxima = 0;  // the first so many have a pass over their largest values
  bool blocks(const Side* s) const {
    for (int i = 0; i < count; ++i)
      if (all[i].s == s) return all[i].field != ~size_t(0);
    return false;
  }
  void add(const float* src, uint32_t rows, uint32_t cols, const Side* straight, const Side* across, uint32_t c0 = 0, int turn = -1) {
    sources[jobs.count++] = {src, rows, cols, straight, across, c0, turn};
    if (across && blocks(across)) return;
    maxima = jobs.count;
    const Reach by = reach(rows, across);
    if (straight) parts += size_t(cdiv(cols, by.cols)) * rows;
    if (across) parts += size_t(cdiv(rows, by.rows)) * cols;
  }
  // The workspace, room for `more` floats at *extra, and the jobs.  `free`: what is there for fp32 when
  // the products are done, up to the sides' end, `least` floats.
  float* free;
  uint32_t* flag;
  bool lay(size_t more, float** extra, size_t least) {
    at.next = std::max(at.next, (least + 63) & ~size_t(63));
    const size_t first = at.take(tops), tail = at.take(more), part = at.take(parts);
    float* ws = workspace(at.next);
    if (!ws) return false;
    *extra = ws + tail;
    free = ws;
    flag = reinterpret_cast<uint32_t*>(ws + first) + words;
    for (int i = 0; i < count; ++i) {
      Side& s = *all[i].s;
      s.p = ws + all[i].p;
      s.top = reinterpret_cast<uint32_t*>(ws + first) + all[i].top;
      s.field = all[i].field == ~size_t(0) ? nullptr : reinterpret_cast<uint8_t*>(ws + all[i].field);
    }
    jobs.clear = reinterpret_cast<uint32_t*>(ws + first);
    jobs.clears = uint32_t(raised);
    uint32_t* next = reinterpret_cast<uint32_t*>(ws + part);
    for (uint32_t i = 0; i < jobs.count; ++i) {
      const Source& f = sources[i];
      Job& j = jobs.j[i];
      j.src = f.src;
      j.rows = f.rows;
      j.cols = f.cols;
      if (f.straight) j.straight = *f.straight;
      if (f.across) j.across = *f.across;
      j.c0 = f.c0;
      j.turn = f.turn;
      if (j.across.field) continue;
      const Reach by = reach(f.rows, f.across);
      if (f.straight) {
        const uint32_t n = cdiv(f.cols, by.cols);
        j.rowPart = next;
        next += size_t(n) * f.rows;
        j.rowFrom = j.rowPart;
        j.rowCount = n;
        if (i && sources[i - 1].straight == f.straight) {  // behind the other's
          Job& o = jobs.j[i - 1];
          o.rowCount += n;
          j.rowFrom = o.rowFrom;
          j.rowCount = o.rowCount;
        }
      }
      if (f.across) {
        j.colPart = next;
        j.colCount = cdiv(f.rows, by.rows);
        next += size_t(j.colCount) * f.cols;
      }
    }
    return true;
  }
};

// The first `maxima` of the jobs, which take their largest values beforehand, come first.
bool run_jobs(Jobs& t, uint32_t maxima) {
  uint32_t n = 0;
  for (uint32_t i = 0; i < maxima; ++i) {
    t.start[i] = n;
    const Reach by = reach(t.j[i].rows, t.j[i].across.p);
    n += cdiv(t.j[i].rows, by.rows) * cdiv(t.j[i].cols, by.cols);
  }
  const uint32_t count = t.count;
  t.count = maxima;
  hipLaunchKernelGGL(k_mlp_max, dim3(n), dim3(kT), 0, stream(), t);
  t.count = count;
  if (!check_launch("gated_mlp")) return false;
  n = 0;
  for (uint32_t i = 0; i < t.count; ++i) {
    t.start[i] = n;
    n += cdiv(std::max(t.j[i].straight.p ? t.j[i].straight.rows : 0, t.j[i].across.p ? t.j[i].across.depth : 0), 128) * cdiv(t.j[i].cols, 128);
  }
  hipLaunchKernelGGL(k_mlp_split, dim3(n), dim3(kT), 0, stream(), t);
  return check_launch("gated_mlp");
}
// Splits of the depths: no workgroup has more than a slot's share of the launch (two a CU),
// or `kSplitLeast` where that is more (backward us with 256, 512, 1024 and 2048, 1024 x 1024 x 4096
// 229, 226, 235 and 232, 400 x 512 x 2048 91, 83, 87 and 107, 256 x 1024 x 2816 113, 112, 109 and
// 126).  Floats of their shares.
constexpr uint32_t kSplitLeast = 512;
template <int N>
size_t split(Prods<N>& t) {
  double all = 0;
  for (uint32_t i = 0; i < t.count; ++i) all += double(t.a[i].p.rows / kTile) * (t.a[i].q.rows / kTile) * t.a[i].depth;
  const double most = std::max<double>(kSplitLeast, all / (2 * num_cus()));
  size_t floats = 0;
  for (uint32_t i = 0; i < t.count; ++i) {
    Prod& a = t.a[i];
    a.splits = std::min(uint32_t(std::ceil(a.depth / most)), a.depth / kTile);
    if (a.splits > 1) floats += (size_t(a.splits) * a.rows * a.cols + 63) & ~size_t(63);
  }
  return floats;
}
// `bytes`: what the launch reads and writes but once (of 4.0e8, g and u: nontemporal accesses
// to them take the gate's product from 454 to 438 us, of 9.4e8 the gradient's from 407 to 377).
// `sums`: what the splits leave to be added up.
template <Op OP, int N>
bool run_products(Prods<N>& t, MlpAct act = kSilu, float* part = nullptr, double bytes = 0, MlpSums* sums = nullptr) {
  uint32_t n = 0;
  for (uint32_t i = 0; i < t.count; ++i) {
    Prod& a = t.a[i];
    a.tm = a.p.rows / kTile;
    a.tn = a.q.rows / kTile;
    a.start = n;
    a.splits = std::max(a.splits, 1u);
    n += a.tm * a.tn * a.splits;
    if (a.splits == 1) continue;
    a.part = part;
    const size_t values = size_t(a.rows) * a.cols;
    part += (size_t(a.splits) * values + 63) & ~size_t(63);
    sums->add(a.part, a.out, uint32_t(values), a.splits);
  }
  by_act(act, [&](auto k) {
    constexpr MlpAct A = OP == STORE ? kSilu : decltype(k)::value;
    if (OP != STORE && stream_nt(bytes))
      hipLaunchKernelGGL((k_mlp_product<OP, A, N, OP != STORE>), dim3(n), dim3(kT), 0, stream(), t);
    else
      hipLaunchKernelGGL((k_mlp_product<OP, A, N, false>), dim3(n), dim3(kT), 0, stream(), t);
  });
  return check_launch("gated_mlp");
}
template <int N>
void add(Prods<N>& t, const Side& p, const Side& q, bool flip, uint32_t block, uint32_t rows, uint32_t cols, float* out) {
  Prod& a = t.a[t.count++];
  a.p = p;
  a.q = q;
  a.flip = flip;
  a.depth = p.depth;
  a.block = block;
  a.rows = rows;
  a.cols = cols;
  a.out = out;
}

}  // namespace

bool mlp_forward_parts(const MlpArgs& a) {
  const uint32_t M = pad(a.rows, kTile), C = pad(a.cols, kTile), F = pad(a.hidden, kTile), O = pad(a.out, kTile);
  Plan plan;
  Side x{}, w{}, d{}, m{};
  // A pass over the weights' largest values less, and exponents of their blocks in the product's
  // loop: worth it for few rows (forward us with and without the pass, 200 x 2048 x 8192 240 and
  // 208, 700 x 1024 x 4096 117 and 116, 4096 x 1024 x 2816 263 and 266, 8192 x 1024 x 4096 640
  // and 650).
  const bool blocks = a.rows <= 2048;
  plan.side(m, M, F, 64);
  plan.flags(3 + M);
  plan.side(w, 2 * F, C, blocks ? 128 : 0);
  plan.side(x, M, C);
  plan.side(d, O, F);
  plan.add(a.x, a.rows, a.cols, &x, nullptr);
  plan.add(a.wd, a.hidden, a.out, nullptr, &d);
  plan.add(a.wg, a.cols, a.hidden, nullptr, &w, 0, 0);
  plan.add(a.wu, a.cols, a.hidden, nullptr, &w, 0, 1);
  ProfScope prof("mlp_parts", 6.0 * a.rows * a.cols * a.hidden, 4.0 * (2.0 * a.rows * a.cols + 3.0 * a.cols * a.hidden));
  // The second product's sides get their places with the others.
  Prods<1> t1{}, t2{};
  add(t2, d, m, true, 64, a.rows, a.out, a.y);
  float* part;
  if (!plan.lay(split(t2), &part, size_t(a.rows) * a.hidden)) return false;
  t2.a[0].p = d;
  t2.a[0].q = m;
  t2.a[0].any = plan.flag;
  t2.a[0].again = plan.flag + 3;
  if (!run_jobs(plan.jobs, plan.maxima)) return false;
  t1.count = 1;
  Prod& g = t1.a[0];
  g.p = x;
  g.q = w;
  g.block = 128;
  g.depth = C;
  g.rows = a.rows;
  g.m = m;
  g.any = plan.flag;
  g.again = plan.flag + 3;
  g.hidden = a.hidden;
  if (a.saved) {
    g.g = a.saved;
    g.u = a.saved + size_t(a.rows) * a.hidden;
  }
  const double bytes = (a.saved ? 12.0 : 4.0) * M * F;
  if (!(blocks ? run_products<BLOCK_GATE>(t1, a.act, nullptr, bytes) : run_products<GATE>(t1, a.act, nullptr, bytes))) return false;
  MlpSums sums{};
  return run_products<STORE>(t2, kSilu, part, 0, &sums) && mlp_forward_again(a, {plan.flag, plan.flag + 3, plan.flag + 1, plan.free}, sums);
}

bool mlp_backward_parts(const MlpArgs& a, const float* dy, float* dx, float* dwg, float* dwu, float* dwd) {
  const uint32_t M = pad(a.rows, kTile), C = pad(a.cols, kTile), F = pad(a.hidden, kTile), O = pad(a.out, kTile);
  Plan plan;
  Side yr{}, yc{}, d{}, xc{}, w{}, dr{}, dgc{}, duc{}, mc{};
  if (dx) plan.side(dr, M, 2 * F, 128);
  if (dwd) plan.side(mc, F, M, 128);
  if (dwg) plan.side(dgc, F, M, 128);
  if (dwu) plan.side(duc, F, M, 128);
  plan.flags(3);
  plan.side(yr, M, O);
  plan.side(d, F, O);
  if (dwd) plan.side(yc, O, M);
  if (dwg || dwu) plan.side(xc, C, M);
  if (dx) plan.side(w, C, 2 * F);
  plan.add(dy, a.rows, a.out, &yr, dwd ? &yc : nullptr);
  plan.add(a.wd, a.hidden, a.out, &d, nullptr);
  if (dwg || dwu) plan.add(a.x, a.rows, a.cols, nullptr, &xc);
  if (dx) {
    plan.add(a.wg, a.cols, a.hidden, &w, nullptr, 0);
    plan.add(a.wu, a.cols, a.hidden, &w, nullptr, F);
  }
  ProfScope prof("mlp_parts", 12.0 * a.rows * a.cols * a.hidden, 8.0 * (2.0 * a.rows * a.cols + 3.0 * a.cols * a.hidden));
  // All that follow dm's in one launch, the deepest first: a last round of few workgroups
  // instead of four.  Twice: their sizes first, their places once they have them.
  Prods<4> t2{};
  auto rest = [&] {
    const Prods<4> had = t2;
    t2 = {};
    if (dx && 2 * F >= M) add(t2, w, dr, true, 128, a.rows, a.cols, dx);
    if (dwd) add(t2, yc, mc, true, 128, a.hidden, a.out, dwd);
    if (dwg) add(t2, xc, dgc, false, 128, a.cols, a.hidden, dwg);
    if (dwu) add(t2, xc, duc, false, 128, a.cols, a.hidden, dwu);
    if (dx && 2 * F < M) add(t2, w, dr, true, 128, a.rows, a.cols, dx);
    for (uint32_t i = 0; i < t2.count; ++i) {
      t2.a[i].splits = had.a[i].splits;
      t2.a[i].any = plan.flag;
    }
  };
  rest();
  float* part;
  if (!plan.lay(split(t2), &part, mlp_again_floats(a))) return false;
  rest();
  if (!run_jobs(plan.jobs, plan.maxima)) return false;
  Prods<1> t1{};
  t1.count = 1;
  Prod& g = t1.a[0];
  g.p = yr;
  g.q = d;
  g.depth = O;
  g.rows = a.rows;
  g.hidden = a.hidden;
  g.g = a.saved;
  g.u = a.saved + size_t(a.rows) * a.hidden;
  g.any = plan.flag;
  g.dr = dr;
  g.dgc = dgc;
  g.duc = duc;
  g.mc = mc;
  if (!run_products<GRAD>(t1, a.act, nullptr, 28.0 * M * F)) return false;
  MlpSums sums{};
  return run_products<STORE>(t2, kSilu, part, 0, &sums) &&
         mlp_backward_again(a, dy, dx, dwg, dwu, dwd, {plan.flag, nullptr, plan.flag + 1, plan.free}, sums);
}

// The parts of the weights are made anew at each call, which few rows do not pay for.
// Microseconds on fp32 MFMAs / on parts, forward: 128 x 4096 x 8192 332 / 363, 160 x 2048 x 8192 262 / 207,
// 192 x 1024 x 4096 72 / 83, 256 of them 84 / 84, 512 x 512 x 2048 48 / 59, 700 of them 71 / 59, 2048 x 256 x
// 1024 49 / 53, 3000 of them 69 / 54, 4096 x 128 x 512 33 / 44, 8192 of them 53 / 47, 16384 x 64 x 256 35 / 42,
// 32768 of them 60 / 54.
// Backward, a fit to such times of 58 sizes (rows of 48 to 65536, widths of 33 to 4096), within 30 % of each; the side it
// takes is the faster one, or within 3 %: on fp32 by the tiles' values, on parts by what dm's epilogue moves, the
// products, the weights' parts and the tokens'.  96 x 2048 x 8192 331 / 352, 128 of them 363 / 356, 128 x 1024 x 4096
// 116 / 115, 192 of them 165 / 127, 150 x 512 x 8192 147 / 123, 500 x 600 x 1000 68 / 81, 256 x 512 x 2048 61 / 78, 400 of
// them 101 / 88, 1024 x 256 x 1024 63 / 76, 2048 of them 130 / 86, 4096 x 128 x 512 67 / 78, 8192 of them 130 / 100, 6112 x 71
// x 5862 1163 / 634, 32768 x 64 x 256 150 / 218, 30000 x 96 x 200 173 / 200.
bool mlp_on_parts(const MlpArgs& a, bool backward) {
  // a tile's rows are reached with 32-bit offsets
  if (std::max({a.rows, a.cols, a.hidden, a.out}) > (1u << 21) || std::min({a.rows, a.cols, a.hidden, a.out}) < 32) return false;
  const double width = std::sqrt(double(a.cols) * a.out);
  if (!backward) return (a.rows - 115.0) * width * a.hidden >= 5.2e8;
  const uint32_t w = uint32_t(width);
  auto values = [&](uint32_t tile) { return 1e-6 * pad(a.rows, tile) * pad(a.hidden, tile); };  // in whole tiles, millions
  const double fp32 = (12 + values(32) * (5.3 + 0.18 * pad(w, 32))) * (w % 8 ? 1 + 14 / width : 1);  // a depth's last octet value by value
  const double parts = 54 + values(kTile) * (7.7 + 0.0256 * pad(w, kTile)) +
                       13e-6 * width * a.hidden * std::min(1.0, 0.3 + width / 2000) + 1.9e-3 * a.rows;
  return parts < fp32;
}

}  // namespace dce
