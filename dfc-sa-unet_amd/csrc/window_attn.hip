// Attention with a sliding window and always-visible first tokens ("sinks"), grouped key heads,
// forward, backward and over a cache (dfcsa.token_ops.window_attention / window_attention_cached).
//
//   O[i] = sum_j P[i][j] V[j],  P[i] = softmax over the visible j of scale * q_i . k_j
//   key j is visible to the query at position p when j < length, j <= p if causal, and
//   |p - j| < window or j < sinks.  A query that sees nothing (padding) gives zeros.
//   backward, with L the log-sum-exp of a row and delta = dO . O:
//   P = exp(scale q.k - L), dV = P^T dO, dS = P (dO V^T - delta), dQ = scale dS K, dK = scale dS^T Q
//
// Work: 4 D flop for each visible pair and head forward, 10 D backward and 4 D to form S and dP again (a
// query-major pass owns dQ, a key-major pass owns dK and dV, so there are no float atomics and the
// results do not depend on the order workgroups run in); only tiles that hold a visible pair are
// visited, so the cost follows N * (window + sinks), not N^2.
//
// Rows.  The G = H / Hk query heads of a key head are packed with the tokens: row r = t * G + g.  A
// tile of 128 rows then spans 128 / G tokens, so a grouped call reads each key once for its group and
// visits fewer half-masked tiles at the window's edges.
//
// Matrix instructions: 32x32x16 bf16, or 32x32x2 fp32 four at a time (fp32 inputs stay fp32 all the
// way).  The accumulator of one product is the B operand of the next without moving between lanes:
// the accumulator's row order (8 g + 4 (lane / 32) + r) is taken as the contraction order, and the A
// operand is read from LDS in that order -- transposed by ds_read_b64_tr_b16 for bf16.  P and dS are
// rounded to bf16 for that second product (bf16 inputs only): at most 2^-8 of each, which the sum over a
// row's keys averages; the results' error is 1.4 times that of rounding the exact ones (measured 0.0024
// against 0.0017 of their norm; with few visible keys up to 1.6 times).  The kernel for few rows waits for
// memory, so it multiplies P as two bf16, the second one what the first rounded off: its error is the
// results' own rounding (cached, 1000 keys: 0.0020 -> 0.0016 of their norm; 101 us before and after at 32
// sequences).  What bounds each kernel, and what was measured, stands at it.
//
// LDS images hold one row per key (or query row) with 16-byte chunks XOR-swizzled by the row, on the
// source side of an LDS-DMA load: rows are read by 16-byte reads and columns by transposing reads
// without bank conflicts from the same image.  Rows no query of the workgroup sees load as zeros (the
// buffer descriptor's bounds check), so what lies in padding is never multiplied.
#include <algorithm>
#include <cmath>

#include "common.h"
#include "dfcsa_internal.h"

namespace {

typedef __bf16 bh8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bh2_t __attribute__((ext_vector_type(2)));
typedef float f2_t __attribute__((ext_vector_type(2)));
typedef short s4_t __attribute__((ext_vector_type(4)));
typedef short s8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));
typedef float f16_t __attribute__((ext_vector_type(16)));
typedef int i4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4_t lds_s4;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();
constexpr float kNaN = __builtin_nanf("");
// The running maximum moves only when a row outgrows it by 2^kGrow (at 8192 tokens, window 1024: 105 us
// against 111).  A row's largest P is then no longer 1 and rounds to bf16 like the others.  Over many keys
// that averages out; with few it does not (2 sinks and a window of 3, width 8: dK's error 0.0031 instead of
// 0.0025 of its norm), so row tiles that visit at most kFewTiles key tiles, and the kernel for few rows,
// which waits for memory anyway, follow the maximum exactly.
constexpr float kGrow = 8.0f;
constexpr int kFewTiles = 8;

struct WArgs {
  int B, T, M, H, Hk, G, D, R;
  int window, sinks, causal, cached;
  float scale, scale2;   // scale2 = scale * log2(e)
  DivMod dmG;
  const void *q, *k, *v;
  int64_t qb, qt, qh, kb, kt, kh, vb, vt, vh;   // bytes
  const int* lengths;
  void* o;
  bf16_t* rest;          // training in bf16: what the rounding of o left, as bf16 (delta needs more than 8 bits of o)
  float* lse;            // [B][Hk][R], log2 of the sum of exp2(scale2 q.k)
  float* part;           // split results: O [splits][B*Hk*R][D], then lse [splits][B*Hk*R]
  int splits, tiles;     // row (or key) tiles per (batch, key head)
  // backward
  const void *dO;
  int64_t ob, ot, oh;    // dO strides, bytes
  float* delta;
  void *dq, *dk, *dv;
  int nsink, cwin;       // key tiles with sinks; row chunks of a key tile (room for them)
  int cmin;              // chunks if no sequence is padded; see chunks_of
  int pack;              // padded sequences: live tiles first; see spot
  int far32, cfar;       // blocks of 32 sinks, and chunks of the rows beyond the window that see them (0: none)
};

// A kernel's second, rare pass gets the kernel's arguments (by address: for kernels whose one argument is a WArgs), the
// thread's index, its place and LDS as values that the compiler takes for others.  What it needs is then formed
// there again, and not held in registers through the first pass (that spilled scalar registers in the first's loop:
// forward 104 -> 111 us at 8192 tokens, key-major pass 162 -> 175; as a function that is called it needs a stack,
// which costs the launch after it 0.45 us).
//
// The waves on a SIMD that a kernel's first pass reaches, which the second must not lower; it may spill for them.
// P: 0 forward, 1 dQ, 2 dK / dV, 3 few rows, 4 far rows; widths 32, 64, 96, 128 in bf16, then in fp32.
template <typename T, int DP> constexpr int simd_waves(int P) {
  constexpr int w[5][8] = {{4, 4, 2, 2, 4, 3, 2, 1}, {4, 3, 2, 2, 4, 2, 2, 1}, {4, 2, 2, 2, 3, 2, 1, 1},
                           {2, 2, 1, 1, 1, 1, 1, 1}, {2, 2, 1, 1, 1, 1, 1, 1}};
  return w[P][(sizeof(T) == 2 ? 0 : 4) + DP / 32 - 1];
}
// Given as the largest number too: the scheduler gives up the order that interleave() asks for where that takes a kernel
// from more waves to fewer (key-major pass, width 64: 28.8 -> 32.7 us).
#define SIMD_WAVES(P) __attribute__((amdgpu_waves_per_eu(simd_waves<T, DP>(P), simd_waves<T, DP>(P))))
struct Again {
  uint64_t args;
  unsigned smem, bad;
  int tid;
};
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ unsigned lds_addr(const void* p) {
  return (unsigned)(size_t)(const __attribute__((address_space(3))) char*)p;
}
__device__ __forceinline__ char* lds_at(unsigned offset) {
  return (char*)(__attribute__((address_space(3))) char*)(size_t)(unsigned)uniform((int)offset);
}
__device__ __forceinline__ Again again(const char* smem, const void* bad, int tid) {
  Again g{(uint64_t)__builtin_amdgcn_kernarg_segment_ptr(), lds_addr(smem), lds_addr(bad), tid};
  asm volatile("" : "+s"(g.args), "+v"(g.tid));
  return g;
}
__device__ __forceinline__ const WArgs& args_of(const Again& g) {
  const uint64_t p = (uint64_t)(unsigned)uniform((int)(g.args >> 32)) << 32 | (unsigned)uniform((int)g.args);
  return *(const WArgs*)(const __attribute__((address_space(4))) WArgs*)p;
}

// two values to bf16 in one instruction
__device__ __forceinline__ uint32_t cvt2(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2_t){a, b}, bh2_t));
}

// the far rows' parts lie behind the window's (floats)
__device__ __host__ __forceinline__ int64_t far_at(const WArgs& a) {
  const int64_t items = a.cwin > 1 ? (int64_t)a.tiles * a.cwin : (a.cfar ? a.nsink : 0);
  return items * a.B * a.Hk * 128 * 2 * a.D;
}

// ------------------------------------------------------------------ which tile a workgroup takes
// Tiles go to the XCDs in runs: neighbours read the same keys, once into that XCD's L2.  Padded sequences
// would leave XCDs with short ones idle (lengths are on the device, the host cannot plan for them), so the
// runs are of live tiles, equally long, and the empty ones, which have zeros to write, come after them.
// Measured at 2 x 8192 tokens, 16 / 4 heads of 128, window 1024, 8192 and 3000 of them valid: forward 179 ->
// 137 us, dQ 231 -> 176; with all of them valid 1 % slower (32 x 1024 tokens, 12 heads of 64: up to 3 %).
constexpr int kPackSeqs = 64;   // sequences, one per lane: more of them are mixed well enough
struct Spot {
  int bh, tile, sub;   // bh < 0: nothing to do
};
// lane i: tiles of sequence i that hold some of its len * mul rows (or keys), and the sum up to it
__device__ __forceinline__ int live_tiles(const WArgs& a, int mul, int& n) {
  const int i = threadIdx.x & 63;
  n = i < a.B ? (min(max(a.lengths[i], 0), a.M) * mul + 127) / 128 : 0;
  int sum = n * a.Hk;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(sum, o, 64);
    if (i >= o) sum += y;
  }
  return sum;
}
// Row chunks of a key tile: where padding leaves tiles empty, the live ones are cut finer, up to the room
// there is.  The same in every workgroup.  Measured in fp32 at 1531, 1000 and 400 tokens, 6 / 2 heads of 80,
// window 300: key-major pass 110 -> 77 us.
__device__ __forceinline__ int chunks_of(const WArgs& a, int live) {
  return a.cwin == a.cmin ? a.cwin : max(a.cmin, min(a.cwin, (a.D <= 64 ? 512 : 256) / max(live, 1)));
}
// tiles: of each (sequence, key head); each is `per` items, or the chunks of a key tile (per = 0, set here)
__device__ __forceinline__ Spot spot(const WArgs& a, int tiles, int mul, int& per) {
  Spot r;
  if (!a.pack) {
    if (per == 0) per = a.cwin;
    const int L = xcd_remap(blockIdx.x, tiles * a.B * a.Hk * per);
    r.sub = L % per;
    r.tile = L / per % tiles;
    r.bh = L < 0 ? -1 : L / (per * tiles);
    return r;
  }
  const int i = threadIdx.x & 63, x = blockIdx.x & 7, s = blockIdx.x >> 3;
  int n;
  const int sum = live_tiles(a, mul, n), live = __builtin_amdgcn_readfirstlane(__shfl(sum, 63, 64));
  if (per == 0) per = chunks_of(a, live);
  const int run = (live * per + 7) >> 3, all = tiles * a.Hk;
  const bool dead = s >= run;
  const int L = dead ? (s - run) * 8 + x : x * run + s;
  r.bh = -1;
  if (L >= (dead ? all * a.B - live : live) * per) return r;
  const int j = L / per, upto = dead ? all * min(i + 1, a.B) - sum : sum, mine = dead ? tiles - n : n;
  const int b = __builtin_ctzll(__ballot(upto > j));
  const int nb = __builtin_amdgcn_readfirstlane(__shfl(mine, b, 64));
  const int rem = j - __builtin_amdgcn_readfirstlane(__shfl(upto, b, 64)) + nb * a.Hk;
  r.sub = L - j * per;
  r.bh = b * a.Hk + rem / nb;
  r.tile = rem % nb + (dead ? tiles - nb : 0);
  return r;
}
__host__ inline int64_t grid_of(const WArgs& a, int64_t items) { return ((items + 7) / 8 + (a.pack ? 2 : 0)) * 8; }

// ------------------------------------------------------------------ matrix instructions
template <typename T> struct Mma;
template <> struct Mma<bf16_t> {
  typedef s8_t frag;
  static constexpr int KS = 16;   // contraction depth of one fragment pair
  __device__ __forceinline__ static f16_t mma(const frag& a, const frag& b, const f16_t& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bh8_t, a), __builtin_bit_cast(bh8_t, b), c, 0, 0, 0);
  }
  // a sum plus a fragment's elements
  __device__ __forceinline__ static float add(const frag& f, float l) {
    union { frag f; uint32_t u[4]; } x;
    x.f = f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bh2_t, x.u[i]), (bh2_t){(__bf16)1.0f, (__bf16)1.0f}, l, false);
    return l;
  }
  // accumulator registers of contraction step st (16 rows of the 32) as a fragment
  __device__ __forceinline__ static frag pack(const f16_t& p, int st) {
    union { uint32_t u[4]; frag f; } r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.u[i] = cvt2(p[8 * st + 2 * i], p[8 * st + 2 * i + 1]);
    return r.f;
  }
  // what pack() rounded off, as a fragment of its own
  __device__ __forceinline__ static frag pack_rest(const f16_t& p, int st, const frag& hi) {
    union { uint32_t u[4]; frag f; } h, r;
    h.f = hi;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r.u[i] = cvt2(p[8 * st + 2 * i] - __uint_as_float(h.u[i] << 16),
                    p[8 * st + 2 * i + 1] - __uint_as_float(h.u[i] & 0xffff0000u));
    return r.f;
  }
};
template <> struct Mma<float> {
  typedef f4_t frag;
  static constexpr int KS = 8;
  __device__ __forceinline__ static f16_t mma(const frag& a, const frag& b, f16_t c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
  __device__ __forceinline__ static float add(const frag& f, float l) { return l + ((f[0] + f[1]) + (f[2] + f[3])); }
  __device__ __forceinline__ static frag pack(const f16_t& p, int st) {
    return frag{p[4 * st], p[4 * st + 1], p[4 * st + 2], p[4 * st + 3]};
  }
};

// ------------------------------------------------------------------ LDS images
// DP: head width rounded up to 32; the row pitch is 64 or 128 elements.
template <typename T, int DP> struct Img {
  static constexpr int ES = (int)sizeof(T);
  static constexpr int PITCH = (DP <= 64 ? 64 : 128) * ES;
  static constexpr int CPR = PITCH / 16;         // 16-byte chunks per row: 8, 16 or 32
  static constexpr int ROWS = ES == 2 ? 64 : 32; // rows of a tile
  static constexpr int BYTES = ROWS * PITCH;
  static constexpr int NS = DP / Mma<T>::KS;     // fragments along the width
  static constexpr int ND = DP / 32;             // 32-column blocks
  // XOR of the chunk index: rows r .. r + 3 (one transposing read) and rows r .. r + 15 of one chunk
  // (one 16-byte read phase) both spread over all banks
  __device__ __forceinline__ static int swz(int row) {
    return CPR == 8 ? ((row >> 1) & 1) << 2 | ((row >> 2) & 3) : (row & 3) << 2 | ((row >> 2) & 3);
  }
  typedef typename Mma<T>::frag frag;
  // A lane's byte offsets into an image for the two kinds of reads.  The swizzle touches only bits that
  // the width step, the column block and the contraction step do not carry out of, so all reads of a tile
  // are an XOR with a constant and a constant offset away from these two.
  unsigned ra, ca;
  __device__ __forceinline__ void init(int lane) {
    const int row = lane & 31, h = lane >> 5;
    ra = (unsigned)(row * PITCH + ((h ^ swz(row)) << 4));
    if constexpr (ES == 2) {
      const int i = lane & 15, r = 4 * h + (i >> 2), col = (lane & 16) + 4 * (i & 3);
      ca = (unsigned)(r * PITCH + (((col >> 3) ^ swz(r)) << 4) + (col & 4) * 2);
    } else {
      ca = (unsigned)(4 * h * PITCH + (((row >> 2) ^ h) << 4) + (row & 3) * 4);
    }
  }
  // fragment st along the width of row r0 + (lane & 31), columns KS st + (KS / 2)(lane / 32) ..
  __device__ __forceinline__ frag row_frag(const char* img, int r0, int st) const {
    return *(const frag*)(img + (ra ^ (unsigned)(st << 5)) + r0 * PITCH);
  }
  // fragment of 32 columns 32 db + (lane & 31) over the contraction rows of step st of rows r0 ..
  __device__ __forceinline__ frag col_frag(const char* img, int r0, int st, int db) const {
    frag f;
    if constexpr (ES == 2) {
      const char* p = img + (r0 + 16 * st) * PITCH;
      const s4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + (ca ^ (unsigned)(db << 6))));
      const s4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + (ca ^ (unsigned)(db << 6 | 32)) + 8 * PITCH));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[e] = lo[e];
        f[4 + e] = hi[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        f[e] = *(const float*)(img + (r0 + 8 * st + e) * PITCH +
                               (ca ^ (unsigned)((db << 7) ^ (e << 6) ^ (((2 * st) & 3) << 4))));
    }
    return f;
  }
};

// ------------------------------------------------------------------ LDS-DMA
// One instruction moves 64 x 16 bytes to consecutive LDS addresses.  Written in inline asm so that the
// compiler does not drain it before the next LDS read; the kernels wait for their DMAs themselves.  An
// offset past num_records reads zeros.
constexpr unsigned kOob = 0x80000000u;
__device__ __forceinline__ i4_t make_rsrc(const void* base) {
  const uint64_t p = (uint64_t)base;
  i4_t r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)p);
  r[1] = __builtin_amdgcn_readfirstlane((int)((uint32_t)(p >> 32) & 0xffffu));
  r[2] = 0x7fffffff;
  r[3] = 0x00020000;
  // a scalar register that a lane read wrote needs five wait states before a memory instruction takes it
  asm volatile("s_nop 4" : "+s"(r));
  return r;
}
// lds: wave-uniform
__device__ __forceinline__ void dma16(const i4_t& rsrc, unsigned voff, unsigned lds) {
  unsigned keep;
  asm volatile(
      "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds\n\ts_mov_b32 m0, %0"
      : "=&s"(keep)
      : "v"(voff), "s"(rsrc), "s"(__builtin_amdgcn_readfirstlane(lds))
      : "memory");
}
template <int N> __device__ __forceinline__ void wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// Key-row DMA of one wave: NI instructions of a tile shared by NW waves (NW == 1: the wave's own tile).
template <typename T, int DP, int ROWS, int NW> struct KeyDma {
  typedef Img<T, DP> I;
  static constexpr int NI = ROWS * I::CPR / 64 / NW;
  int row[NI];
  unsigned chunk[NI];   // byte offset of the chunk within its row, or out of range
  __device__ __forceinline__ void init(int wave, int lane, int D) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int c = (i * NW + wave) * 64 + lane;
      row[i] = c / I::CPR;
      const int ch = (c % I::CPR) ^ I::swz(row[i]);
      chunk[i] = ch * 16 < D * I::ES ? (unsigned)ch * 16 : kOob;
    }
  }
  // rows key0 + row of base into the image at lds; a row is valid if in [lo, hi) or below sl
  __device__ __forceinline__ void issue(const char* base, int64_t stride, int key0, int lo, int hi, int sl, unsigned lds,
                                        int wave) const {
    const i4_t rs = make_rsrc(base + (int64_t)key0 * stride);
    if (key0 + ROWS <= sl || (key0 >= lo && key0 + ROWS <= hi)) {
#pragma unroll
      for (int i = 0; i < NI; ++i)
        dma16(rs, chunk[i] + (unsigned)row[i] * (unsigned)stride, lds + (i * NW + wave) * 1024);
    } else {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int key = key0 + row[i];
        const bool ok = (key >= lo && key < hi) || key < sl;
        dma16(rs, (ok ? 0u : kOob) | (chunk[i] & kOob) | (chunk[i] + (unsigned)row[i] * (unsigned)stride),
              lds + (i * NW + wave) * 1024);
      }
    }
  }
};

// ------------------------------------------------------------------ masks
struct RowMask {   // of this lane's row: visible(key) = key in [lo, lo + span] or key < sl
  int lo;
  unsigned span;
  int sl;
  __device__ __forceinline__ bool sees(int key) const { return (unsigned)(key - lo) <= span || key < sl; }
  // accumulator rows (keys key0 + 8 (e / 4) + e % 4) that the row does not see become `by`
  __device__ __forceinline__ void hide(f16_t& s, int key0, float by) const {
    const unsigned k = (unsigned)(key0 - lo);
    const int left = sl - key0;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int c = 8 * (e >> 2) + (e & 3);
      s[e] = ((k + c <= span) | (c < left)) ? s[e] : by;
    }
  }
};
struct Seq {       // of the workgroup's sequence
  int len, off;    // valid keys; position of token 0
};
__device__ __forceinline__ Seq seq_of(const WArgs& a, int b) {
  Seq s;
  s.len = a.M;
  if (a.lengths) s.len = min(max(a.lengths[b], 0), a.M);
  s.off = a.cached ? s.len - a.T : 0;
  return s;
}
__device__ __forceinline__ bool alive(const WArgs& a, const Seq& s, int r, int& p) {
  p = dm_div(a.dmG, r) + s.off;
  return r < a.R && p >= 0 && p < s.len;
}
__device__ __forceinline__ RowMask row_mask(const WArgs& a, const Seq& s, int r) {
  int p;
  RowMask m;
  m.lo = 0x7fffffff;   // above every key
  m.span = 0;
  m.sl = 0;
  if (alive(a, s, min(r, a.R - 1), p) && r < a.R) {
    const int hi = a.causal ? p : min(p + a.window - 1, s.len - 1);
    m.lo = p - a.window + 1;
    m.span = (unsigned)(hi - m.lo);
    m.sl = min(a.sinks, a.causal ? p + 1 : s.len);
  }
  return m;
}
// keys that the rows [r0, r1] see: [lo, hi) and [0, sl); pmin > pmax: none
struct Span {
  int pmin, pmax, lo, hi, sl;
  bool cut;   // some of the rows are padding
};
__device__ __forceinline__ Span span_of(const WArgs& a, const Seq& s, int r0, int r1) {
  Span v;
  r1 = min(r1, a.R - 1);
  const int first = dm_div(a.dmG, min(r0, a.R - 1)) + s.off, last = dm_div(a.dmG, r1) + s.off;
  v.pmin = max(first, 0);
  v.pmax = min(last, s.len - 1);
  v.cut = first < 0 || last >= s.len;
  if (r0 > r1 || v.pmin > v.pmax) {
    v.pmin = 1;
    v.pmax = 0;
    v.lo = v.hi = v.sl = 0;
    return v;
  }
  v.lo = max(v.pmin - a.window + 1, 0);
  v.hi = a.causal ? v.pmax + 1 : min(v.pmax + a.window, s.len);
  v.sl = min(a.sinks, a.causal ? v.pmax + 1 : s.len);
  return v;
}
// does every row of the span see every key in [k0, k1)?  is there one that sees one?
__device__ __forceinline__ bool sees_all(const WArgs& a, const Seq& s, const Span& v, int k0, int k1) {
  if (v.cut || v.pmin > v.pmax || k1 > s.len || (a.causal && k1 - 1 > v.pmin)) return false;
  if (k1 <= a.sinks) return true;
  return v.pmax - k0 < a.window && (a.causal || k1 - 1 - v.pmin < a.window);
}
__device__ __forceinline__ bool sees_any(const Span& v, int k0, int k1) {
  return v.pmin <= v.pmax && ((k0 < v.hi && k1 > v.lo) || k0 < v.sl);
}
// the key tiles of a span: sink tiles [0, ns), then window tiles [w0, w1)
struct TileList {
  int ns, w0, n;
  __device__ __forceinline__ int operator[](int i) const { return i < ns ? i : w0 + i - ns; }
};
template <int KT> __device__ __forceinline__ TileList tiles_of(const Span& v) {
  TileList t;
  t.ns = (v.sl + KT - 1) / KT;
  t.w0 = max(v.lo / KT, t.ns);
  t.n = t.ns + max((v.hi + KT - 1) / KT - t.w0, 0);
  return t;
}

// Order of a block's LDS reads and matrix instructions: AHEAD reads, then MM products and READS reads in
// turn, so that a product's operands are under way while the ones before it run.  Left alone the
// compiler reads each operand just before its product and waits for it.
template <int AHEAD, int MM, int READS, int N> __device__ __forceinline__ void interleave() {
  __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, MM, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
  }
}

__device__ __forceinline__ f16_t zero16() {
  f16_t z;
#pragma unroll
  for (int e = 0; e < 16; ++e) z[e] = 0.f;
  return z;
}

// ------------------------------------------------------------------ values that are not finite
// A product of matrix tiles multiplies every element of both: where a hidden key's P is 0 and its V (or K,
// or a hidden row's Q or dO) is infinite or NaN, the 0 * inf reaches rows that do not see it.  Nothing is
// tested for that in the loops; a workgroup that ends with a sum that is not finite runs its tiles once
// more with strict_product, and the waves concerned write again.
//
// There the product takes the finite elements of A; what the others add follows from three cases.  With t
// the number of visible pairs whose A is not finite, and s the sum of sign(A) sign(B) over them (0 for a
// NaN A and for a B of 0, whose product is NaN): t > s where something adds -inf or NaN, t > -s where
// something adds +inf or NaN.  Both are small whole numbers, exact as matrix products of -1, 0 and 1.  So
// inputs of nothing but NaN or infinities cost up to 6 times what others do (8192 tokens, 16 / 4 heads of 128,
// window 1024, forward and backward: 0.42 ms; a row of NaN among the sinks' values 1.1, nothing but NaN in
// q, v or dO 1.6, 1.5 and 1.4; one row and key after the other, without matrix products, they took up to 160).
__device__ __forceinline__ bool finite_all(const f16_t& v) {
  bool ok = true;
#pragma unroll
  for (int e = 0; e < 16; ++e) ok = ok && (__float_as_uint(v[e]) & 0x7f800000u) != 0x7f800000u;
  return ok;
}
// a fragment's finite elements, the others 0; all: were they all finite
__device__ __forceinline__ s8_t finite_part(s8_t a, bool& all) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const bool bad = (a[e] & 0x7f80) == 0x7f80;
    all = all && !bad;
    a[e] = bad ? (short)0 : a[e];
  }
  return a;
}
__device__ __forceinline__ f4_t finite_part(f4_t a, bool& all) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const bool bad = (__float_as_uint(a[e]) & 0x7f800000u) == 0x7f800000u;
    all = all && !bad;
    a[e] = bad ? 0.f : a[e];
  }
  return a;
}
// 1 where an element is not finite (kind), its sign where it is infinite (sign)
__device__ __forceinline__ void classes(const s8_t& a, s8_t& kind, s8_t& sign) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    kind[e] = (a[e] & 0x7f80) == 0x7f80 ? (short)0x3f80 : (short)0;
    sign[e] = (a[e] & 0x7fff) == 0x7f80 ? (short)(0x3f80 | (a[e] & 0x8000)) : (short)0;
  }
}
__device__ __forceinline__ void classes(const f4_t& a, f4_t& kind, f4_t& sign) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t b = __float_as_uint(a[e]);
    kind[e] = (b & 0x7f800000u) == 0x7f800000u ? 1.f : 0.f;
    sign[e] = (b & 0x7fffffffu) == 0x7f800000u ? (b >> 31 ? -1.f : 1.f) : 0.f;
  }
}
// o += A^T b over the 32 rows of img from r0; b is 0 at hidden pairs, see(e): is accumulator element e's visible
template <typename T, int DP, bool FINE, typename See>
__device__ __forceinline__ void strict_product(const Img<T, DP>& im, const char* img, int r0, const f16_t& b,
                                               f16_t (&o)[Img<T, DP>::ND], See see) {
  typedef Img<T, DP> I;
  typedef typename I::frag frag;
  constexpr int NST = 32 / Mma<T>::KS;
  bool all = true;
#pragma unroll
  for (int st = 0; st < NST; ++st) {
    const frag p = Mma<T>::pack(b, st);
    frag low = p;
    if constexpr (FINE && sizeof(T) == 2) low = Mma<T>::pack_rest(b, st, p);
#pragma unroll
    for (int d = 0; d < I::ND; ++d) {
      __builtin_amdgcn_sched_barrier(0);   // one fragment's registers at a time: this is the rare path
      const frag a = finite_part(im.col_frag(img, r0, st, d), all);
      o[d] = Mma<T>::mma(a, p, o[d]);
      if constexpr (FINE && sizeof(T) == 2) o[d] = Mma<T>::mma(a, low, o[d]);
    }
  }
  __builtin_amdgcn_sched_barrier(0);
  if (!__any(!all)) return;
#pragma unroll 1
  for (int neg = 0; neg < 2; ++neg) {   // t > -s, then t > s
    const float by = neg ? -1.f : 1.f;
    frag sg[NST], vis[NST];
#pragma unroll
    for (int st = 0; st < NST; ++st) {
      f16_t x, y;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        x[e] = b[e] > 0.f ? by : (b[e] < 0.f ? -by : 0.f);
        y[e] = see(e) ? 1.f : 0.f;
      }
      sg[st] = Mma<T>::pack(x, st);
      vis[st] = Mma<T>::pack(y, st);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int d = 0; d < I::ND; ++d) {
      f16_t t = zero16();
#pragma unroll
      for (int st = 0; st < NST; ++st) {
        __builtin_amdgcn_sched_barrier(0);
        frag kind, sign;
        classes(im.col_frag(img, r0, st, d), kind, sign);
        t = Mma<T>::mma(sign, sg[st], Mma<T>::mma(kind, vis[st], t));
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] -= t[e] > 0.f ? by * kNegInf : 0.f;
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// ------------------------------------------------------------------ softmax state of 32 rows (one per lane column)
template <typename T, int DP> struct Online {
  typedef Img<T, DP> I;
  typedef typename I::frag frag;
  float m, l;        // maximum (log2 units), this half's sum
  f16_t o[I::ND];    // O^T: column = row of the tile, rows = head columns
  __device__ __forceinline__ void init() {
    m = kNegInf;
    l = 0.f;
#pragma unroll
    for (int d = 0; d < I::ND; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
  }
  // NSUB blocks of 32 keys from key0; the maximum lags by at most grow.  FINE: P as two bf16
  template <int NSUB, bool FINE = false>
  __device__ __forceinline__ void step(const I& im, const char* kimg, const char* vimg, int key0, const frag (&q)[I::NS],
                                       float scale2, bool masked, const RowMask& mask, int lane, float grow) {
    f16_t s[NSUB];
    float mx = kNegInf;
#pragma unroll
    for (int b = 0; b < NSUB; ++b) {
      s[b] = zero16();
#pragma unroll
      for (int st = 0; st < I::NS; ++st) s[b] = Mma<T>::mma(im.row_frag(kimg, 32 * b, st), q[st], s[b]);
    }
    if constexpr (sizeof(T) == 2) interleave<NSUB == 2 ? 4 : 3, NSUB, NSUB, I::NS>();
    if (masked) {
      asm volatile("");   // a branch around the selects, not selects every time
#pragma unroll
      for (int b = 0; b < NSUB; ++b) mask.hide(s[b], key0 + 32 * b + 4 * (lane >> 5), kNegInf);
    }
#pragma unroll
    for (int b = 0; b < NSUB; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[b][e]);
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * scale2;
    if (__any(mx > m + grow || (m == kNegInf && mx > kNegInf))) {
      asm volatile("");   // keeps this a branch: as selects, the 16 ND products would run every time
      const float mn = fmaxf(m, mx);
      const float al = mn == kNegInf ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      l *= al;
#pragma unroll
      for (int d = 0; d < I::ND; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] *= al;
      m = mn;
    }
    const float ms = m == kNegInf ? 0.f : m;
    __builtin_amdgcn_s_setprio(1);   // ahead of the SIMD's other waves while the matrix unit has work (113 -> 110 us)
#pragma unroll
    for (int b = 0; b < NSUB; ++b) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[b][e] = __builtin_amdgcn_exp2f(fmaf(s[b][e], scale2, -ms));
#pragma unroll
      for (int st = 0; st < 32 / Mma<T>::KS; ++st) {
        const frag p = Mma<T>::pack(s[b], st);
        l = Mma<T>::add(p, l);   // of P as it is multiplied
#pragma unroll
        for (int d = 0; d < I::ND; ++d) o[d] = Mma<T>::mma(im.col_frag(vimg, 32 * b, st, d), p, o[d]);
        if constexpr (FINE && sizeof(T) == 2) {
          const frag low = Mma<T>::pack_rest(s[b], st, p);
          l = Mma<T>::add(low, l);
#pragma unroll
          for (int d = 0; d < I::ND; ++d) o[d] = Mma<T>::mma(im.col_frag(vimg, 32 * b, st, d), low, o[d]);
        }
      }
    }
    __builtin_amdgcn_s_setprio(0);
  }
  // the same with lse, the row's log-sum over all its keys (log2; +inf: it sees none), and strict products
  template <int NSUB, bool FINE = false>
  __device__ __forceinline__ void again(const I& im, const char* kimg, const char* vimg, int key0, const frag (&q)[I::NS],
                                        float scale2, const RowMask& mask, int lane, float lse) {
#pragma unroll 1
    for (int b = 0; b < NSUB; ++b) {
      f16_t s = zero16();
#pragma unroll
      for (int st = 0; st < I::NS; ++st) s = Mma<T>::mma(im.row_frag(kimg, 32 * b, st), q[st], s);
      const int k0 = key0 + 32 * b + 4 * (lane >> 5);
      mask.hide(s, k0, kNegInf);
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], scale2, -lse));
      if constexpr (!FINE)   // lse is of the P that were multiplied then: the sum of these is nearly 1
#pragma unroll
        for (int st = 0; st < 32 / Mma<T>::KS; ++st) l = Mma<T>::add(Mma<T>::pack(s, st), l);
      strict_product<T, DP, FINE>(im, vimg, 32 * b, s, o, [&](int e) { return mask.sees(k0 + 8 * (e >> 2) + (e & 3)); });
    }
  }
};

// this lane's row of a [token][head] tensor as fragments (rows that are not ok: zeros).  ALL: the row is there
// whether ok or not, and is loaded without branches (the dQ pass in fp32 spills beside them, 53 -> 57 us at width
// 64; in bf16 they are the faster form, 137 against 141 us at 8192 tokens)
template <typename T, int DP, bool ALL = false>
__device__ __forceinline__ void load_frags(const char* row, bool ok, int D, int lane,
                                           typename Mma<T>::frag (&f)[Img<T, DP>::NS]) {
  constexpr int KS = Mma<T>::KS;
#pragma unroll
  for (int st = 0; st < Img<T, DP>::NS; ++st) {
    const int d = KS * st + KS / 2 * (lane >> 5);
    constexpr int NE = sizeof(f[0]) / sizeof(f[0][0]);
    if constexpr (ALL) {
      const auto x = *(const typename Mma<T>::frag*)(row + (d < D ? d : 0) * (int)sizeof(T));
#pragma unroll
      for (int e = 0; e < NE; ++e) f[st][e] = ok && d < D ? x[e] : 0;
    } else {
#pragma unroll
      for (int e = 0; e < NE; ++e) f[st][e] = 0;
      if (ok && d < D) f[st] = *(const typename Mma<T>::frag*)(row + d * (int)sizeof(T));
    }
  }
}
template <typename T> __device__ __forceinline__ void store4(T* p, float a, float b, float c, float d);
template <> __device__ __forceinline__ void store4<float>(float* p, float a, float b, float c, float d) {
  *(float4*)p = make_float4(a, b, c, d);
}
template <> __device__ __forceinline__ void store4<bf16_t>(bf16_t* p, float a, float b, float c, float d) {
  *(uint2*)p = make_uint2(cvt2(a, b), cvt2(c, d));
}
// column `lane & 31` of an accumulated [head column][row] tile to the row at p
template <typename T, int ND>
__device__ __forceinline__ void store_col(T* p, const f16_t (&o)[ND], float f, int D, int lane) {
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = 32 * d + 8 * g + 4 * (lane >> 5);
      if (32 * ND == D || c < D) store4<T>(p + c, o[d][4 * g] * f, o[d][4 * g + 1] * f, o[d][4 * g + 2] * f, o[d][4 * g + 3] * f);
    }
}

// what the rounding of four values to bf16 left, as bf16
__device__ __forceinline__ void store4_rest(bf16_t* p, float a, float b, float c, float d) {
  store4<bf16_t>(p, a - bf2f(f2bf(a)), b - bf2f(f2bf(b)), c - bf2f(f2bf(c)), d - bf2f(f2bf(d)));
}

// The 32 rows of a wave's accumulated [head column][row] tile, times f, to global rows at(row) (null:
// none).  A lane holds 4 columns of a row at a time, 8 bytes in bf16: written straight, the stores of
// one instruction touch 32 rows (measured: 20 of the forward's 113 us at 8192 tokens, 16 heads of 128).
// bf16 tiles go through LDS (wave-private, 32 * kOutPitch bytes) and leave as 16-byte pieces of whole rows.
template <int DP> constexpr int out_pitch() { return DP * 2 + 16; }
template <typename T, int DP, bool REST, typename At>
__device__ __forceinline__ void store_rows(char* lds, const f16_t (&o)[DP / 32], float f, int D, int lane, At at) {
  if constexpr (sizeof(T) == 4) {
    float* p = at(lane & 31);
    if (p) store_col<float, DP / 32>(p, o, f, D, lane);
  } else {
    constexpr int P = out_pitch<DP>(), CPR = DP / 8;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        bf16_t* p = (bf16_t*)(lds + (lane & 31) * P) + 32 * d + 8 * g + 4 * (lane >> 5);
        if constexpr (REST) store4_rest(p, o[d][4 * g] * f, o[d][4 * g + 1] * f, o[d][4 * g + 2] * f, o[d][4 * g + 3] * f);
        else store4<bf16_t>(p, o[d][4 * g] * f, o[d][4 * g + 1] * f, o[d][4 * g + 2] * f, o[d][4 * g + 3] * f);
      }
#pragma unroll
    for (int i = 0; i < 32 * CPR / 64; ++i) {
      const int e = i * 64 + lane, row = e / CPR, c = e % CPR;
      bf16_t* p = at(row);
      if (p && c * 8 < D) *(uint4*)(p + c * 8) = *(const uint4*)(lds + row * P + c * 16);
    }
  }
}

// The results of a wave's 32 rows from rw over (part of) their keys: straight to o and lse, or to the
// split's partial.  lds: 32 * out_pitch bytes of the wave's own.
template <typename T, int DP>
__device__ __forceinline__ void finish_rows(const WArgs& a, int bh, int split, int rw, const f16_t (&o)[DP / 32], float lsum,
                                            float lse, char* lds, int lane) {
  const float inv = lsum > 0.f ? 1.0f / lsum : (lsum == 0.f ? 0.f : lsum);   // NaN sums stay NaN
  const int64_t row0 = (int64_t)bh * a.R, rows = (int64_t)a.B * a.Hk * a.R;
  const int r = rw + (lane & 31);
  if (a.splits == 1) {
    const int b = bh / a.Hk, hk = bh - b * a.Hk;
    const int64_t base = ((int64_t)b * a.T * a.H + hk * a.G) * a.D;
    auto at = [&](int i) -> int64_t {   // element offset of row rw + i
      const int t = dm_div(a.dmG, rw + i), g = rw + i - t * a.G;
      return base + ((int64_t)t * a.H + g) * a.D;
    };
    // the row's own scale has to be applied before the rows change lanes
    f16_t n[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) n[d][e] = o[d][e] * inv;
    store_rows<T, DP, false>(lds, n, 1.f, a.D, lane, [&](int i) { return rw + i < a.R ? (T*)a.o + at(i) : nullptr; });
    if constexpr (sizeof(T) == 2)
      if (a.rest)
        store_rows<T, DP, true>(lds, n, 1.f, a.D, lane, [&](int i) { return rw + i < a.R ? (T*)a.rest + at(i) : nullptr; });
    if (a.lse && lane < 32 && r < a.R) a.lse[row0 + r] = lse;
  } else if (r < a.R) {
    store_col<float, DP / 32>(a.part + (split * rows + row0 + r) * a.D, o, inv, a.D, lane);
    if (lane < 32) a.part[a.splits * rows * a.D + split * rows + row0 + r] = lse;
  }
}

// ============================================================================ forward
// 128 rows per workgroup, 32 per wave; key tiles double-buffered in LDS, one barrier a tile: a tile's DMA
// runs while the one before it is worked on.  64 KB of LDS and up to 256 registers leave two workgroups
// on a CU, two waves on a SIMD (three with 32-key tiles measured no faster: 118 against 113 us).
// Measured at 8192 tokens, 16 / 4 heads of 128, window 1024: 104 us, 620 TFLOP/s of the 1145 that a large
// library product reaches here; 25 us of it are the reads of q and the writes of o, its rest and lse, the
// matrix unit is busy 30 % of the time, the vector unit (exponentials, maxima, sums) 36 % (counters, 2.4 GHz).
//
// A pass: all tiles, their results written; true: some are not finite.  lse: of the lane's row, formed by the first pass
template <typename T, int DP, bool strict>
__device__ __forceinline__ bool fwd_pass(const WArgs& a, const Spot& at, int tid, char* smem, int* s_bad, float& lse) {
  typedef Img<T, DP> I;
  constexpr int KT = I::ROWS;
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int split = at.sub, tile = at.tile, bh = at.bh;
  const int b = bh / a.Hk, hk = bh - b * a.Hk;
  const Seq seq = seq_of(a, b);
  const int r0 = tile * 128, rw = r0 + wave * 32;
  const Span wg = span_of(a, seq, r0, r0 + 127), my = span_of(a, seq, rw, rw + 31);
  const TileList tl = tiles_of<KT>(wg);
  const int it0 = (int)((int64_t)tl.n * split / a.splits), it1 = (int)((int64_t)tl.n * (split + 1) / a.splits);

  const char* kbase = (const char*)a.k + b * a.kb + hk * a.kh;
  const char* vbase = (const char*)a.v + b * a.vb + hk * a.vh;
  KeyDma<T, DP, KT, 4> dma;
  dma.init(wave, lane, a.D);
  const int r = rw + (lane & 31);
  const RowMask mask = row_mask(a, seq, r);
  typename I::frag q[I::NS];
  {
    const int t = dm_div(a.dmG, min(r, a.R - 1)), g = min(r, a.R - 1) - t * a.G;
    load_frags<T, DP>((const char*)a.q + b * a.qb + t * a.qt + (hk * a.G + g) * a.qh, mask.lo != 0x7fffffff, a.D, lane, q);
  }
  I im;
  im.init(lane);
  bool bad = strict && __builtin_amdgcn_readfirstlane(s_bad[wave]);
  Online<T, DP> st;
  st.init();
  if (it0 < it1) {
    dma.issue(kbase, a.kt, tl[it0] * KT, wg.lo, wg.hi, wg.sl, lds_addr(smem), wave);
    dma.issue(vbase, a.vt, tl[it0] * KT, wg.lo, wg.hi, wg.sl, lds_addr(smem) + I::BYTES, wave);
  }
  for (int it = it0; it < it1; ++it) {
    char* cur = smem + ((it - it0) & 1) * 2 * I::BYTES;
    const unsigned nxt = lds_addr(smem) + ((it - it0 + 1) & 1) * 2 * I::BYTES;
    wait_vm<0>();
    lds_barrier();   // this tile is there, and every wave is done with the other buffer
    if (it + 1 < it1) {
      dma.issue(kbase, a.kt, tl[it + 1] * KT, wg.lo, wg.hi, wg.sl, nxt, wave);
      dma.issue(vbase, a.vt, tl[it + 1] * KT, wg.lo, wg.hi, wg.sl, nxt + I::BYTES, wave);
    }
    const int key0 = tl[it] * KT;
    if (!sees_any(my, key0, key0 + KT)) continue;
    if constexpr (!strict)
      st.template step<KT / 32>(im, cur, cur + I::BYTES, key0, q, a.scale2, !sees_all(a, seq, my, key0, key0 + KT), mask, lane,
                                tl.n <= kFewTiles ? 0.f : kGrow);
    else if (bad)
      st.template again<KT / 32>(im, cur, cur + I::BYTES, key0, q, a.scale2, mask, lane, lse == kNegInf ? -kNegInf : lse);
  }
  float lsum = st.l + __shfl_xor(st.l, 32, 64);
  if constexpr (!strict) {
    // a live row sees its own position's key at least: a sum of 0 has only scores of -inf in it
    if (a.splits == 1 && lsum == 0.f && mask.lo != 0x7fffffff) lsum = kNaN;
    lse = lsum == 0.f ? kNegInf : st.m + __builtin_amdgcn_logf(lsum);
    bool ok = true;
#pragma unroll
    for (int d = 0; d < I::ND; ++d) ok = ok && finite_all(st.o[d]);
    bad = __any(!ok && r < a.R);
    if (lane == 0) s_bad[wave] = bad;
  }
  lds_barrier();   // the tiles are read, the waves' results known
  if (!strict || bad) finish_rows<T, DP>(a, bh, split, rw, st.o, lsum, lse, smem + wave * 32 * out_pitch<DP>(), lane);
  if (strict || !(s_bad[0] | s_bad[1] | s_bad[2] | s_bad[3])) return false;
  wait_vm<0>();   // the stores that the next ones replace
  lds_barrier();
  return true;
}
template <typename T, int DP>
__device__ __forceinline__ void fwd_again(Again g, Spot at, float lse) {
  at = Spot{uniform(at.bh), uniform(at.tile), uniform(at.sub)};
  fwd_pass<T, DP, true>(args_of(g), at, g.tid, lds_at(g.smem), (int*)lds_at(g.bad), lse);
}
template <typename T, int DP>
__global__ void __launch_bounds__(256) SIMD_WAVES(0) wattn_fwd_kernel(const WArgs a) {
  __shared__ __attribute__((aligned(16))) char smem[4 * Img<T, DP>::BYTES];
  __shared__ int s_bad[4];
  int per = a.splits;
  const Spot at = spot(a, a.tiles, a.G, per);
  if (at.bh < 0) return;
  float lse = 0.f;
  if (fwd_pass<T, DP, false>(a, at, threadIdx.x, smem, s_bad, lse)) fwd_again<T, DP>(again(smem, s_bad, threadIdx.x), at, lse);
}

// weights and sum of one row's results of four waves
__device__ __forceinline__ void join_waves(const float (&m)[4][32], const float (&l)[4][32], int row, float (&f)[4], float& inv,
                                           float& lse) {
  float mm = kNegInf, ls = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) mm = fmaxf(mm, m[w][row]);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[w] = mm == kNegInf ? (l[w][row] == 0.f ? 0.f : l[w][row]) : __builtin_amdgcn_exp2f(m[w][row] - mm);
    ls += f[w] * l[w][row];
  }
  inv = ls > 0.f ? 1.0f / ls : (ls == 0.f ? 0.f : ls);
  lse = ls == 0.f ? kNegInf : mm + __builtin_amdgcn_logf(ls);
}

// Few rows (at most 32 per tile): the four waves share the rows and split the keys, each with its own
// LDS ring of 32-key tiles and no barrier in the loop; joined at the end.  Bound by the caches' bytes:
// 32 sequences, one token each over 4096 + 16 keys of 8 heads of 128 in bf16 (539 MB) take 99 us, 5.4 TB/s
// (a large copy: 5.0).  One sequence over 1024 + 4 keys of 4 heads, split over 36 workgroups: 7.3 us + 4.1
// for the join, all of it latency.
template <typename T, int DP> struct Few {
  typedef Img<T, DP> I;
  static constexpr int KT = 32, IB = KT * I::PITCH;
  static constexpr int STG = IB <= 8192 ? 2 : 1;   // stages of K and V per wave (wide fp32: one fits)
  static constexpr int RING = STG * 2 * IB;
  static constexpr int OUT = 32 * (DP + 4) * 4;
  static constexpr int PER = RING > OUT ? RING : OUT;
};
// all tiles, their results written; true: some are not finite.  lse: of row lane & 31 over these keys, for the second time
template <typename T, int DP, bool strict>
__device__ __forceinline__ bool few_pass(const WArgs& a, int L, int tid, char* smem, float (&sm_m)[4][32], float (&sm_l)[4][32],
                                         float& lse) {
  typedef Few<T, DP> F;
  typedef Img<T, DP> I;
  constexpr int KT = F::KT, IB = F::IB, STG = F::STG, PER = F::PER;
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int split = L % a.splits, tile = (L / a.splits) % a.tiles, bh = L / (a.splits * a.tiles);
  const int b = bh / a.Hk, hk = bh - b * a.Hk;
  const Seq seq = seq_of(a, b);
  const int r0 = tile * 32;
  const Span my = span_of(a, seq, r0, r0 + 31);
  const TileList tl = tiles_of<KT>(my);
  const int it0 = (int)((int64_t)tl.n * split / a.splits) + wave, it1 = (int)((int64_t)tl.n * (split + 1) / a.splits);

  const char* kbase = (const char*)a.k + b * a.kb + hk * a.kh;
  const char* vbase = (const char*)a.v + b * a.vb + hk * a.vh;
  char* ring = smem + wave * PER;
  KeyDma<T, DP, KT, 1> dma;
  dma.init(0, lane, a.D);
  const int r = r0 + (lane & 31);
  const RowMask mask = row_mask(a, seq, r);
  typename I::frag q[I::NS];
  {
    const int t = dm_div(a.dmG, min(r, a.R - 1)), g = min(r, a.R - 1) - t * a.G;
    load_frags<T, DP>((const char*)a.q + b * a.qb + t * a.qt + (hk * a.G + g) * a.qh, mask.lo != 0x7fffffff, a.D, lane, q);
  }
  I im;
  im.init(lane);
  const int row = tid >> 3, c0 = (tid & 7) * (DP / 8), rr = r0 + row;   // of the join: 8 threads a row
  Online<T, DP> st;
  st.init();
  if (it0 < it1) {
    dma.issue(kbase, a.kt, tl[it0] * KT, my.lo, my.hi, my.sl, lds_addr(ring), 0);
    dma.issue(vbase, a.vt, tl[it0] * KT, my.lo, my.hi, my.sl, lds_addr(ring) + IB, 0);
  }
  int cur = 0;
  for (int it = it0; it < it1; it += 4, cur = (cur + 1) % STG) {
    char* c = ring + cur * 2 * IB;
    const unsigned n = lds_addr(ring) + (cur + 1) % STG * 2 * IB;
    if (STG == 2 && it + 4 < it1) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the reads of the buffer filled next are done
      dma.issue(kbase, a.kt, tl[it + 4] * KT, my.lo, my.hi, my.sl, n, 0);
      dma.issue(vbase, a.vt, tl[it + 4] * KT, my.lo, my.hi, my.sl, n + IB, 0);
      wait_vm<2 * KeyDma<T, DP, KT, 1>::NI>();
    } else {
      wait_vm<0>();
    }
    const int key0 = tl[it] * KT;
    if constexpr (!strict)
      st.template step<1, true>(im, c, c + IB, key0, q, a.scale2, !sees_all(a, seq, my, key0, key0 + KT), mask, lane, 0.f);
    else
      st.template again<1, true>(im, c, c + IB, key0, q, a.scale2, mask, lane, lse);
    if (STG == 1 && it + 4 < it1) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      dma.issue(kbase, a.kt, tl[it + 4] * KT, my.lo, my.hi, my.sl, n, 0);
      dma.issue(vbase, a.vt, tl[it + 4] * KT, my.lo, my.hi, my.sl, n + IB, 0);
    }
  }
  // join: O of wave w at ring w as [row][DP + 4] floats
  const float lsum = st.l + __shfl_xor(st.l, 32, 64);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  float* mine = (float*)ring + (lane & 31) * (DP + 4);
#pragma unroll
  for (int d = 0; d < I::ND; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *(float4*)(mine + 32 * d + 8 * g + 4 * (lane >> 5)) =
          make_float4(st.o[d][4 * g], st.o[d][4 * g + 1], st.o[d][4 * g + 2], st.o[d][4 * g + 3]);
  if (!strict && lane < 32) {
    sm_m[wave][lane] = st.m;
    sm_l[wave][lane] = lsum;
  }
  __syncthreads();
  float f[4], inv, out_lse;
  if constexpr (strict) f[0] = f[1] = f[2] = f[3] = inv = 1.f;   // P came with the row's sum taken off
  else join_waves(sm_m, sm_l, row, f, inv, out_lse);
  int p;
  if (!strict && a.splits == 1 && out_lse == kNegInf && alive(a, seq, rr, p)) inv = out_lse = kNaN;   // scores of -inf alone
  bool ok = true;
  const int64_t orow = (int64_t)bh * a.R + rr, rows = (int64_t)a.B * a.Hk * a.R;
  const int t = dm_div(a.dmG, min(rr, a.R - 1)), g = rr - t * a.G;
  const int64_t at = (((int64_t)b * a.T + t) * a.H + hk * a.G + g) * a.D;
  T* po = (T*)a.o + at;
  float* pp = a.splits == 1 ? nullptr : a.part + (split * rows + orow) * a.D;
#pragma unroll
  for (int c = 0; c < DP / 8; c += 4) {
    if (rr < a.R && c0 + c < a.D) {
      float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float4 x = *(const float4*)((const float*)(smem + w * PER) + row * (DP + 4) + c0 + c);
        s[0] += f[w] * x.x;
        s[1] += f[w] * x.y;
        s[2] += f[w] * x.z;
        s[3] += f[w] * x.w;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) ok = ok && (__float_as_uint(s[e]) & 0x7f800000u) != 0x7f800000u;
      if (pp) {
        store4<float>(pp + c0 + c, s[0] * inv, s[1] * inv, s[2] * inv, s[3] * inv);
      } else {
        store4<T>(po + c0 + c, s[0] * inv, s[1] * inv, s[2] * inv, s[3] * inv);
        if (sizeof(T) == 2 && a.rest) store4_rest(a.rest + at + c0 + c, s[0] * inv, s[1] * inv, s[2] * inv, s[3] * inv);
      }
    }
  }
  if (!strict && (tid & 7) == 0 && rr < a.R) {
    if (pp) a.part[a.splits * rows * a.D + split * rows + orow] = out_lse;
    else if (a.lse) a.lse[orow] = out_lse;
  }
  if (strict || !__syncthreads_or(!ok)) return false;
  join_waves(sm_m, sm_l, lane & 31, f, inv, lse);
  if (lse == kNegInf) lse = a.splits == 1 && mask.lo != 0x7fffffff ? kNaN : -kNegInf;   // or: sees nothing
  return true;
}
template <typename T, int DP> __device__ __forceinline__ void few_again(Again g, int L, float lse) {
  typedef float Stat[4][32];
  Stat& unused = *(Stat*)lds_at(g.bad);
  few_pass<T, DP, true>(args_of(g), uniform(L), g.tid, lds_at(g.smem), unused, unused, lse);
}
template <typename T, int DP>
__global__ void __launch_bounds__(256) SIMD_WAVES(3) wattn_few_kernel(const WArgs a) {
  __shared__ __attribute__((aligned(16))) char smem[4 * Few<T, DP>::PER];
  __shared__ float sm_m[4][32], sm_l[4][32];
  const int L = xcd_remap(blockIdx.x, a.tiles * a.B * a.Hk * a.splits);
  if (L < 0) return;
  float lse = 0.f;
  if (few_pass<T, DP, false>(a, L, threadIdx.x, smem, sm_m, sm_l, lse))
    few_again<T, DP>(again(smem, sm_m, threadIdx.x), L, lse);
}

// One row per 32 threads: the splits' results weighted by their sums, in split order.  At most 64
// splits; their 2 x 32 sums are read at once, then four results are in flight at a time.
template <typename T>
__global__ void __launch_bounds__(256) wattn_join_kernel(const WArgs a) {
  const int64_t rows = (int64_t)a.B * a.Hk * a.R, row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int i = threadIdx.x & 31, c = i * 4;
  const float* lp = a.part + a.splits * rows * a.D + row;
  const float l0 = i < a.splits ? lp[i * rows] : kNegInf, l1 = i + 32 < a.splits ? lp[(i + 32) * rows] : kNegInf;
  float mm = fmaxf(l0, l1);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor(mm, o, 32));
  // A NaN sum has to reach the result: the maximum drops it, its weight does not.  Below 0: a split that saw
  // nothing.  One whose weight rounds to 0 saw something, and 0 times its infinity or NaN is NaN as in one piece.
  const float f0 = l0 == kNegInf ? -1.f : __builtin_amdgcn_exp2f(l0 - mm);
  const float f1 = l1 == kNegInf ? -1.f : __builtin_amdgcn_exp2f(l1 - mm);
  float s[4] = {0.f, 0.f, 0.f, 0.f}, ls = 0.f;
  const float* p = a.part + row * a.D + (c < a.D ? c : 0);
  for (int z0 = 0; z0 < a.splits; z0 += 4) {
    float4 x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = *(const float4*)(p + (int64_t)min(z0 + k, a.splits - 1) * rows * a.D);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int z = z0 + k;
      const float f = z < a.splits ? __shfl(z < 32 ? f0 : f1, z & 31, 32) : -1.f;
      if (f < 0.f) continue;
      ls += f;
      s[0] += f * x[k].x;
      s[1] += f * x[k].y;
      s[2] += f * x[k].z;
      s[3] += f * x[k].w;
    }
  }
  const int bh = (int)(row / a.R), r = (int)(row - (int64_t)bh * a.R);
  const int b = bh / a.Hk, hk = bh - b * a.Hk, t = dm_div(a.dmG, r), g = r - t * a.G;
  int pos;
  if (ls == 0.f && alive(a, seq_of(a, b), r, pos)) ls = kNaN;   // sees keys, with scores of -inf alone
  const float inv = ls == 0.f ? 0.f : 1.0f / ls;
  if (c < a.D) {
    const int64_t at = (((int64_t)b * a.T + t) * a.H + hk * a.G + g) * a.D + c;
    store4<T>((T*)a.o + at, s[0] * inv, s[1] * inv, s[2] * inv, s[3] * inv);
    if (sizeof(T) == 2 && a.rest) store4_rest(a.rest + at, s[0] * inv, s[1] * inv, s[2] * inv, s[3] * inv);
  }
  if (a.lse && i == 0) a.lse[row] = ls == 0.f ? kNegInf : mm + __builtin_amdgcn_logf(ls);
}

// ============================================================================ backward: dQ
// As the forward, with S and dP per key tile; also writes delta = dO . O for the key-major pass.
// Measured as above: 135 us, 720 TFLOP/s over its three products; its rows' q, dO, O and O's rest are
// 134 MB of the 250 that the whole call has to move.
//
// A pass: all tiles, their results written; true: some are not finite
template <typename T, int DP, bool strict>
__device__ __forceinline__ bool dq_pass(const WArgs& a, const Spot& at, int tid, char* smem, int* s_bad) {
  typedef Img<T, DP> I;
  typedef typename I::frag frag;
  constexpr int KT = I::ROWS;
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool bad = !strict || __builtin_amdgcn_readfirstlane(s_bad[wave]);   // are these the wave's results
  const int tile = at.tile, bh = at.bh;
  const int b = bh / a.Hk, hk = bh - b * a.Hk;
  const Seq seq = seq_of(a, b);
  const int r0 = tile * 128, rw = r0 + wave * 32;
  const Span wg = span_of(a, seq, r0, r0 + 127), my = span_of(a, seq, rw, rw + 31);
  const TileList tl = tiles_of<KT>(wg);

  const char* kbase = (const char*)a.k + b * a.kb + hk * a.kh;
  const char* vbase = (const char*)a.v + b * a.vb + hk * a.vh;
  KeyDma<T, DP, KT, 4> dma;
  dma.init(wave, lane, a.D);
  const int r = rw + (lane & 31);
  const RowMask mask = row_mask(a, seq, r);
  const bool live = mask.lo != 0x7fffffff;
  const int t = dm_div(a.dmG, min(r, a.R - 1)), g = min(r, a.R - 1) - t * a.G;
  const int64_t orow = (((int64_t)b * a.T + t) * a.H + hk * a.G + g) * a.D;
  frag q[I::NS], dof[I::NS];
  constexpr bool ALL = sizeof(T) == 4 && DP <= 96;
  load_frags<T, DP, ALL>((const char*)a.q + b * a.qb + t * a.qt + (hk * a.G + g) * a.qh, live, a.D, lane, q);
  load_frags<T, DP, ALL>((const char*)a.dO + b * a.ob + t * a.ot + (hk * a.G + g) * a.oh, live, a.D, lane, dof);
  float dl = 0.f, lse = 0.f;
  {
    frag of[I::NS];
    load_frags<T, DP, ALL>((const char*)((const T*)a.o + orow), live, a.D, lane, of);
    constexpr int NE = sizeof(frag) / sizeof(T);
    if (sizeof(T) == 2 && a.rest) {
      frag rf[I::NS];
      load_frags<T, DP, ALL>((const char*)(a.rest + orow), live, a.D, lane, rf);
#pragma unroll
      for (int st = 0; st < I::NS; ++st)
#pragma unroll
        for (int e = 0; e < NE; ++e) dl += bf2f((bf16_t)rf[st][e]) * bf2f((bf16_t)dof[st][e]);
    }
#pragma unroll
    for (int st = 0; st < I::NS; ++st)
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        if constexpr (sizeof(T) == 2) dl += bf2f((bf16_t)of[st][e]) * bf2f((bf16_t)dof[st][e]);
        else dl += of[st][e] * dof[st][e];
      }
    dl += __shfl_xor(dl, 32, 64);
    const int64_t row = (int64_t)bh * a.R + r;
    if (live) lse = a.lse[row];
    if (!strict && r < a.R && lane < 32) a.delta[row] = dl;
  }
  f16_t dq[I::ND];
  I im;
  im.init(lane);
  auto body = [&](const char* cur, int key0, bool masked) __attribute__((always_inline)) {
#pragma unroll 1   // one 32 x 32 block's registers at a time; the other wave of the SIMD fills the gaps
    for (int kb = 0; kb < KT / 32; ++kb) {
      f16_t s = zero16(), dp = zero16();
      __builtin_amdgcn_s_setprio(1);   // 146 -> 142 us
#pragma unroll
      for (int st = 0; st < I::NS; ++st) {   // two chains of dependent products, side by side
        s = Mma<T>::mma(im.row_frag(cur, 32 * kb, st), q[st], s);
        dp = Mma<T>::mma(im.row_frag(cur + I::BYTES, 32 * kb, st), dof[st], dp);
      }
      if constexpr (sizeof(T) == 2) interleave<4, 2, 2, I::NS>();
      __builtin_amdgcn_s_setprio(0);
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale2, -lse)) * (dp[e] - dl);
      if (masked) {
        asm volatile("");
        mask.hide(s, key0 + 32 * kb + 4 * (lane >> 5), 0.f);
      }
      if constexpr (strict) {
        strict_product<T, DP, false>(im, cur, 32 * kb, s, dq,
                                     [&](int e) { return mask.sees(key0 + 32 * kb + 4 * (lane >> 5) + 8 * (e >> 2) + (e & 3)); });
      } else {
#pragma unroll
        for (int st = 0; st < 32 / Mma<T>::KS; ++st) {
          const frag ds = Mma<T>::pack(s, st);
#pragma unroll
          for (int d = 0; d < I::ND; ++d) dq[d] = Mma<T>::mma(im.col_frag(cur, 32 * kb, st, d), ds, dq[d]);
        }
        if constexpr (sizeof(T) == 2) interleave<8, 1, 2, 2 * I::ND>();
      }
    }
  };
  const int64_t obase = ((int64_t)b * a.T * a.H + hk * a.G) * a.D;
#pragma unroll
  for (int d = 0; d < I::ND; ++d) dq[d] = zero16();
  if (tl.n > 0) {
    dma.issue(kbase, a.kt, tl[0] * KT, wg.lo, wg.hi, wg.sl, lds_addr(smem), wave);
    dma.issue(vbase, a.vt, tl[0] * KT, wg.lo, wg.hi, wg.sl, lds_addr(smem) + I::BYTES, wave);
  }
  for (int it = 0; it < tl.n; ++it) {
    char* cur = smem + (it & 1) * 2 * I::BYTES;
    const unsigned nxt = lds_addr(smem) + ((it + 1) & 1) * 2 * I::BYTES;
    wait_vm<0>();
    lds_barrier();
    if (it + 1 < tl.n) {
      dma.issue(kbase, a.kt, tl[it + 1] * KT, wg.lo, wg.hi, wg.sl, nxt, wave);
      dma.issue(vbase, a.vt, tl[it + 1] * KT, wg.lo, wg.hi, wg.sl, nxt + I::BYTES, wave);
    }
    const int key0 = tl[it] * KT;
    if (bad && sees_any(my, key0, key0 + KT)) body(cur, key0, strict || !sees_all(a, seq, my, key0, key0 + KT));
  }
  if constexpr (!strict) {
    bool ok = true;
#pragma unroll
    for (int d = 0; d < I::ND; ++d) ok = ok && finite_all(dq[d]);
    const int any = __any(!ok && r < a.R);
    if (lane == 0) s_bad[wave] = any;
  }
  lds_barrier();
  if (bad)
    store_rows<T, DP, false>(smem + wave * 32 * out_pitch<DP>(), dq, a.scale, a.D, lane, [&](int i) -> T* {
      const int ti = dm_div(a.dmG, min(rw + i, a.R - 1)), gi = rw + i - ti * a.G;
      return rw + i < a.R ? (T*)a.dq + obase + ((int64_t)ti * a.H + gi) * a.D : nullptr;
    });
  if (strict || !(s_bad[0] | s_bad[1] | s_bad[2] | s_bad[3])) return false;
  wait_vm<0>();   // the stores that the next ones replace
  lds_barrier();
  return true;
}
template <typename T, int DP> __device__ __forceinline__ void dq_again(Again g, Spot at) {
  at = Spot{uniform(at.bh), uniform(at.tile), uniform(at.sub)};
  dq_pass<T, DP, true>(args_of(g), at, g.tid, lds_at(g.smem), (int*)lds_at(g.bad));
}
template <typename T, int DP>
__global__ void __launch_bounds__(256) SIMD_WAVES(1) wattn_dq_kernel(const WArgs a) {
  __shared__ __attribute__((aligned(16))) char smem[4 * Img<T, DP>::BYTES];
  __shared__ int s_bad[4];
  int per = 1;
  const Spot at = spot(a, a.tiles, a.G, per);
  if (at.bh < 0) return;
  if (dq_pass<T, DP, false>(a, at, threadIdx.x, smem, s_bad)) dq_again<T, DP>(again(smem, s_bad, threadIdx.x), at);
}

// ============================================================================ backward: dK, dV
// 128 keys per workgroup, 32 per wave (lane column = key); row tiles of Q and dO double-buffered in
// LDS.  bf16 wider than 64: eight waves, two for each 32 keys, which take the two 32-row halves of a
// tile and add up at the end through LDS (one such workgroup fills a CU: measured 284 -> 225 us at 8192
// tokens, 16 / 4 heads of 128, window 1024, against four waves with one tile per CU; 162 us with the far
// rows taken out and the operands read ahead: 800 TFLOP/s over four products).  LDS reads bound it next
// (K is read again for every row block: 320 of about 1024 cycles of a CU's LDS a block, beside the
// products' own).  Running the two waves of a SIMD half a tile apart measured slower (185 us).
// A workgroup takes the rows whose window reaches its keys, or one of cwin chunks of them; the rows
// further away that see sinks are wattn_far_kernel's.  fp32 parts are added in order by wattn_dkv_join.
__device__ __forceinline__ void key_rows(const WArgs& a, const Seq& seq, int kt, int rt, int& i0, int& i1) {
  const int k0 = kt * 128, k1 = min(k0 + 128, seq.len);
  int p0 = a.causal ? k0 : max(k0 - a.window + 1, 0), p1 = min(k1 - 1 + a.window - 1, seq.len - 1);
  if (k0 < a.sinks && !a.cfar) {   // few rows are further away: no pass of their own
    p0 = a.causal ? k0 : 0;
    p1 = seq.len - 1;
  }
  i0 = i1 = 0;   // tiles of rt rows
  if (k0 < k1 && p0 <= p1) {
    i0 = p0 * a.G / rt;
    i1 = ((p1 + 1) * a.G + rt - 1) / rt;
  }
}
constexpr int kBoth = 0, kDv = 1, kDk = 2;
template <typename T, int DP> constexpr int dkv_waves() { return sizeof(T) == 2 && DP > 64 ? 8 : 4; }
template <typename T, int DP> struct Dkv {
  typedef Img<T, DP> I;
  // bf16 heads wider than 64: K (32 registers) stays in LDS, so that two waves fit on a SIMD beside the
  // 128 accumulators
  static constexpr bool KLDS = sizeof(T) == 2 && DP > 64;
  static constexpr int NW = dkv_waves<T, DP>();
  static constexpr int RT = I::ROWS, RB = RT * I::PITCH;
  static constexpr int OUT = NW == 8 ? 4 * 64 * (DP / 2) * 4 : 0;   // one wave's dK or dV, four times
  static constexpr int NB = 2;   // row tiles in LDS
  static constexpr int MAIN = 2 * NB * RB + (KLDS ? 128 * I::PITCH : 0);
  static constexpr int LDS = MAIN > OUT ? MAIN : OUT;
  struct Stats {
    float l[NB][RT], d[NB][RT];
  };
};
// the row tiles for both sums, or strictly for one (its registers, and no more); true: some are not finite
template <typename T, int DP, int which>
__device__ __forceinline__ bool dkv_pass(const WArgs& a, const Spot& place, int nch, int tid, char* smem,
                                         typename Dkv<T, DP>::Stats& stats, int* s_bad) {
  typedef Img<T, DP> I;
  typedef Dkv<T, DP> P;
  typedef typename I::frag frag;
  constexpr bool KLDS = P::KLDS, strict = which != kBoth, k_sum = which != kDv, v_sum = which != kDk;
  constexpr int NW = P::NW, RT = P::RT, RB = P::RB, NB = P::NB;
  constexpr int NI = RT * I::CPR / 64 / NW;
  auto &s_l = stats.l, &s_d = stats.d;
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int bh = place.bh, kt = place.tile, ch = place.sub, item = kt * a.cwin + ch;
  const int b = bh / a.Hk, hk = bh - b * a.Hk;
  const Seq seq = seq_of(a, b);
  const int k0 = kt * 128;
  int i0, i1;
  key_rows(a, seq, kt, RT, i0, i1);
  const int n = i1 - i0;
  const int c0 = i0 + (int)((int64_t)n * ch / nch), c1 = i0 + (int)((int64_t)n * (ch + 1) / nch);

  const int kb = wave & 3, half = wave >> 2;
  const bool bad = !strict || __builtin_amdgcn_readfirstlane(s_bad[kb]);   // are these the wave's results
  const int kw = k0 + kb * 32, key = kw + (lane & 31);
  const bool kok = key < seq.len;
  frag kf[KLDS ? 1 : I::NS], vf[I::NS];
  const char* kimg = smem + 2 * NB * RB;
  {
    const int kk = min(key, a.M - 1);
    if constexpr (KLDS) {
      KeyDma<T, DP, 128, NW> dma;
      dma.init(wave, lane, a.D);
      if (k0 < seq.len) dma.issue((const char*)a.k + b * a.kb + hk * a.kh, a.kt, k0, 0, seq.len, 0, lds_addr(smem) + 2 * NB * RB, wave);
    } else {
      load_frags<T, DP>((const char*)a.k + b * a.kb + (int64_t)kk * a.kt + hk * a.kh, kok, a.D, lane, kf);
    }
    load_frags<T, DP>((const char*)a.v + b * a.vb + (int64_t)kk * a.vt + hk * a.vh, kok, a.D, lane, vf);
  }
  // rows that see this lane's key: [vlo, vhi)
  int vlo = 0x7fffffff, vhi = 0;
  if (kok) {
    vlo = a.causal ? key * a.G : max(key - a.window + 1, 0) * a.G;
    vhi = (key + a.window) * a.G;
    if (key < a.sinks) {
      vhi = 0x7fffffff;
      if (!a.causal) vlo = 0;
    }
  }
  // rows that see all, or any, of the wave's keys
  const int klast = kw + 31;
  int alo = a.causal ? klast * a.G : max(klast - a.window + 1, 0) * a.G, ahi = (kw + a.window) * a.G;
  int nlo = a.causal ? kw * a.G : max(kw - a.window + 1, 0) * a.G, nhi = (klast + a.window) * a.G;
  if (klast < a.sinks) {
    ahi = 0x7fffffff;
    if (!a.causal) alo = 0;
  }
  if (kw < a.sinks) {
    nhi = 0x7fffffff;
    if (!a.causal) nlo = 0;
  }
  if (klast >= seq.len) alo = 0x7fffffff;
  if (kw >= seq.len) nhi = 0;

  int drow[NI];
  unsigned dch[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int c = (i * NW + wave) * 64 + lane;
    drow[i] = c / I::CPR;
    const int cc = (c % I::CPR) ^ I::swz(drow[i]);
    dch[i] = cc * 16 < a.D * I::ES ? (unsigned)cc * 16 : kOob;
  }
  const char* qbase = (const char*)a.q + b * a.qb + hk * a.G * a.qh;
  const char* obase = (const char*)a.dO + b * a.ob + hk * a.G * a.oh;
  const int rlim = min(seq.len * a.G, a.R);   // live rows
  auto issue = [&](int tile, unsigned img) __attribute__((always_inline)) {
    const int r0 = tile * RT, t0 = dm_div(a.dmG, r0);
    const i4_t rq = make_rsrc(qbase + t0 * a.qt), ro = make_rsrc(obase + t0 * a.ot);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = r0 + drow[i], t = dm_div(a.dmG, r), g = r - t * a.G;
      const unsigned bad = (r < rlim ? 0u : kOob) | (dch[i] & kOob);
      dma16(rq, bad | (dch[i] + (unsigned)((t - t0) * (int)a.qt + g * (int)a.qh)), img + (i * NW + wave) * 1024);
      dma16(ro, bad | (dch[i] + (unsigned)((t - t0) * (int)a.ot + g * (int)a.oh)), img + RB + (i * NW + wave) * 1024);
    }
  };
  const float* lbase = a.lse + (int64_t)bh * a.R;
  const float* dbase = a.delta + (int64_t)bh * a.R;
  auto stat = [&](int tile) __attribute__((always_inline)) {   // threads [0, RT): lse, [64, 64 + RT): delta
    const int i = tid & 63, r = tile * RT + i;
    if (i >= RT || wave > 1) return 0.f;
    if (wave == 0) return r < rlim ? lbase[r] : __builtin_inff();   // exp2(. - inf) = 0
    return r < rlim ? dbase[r] : 0.f;
  };
  auto put = [&](float v, int buf) __attribute__((always_inline)) {
    const int i = tid & 63;
    if (i < RT && wave == 0) s_l[buf][i] = v;
    if (i < RT && wave == 1) s_d[buf][i] = v;
  };
  f16_t dk[I::ND], dv[I::ND];
  I im;
  im.init(lane);
  // one 32 x 32 block in two phases: S and dP; then P, dS and the products with them
  f16_t s, dp;
  auto scores = [&](const char* cur, int rb) __attribute__((always_inline)) {
    s = zero16();
    dp = zero16();
#pragma unroll
    for (int st = 0; st < I::NS; ++st) {
      frag kk;
      if constexpr (KLDS) kk = im.row_frag(kimg + kb * 32 * I::PITCH, 0, st);
      else kk = kf[st];
      s = Mma<T>::mma(im.row_frag(cur, 32 * rb, st), kk, s);
      dp = Mma<T>::mma(im.row_frag(cur + RB, 32 * rb, st), vf[st], dp);
    }
    if constexpr (sizeof(T) == 2) interleave<(KLDS ? 6 : 4), 2, (KLDS ? 3 : 2), I::NS>();
  };
  auto products = [&](const char* cur, int buf, int r0, int rb, bool masked) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int rr = 32 * rb + 8 * g + 4 * (lane >> 5);
      const f4_t l4 = *(const f4_t*)&s_l[buf][rr], d4 = *(const f4_t*)&s_d[buf][rr];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[4 * g + e] = __builtin_amdgcn_exp2f(fmaf(s[4 * g + e], a.scale2, -l4[e]));
        dp[4 * g + e] = s[4 * g + e] * (dp[4 * g + e] - d4[e]);
      }
    }
    if (masked) {
      asm volatile("");
      const int rr = r0 + 4 * (lane >> 5), ge = vlo - rr, lt = (strict ? min(vhi, rlim) : vhi) - rr;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int c = 8 * (e >> 2) + (e & 3);
        const bool see = (c >= ge) & (c < lt);
        s[e] = see ? s[e] : 0.f;
        dp[e] = see ? dp[e] : 0.f;
      }
    }
    if constexpr (strict) {
      auto see = [&](int e) {
        const int row = r0 + 4 * (lane >> 5) + 8 * (e >> 2) + (e & 3);
        return row >= vlo && row < min(vhi, rlim);
      };
      if constexpr (which == kDv) strict_product<T, DP, false>(im, cur + RB, 32 * rb, s, dv, see);
      else strict_product<T, DP, false>(im, cur, 32 * rb, dp, dk, see);
    } else {
      __builtin_amdgcn_s_setprio(1);   // 220 -> 215 us
#pragma unroll
      for (int st = 0; st < 32 / Mma<T>::KS; ++st) {
        const frag pf = Mma<T>::pack(s, st), df = Mma<T>::pack(dp, st);
#pragma unroll
        for (int d = 0; d < I::ND; ++d) {
          dv[d] = Mma<T>::mma(im.col_frag(cur + RB, 32 * rb, st, d), pf, dv[d]);
          dk[d] = Mma<T>::mma(im.col_frag(cur, 32 * rb, st, d), df, dk[d]);
        }
      }
      if constexpr (sizeof(T) == 2) interleave<8, 1, 2, 4 * I::ND>();
      __builtin_amdgcn_s_setprio(0);
    }
  };

#pragma unroll
  for (int d = 0; d < I::ND; ++d) {
    if constexpr (k_sum) dk[d] = zero16();
    if constexpr (v_sum) dv[d] = zero16();
  }
  if (c0 < c1) {
    put(stat(c0), 0);
    issue(c0, lds_addr(smem));
  }
  for (int it = c0; it < c1; ++it) {
    const int buf = (it - c0) & 1;
    char* cur = smem + buf * 2 * RB;
    wait_vm<0>();
    lds_barrier();
    float nx = 0.f;
    const bool more = it + 1 < c1;
    if (more) {
      nx = stat(it + 1);
      issue(it + 1, lds_addr(smem) + (buf ^ 1) * 2 * RB);
    }
#pragma unroll 1   // one block's registers at a time; the other waves of the SIMD fill the gaps
    for (int rb = NW == 8 ? half : 0; rb < RT / 32; rb += NW == 8 ? 2 : 1) {
      const int r0 = it * RT + 32 * rb;
      if (bad && r0 < nhi && r0 + 32 > nlo) {
        scores(cur, rb);
        products(cur, buf, r0, rb, strict || r0 < alo || r0 + 32 > ahi);
      }
    }
    if (more) put(nx, buf ^ 1);
  }
  wait_vm<0>();   // K's DMA, where no row tile waited for it
  auto check = [&]() __attribute__((always_inline)) {
    if constexpr (!strict) {
      bool ok = true;
#pragma unroll
      for (int d = 0; d < I::ND; ++d) ok = ok && finite_all(dk[d]) && finite_all(dv[d]);
      const int any = __any(!ok);
      if (lane == 0 && half == 0) s_bad[kb] = any;
    }
  };
  if constexpr (NW != 8) check();
  __syncthreads();
  if constexpr (NW == 8) {
    // the second half's sums: [register group of 4][lane] in LDS, dK then dV
    float* x = (float*)smem + kb * 64 * (DP / 2) + lane * 4;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (i ? !v_sum : !k_sum) continue;
      f16_t(&acc)[I::ND] = i ? dv : dk;
      if (half == 1)
#pragma unroll
        for (int d = 0; d < I::ND; ++d)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *(float4*)(x + (d * 4 + g) * 256) = make_float4(acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2], acc[d][4 * g + 3]);
      __syncthreads();
      if (half == 0)
#pragma unroll
        for (int d = 0; d < I::ND; ++d)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const float4 v = *(const float4*)(x + (d * 4 + g) * 256);
            acc[d][4 * g] += v.x;
            acc[d][4 * g + 1] += v.y;
            acc[d][4 * g + 2] += v.z;
            acc[d][4 * g + 3] += v.w;
          }
      if (i == 1) check();
      __syncthreads();
    }
  }
  if (half == 0 && bad) {   // these are the wave's results
    if (a.cwin == 1 && !(kt < a.nsink && a.cfar)) {
      char* lds = smem + kb * 32 * out_pitch<DP>();
      auto at = [&](void* p) {
        return [&, p](int i) { return kw + i < a.M ? (T*)p + (((int64_t)b * a.M + kw + i) * a.Hk + hk) * a.D : nullptr; };
      };
      if constexpr (k_sum) store_rows<T, DP, false>(lds, dk, a.scale, a.D, lane, at(a.dk));
      if constexpr (v_sum) store_rows<T, DP, false>(lds, dv, 1.f, a.D, lane, at(a.dv));
    } else if (key < a.M) {
      const int items = a.cwin > 1 ? a.tiles * a.cwin : a.nsink;   // as in the join
      float* p = a.part + (((int64_t)bh * items + item) * 128 + kb * 32 + (lane & 31)) * 2 * a.D;
      if constexpr (k_sum) store_col<float, I::ND>(p, dk, a.scale, a.D, lane);
      if constexpr (v_sum) store_col<float, I::ND>(p + a.D, dv, 1.f, a.D, lane);
    }
  }
  if (!(s_bad[0] | s_bad[1] | s_bad[2] | s_bad[3])) return false;
  wait_vm<0>();   // the stores that the next ones replace
  lds_barrier();
  return true;
}
template <typename T, int DP, int which>
__device__ __forceinline__ void dkv_again(Again g, Spot place, int nch, unsigned stats) {
  place = Spot{uniform(place.bh), uniform(place.tile), uniform(place.sub)};
  dkv_pass<T, DP, which>(args_of(g), place, uniform(nch), g.tid, lds_at(g.smem),
                         *(typename Dkv<T, DP>::Stats*)lds_at(stats), (int*)lds_at(g.bad));
}
template <typename T, int DP>
__global__ void __launch_bounds__((64 * dkv_waves<T, DP>())) SIMD_WAVES(2) wattn_dkv_kernel(const WArgs a) {
  __shared__ __attribute__((aligned(256))) char smem[Dkv<T, DP>::LDS];
  __shared__ __attribute__((aligned(16))) typename Dkv<T, DP>::Stats stats;
  __shared__ int s_bad[4];
  int nch = 0;
  const Spot place = spot(a, a.tiles, 1, nch);
  if (place.bh < 0) return;
  if (dkv_pass<T, DP, kBoth>(a, place, nch, threadIdx.x, smem, stats, s_bad)) {
    dkv_again<T, DP, kDv>(again(smem, s_bad, threadIdx.x), place, nch, lds_addr(&stats));
    dkv_again<T, DP, kDk>(again(smem, s_bad, threadIdx.x), place, nch, lds_addr(&stats));
  }
}

// Rows beyond the window of the sinks' key tiles: they see `sinks` keys only.  A workgroup has one block
// of 32 sink keys (a.far32 of them) and one of cfar chunks of the rows; each wave runs through its own
// row blocks with its own LDS ring, without barriers; the waves' sums are added at the end into part.
// Measured as above (28 000 rows, 4 sinks): 18 us; as chunks of the key-major kernel the rows cost 40.
// all row blocks, their sums written; true: some are not finite
template <typename T, int DP, bool strict>
__device__ __forceinline__ bool far_pass(const WArgs& a, int L, int tid, char* smem, float (&s_st)[4][64]) {
  typedef Img<T, DP> I;
  typedef typename I::frag frag;
  constexpr int RB = 32 * I::PITCH, STG = RB <= 8192 ? 2 : 1, RING = STG * 2 * RB;
  constexpr int NI = RB / 1024;
  static_assert(RING >= 64 * DP * 4, "the sums fit a wave's ring");
  constexpr int RT = I::ROWS;   // as wattn_dkv_kernel
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ch = L % a.cfar, sb = L / a.cfar % a.far32, bh = L / (a.cfar * a.far32);
  const int b = bh / a.Hk, hk = bh - b * a.Hk;
  const Seq seq = seq_of(a, b);
  const int rlim = min(seq.len * a.G, a.R);   // live rows
  int i0, i1;
  key_rows(a, seq, sb / 4, RT, i0, i1);
  // row blocks [0, nlo) (causal: those rows come before the keys) and [hi0, hi0 + nhi)
  const int kw = sb * 32, key = kw + (lane & 31);
  const int nlo = a.causal || i0 == i1 ? 0 : i0 * (RT / 32);
  const int hi0 = i1 * (RT / 32), nhi = i0 == i1 ? 0 : max((rlim + 31) / 32 - hi0, 0);
  const int nb = kw < seq.len ? nlo + nhi : 0;
  const int c0 = (int)((int64_t)nb * ch / a.cfar) + wave, c1 = (int)((int64_t)nb * (ch + 1) / a.cfar);
  const bool kok = key < seq.len && key < a.sinks;

  frag kf[I::NS], vf[I::NS];
  {
    const int kk = min(key, a.M - 1);
    load_frags<T, DP>((const char*)a.k + b * a.kb + (int64_t)kk * a.kt + hk * a.kh, kok, a.D, lane, kf);
    load_frags<T, DP>((const char*)a.v + b * a.vb + (int64_t)kk * a.vt + hk * a.vh, kok, a.D, lane, vf);
  }
  const char* qbase = (const char*)a.q + b * a.qb + hk * a.G * a.qh;
  const char* obase = (const char*)a.dO + b * a.ob + hk * a.G * a.oh;
  char* ring = smem + wave * RING;
  auto row_of = [&](int i) __attribute__((always_inline)) { return (i < nlo ? i : hi0 + i - nlo) * 32; };
  float st_v = 0.f;   // lanes [0, 32): lse of the block in flight, [32, 64): delta
  auto issue = [&](int i, unsigned img) __attribute__((always_inline)) {
    const int r0 = row_of(i), t0 = dm_div(a.dmG, r0);
    const int rs = r0 + (lane & 31);
    st_v = lane < 32 ? __builtin_inff() : 0.f;   // exp2(. - inf) = 0
    if (rs < rlim) st_v = (lane < 32 ? a.lse : a.delta)[(int64_t)bh * a.R + rs];
    const i4_t rq = make_rsrc(qbase + t0 * a.qt), ro = make_rsrc(obase + t0 * a.ot);
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int c = j * 64 + lane, row = c / I::CPR, cc = (c % I::CPR) ^ I::swz(row);
      const int r = r0 + row, t = dm_div(a.dmG, r), g = r - t * a.G;
      const unsigned bad = r < rlim && cc * 16 < a.D * I::ES ? 0u : kOob;
      dma16(rq, bad | (unsigned)(cc * 16 + (t - t0) * (int)a.qt + g * (int)a.qh), img + j * 1024);
      dma16(ro, bad | (unsigned)(cc * 16 + (t - t0) * (int)a.ot + g * (int)a.oh), img + RB + j * 1024);
    }
  };
  f16_t dk[I::ND], dv[I::ND];
  I im;
  im.init(lane);
  float* out = a.part + far_at(a) + ((int64_t)bh * a.far32 * a.cfar + sb * a.cfar + ch) * 32 * 2 * a.D;
#pragma unroll
  for (int d = 0; d < I::ND; ++d) dk[d] = dv[d] = zero16();
  if (c0 < c1) issue(c0, lds_addr(ring));
  int cur = 0;
  for (int i = c0; i < c1; i += 4, cur = (cur + 1) % STG) {
    const char* q = ring + cur * 2 * RB;
    const unsigned nx = lds_addr(ring) + (cur + 1) % STG * 2 * RB;
    wait_vm<0>();   // this block is there (the wave has the other one in flight only from here on)
    s_st[wave][lane] = st_v;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // and the reads of the buffer filled next are done
    if (STG == 2 && i + 4 < c1) issue(i + 4, nx);
    f16_t s = zero16(), dp = zero16();
#pragma unroll
    for (int st = 0; st < I::NS; ++st) s = Mma<T>::mma(im.row_frag(q, 0, st), kf[st], s);
#pragma unroll
    for (int st = 0; st < I::NS; ++st) dp = Mma<T>::mma(im.row_frag(q + RB, 0, st), vf[st], dp);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f4_t l4 = *(const f4_t*)&s_st[wave][8 * g + 4 * (lane >> 5)], d4 = *(const f4_t*)&s_st[wave][32 + 8 * g + 4 * (lane >> 5)];
#pragma unroll
      for (int e = 0; e < 4; ++e) {   // every live row sees the lane's key if it is a sink: a select for the others
        const float p = __builtin_amdgcn_exp2f(fmaf(s[4 * g + e], a.scale2, -l4[e]));
        dp[4 * g + e] = kok ? p * (dp[4 * g + e] - d4[e]) : 0.f;
        s[4 * g + e] = kok ? p : 0.f;
      }
    }
    if constexpr (strict) {
      const int left = rlim - row_of(i) - 4 * (lane >> 5);
      auto see = [&](int e) { return kok && 8 * (e >> 2) + (e & 3) < left; };
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[e] = see(e) ? s[e] : 0.f;
        dp[e] = see(e) ? dp[e] : 0.f;
      }
      strict_product<T, DP, false>(im, q + RB, 0, s, dv, see);
      strict_product<T, DP, false>(im, q, 0, dp, dk, see);
    } else {
#pragma unroll
      for (int st = 0; st < 32 / Mma<T>::KS; ++st) {
        const frag pf = Mma<T>::pack(s, st), df = Mma<T>::pack(dp, st);
#pragma unroll
        for (int d = 0; d < I::ND; ++d) {
          dv[d] = Mma<T>::mma(im.col_frag(q + RB, 0, st, d), pf, dv[d]);
          dk[d] = Mma<T>::mma(im.col_frag(q, 0, st, d), df, dk[d]);
        }
      }
    }
    if (STG == 1 && i + 4 < c1) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      issue(i + 4, nx);
    }
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  float* x = (float*)ring + lane * 4;   // [dK, dV][register group of 4][lane]
#pragma unroll
  for (int d = 0; d < I::ND; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      *(float4*)(x + (d * 4 + g) * 256) = make_float4(dk[d][4 * g], dk[d][4 * g + 1], dk[d][4 * g + 2], dk[d][4 * g + 3]);
      *(float4*)(x + ((I::ND + d) * 4 + g) * 256) = make_float4(dv[d][4 * g], dv[d][4 * g + 1], dv[d][4 * g + 2], dv[d][4 * g + 3]);
    }
  __syncthreads();
  bool ok = true;
  for (int e = tid; e < 2 * I::ND * 4 * 64; e += 256) {
    const int ln = e & 63, grp = e >> 6, which = grp / (I::ND * 4), c = grp % (I::ND * 4) * 8 + 4 * (ln >> 5);
    float4 v = *(const float4*)((const float*)smem + e * 4);
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      const float4 y = *(const float4*)((const float*)(smem + w * RING) + e * 4);
      v.x += y.x;
      v.y += y.y;
      v.z += y.z;
      v.w += y.w;
    }
    const float f = which ? 1.f : a.scale;
    const float t = v.x * 0.f + v.y * 0.f + v.z * 0.f + v.w * 0.f;   // NaN where one is not finite
    ok = ok && (t == 0.f || kw + (ln & 31) >= a.sinks);              // (the join reads the sinks' alone)
    if (c < a.D) *(float4*)(out + (ln & 31) * 2 * a.D + which * a.D + c) = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
  }
  return !strict && __syncthreads_or(!ok);
}
template <typename T, int DP> __device__ __forceinline__ void far_again(Again g, int L) {
  typedef float Stat[4][64];
  far_pass<T, DP, true>(args_of(g), uniform(L), g.tid, lds_at(g.smem), *(Stat*)lds_at(g.bad));
}
template <typename T, int DP>
__global__ void __launch_bounds__(256) SIMD_WAVES(4) wattn_far_kernel(const WArgs a) {
  constexpr int RB = 32 * Img<T, DP>::PITCH, RING = (RB <= 8192 ? 2 : 1) * 2 * RB;
  __shared__ __attribute__((aligned(256))) char smem[4 * RING];
  __shared__ __attribute__((aligned(16))) float s_st[4][64];   // lse, delta of the block
  const int L = xcd_remap(blockIdx.x, a.far32 * a.cfar * a.B * a.Hk);
  if (L < 0) return;
  if (far_pass<T, DP, false>(a, L, threadIdx.x, smem, s_st)) far_again<T, DP>(again(smem, s_st, threadIdx.x), L);
}

// dK and dV of the key tiles in parts: the window's chunks, then the far rows' (sinks only), in order.
// One 4-column piece of dK or dV per thread.
template <typename T>
__global__ void __launch_bounds__(256) wattn_dkv_join_kernel(const WArgs a) {
  const int q = 2 * a.D / 4, ntile = a.cwin > 1 ? a.tiles : a.nsink, items = ntile * a.cwin;
  int nch = a.cwin;
  if (a.cwin != a.cmin) {   // then lengths are there, of at most kPackSeqs sequences
    int n;
    nch = chunks_of(a, __shfl(live_tiles(a, 1, n), 63, 64));
  }
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x, per = (int64_t)ntile * 128 * q;
  if (e >= per * a.B * a.Hk) return;
  const int bh = (int)(e / per);
  const int64_t rem = e - bh * per;
  const int c = (int)(rem % q) * 4, key = (int)(rem / q);
  if (key >= a.M) return;
  const float* p = a.part + (((int64_t)bh * items + key / 128 * a.cwin) * 128 + key % 128) * 2 * a.D + c;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < nch; ++i) {
    const float4 x = *(const float4*)(p + (int64_t)i * 128 * 2 * a.D);
    s[0] += x.x;
    s[1] += x.y;
    s[2] += x.z;
    s[3] += x.w;
  }
  if (a.cfar && key < a.sinks) {
    const float* f = a.part + far_at(a) + (((int64_t)bh * a.far32 + key / 32) * a.cfar * 32 + key % 32) * 2 * a.D + c;
    // sixteen in flight; of the last, fewer, the bits of what is there twice are off (0 times an infinity is NaN, and
    // what the compiler sees to be a select it makes branches around the loads: 6 -> 8 us)
    auto add = [&](int i, bool all) {
      float4 x[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = *(const float4*)(f + (int64_t)(all ? i + j : min(i + j, a.cfar - 1)) * 32 * 2 * a.D);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        unsigned in = all || i + j < a.cfar ? ~0u : 0u;
        if (!all) asm("" : "+v"(in));
        s[0] += __uint_as_float(__float_as_uint(x[j].x) & in);
        s[1] += __uint_as_float(__float_as_uint(x[j].y) & in);
        s[2] += __uint_as_float(__float_as_uint(x[j].z) & in);
        s[3] += __uint_as_float(__float_as_uint(x[j].w) & in);
      }
    };
    int i = 0;
    for (; i + 16 <= a.cfar; i += 16) add(i, true);
    if (i < a.cfar) add(i, false);
  }
  const int b = bh / a.Hk, hk = bh - b * a.Hk;
  T* dst = (T*)(c < a.D ? a.dk : a.dv) + (((int64_t)b * a.M + key) * a.Hk + hk) * a.D + (c < a.D ? c : c - a.D);
  store4<T>(dst, s[0], s[1], s[2], s[3]);
}

// ============================================================================ host
bool fill(const dfcsa_wattn_desc* d, WArgs& a, bool backward) {
  if (!d || (d->dtype != DFCSA_DT_F32 && d->dtype != DFCSA_DT_BF16)) return false;
  if (d->B <= 0 || d->T <= 0 || d->M <= 0 || d->H <= 0 || d->Hk <= 0 || d->H > 65536 || d->H % d->Hk || d->D < 8 || d->D % 8 ||
      d->D > 128 || d->window < 1 || d->sinks < 0 || !(d->scale > 0.f) || !std::isfinite(d->scale * kLog2e) || !d->q || !d->k || !d->v || !d->o)
    return false;
  if (!d->cached && d->T != d->M) return false;
  if (d->cached && (!d->lengths || backward || !d->causal)) return false;
  a.B = d->B; a.T = d->T; a.M = d->M; a.H = d->H; a.Hk = d->Hk; a.G = d->H / d->Hk; a.D = d->D;
  const int64_t R = (int64_t)d->T * a.G;
  // row and key arithmetic is 32 bits wide, up to (M + window) * G
  if (R > (1 << 29) || (int64_t)d->M * a.G > (1 << 29) || (int64_t)d->B * d->Hk > (1 << 24)) return false;
  a.R = (int)R;
  a.window = std::min(d->window, d->M);   // a window of M keys hides nothing
  a.sinks = std::min(d->sinks, d->M);
  a.causal = d->causal != 0;
  a.cached = d->cached != 0;
  a.scale = d->scale;
  a.scale2 = d->scale * kLog2e;
  a.dmG = make_divmod(a.G);
  const int es = d->dtype == DFCSA_DT_F32 ? 4 : 2;
  const void* ptr[4] = {d->q, d->k, d->v, backward ? d->dout : nullptr};
  const int64_t* str[4] = {d->q_stride, d->k_stride, d->v_stride, d->dout_stride};
  for (int i = 0; i < (backward ? 4 : 3); ++i) {
    if (!ptr[i] || (uintptr_t)ptr[i] % 16) return false;
    for (int j = 0; j < 3; ++j)
      if (str[i][j] < 0 || (str[i][j] * es) % 16) return false;
    // offsets within one tile are 32 bits wide (a tile of q or dout spans heads, one of k or v does not)
    const bool rows = i == 0 || i == 3;
    if (str[i][1] * es >= (1 << 23) || (rows && str[i][2] * es * a.G >= (1 << 29))) return false;
  }
  a.q = d->q; a.k = d->k; a.v = d->v;
  a.qb = d->q_stride[0] * es; a.qt = d->q_stride[1] * es; a.qh = d->q_stride[2] * es;
  a.kb = d->k_stride[0] * es; a.kt = d->k_stride[1] * es; a.kh = d->k_stride[2] * es;
  a.vb = d->v_stride[0] * es; a.vt = d->v_stride[1] * es; a.vh = d->v_stride[2] * es;
  a.lengths = d->lengths;
  a.o = d->o;
  a.rest = d->dtype == DFCSA_DT_BF16 ? (bf16_t*)d->o_rest : nullptr;
  a.lse = d->lse;
  a.part = d->work;
  a.splits = 1;
  a.dO = d->dout; a.ob = a.ot = a.oh = 0;
  a.delta = d->delta;
  a.dq = d->dq; a.dk = d->dk; a.dv = d->dv;
  a.nsink = a.cwin = a.cmin = a.far32 = a.cfar = a.tiles = 0;
  a.pack = a.lengths && !a.cached && a.B <= kPackSeqs;
  if (backward) {
    a.ob = d->dout_stride[0] * es; a.ot = d->dout_stride[1] * es; a.oh = d->dout_stride[2] * es;
    if (!d->lse || !d->delta || !d->dq || !d->dk != !d->dv) return false;   // dk and dv: both or neither
  }
  return true;
}

// a launch counts its threads in 32 bits (groups are padded, see grid_of)
bool fits(int64_t groups, int threads) { return (groups + 24) * threads < (int64_t)1 << 32; }
int dkv_threads(const WArgs& a, bool f32) { return !f32 && a.D > 64 ? 512 : 256; }
// threads of the join over ntile key tiles
int64_t join_items(const WArgs& a, int64_t ntile) { return ntile * 128 * (2 * a.D / 4) * a.B * a.Hk; }

// The forward's plan: few = the kernel whose waves split the keys of 32 rows; splits over the keys
// where the row tiles alone do not fill the card.  The estimate is in rounds of the waves (few: 128
// keys, else a tile of 64 or 32), 3 of which a workgroup takes to start and end, and the join about as
// long as 3: workgroups beyond one for each CU share it (wide and fp32 ones: the LDS or the matrix
// unit is then full, so two take twice as long; else two run in 1.4 times the time of one).
void plan_fwd(WArgs& a, bool f32, bool& few) {
  const int bh = a.B * a.Hk;
  few = a.R <= 64;
  a.tiles = few ? (a.R + 31) / 32 : (a.R + 127) / 128;
  const int64_t base = (int64_t)a.tiles * bh;
  // keys a row tile can see, whatever the lengths are
  const int64_t tok = std::min<int64_t>(((few ? 32 : 128) + a.G - 1) / a.G + 1, a.T);
  const int64_t span = std::min<int64_t>(a.M, (int64_t)a.window * (a.causal ? 1 : 2) + tok + a.sinks);
  const int64_t step = few ? 128 : (f32 ? 32 : 64), rounds = (span + step - 1) / step;
  const double two = few ? (a.D > 64 || f32 ? 2.0 : 1.4) : (f32 ? 2.0 : 1.4);
  double best = 0;
  a.splits = 1;
  for (int s = 1; s <= 64 && s <= rounds; ++s) {
    const int64_t per = (base * s + 255) / 256;   // workgroups of the fullest CU
    const double load = per <= 1 ? 1.0 : two * (double)per / 2.0;
    const double t = ((double)((rounds + s - 1) / s) + 3) * load + (s > 1 ? 3 + 0.05 * s : 0);
    if (s == 1 || t < best) {
      best = t;
      a.splits = s;
    }
  }
}
int64_t fwd_work(const WArgs& a) { return a.splits == 1 ? 0 : (int64_t)a.splits * a.B * a.Hk * a.R * (a.D + 1); }

// The backward's key tiles, and how many chunks their rows are split into.  A tile has `win` rows; more
// workgroups than run at once cost a second round of them all, too few leave CUs idle, and more than
// one chunk costs the fp32 parts' way to memory and back.  Estimated in microseconds: a row tile is 2
// (bf16, width 128; 64 x 128 pairs) or 6 (fp32, 32 x 128), a workgroup starts and ends in 4 of them, the
// parts move at 5 TB/s behind a 4 us launch.  The far rows are cut to a workgroup for each CU, a block of 32
// rows for each of its waves (two blocks: 21 instead of 14 us in fp32, 3 x 1531 tokens, 6 / 2 heads of 80).
void plan_bwd(WArgs& a, bool f32) {
  a.tiles = (a.M + 127) / 128;
  a.nsink = (a.sinks + 127) / 128;
  const int64_t bh = (int64_t)a.B * a.Hk, rt = f32 ? 32 : 64;
  const int slots = a.D <= 64 ? 512 : 256;
  const double tile = (f32 ? 6.0 : 2.0) * std::max(a.D, 32) / 128;
  const int64_t win = std::min<int64_t>(a.M, (int64_t)a.window * (a.causal ? 1 : 2) + 127) * a.G;
  const int64_t wt = (win + rt - 1) / rt;
  double best = 0;
  a.cwin = 1;
  for (int c = 1; c <= 8 && c <= std::max<int64_t>(1, wt / 2); ++c) {
    if (c > 1 && !(fits(a.tiles * bh * c, 512) && join_items(a, a.tiles) < (int64_t)1 << 30)) break;
    const double rounds = (double)((a.tiles * bh * c + slots - 1) / slots);
    double t = rounds * ((double)((wt + c - 1) / c) + 4) * tile;
    if (c > 1) t += 4 + (double)c * a.M * bh * a.D * 16 / 5e6;
    if (c == 1 || t < best) {
      best = t;
      a.cwin = c;
    }
  }
  // room for more chunks where padding may empty tiles; a single chunk has no join to add them in
  a.cmin = a.cwin;
  if (a.pack && a.cwin > 1 && fits(a.tiles * bh * 8, 512))
    a.cwin = (int)std::max<int64_t>(a.cwin, std::min<int64_t>(8, wt / 2));
  // tokens beyond the window of the first sink tile, and (two-sided) before that of the last
  const int64_t high = (int64_t)a.M - 127 - a.window;
  const int64_t low = a.causal ? 0 : (int64_t)(a.nsink - 1) * 128 - a.window + 1;
  const int64_t far = std::max<int64_t>(high, 0) + std::max<int64_t>(low, 0);
  a.far32 = a.cfar = 0;
  // a pass of their own costs two launches, about 12 us; without it the sinks' tiles take the far rows too
  if (a.sinks > 0 && (double)(far * a.G / rt) * tile > 12 && join_items(a, a.nsink) < (int64_t)1 << 30) {
    a.far32 = (a.sinks + 31) / 32;
    const int64_t blocks = (far * a.G + 31) / 32, base = bh * a.far32;
    a.cfar = (int)std::max<int64_t>(1, std::min<int64_t>({(256 + base - 1) / base, blocks / 4, 64}));
  }
}
int64_t bwd_work(const WArgs& a) { return !a.dk ? 0 : far_at(a) + (int64_t)a.B * a.Hk * a.far32 * a.cfar * 32 * 2 * a.D; }

#define BY_WIDTH(KERNEL, GRID, THREADS, ARGS)                                                        \
  do {                                                                                               \
    if (a.D <= 32) hipLaunchKernelGGL((KERNEL<T, 32>), GRID, dim3(THREADS), 0, st, ARGS);            \
    else if (a.D <= 64) hipLaunchKernelGGL((KERNEL<T, 64>), GRID, dim3(THREADS), 0, st, ARGS);       \
    else if (a.D <= 96) hipLaunchKernelGGL((KERNEL<T, 96>), GRID, dim3(THREADS), 0, st, ARGS);       \
    else hipLaunchKernelGGL((KERNEL<T, 128>), GRID, dim3(THREADS), 0, st, ARGS);                     \
  } while (0)

template <typename T>
int run_fwd(const WArgs& a, bool few, hipStream_t st) {
  const int items = a.tiles * a.B * a.Hk * a.splits;
  const dim3 grid((unsigned)(few ? xcd_pad(items) : grid_of(a, items)));
  if (few) BY_WIDTH(wattn_few_kernel, grid, 256, a);
  else BY_WIDTH(wattn_fwd_kernel, grid, 256, a);
  DFCSA_CHECK_LAUNCH();
  if (a.splits > 1) {
    const int64_t rows = (int64_t)a.B * a.Hk * a.R;
    hipLaunchKernelGGL((wattn_join_kernel<T>), dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, st, a);
    DFCSA_CHECK_LAUNCH();
  }
  return 0;
}
template <typename T>
int run_bwd(WArgs a, hipStream_t st) {
  WArgs q = a;
  q.tiles = (a.R + 127) / 128;
  {
    const WArgs& a = q;
    BY_WIDTH(wattn_dq_kernel, dim3((unsigned)grid_of(a, (int64_t)a.tiles * a.B * a.Hk)), 256, a);
  }
  DFCSA_CHECK_LAUNCH();
  if (!a.dk) return 0;
  const int bh = a.B * a.Hk;
  BY_WIDTH(wattn_dkv_kernel, dim3((unsigned)grid_of(a, (int64_t)a.tiles * a.cwin * bh)), dkv_threads(a, sizeof(T) == 4), a);
  DFCSA_CHECK_LAUNCH();
  if (a.cfar) {
    BY_WIDTH(wattn_far_kernel, dim3((unsigned)xcd_pad(a.far32 * a.cfar * bh)), 256, a);
    DFCSA_CHECK_LAUNCH();
  }
  const int ntile = a.cwin > 1 ? a.tiles : (a.cfar ? a.nsink : 0);
  if (ntile) {
    const int64_t e = join_items(a, ntile);
    hipLaunchKernelGGL((wattn_dkv_join_kernel<T>), dim3((unsigned)((e + 255) / 256)), dim3(256), 0, st, a);
    DFCSA_CHECK_LAUNCH();
  }
  return 0;
}

}  // namespace

extern "C" {

int dfcsa_wattn_work_floats(const dfcsa_wattn_desc* d, int backward, int64_t* floats) {
  WArgs a;
  if (!floats || !fill(d, a, backward != 0)) return DFCSA_EINVAL;
  if (backward) {
    plan_bwd(a, d->dtype == DFCSA_DT_F32);
    *floats = bwd_work(a);
  } else {
    bool few;
    plan_fwd(a, d->dtype == DFCSA_DT_F32, few);
    *floats = fwd_work(a);
  }
  return 0;
}

int dfcsa_wattn_fwd(const dfcsa_wattn_desc* d, void* stream) {
  WArgs a;
  if (!fill(d, a, false)) return DFCSA_EINVAL;
  bool few;
  plan_fwd(a, d->dtype == DFCSA_DT_F32, few);
  if (!fits((int64_t)a.tiles * a.B * a.Hk * a.splits, 256)) return DFCSA_EINVAL;
  if (a.splits > 1 && !fits(((int64_t)a.B * a.Hk * a.R + 7) / 8, 256)) return DFCSA_EINVAL;
  if (fwd_work(a) > 0 && (!d->work || d->work_floats < fwd_work(a))) return DFCSA_EINVAL;
  return d->dtype == DFCSA_DT_F32 ? run_fwd<float>(a, few, (hipStream_t)stream) : run_fwd<bf16_t>(a, few, (hipStream_t)stream);
}

int dfcsa_wattn_bwd(const dfcsa_wattn_desc* d, void* stream) {
  WArgs a;
  if (!fill(d, a, true)) return DFCSA_EINVAL;
  plan_bwd(a, d->dtype == DFCSA_DT_F32);
  const int64_t bh = (int64_t)a.B * a.Hk;
  if (!fits((a.R + 127) / 128 * bh, 256) || !fits((int64_t)a.tiles * a.cwin * bh, dkv_threads(a, d->dtype == DFCSA_DT_F32)) ||
      !fits((int64_t)a.far32 * a.cfar * bh, 256))
    return DFCSA_EINVAL;
  if (bwd_work(a) > 0 && (!d->work || d->work_floats < bwd_work(a))) return DFCSA_EINVAL;
  return d->dtype == DFCSA_DT_F32 ? run_bwd<float>(a, (hipStream_t)stream) : run_bwd<bf16_t>(a, (hipStream_t)stream);
}

}  // extern "C"
