// Attention of a drafted tree over the page pool for MI355X (gfx950), behind include/barq_ragged.h:
//
//   out[b, h, i, :] = softmax_x(scale * q[b, h, i, :] . K_x) V_x   over the cached positions of row b (read
//   from the pages through the block table) and the tree's nodes j with mask[b, i, j] (read from the node
//   tensors), h of KV head h / G.
//
// Split.  The G * T query rows of a (row, KV head) pair share every key and value, so a workgroup takes a block of
// 32 * WQ of them and a range of the pair's tiles of positions: the cached ones, then the nodes.  Its four waves
// are WQ groups of 32 query rows by WK = 4 / WQ groups of a tile's positions.  Ranges of one pair are joined by a
// second launch from their unnormalised sums, maxima and sums (32 bits), or the one range writes the output.
//
// A tile's keys and values go through registers into LDS, the next tile's loads in flight while this one is
// computed, the block table's entries one tile further ahead.
//
// Arithmetic.  S^T = K Q^T and O^T = V^T P^T on the 32x32x16 MFMA, so that a lane holds 16 positions' scores of ONE
// query row: the softmax needs no lane exchange but with lane ^ 32, and the lane's scores are, as they stand, its
// operand of the second product, whose positions are taken in the order 16k + {0-3, 8-11} (lanes below 32) and
// 16k + {4-7, 12-15}.  V^T comes from LDS by the transposing read of four positions at a time.  Both products of
// 16-bit numbers are exact in the MFMA's 32-bit sums.  Probabilities are handed over as two 16-bit numbers each,
// the rounded value and the rounded remainder (2^-17 of the value is lost in bf16): one alone would add an error
// as large as the output's own rounding.  Running maximum and sum per query row in base 2, 32 bits; the sums are
// rescaled only when a maximum grows by more than 2^8, which every exponent here holds.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

#include "barq_kv.h"
#include "barq_kv_fp8.h"
#include "barq_ragged.h"
#include "fastdiv.h"

namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kWords = BARQ_TREE_MAX_NODES / 32;  // mask words of a node
constexpr int64_t kI32Max = 0x7fffffff;
enum : int { kBF16 = BARQ_KV_BF16, kF16 = BARQ_KV_FP16 };

struct TreeArgs {
  const char* kpages;
  const char* vpages;
  const int32_t* block_table;
  const int32_t* seq_lens;
  int32_t* errors;
  int64_t page_bytes;
  const char* q;
  const char* nk;
  const char* nv;
  const uint8_t* mask;
  char* out;
  int64_t q_sb, q_sh, q_st;  // bytes
  int64_t n_sb, n_sh, n_st;
  int64_t m_sb, m_si, m_sj;
  int64_t o_sb, o_sh, o_st;
  float* part;               // unnormalised sums [pair, split, row, dim], then maxima and sums [pair, split, row, 2]
  float* part_ml;
  FastDiv div_page, div_group;
  int32_t row_bytes;         // bytes between positions of a page
  int32_t head_bytes;
  int32_t num_pages, max_blocks, kv_heads, group, nodes, rows, max_seq;
  int32_t row_blocks;        // blocks of query rows of a pair
  int32_t splits;            // ranges of a pair, at most
  int32_t range;             // tiles of a range
  int32_t units;             // pairs * splits
  int32_t pairs;
  float scale_log2;
  // fp8 cold store: a table entry -2 - c names cold page c
  const uint8_t* kcodes;
  const uint8_t* vcodes;
  const uint8_t* kscales;
  const uint8_t* vscales;
  int32_t num_cold, page_size;
};

// What a workgroup takes, by head size and groups of query rows.
template <int HD, int WQ>
struct Shape {
  static constexpr int kWK = 4 / WQ;
  static constexpr int kSub = WQ == 4 ? 2 : 1;       // 32-position pieces of a tile that a wave takes
  static constexpr int kTile = 32 * kWK * kSub;      // positions of a tile
  static constexpr int kRows = 32 * WQ;              // query rows
  static constexpr int kChunks = HD / 8;             // 16-byte pieces of a position's head
  static constexpr int kStep = kThreads / kChunks;   // positions that the workgroup loads at once
  static constexpr int kLoads = kTile / kStep;
  static constexpr int kRowBytes = HD * 2;
  static constexpr int kTileBytes = kTile * kRowBytes;
};

template <int E>
__device__ __forceinline__ f32x16 mfma(const u32x4 a, const u32x4 b, f32x16 c) {
  if constexpr (E == kBF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
}

template <int E>
__device__ __forceinline__ uint32_t pack2(float x, float y) {  // both rounded to nearest even
  const f32x2 v = {x, y};
  if constexpr (E == kBF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}
template <int E>
__device__ __forceinline__ float low_of(uint32_t w) {
  if constexpr (E == kBF16) return __uint_as_float(w << 16);
  else return (float)__builtin_bit_cast(_Float16, (uint16_t)w);
}
template <int E>
__device__ __forceinline__ float high_of(uint32_t w) {
  if constexpr (E == kBF16) return __uint_as_float(w & 0xffff0000u);
  else return (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16));
}

// Whether any of a 16-byte vector's 8 elements is an infinity or a NaN.
template <int E>
__device__ __forceinline__ bool nonfinite8(const u32x4 w) {
  constexpr uint32_t ex = E == kBF16 ? 0x7F80u : 0x7C00u;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) bad |= (w[i] & ex) == ex || ((w[i] >> 16) & ex) == ex;
  return bad;
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// The values of lanes l & 31 and (l & 31) + 32, in every lane.
__device__ __forceinline__ f32x2 halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return f32x2{__uint_as_float(r[0]), __uint_as_float(r[1])};
}

// LDS of the workgroup is ordered around a barrier; loads from memory stay in flight.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Places of 16-byte piece c of position p in a tile's rows, such that the lanes of a read -- 8 positions' same
// piece of keys, 4 adjacent positions' 64 bytes of values -- fall on different banks.
template <int HD>
__device__ __forceinline__ int key_at(int p, int c) {
  return p * (HD * 2) + ((c ^ (p & (HD == 64 ? 7 : 15))) << 4);
}
template <int HD>
__device__ __forceinline__ int value_at(int p, int c) {
  return p * (HD * 2) + ((c ^ ((HD == 64 ? (p >> 1) & 1 : p & 3) << 2)) << 4);
}

// A page's entry as an index of pages (or, cold, -2 - cold page), 0 and flagged where it names none.
template <bool COLD>
__device__ __forceinline__ int checked_entry(const TreeArgs& a, int e) {
  if (e >= 0 && e < a.num_pages) return e;
  if (COLD && e <= -2 && -2 - e < a.num_cold) return e;
  atomicOr(a.errors, BARQ_KV_ERRBIT_BAD_INDEX);
  return 0;
}

template <int E, typename OutT>
__device__ __forceinline__ void store4(char* p, const f32x4 v) {
  if constexpr (sizeof(OutT) == 4) *(f32x4*)p = v;
  else *(u32x2*)p = u32x2{pack2<E>(v[0], v[1]), pack2<E>(v[2], v[3])};
}

template <int E, int HD, int WQ, bool COLD, typename OutT>
__global__ void __launch_bounds__(kThreads, HD == 256 ? 1 : 2) tree_kernel(const TreeArgs a) {
  using S = Shape<HD, WQ>;
  constexpr int kDT = HD / 32;     // 32-dim tiles of the output
  constexpr int kKS = HD / 16;     // k-steps of the scores
  // keys, then values, of one tile; at the end the other position groups' sums
  constexpr int kJoin = (S::kWK - 1) * WQ * (kDT * 16 + 2) * 64 * 4;
  constexpr int kLds = 2 * S::kTileBytes > kJoin ? 2 * S::kTileBytes : kJoin;
  __shared__ __attribute__((aligned(16))) char s_tile[kLds];
  __shared__ uint32_t s_mask[S::kRows][kWords];
  __shared__ uint32_t s_bad[kWords];  // nodes whose V holds an infinity or a NaN: stored as zeros in the tile

  const int id = (int)blockIdx.x;
  // Row blocks of one unit read the same pages: 8 ids apart they run on one XCD and share its L2.
  const int unit = id / (8 * a.row_blocks) * 8 + (id & 7);
  const int rb = (id >> 3) % a.row_blocks;
  if (unit >= a.units) return;
  const int kvh = unit % a.kv_heads;
  const int bs = unit / a.kv_heads;
  const int b = bs / a.splits;
  const int split = bs - b * a.splits;
  int len = a.seq_lens[b];
  if (len > a.max_seq) {
    if (split == 0 && kvh == 0 && rb == 0 && threadIdx.x == 0) atomicOr(a.errors, BARQ_KV_ERRBIT_ATTN_SHORT);
    len = a.max_seq;
  }
  len = max(len, 0);
  const int ctiles = (len + S::kTile - 1) / S::kTile;
  const int tiles = ctiles + (a.nodes + S::kTile - 1) / S::kTile;
  const int tile0 = split * a.range, tile1 = min(tile0 + a.range, tiles);
  if (tile0 >= tile1) return;

  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int qg = wave % WQ, kg = wave / WQ;
  const int l32 = lane & 31, half = lane >> 5;
  const int row = rb * S::kRows + qg * 32 + l32;    // query row: node * G + head of the group
  const int node_row = (int)a.div_group.div((uint32_t)min(row, a.rows - 1));
  const int head = kvh * a.group + min(row, a.rows - 1) - node_row * a.group;
  const bool wave_live = rb * S::kRows + qg * 32 < a.rows;

  u32x4 q[kKS];
  {
    const char* qp = a.q + (int64_t)b * a.q_sb + (int64_t)head * a.q_sh + (int64_t)node_row * a.q_st + half * 16;
#pragma unroll
    for (int k = 0; k < kKS; ++k) q[k] = *(const u32x4*)(qp + k * 32);
  }

  const int node_lo = (int)a.div_group.div((uint32_t)(rb * S::kRows));
  if (tile1 > ctiles) {  // the tree's mask as bits
    const int count = (int)a.div_group.div((uint32_t)min(rb * S::kRows + S::kRows - 1, a.rows - 1)) - node_lo + 1;
    for (int i = wave; i < count; i += 4) {
      const int n = node_lo + i;
      for (int j0 = 0; j0 < a.nodes; j0 += 64) {
        const int j = j0 + lane;
        bool sees = j <= n;
        if (a.mask && j < a.nodes)
          sees = a.mask[(int64_t)b * a.m_sb + (int64_t)n * a.m_si + (int64_t)j * a.m_sj] != 0;
        const uint64_t bits = __ballot(sees && j < a.nodes);
        if (lane == 0) {
          s_mask[i][j0 / 32] = (uint32_t)bits;
          s_mask[i][j0 / 32 + 1] = (uint32_t)(bits >> 32);
        }
      }
    }
    if (tid < kWords) s_bad[tid] = 0;
  }

  // ---- loads: thread t takes piece t % kChunks of positions t / kChunks + i * kStep
  const int c = tid % S::kChunks, p0 = tid / S::kChunks;
  const int32_t* table = a.block_table + (int64_t)b * a.max_blocks;
  int entry[S::kLoads];
  u32x4 kreg[S::kLoads], vreg[S::kLoads];
  uint32_t cold_mask = 0, vshift = 0;  // of the tile in the registers
  (void)vshift;
  auto load_entries = [&](int tile) {
    if (tile >= ctiles) return;
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i)
      entry[i] = table[a.div_page.div((uint32_t)min(tile * S::kTile + p0 + i * S::kStep, len - 1))];
  };
  auto load_tile = [&](int tile) {
    cold_mask = 0;
    if (tile < ctiles) {
      int64_t at[S::kLoads];
#pragma unroll
      for (int i = 0; i < S::kLoads; ++i) {
        const int pos = min(tile * S::kTile + p0 + i * S::kStep, len - 1);
        const int e = checked_entry<COLD>(a, entry[i]);
        const int off = pos - (int)a.div_page.div((uint32_t)pos) * (int)a.div_page.d;
        if constexpr (COLD) {
          const bool cold = e < 0;
          const int64_t cp = -2 - (int64_t)e;
          cold_mask |= (uint32_t)cold << i;
          // 8 bytes of codes and 8 of scales, or 16 of elements
          const int64_t el = (cp * a.page_size + off) * (a.row_bytes / 2) + (int64_t)kvh * HD + c * 8;
          const int64_t ks = (cp * a.kv_heads + kvh) * HD + c * 8;
          const int64_t vs = ((cp * a.page_size + off) * a.kv_heads + kvh);
          const int64_t hot = (int64_t)e * a.page_bytes + (int64_t)off * a.row_bytes + (int64_t)kvh * a.head_bytes + c * 16;
          const char* k0 = cold ? (const char*)a.kcodes + el : a.kpages + hot;
          const char* k1 = cold ? (const char*)a.kscales + ks : a.kpages + hot + 8;
          const char* v0 = cold ? (const char*)a.vcodes + el : a.vpages + hot;
          const char* v1 = cold ? (const char*)a.vscales + (vs & ~(int64_t)7) : a.vpages + hot + 8;
          const u32x2 ka = *(const u32x2*)k0, kb = *(const u32x2*)k1;
          const u32x2 va = *(const u32x2*)v0, vb = *(const u32x2*)v1;
          kreg[i] = u32x4{ka[0], ka[1], kb[0], kb[1]};
          vreg[i] = u32x4{va[0], va[1], vb[0], vb[1]};
          at[i] = 0;
        } else {
          at[i] = (int64_t)e * a.page_bytes + (int64_t)off * a.row_bytes + (int64_t)kvh * a.head_bytes + c * 16;
        }
      }
      if constexpr (!COLD) {
#pragma unroll
        for (int i = 0; i < S::kLoads; ++i) {
          kreg[i] = *(const u32x4*)(a.kpages + at[i]);
          vreg[i] = *(const u32x4*)(a.vpages + at[i]);
        }
      }
    } else {
      const int64_t base = (int64_t)b * a.n_sb + (int64_t)kvh * a.n_sh + c * 16;
#pragma unroll
      for (int i = 0; i < S::kLoads; ++i) {
        const int64_t at = base + (int64_t)min((tile - ctiles) * S::kTile + p0 + i * S::kStep, a.nodes - 1) * a.n_st;
        kreg[i] = *(const u32x4*)(a.nk + at);
        vreg[i] = *(const u32x4*)(a.nv + at);
      }
    }
  };
  auto store_tile = [&](int tile) {
    const int limit = tile < ctiles ? len - tile * S::kTile : a.nodes - (tile - ctiles) * S::kTile;
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      const int p = p0 + i * S::kStep;
      u32x4 k = kreg[i], v = vreg[i];
      if constexpr (COLD) {
        if (cold_mask >> i & 1) {
          uint32_t w[4];
          barq_fp8::dequant8<E>(k[0], k[1], k[2], k[3], w);
          k = u32x4{w[0], w[1], w[2], w[3]};
          const int pos = min(tile * S::kTile + p, len - 1);
          const int off = pos - (int)a.div_page.div((uint32_t)pos) * (int)a.div_page.d;
          const int byte = (off * a.kv_heads + kvh) & 7;  // a page's scales begin at a multiple of 8
          const uint32_t s = ((byte & 4 ? v[3] : v[2]) >> (byte & 3) * 8 & 0xFFu) * 0x01010101u;
          barq_fp8::dequant8<E>(v[0], v[1], s, s, w);
          v = u32x4{w[0], w[1], w[2], w[3]};
        }
      }
      bool keep = p < limit;
      if (tile >= ctiles && keep && nonfinite8<E>(v)) {
        const int j = (tile - ctiles) * S::kTile + p;
        atomicOr(&s_bad[j / 32], 1u << (j % 32));
        keep = false;
      }
      *(u32x4*)(s_tile + key_at<HD>(p, c)) = k;
      *(u32x4*)(s_tile + S::kTileBytes + value_at<HD>(p, c)) = keep ? v : u32x4{0, 0, 0, 0};
    }
  };

  f32x16 o[kDT];
#pragma unroll
  for (int d = 0; d < kDT; ++d) o[d] = f32x16{0};
  float m = -INFINITY, l = 0.0f;

  // V's transposing read: lane i of 16 gives the address of position i / 4 and dims 4 (i % 4), and gets dim i of
  // the four positions.
  const int vp = (lane & 15) >> 2, vc = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1), vb = (lane & 1) * 8;

  auto compute = [&](int tile) {
    f32x16 s[S::kSub];
    uint32_t seen[S::kSub];
#pragma unroll
    for (int u = 0; u < S::kSub; ++u) {
      const int pb = (kg * S::kSub + u) * 32;
      if (tile < ctiles) {
        const int n = len - tile * S::kTile - pb;
        seen[u] = n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u;
      } else {
        const int jb = (tile - ctiles) * S::kTile + pb;
        seen[u] = jb < a.nodes && row < a.rows ? s_mask[node_row - node_lo][jb / 32] : 0u;
      }
      s[u] = f32x16{0};
#pragma unroll
      for (int k = 0; k < kKS; ++k)
        s[u] = mfma<E>(*(const u32x4*)(s_tile + key_at<HD>(pb + l32, 2 * k + half)), q[k], s[u]);
    }
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < S::kSub; ++u) {
      if (__any(seen[u] != ~0u)) {
        const uint32_t w = seen[u] >> (4 * half);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[u][i] = w >> (8 * (i / 4) + i % 4) & 1 ? s[u][i] : -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[u][i]);
    }
    const f32x2 tops = halves(top);
    top = fmaxf(tops[0], tops[1]) * a.scale_log2;
    if (__any(top > m + 8.0f)) {
      const float fresh = fmaxf(m, top);
      const float by = fresh == -INFINITY ? 1.0f : exp2_(m - fresh);
      m = fresh;
      l *= by;
#pragma unroll
      for (int d = 0; d < kDT; ++d) o[d] *= by;
    }
    const float shift = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int u = 0; u < S::kSub; ++u) {
      const int pb = (kg * S::kSub + u) * 32;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[u][i] = exp2_(fmaf(s[u][i], a.scale_log2, -shift));
        l += s[u][i];
      }
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        u32x4 hi, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = s[u][8 * kk + 2 * e], y = s[u][8 * kk + 2 * e + 1];
          hi[e] = pack2<E>(x, y);
          lo[e] = pack2<E>(x - low_of<E>(hi[e]), y - high_of<E>(hi[e]));
        }
        const int at = pb + 16 * kk + 4 * half + vp;
#pragma unroll
        for (int d = 0; d < kDT; ++d) {
          typedef __attribute__((address_space(3))) s16x4 lds4;
          const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds4*)(s_tile + S::kTileBytes + value_at<HD>(at, d * 4 + vc) + vb));
          const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds4*)(s_tile + S::kTileBytes + value_at<HD>(at + 8, d * 4 + vc) + vb));
          const u32x2 w0 = __builtin_bit_cast(u32x2, v0), w1 = __builtin_bit_cast(u32x2, v1);
          const u32x4 v = {w0[0], w0[1], w1[0], w1[1]};
          o[d] = mfma<E>(v, lo, o[d]);
          o[d] = mfma<E>(v, hi, o[d]);
        }
      }
      // Nodes whose V is not finite, for the rows that see them alone.
      if (tile >= ctiles) {
        const int jb = (tile - ctiles) * S::kTile + pb;
        uint32_t bad = jb < a.nodes ? __builtin_amdgcn_readfirstlane(s_bad[jb / 32]) : 0u;
        while (bad) {
          const int j = __builtin_ctz(bad);
          bad &= bad - 1;
          float p = 0.0f;
#pragma unroll
          for (int i = 0; i < 16; ++i) p = (j >> 3) * 4 + (j & 3) == i ? s[u][i] : p;
          const f32x2 both = halves(p);
          p = j & 4 ? both[1] : both[0];
          const char* vrow = a.nv + (int64_t)b * a.n_sb + (int64_t)kvh * a.n_sh + (int64_t)(jb + j) * a.n_st + half * 8;
#pragma unroll
          for (int d = 0; d < kDT; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const u32x2 w = *(const u32x2*)(vrow + d * 64 + g * 16);
              if (p > 0.0f) {
                o[d][4 * g] += p * low_of<E>(w[0]);
                o[d][4 * g + 1] += p * high_of<E>(w[0]);
                o[d][4 * g + 2] += p * low_of<E>(w[1]);
                o[d][4 * g + 3] += p * high_of<E>(w[1]);
              }
            }
        }
      }
    }
  };

  load_entries(tile0);
  load_tile(tile0);
  load_entries(tile0 + 1);
  for (int tile = tile0; tile < tile1; ++tile) {
    if (tile > tile0 || tile1 > ctiles) lds_barrier();  // the tile before is read; the mask is written
    store_tile(tile);
    if (tile + 1 < tile1) {
      load_tile(tile + 1);
      load_entries(tile + 2);
    }
    lds_barrier();
    if (wave_live) compute(tile);
  }
  const f32x2 ls = halves(l);
  l = ls[0] + ls[1];

  if constexpr (S::kWK > 1) {  // join the groups of positions
    lds_barrier();
    float* s_join = (float*)s_tile;
    constexpr int kPer = kDT * 16 + 2;
    if (kg > 0) {
      float* to = s_join + (int64_t)((kg - 1) * WQ + qg) * kPer * 64;
#pragma unroll
      for (int d = 0; d < kDT; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *(f32x4*)(to + (d * 4 + g) * 256 + lane * 4) =
              f32x4{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
      to[kDT * 1024 + lane] = m;
      to[kDT * 1024 + 64 + lane] = l;
    }
    lds_barrier();
    if (kg > 0) return;
    float top = m, ms[S::kWK], scale[S::kWK];
    ms[0] = m;
#pragma unroll
    for (int k = 1; k < S::kWK; ++k) {
      ms[k] = s_join[(int64_t)((k - 1) * WQ + qg) * kPer * 64 + kDT * 1024 + lane];
      top = fmaxf(top, ms[k]);
    }
#pragma unroll
    for (int k = 0; k < S::kWK; ++k) scale[k] = ms[k] == -INFINITY ? 0.0f : exp2_(ms[k] - top);
    m = top;
    l *= scale[0];
#pragma unroll
    for (int d = 0; d < kDT; ++d) o[d] *= scale[0];
#pragma unroll
    for (int k = 1; k < S::kWK; ++k) {
      const float* from = s_join + (int64_t)((k - 1) * WQ + qg) * kPer * 64;
      l += scale[k] * from[kDT * 1024 + 64 + lane];
#pragma unroll
      for (int d = 0; d < kDT; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 v = *(const f32x4*)(from + (d * 4 + g) * 256 + lane * 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[d][4 * g + e] += scale[k] * v[e];
        }
    }
  }
  if (row >= a.rows) return;
  const int parts = (tiles + a.range - 1) / a.range;
  if (parts == 1) {
    const float by = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    char* op = a.out + (int64_t)b * a.o_sb + (int64_t)head * a.o_sh + (int64_t)node_row * a.o_st +
               half * 4 * (int)sizeof(OutT);
#pragma unroll
    for (int d = 0; d < kDT; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        store4<E, OutT>(op + (d * 32 + g * 8) * (int)sizeof(OutT),
                        f32x4{o[d][4 * g] * by, o[d][4 * g + 1] * by, o[d][4 * g + 2] * by, o[d][4 * g + 3] * by});
  } else {
    const int64_t rec = ((int64_t)(b * a.kv_heads + kvh) * a.splits + split) * a.rows + row;
    float* to = a.part + rec * HD + half * 4;
#pragma unroll
    for (int d = 0; d < kDT; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *(f32x4*)(to + d * 32 + g * 8) = f32x4{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
    if (half == 0) *(f32x2*)(a.part_ml + rec * 2) = f32x2{m, l};
  }
}

// Joins the ranges of a pair, in their order: HD / 4 threads a query row.
template <int E, int HD, typename OutT>
__global__ void __launch_bounds__(kThreads) tree_join_kernel(const TreeArgs a, int tile_positions) {
  constexpr int kPer = kThreads / (HD / 4);
  const int pair = (int)blockIdx.x;
  const int row = (int)blockIdx.y * kPer + (int)threadIdx.x / (HD / 4);
  const int d = ((int)threadIdx.x % (HD / 4)) * 4;
  if (row >= a.rows) return;
  const int b = pair / a.kv_heads, kvh = pair - b * a.kv_heads;
  const int len = max(min(a.seq_lens[b], a.max_seq), 0);
  const int tiles = (len + tile_positions - 1) / tile_positions + (a.nodes + tile_positions - 1) / tile_positions;
  const int parts = (tiles + a.range - 1) / a.range;
  if (parts == 1) return;
  const int64_t rec = (int64_t)pair * a.splits * a.rows + row;
  float top = -INFINITY;
  for (int s = 0; s < parts; ++s) top = fmaxf(top, a.part_ml[(rec + (int64_t)s * a.rows) * 2]);
  f32x4 sum = {0, 0, 0, 0};
  float l = 0.0f;
  for (int s = 0; s < parts; ++s) {
    const int64_t at = rec + (int64_t)s * a.rows;
    const f32x2 ml = *(const f32x2*)(a.part_ml + at * 2);
    const float by = ml[0] == -INFINITY ? 0.0f : exp2_(ml[0] - top);
    sum += by * *(const f32x4*)(a.part + at * HD + d);
    l += by * ml[1];
  }
  const float by = l > 0.0f || l != l ? 1.0f / l : 0.0f;
  const int node = (int)a.div_group.div((uint32_t)row);
  store4<E, OutT>(a.out + (int64_t)b * a.o_sb + (int64_t)(kvh * a.group + row - node * a.group) * a.o_sh +
                      (int64_t)node * a.o_st + d * (int)sizeof(OutT),
                  sum * by);
}

struct Plan {
  int wq, tile, row_blocks;
  int64_t splits, range, pairs, rows;
};

// How a call is cut: query rows by the fewest blocks, then ranges of tiles so that the launch fills the GPU.
bool plan_of(const barq_kv_pool* p, int64_t batch, int64_t q_heads, int64_t nodes, int64_t max_seq, int64_t mean_seq,
             Plan* out) {
  if (!p || p->elem_bytes != 2 || (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256)) return false;
  if (p->kv_heads < 1 || batch < 1 || batch > p->max_batch || q_heads < 1 || q_heads % p->kv_heads || nodes < 1 ||
      nodes > BARQ_TREE_MAX_NODES || max_seq < 0 || mean_seq < 0)
    return false;
  const int64_t cap = p->max_blocks * p->page_size;
  const int64_t longest = max_seq == 0 ? cap : std::min(max_seq, cap);
  const int64_t rows = q_heads / p->kv_heads * nodes;
  if (rows > (int64_t(1) << 17)) return false;
  const int wq = rows > 64 ? 4 : rows > 32 || p->head_dim == 256 ? 2 : 1;
  const int tile = wq == 1 ? 128 : 64;
  const int64_t pairs = batch * p->kv_heads, blocks = (rows + 32 * wq - 1) / (32 * wq);
  const auto tiles_of = [&](int64_t n) { return (n + tile - 1) / tile + (nodes + tile - 1) / tile; };
  const int64_t most = tiles_of(longest), mean = tiles_of(mean_seq ? std::min(mean_seq, longest) : longest);
  const int64_t want = p->head_dim == 256 ? 256 : 512;  // workgroups that are resident at once
  // A range keeps two tiles at least; mean tiles a pair over all of the launch's ranges.
  int64_t range = std::max<int64_t>(2, (mean * pairs * blocks + want - 1) / want);
  range = std::min(range, most);
  out->wq = wq;
  out->tile = tile;
  out->row_blocks = (int)blocks;
  out->range = range;
  out->splits = (most + range - 1) / range;
  out->pairs = pairs;
  out->rows = rows;
  return pairs * out->splits * blocks < (int64_t(1) << 30);
}

int64_t workspace_of(const Plan& p, int64_t hd) {
  return p.splits == 1 ? 0 : p.pairs * p.splits * p.rows * (hd + 2) * 4;
}

using Kernel = const void*;
template <int E, int HD, bool COLD, typename OutT>
Kernel by_shape(int wq) {
  if constexpr (HD != 256)
    if (wq == 1) return (Kernel)&tree_kernel<E, HD, 1, COLD, OutT>;
  return wq == 2 ? (Kernel)&tree_kernel<E, HD, 2, COLD, OutT> : (Kernel)&tree_kernel<E, HD, 4, COLD, OutT>;
}
template <int E, typename OutT>
Kernel by_head(int64_t hd, bool cold, int wq) {
  if (hd == 256) return by_shape<E, 256, false, OutT>(wq);
  if (hd == 128) return cold ? by_shape<E, 128, true, OutT>(wq) : by_shape<E, 128, false, OutT>(wq);
  return cold ? by_shape<E, 64, true, OutT>(wq) : by_shape<E, 64, false, OutT>(wq);
}
template <int E, typename OutT>
Kernel join_of(int64_t hd) {
  return hd == 256   ? (Kernel)&tree_join_kernel<E, 256, OutT>
         : hd == 128 ? (Kernel)&tree_join_kernel<E, 128, OutT>
                     : (Kernel)&tree_join_kernel<E, 64, OutT>;
}

int launch(Kernel kernel, dim3 grid, void** args, void* stream) {
  if (hipLaunchKernel(kernel, grid, dim3(kThreads), args, 0, (hipStream_t)stream) == hipSuccess) return BARQ_KV_OK;
  (void)hipGetLastError();
  return BARQ_KV_ERR_LAUNCH;
}

}  // namespace

extern "C" {

int64_t barq_tree_attention_workspace_bytes(const barq_kv_pool* pool, int64_t batch, int64_t q_heads, int64_t nodes,
                                            int64_t max_seq, int64_t mean_seq) {
  Plan p;
  return plan_of(pool, batch, q_heads, nodes, max_seq, mean_seq, &p) ? workspace_of(p, pool->head_dim) : -1;
}

int barq_tree_attention(const barq_kv_pool* pool, const barq_kv_cold* cold, const void* query, int64_t batch,
                        int64_t q_heads, int64_t nodes, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_t,
                        const void* node_key, const void* node_value, int64_t node_stride_b, int64_t node_stride_h,
                        int64_t node_stride_t, const uint8_t* mask, int64_t mask_stride_b, int64_t mask_stride_i,
                        int64_t mask_stride_j, void* out, int64_t out_stride_b, int64_t out_stride_h,
                        int64_t out_stride_t, float scale, int64_t max_seq, int64_t mean_seq, int64_t flags,
                        void* workspace, int64_t workspace_bytes, void* stream) {
  Plan plan;
  if (!pool || !pool->key_pages || !pool->value_pages || !pool->block_table || !pool->seq_lens || !pool->ctrl ||
      !query || !node_key || !node_value || !out || (flags & ~(int64_t)(BARQ_KV_ATTN_FP16 | BARQ_KV_ATTN_OUT_F32)) ||
      pool->num_pages < 1 || pool->num_pages > kI32Max || pool->page_size < 1 || pool->max_blocks < 1 ||
      pool->max_blocks * pool->page_size > kI32Max || pool->kv_heads * pool->head_dim * 2 > kI32Max ||
      !plan_of(pool, batch, q_heads, nodes, max_seq, mean_seq, &plan))
    return BARQ_KV_ERR_INVALID;
  const bool f16 = flags & BARQ_KV_ATTN_FP16, f32 = flags & BARQ_KV_ATTN_OUT_F32;
  const int64_t os = f32 ? 4 : 2, hd = pool->head_dim;
  const uint64_t in_bits = (uint64_t)(uintptr_t)query | (uint64_t)(uintptr_t)node_key | (uint64_t)(uintptr_t)node_value |
                           (uint64_t)(uintptr_t)pool->key_pages | (uint64_t)(uintptr_t)pool->value_pages |
                           (uint64_t)((q_stride_b | q_stride_h | q_stride_t | node_stride_b | node_stride_h | node_stride_t) * 2);
  if ((in_bits & 15) || ((uint64_t)(uintptr_t)out | (uint64_t)((out_stride_b | out_stride_h | out_stride_t) * os)) & (uint64_t)(4 * os - 1))
    return BARQ_KV_ERR_INVALID;
  if (q_stride_b < 0 || q_stride_h < 0 || q_stride_t < 0 || node_stride_b < 0 || node_stride_h < 0 || node_stride_t < 0 ||
      out_stride_b < 0 || out_stride_h < 0 || out_stride_t < 0 || mask_stride_b < 0 || mask_stride_i < 0 || mask_stride_j < 0)
    return BARQ_KV_ERR_INVALID;
  if (cold && (hd == 256 || pool->page_size % 16 || !cold->key_codes || !cold->value_codes || !cold->key_scales ||
               !cold->value_scales || cold->num_cold < 1 || cold->num_cold >= kI32Max - 2 ||
               cold->element_type != (f16 ? BARQ_KV_FP16 : BARQ_KV_BF16) ||
               (((uintptr_t)cold->key_codes | (uintptr_t)cold->value_codes | (uintptr_t)cold->key_scales |
                 (uintptr_t)cold->value_scales) & 7)))
    return BARQ_KV_ERR_INVALID;
  const int64_t need = workspace_of(plan, hd);
  if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))) return BARQ_KV_ERR_INVALID;
  const int64_t cap = pool->max_blocks * pool->page_size;
  TreeArgs a = {};
  a.kpages = (const char*)pool->key_pages;
  a.vpages = (const char*)pool->value_pages;
  a.block_table = pool->block_table;
  a.seq_lens = pool->seq_lens;
  a.errors = pool->ctrl + BARQ_KV_CTRL_ERRORS;
  a.head_bytes = (int32_t)(hd * 2);
  a.row_bytes = (int32_t)(pool->kv_heads * hd * 2);
  a.page_bytes = pool->page_size * (int64_t)a.row_bytes;
  a.q = (const char*)query;
  a.nk = (const char*)node_key;
  a.nv = (const char*)node_value;
  a.mask = mask;
  a.out = (char*)out;
  a.q_sb = q_stride_b * 2, a.q_sh = q_stride_h * 2, a.q_st = q_stride_t * 2;
  a.n_sb = node_stride_b * 2, a.n_sh = node_stride_h * 2, a.n_st = node_stride_t * 2;
  a.m_sb = mask_stride_b, a.m_si = mask_stride_i, a.m_sj = mask_stride_j;
  a.o_sb = out_stride_b * os, a.o_sh = out_stride_h * os, a.o_st = out_stride_t * os;
  a.part = (float*)workspace;
  a.part_ml = a.part + plan.pairs * plan.splits * plan.rows * hd;
  a.group = (int32_t)(q_heads / pool->kv_heads);
  a.div_page = FastDiv::make((uint32_t)pool->page_size);
  a.div_group = FastDiv::make((uint32_t)a.group);
  a.num_pages = (int32_t)pool->num_pages;
  a.max_blocks = (int32_t)pool->max_blocks;
  a.kv_heads = (int32_t)pool->kv_heads;
  a.nodes = (int32_t)nodes;
  a.rows = (int32_t)plan.rows;
  a.max_seq = (int32_t)(max_seq == 0 ? cap : std::min(max_seq, cap));
  a.row_blocks = plan.row_blocks;
  a.splits = (int32_t)plan.splits;
  a.range = (int32_t)plan.range;
  a.pairs = (int32_t)plan.pairs;
  a.units = (int32_t)(plan.pairs * plan.splits);
  a.scale_log2 = scale * 1.44269504088896340736f;
  a.page_size = (int32_t)pool->page_size;
  if (cold) {
    a.kcodes = (const uint8_t*)cold->key_codes;
    a.vcodes = (const uint8_t*)cold->value_codes;
    a.kscales = (const uint8_t*)cold->key_scales;
    a.vscales = (const uint8_t*)cold->value_scales;
    a.num_cold = (int32_t)cold->num_cold;
  }
  const Kernel kernel = f16 ? (f32 ? by_head<kF16, float>(hd, cold, plan.wq) : by_head<kF16, uint16_t>(hd, cold, plan.wq))
                            : (f32 ? by_head<kBF16, float>(hd, cold, plan.wq) : by_head<kBF16, uint16_t>(hd, cold, plan.wq));
  void* args[] = {&a};
  int rc = launch(kernel, dim3((uint32_t)((a.units + 7) / 8 * 8 * plan.row_blocks)), args, stream);
  if (rc == BARQ_KV_OK && plan.splits > 1) {
    const Kernel join = f16 ? (f32 ? join_of<kF16, float>(hd) : join_of<kF16, uint16_t>(hd))
                            : (f32 ? join_of<kBF16, float>(hd) : join_of<kBF16, uint16_t>(hd));
    int32_t tile = plan.tile;
    void* jargs[] = {&a, &tile};
    const int64_t per = kThreads / (hd / 4);
    rc = launch(join, dim3((uint32_t)plan.pairs, (uint32_t)((plan.rows + per - 1) / per)), jargs, stream);
  }
  return rc;
}

}  // extern "C"
