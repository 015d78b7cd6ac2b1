// Attention of a drafted tree over the page pool for MI355X (gfx950), behind include/barq_ragged.h:
//
//   out[b, h, i, :] = softmax_x(scale * q[b, h, i, :] . K_x) V_x   over the cached positions of row b (read
//   from the pages through the block table) and the tree's nodes j with mask[b, i, j] (read from the node
//   tensors), h of KV head h / G.
//
// Split.  The G * T query rows of a (row, KV head) pair share every key and value, so a workgroup takes a block of
// 32 * WQ of them and a range of the pair's tiles of positions: the cached ones and the nodes.  Its waves are WQ
// groups of 32 query rows by WK groups of a tile's positions.  Ranges of one pair are joined by a second launch from
// their unnormalised sums, maxima and sums (32 bits), or the one range writes the output.  Two kernels:
//   tree_kernel       little work, page sizes and trees that the other does not take: the host cuts each pair into
//                     equal ranges; tiles go through registers into LDS, the next one's loads in flight while this
//                     one is computed, the block table's entries one tile further ahead.
//   tree_flat_kernel  the rest, and fp8 pages: the device cuts the list of all pairs' tiles; tiles go straight to LDS.
//
// Arithmetic.  S^T = K Q^T and O^T = V^T P^T on the 32x32x16 MFMA, so that a lane holds 16 positions' scores of ONE
// query row: the softmax needs no lane exchange but with lane ^ 32, and the lane's scores are, as they stand, its
// operand of the second product, whose positions are taken in the order 16k + {0-3, 8-11} (lanes below 32) and
// 16k + {4-7, 12-15}.  V^T comes from LDS by the transposing read of four positions at a time.  Both products of
// 16-bit numbers are exact in the MFMA's 32-bit sums.  Probabilities are handed over as two 16-bit numbers each,
// the rounded value and the rounded remainder (2^-17 of the value is lost in bf16): one alone would add an error
// as large as the output's own rounding.  Running maximum and sum per query row in base 2, 32 bits; the sums are
// rescaled only when a maximum grows by more than 2^8, which every exponent here holds.
//
// What bounds it.  Few query rows: the pages' bytes.  From about 64 query rows a pair the matrix units: with the
// remainders' product a key costs 1.5 times the two products' operations.  64 nodes of 8 heads a KV head over 32 rows
// of up to 4,096 positions run at 960 TFLOP/s, three quarters of what one large product reaches on the card; deeper
// prefetch, another order of products and softmax, wave priorities and other batches of reads changed that by 2% at
// most, and the remainders' share is the price of errors as small as the rounding of the output.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "barq_kv.h"
#include "barq_kv_commit.h"
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
  int32_t batch, groups;     // of the flat schedule: rows, groups of workgroups
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

// A page's entry as an index of pages, 0 and flagged where it names none.
__device__ __forceinline__ int checked_entry(const TreeArgs& a, int e) {
  if (e >= 0 && e < a.num_pages) return e;
  atomicOr(a.errors, BARQ_KV_ERRBIT_BAD_INDEX);
  return 0;
}

template <int E, typename OutT>
__device__ __forceinline__ void store4(char* p, const f32x4 v) {
  if constexpr (sizeof(OutT) == 4) *(f32x4*)p = v;
  else *(u32x2*)p = u32x2{pack2<E>(v[0], v[1]), pack2<E>(v[2], v[3])};
}

template <int E, int HD, int WQ, typename OutT>
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
  auto load_entries = [&](int tile) {
    if (tile >= ctiles) return;
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i)
      entry[i] = table[a.div_page.div((uint32_t)min(tile * S::kTile + p0 + i * S::kStep, len - 1))];
  };
  auto load_tile = [&](int tile) {
    if (tile < ctiles) {
      int64_t at[S::kLoads];
#pragma unroll
      for (int i = 0; i < S::kLoads; ++i) {
        const int pos = min(tile * S::kTile + p0 + i * S::kStep, len - 1);
        const int off = pos - (int)a.div_page.div((uint32_t)pos) * (int)a.div_page.d;
        at[i] = (int64_t)checked_entry(a, entry[i]) * a.page_bytes + (int64_t)off * a.row_bytes + (int64_t)kvh * a.head_bytes + c * 16;
      }
#pragma unroll
      for (int i = 0; i < S::kLoads; ++i) {
        kreg[i] = *(const u32x4*)(a.kpages + at[i]);
        vreg[i] = *(const u32x4*)(a.vpages + at[i]);
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
      const u32x4 k = kreg[i], v = vreg[i];
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

// ------------------------------------------------------------------- two-byte pages, asynchronous tiles
// The flat schedule: every (row, KV head) pair's tiles, the tree's nodes first and then the cached positions, form
// one list; group g of row_blocks workgroups takes the g-th equal range of it, whatever the rows' lengths.
// A range's piece of a pair that is not the whole pair leaves a record (slot 2g for a piece that begins inside its
// pair, else 2g + 1: a range has at most one of each), joined by a second launch in the order of the groups.
//
// A tile's keys and values go to LDS by asynchronous loads, 128 KB of them: the stages but one are in flight while
// one is computed.  Each step a wave waits for its own loads of the next
// tile, decodes what codes it loaded, and meets the others at one barrier; nothing else waits for memory.
// Whole calls, host's cut and tiles through registers -> this (us; 8 KV heads of 128): 16 rows of 512 to 2,048
// positions, 24 nodes x 4 query heads 53.6 -> 39.6; one row of 32,749, 64 x 4 95.9 -> 77.0; 32 rows of 512 to 4,096,
// 64 x 8 355 -> 265; 4 heads of 256, 12 rows of 1,500, 7 x 2 31.4 -> 27.7; 16 rows of 2,000, fp8 pages, 16 x 4
// 96.1 -> 43.0.
template <int HD, int TILE>
struct Ring {
  static constexpr int kTile = TILE;                 // positions of a tile
  static constexpr int kBytes = kTile * HD * 2;      // of its keys, or values
  static constexpr int kStages = 65536 / kBytes;     // tiles in LDS: 128 KB of them
  static constexpr int kChunks = HD / 8;
  static constexpr int kGroup = 64 / kChunks;        // positions that one load of a wave covers
};

__device__ __forceinline__ int row_length(const TreeArgs& a, int b) { return max(min(a.seq_lens[b], a.max_seq), 0); }

template <int KT>
__device__ __forceinline__ int pair_tiles(const TreeArgs& a, int len) {
  return (len + KT - 1) / KT + (a.nodes + KT - 1) / KT;
}

// The list's length of one KV head's pair of row b: its tiles, after kPairCost places for what a pair costs besides
// (query, table, mask, nodes, record: 9 to 12 us with 256 query rows, where a tile takes 2.3).  With 2 places the workgroup with a row of
// no positions took 283 us where the average took 190; with 5 all 32 rows take 250; 4, 6 and 8 within 2%.
constexpr int kPairCost = 5;
template <int KT>
__device__ __forceinline__ int pair_places(const TreeArgs& a, int len) {
  return pair_tiles<KT>(a, len) + kPairCost;
}

// Places of one KV head of rows [0, b), and of all rows.  Run by a whole wave.
template <int KT>
__device__ __forceinline__ void count_places(const TreeArgs& a, int b, int lane, int* before, int* all) {
  int upto = 0, sum = 0;
  for (int r0 = 0; r0 < a.batch; r0 += 64) {
    const int r = r0 + lane;
    const int t = r < a.batch ? pair_places<KT>(a, row_length(a, r)) : 0;
    sum += barq_commit::wave_sum(t);
    upto += barq_commit::wave_sum(r < b ? t : 0);
  }
  *before = upto;
  *all = sum;
}

__device__ __forceinline__ int range_of(const TreeArgs& a, int all) {
  return max(1, (all * a.kv_heads + a.groups - 1) / a.groups);
}

// 16 bytes a lane from `key` + `key_at` to LDS at `to` + 16 * lane, and from `value` + `value_at` to `gap` bytes
// further, asynchronously: counted by vmcnt, with no register in flight.  (As a builtin, every LDS read would wait
// for all of them.)  The idle cycles cover a scalar register that a vector instruction has just written, and m0.
__device__ __forceinline__ void load_lds(const char* key, uint32_t key_at, const char* value, uint32_t value_at,
                                         uint32_t to, uint32_t gap) {
  asm volatile(
      "s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\t"
      "global_load_lds_dwordx4 %4, %5" ::"s"(to), "v"(key_at), "s"(key), "s"(to + gap), "v"(value_at), "s"(value)
      : "memory");
}

// The same of 4 bytes a lane, or of 16 bytes a lane from one place.
__device__ __forceinline__ void load_lds1(const char* from, uint32_t at, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dword %1, %2" ::"s"(to), "v"(at), "s"(from) : "memory");
}
__device__ __forceinline__ void load_lds4(const char* from, uint32_t at, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(at), "s"(from) : "memory");
}

// Wait for all but the newest N of the wave's loads (then BARRIER: for the workgroup); LDS is ordered around it.
template <int N, bool BARRIER>
__device__ __forceinline__ void wait_loads() {
  if constexpr (BARRIER) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
  else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// All but the newest `tiles` (at most MOST) of PER loads each.
template <int PER, int MOST, bool BARRIER>
__device__ __forceinline__ void wait_tiles(int tiles) {
  if constexpr (MOST > 0)
    if (tiles < MOST) return wait_tiles<PER, MOST - 1, BARRIER>(tiles);
  wait_loads<PER * MOST, BARRIER>();
}
// The same of LDS alone: loads stay in flight.
__device__ __forceinline__ void lds_only_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// A scale byte as a float, 2^(s - 127).
__device__ __forceinline__ float scale_of(uint32_t s) { return __uint_as_float(max(s << 23, 0x00400000u)); }

// Codes 0 and 1 (HIGH: 2 and 3) of four E4M3 codes times a scale, as two 16-bit numbers.  The instruction's products
// are exact wherever the 16-bit type holds them, and rounded to nearest even elsewhere: equal to barq_kv_fp8.h's
// element by element for all 256 codes at all scale bytes but 255 (compared one by one on the GPU), which is E8M0's
// NaN and stored by no quantiser.
template <int E, bool HIGH>
__device__ __forceinline__ uint32_t scaled2(uint32_t codes, float scale) {
  if constexpr (E == kBF16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, HIGH));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, HIGH));
}

template <int E, int HD, int WQ, int WK, int TILE, bool COLD, typename OutT>
__global__ void __launch_bounds__(64 * WQ * WK, WQ * WK == 8 ? 2 : 1) tree_flat_kernel(const TreeArgs a) {
  using R = Ring<HD, TILE>;
  constexpr int kNW = WQ * WK, kTile = R::kTile, kRows = 32 * WQ, kStages = R::kStages;
  constexpr int kSub = kTile / (32 * WK);  // 32-position pieces of a tile that a wave takes
  constexpr int kDT = HD / 32, kKS = HD / 16;
  constexpr int kPos = kTile / kNW, kLoads = kPos / R::kGroup;  // a wave's positions of a tile, loads of K and of V
  static_assert(kSub >= 1 && kLoads >= 1 && 2 * kLoads * (kStages - 1) < 64, "loads in flight that a wait can count");
  constexpr int kKeys = 2;  // pieces of keys read at once
  constexpr int kPer = kDT * 16 + 2;
  static_assert((WK - 1) * WQ * kPer * 256 <= kStages * 2 * R::kBytes, "the joined sums fit the ring");
  __shared__ __attribute__((aligned(1024))) char s_ring[2 * kStages * R::kBytes];  // stages of keys and of values
  __shared__ __attribute__((aligned(8))) uint32_t s_mask[kRows][kWords];
  __shared__ uint32_t s_bad[kWords];

  const int id = (int)blockIdx.x;
  const int group = id / (8 * a.row_blocks) * 8 + (id & 7);
  const int rb = (id >> 3) % a.row_blocks;
  if (group >= a.groups) return;
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int qg = wave % WQ, kg = wave / WQ;
  const int l32 = lane & 31, half = lane >> 5;
  if (id == 0)
    for (int b = tid; b < a.batch; b += 64 * kNW)
      if (a.seq_lens[b] > a.max_seq) atomicOr(a.errors, BARQ_KV_ERRBIT_ATTN_SHORT);

  // ---- this group's range: [at, end) of the list; it begins in row b
  int len_lane = lane < a.batch ? row_length(a, lane) : 0;  // of the 64 rows from len_row on
  int len_row = 0;
  asm volatile("" : "+v"(len_lane));  // waited for here, as below
  int all = barq_commit::wave_sum(lane < a.batch ? pair_places<kTile>(a, len_lane) : 0);
  for (int r0 = 64; r0 < a.batch; r0 += 64)
    all += barq_commit::wave_sum(r0 + lane < a.batch ? pair_places<kTile>(a, row_length(a, r0 + lane)) : 0);
  const int range = range_of(a, all);
  int at = group * range;
  const int end = min(at + range, all * a.kv_heads);
  if (at >= end) return;
  int b = 0, row_start = 0;  // row b's first place in the list
  for (;;) {
    const int here = len_row + lane < a.batch ? pair_places<kTile>(a, len_lane) * a.kv_heads : 0;
    const int incl = barq_commit::wave_incl_scan(here);
    const uint64_t past = __ballot(row_start + incl > at && here > 0);
    if (past) {
      const int k = __builtin_ctzll(past);
      b = len_row + k;
      row_start += __builtin_amdgcn_readlane(incl - here, k);
      break;
    }
    row_start += __builtin_amdgcn_readlane(incl, 63);
    len_row += 64;
    len_lane = len_row + lane < a.batch ? row_length(a, len_row + lane) : 0;
    asm volatile("" : "+v"(len_lane));
  }

  const int row = rb * kRows + qg * 32 + l32;  // query row: node * G + head of the group
  const int node_row = (int)a.div_group.div((uint32_t)min(row, a.rows - 1));
  const int group_head = min(row, a.rows - 1) - node_row * a.group;
  const int node_lo = (int)a.div_group.div((uint32_t)(rb * kRows));
  const bool wave_live = rb * kRows + qg * 32 < a.rows;
  const int ntiles = (a.nodes + kTile - 1) / kTile;
  // a lane's place in a load: position lane / kChunks of the group, and for the place of a piece in LDS the piece
  // that belongs there
  const int lp = lane / R::kChunks, slot_c = lane % R::kChunks;
  const int node_c = tid % R::kChunks, node_p = tid / R::kChunks;
  constexpr int kNodeStep = 64 * kNW / R::kChunks, kNodeLoads = kTile / kNodeStep;
  // The lanes' places in a tile: of their key's piece of k-step 0 (step k: bits of k << 5 turned over) and of V's
  // transposing read of dims 0 .. 31 (dims 32 d ..: bits of d << 6).  For that lane i of 16 gives the address of
  // position i / 4 and dims 4 (i % 4), and gets dim i of the four positions.
  const int vp = (lane & 15) >> 2;
  const uint32_t key_lane = (uint32_t)key_at<HD>(kg * kSub * 32 + l32, half);
  const uint32_t value_lane = (uint32_t)(R::kBytes + value_at<HD>(kg * kSub * 32 + 4 * half + vp,
                                                                 ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) +
                                         (lane & 1) * 8);
  // and, from a wave's first position of a tile on, of what it loads: of a load's group of positions its own, and of
  // that the piece that belongs in its place
  const uint32_t key_from = (uint32_t)(lp * a.row_bytes) + (uint32_t)(slot_c ^ ((wave * kPos + lp) & (HD == 64 ? 7 : 15))) * 16;
  const uint32_t value_from = (uint32_t)(lp * a.row_bytes) +
                              (uint32_t)(slot_c ^ ((HD == 64 ? (lp >> 1) & 1 : (wave * kPos + lp) & 3) << 2)) * 16;
  // turned over in these for the i-th group
  constexpr auto key_turn = [](int i) { return (uint32_t)((i * R::kGroup) & (HD == 64 ? 7 : 15)) << 4; };
  constexpr auto value_turn = [](int i) { return HD == 64 ? 0u : (uint32_t)((i * R::kGroup) & 3) << 6; };
  const int block_step = kTile / (int)a.div_page.d, place_step = kTile % (int)a.div_page.d;  // of a tile
  // Cold pages: a wave takes its positions of a tile in units of two loads' groups, of which each lies in one page and
  // has as many loads of codes and scales as of elements.  A unit's codes go to the front of its keys' (values') place
  // in LDS, its scales 1 KB behind, and the wave decodes them where they are before the tile's step.
  constexpr int kUnit = 2 * R::kGroup, kUnits = kPos / kUnit;
  static_assert(!COLD || (kPos % kUnit == 0 && kUnits <= 4 && kStages <= 4), "units of a tile in four bits");
  const int code_p = lane / (HD / 16);  // the position of a unit that a lane loads the codes of, from `code_from` on
  const uint32_t code_from = (uint32_t)(code_p * (a.row_bytes / 2) + lane % (HD / 16) * 16);
  uint32_t colds = 0;  // the units of the stages' tiles that hold codes
  constexpr int kWhole = 8;
  static_assert(kPos % kWhole == 0 && kWhole % R::kGroup == 0, "whole parts of a wave's positions");
  const bool whole = (int)a.div_page.d % kWhole == 0;  // so many of a wave's positions of a tile lie in one page

  for (bool first = true; at < end;) {
    if (b >= len_row + 64) {
      len_row += 64;
      len_lane = len_row + lane < a.batch ? row_length(a, len_row + lane) : 0;
      asm volatile("" : "+v"(len_lane));
    }
    const int len = __builtin_amdgcn_readlane(len_lane, b - len_row);
    const int tiles = pair_tiles<kTile>(a, len), places = tiles + kPairCost;
    const int kvh = (at - row_start) / places;
    if (kvh >= a.kv_heads) {  // the next row
      row_start += places * a.kv_heads;
      ++b;
      continue;
    }
    const int pair_start = row_start + kvh * places + kPairCost;  // its first tile's place
    const int t0 = max(at - pair_start, 0), t1 = min(tiles, end - pair_start);
    at = pair_start + max(t1, 0);
    if (t1 <= t0) break;  // the range ends before the pair's first tile
    const int head = kvh * a.group + group_head;
    const int count = t1 - t0, nodes_here = max(min(t1, ntiles) - t0, 0);  // tiles, and those of nodes, first
    const int c0 = max(t0 - ntiles, 0);                                    // the first cached tile

    // What a piece needs once is read again from the kernel's arguments: scalar registers are for the tiles.
    const __attribute__((address_space(4))) TreeArgs* rare =
        (const __attribute__((address_space(4))) TreeArgs*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(rare));

    u32x4 q[kKS];
    {
      const char* qp = rare->q + (int64_t)b * rare->q_sb + (int64_t)head * rare->q_sh + (int64_t)node_row * rare->q_st + half * 16;
#pragma unroll
      for (int k = 0; k < kKS; ++k) q[k] = *(const u32x4*)(qp + k * 32);
    }

    // ---- cached tiles: each wave loads kPos positions of a tile, a group of kGroup in one load
    const int32_t* table = rare->block_table + (int64_t)b * rare->max_blocks;
    const int last_blk = count > nodes_here ? (int)a.div_page.div((uint32_t)(len - 1)) : 0;
    const auto entries = [&](int blk0) __attribute__((always_inline)) {  // a window of the block table, one entry a lane
      const int e = blk0 + lane <= last_blk ? table[blk0 + lane] : 0;
      if (e >= 0 && e < rare->num_pages) return e;
      if (COLD && e <= -2 && -2 - e < rare->num_cold) return e;
      atomicOr(rare->errors, BARQ_KV_ERRBIT_BAD_INDEX);
      return 0;
    };
    // The wave's block (place in it) of the next tile to load; the entries of 64 blocks from blk0 on and of the 64
    // after them, one a lane.
    int blk0 = 0, blk = 0, place = 0, window = 0, ahead = 0;
    if (count > nodes_here) {
      const int pos = c0 * kTile + wave * kPos;
      blk = (int)a.div_page.div((uint32_t)pos);
      place = pos - blk * (int)a.div_page.d;
      blk0 = min(blk, last_blk);
      window = entries(blk0);
      ahead = entries(blk0 + 64);
    }
    // The query has come when the table has: waited for here, and not in the loop.
#pragma unroll
    for (int k = 0; k < kKS; ++k) asm volatile("" : "+v"(q[k]));
    asm volatile("" : "+v"(window), "+v"(ahead));
    const int64_t head_at = (int64_t)kvh * a.head_bytes;
    // The piece's tile t of keys (V: of values) into its stage.  Nodes go through registers.
    const auto load_nodes = [&](int t, bool v) __attribute__((always_inline)) {
      char* const stage = s_ring + (2 * (t & (kStages - 1)) + (v ? 1 : 0)) * R::kBytes;
      const char* const from = (v ? rare->nv : rare->nk) + (int64_t)b * rare->n_sb + (int64_t)kvh * rare->n_sh + node_c * 16;
      u32x4 reg[kNodeLoads];
#pragma unroll
      for (int i = 0; i < kNodeLoads; ++i)
        reg[i] = *(const u32x4*)(from + (int64_t)min((t0 + t) * kTile + node_p + i * kNodeStep, rare->nodes - 1) * rare->n_st);
#pragma unroll
      for (int i = 0; i < kNodeLoads; ++i) asm volatile("" : "+v"(reg[i]));  // waited for in any case
#pragma unroll
      for (int i = 0; i < kNodeLoads; ++i) {
        const int p = node_p + i * kNodeStep, j = (t0 + t) * kTile + p;
        if (v) {
          bool keep = j < rare->nodes;
          if (keep && nonfinite8<E>(reg[i])) {  // a V that is not finite is kept apart
            atomicOr(&s_bad[j / 32], 1u << (j % 32));
            keep = false;
          }
          *(u32x4*)(stage + value_at<HD>(p, node_c)) = keep ? reg[i] : u32x4{0, 0, 0, 0};
        } else {
          *(u32x4*)(stage + key_at<HD>(p, node_c)) = reg[i];
        }
      }
    };
    const char* const kbase = a.kpages + head_at;
    const int64_t to_values = a.vpages - a.kpages;
    typedef __attribute__((address_space(3))) char lds_char;
    lds_char* const ring = (lds_char*)s_ring;
    const uint32_t ring_at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)ring);
    const auto entry_of = [&](int i) __attribute__((always_inline)) {  // a block's entry, i blocks after blk0
      return __builtin_amdgcn_readlane(i < 64 ? window : ahead, i & 63);
    };
    const auto page_of = [&](int i) __attribute__((always_inline)) { return (int64_t)entry_of(i) * a.page_bytes; };
    const auto load_cached = [&](int t) __attribute__((always_inline)) {  // tile t of the piece; in order
      const uint32_t to = ring_at + (uint32_t)(t & (kStages - 1)) * (2 * R::kBytes) + (uint32_t)(wave * kPos * HD * 2);
      const int base = (c0 + t - nodes_here) * kTile + wave * kPos;
      if (blk >= blk0 + 64 && blk0 + 64 <= last_blk) {
        blk0 += 64;
        window = ahead;
        ahead = entries(blk0 + 64);
      }
      if constexpr (COLD) {
        uint32_t codes = 0;
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
          // past the row's end: its last unit again, and in that its last position
          const int pos = min(base + u * kUnit, (len - 1) / kUnit * kUnit), last = len - 1 - pos;
          const int bi = (int)a.div_page.div((uint32_t)pos), off = pos - bi * (int)a.div_page.d;
          const int e = entry_of(bi - blk0);
          const uint32_t at = to + u * 2048;
          if (e >= 0) {
            const char* const k0 = kbase + ((int64_t)e * a.page_bytes + (int64_t)off * a.row_bytes);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              const int back = (g * R::kGroup + min(lp, last - g * R::kGroup) - lp) * a.row_bytes;
              const int i = 2 * u + g;
              load_lds(k0, (key_from ^ key_turn(i)) + (uint32_t)back, k0 + to_values,
                       (value_from ^ value_turn(i)) + (uint32_t)back, at + g * 1024, R::kBytes);
            }
          } else {
            asm volatile("" : "+s"(rare));
            const int64_t cp = -2 - (int64_t)e, p = cp * rare->page_size + off;
            const int64_t el = p * (a.row_bytes / 2) + kvh * HD;
            load_lds((const char*)rare->kcodes + el, code_from, (const char*)rare->vcodes + el, code_from, at, R::kBytes);
            load_lds4((const char*)rare->kscales + (cp * a.kv_heads + kvh) * HD, (uint32_t)(lane % (HD / 16) * 16),
                      at + 1024);
            // a position's scale is one byte of these four (p times the heads is a multiple of 8)
            load_lds1((const char*)rare->vscales + p * a.kv_heads, (uint32_t)((code_p * a.kv_heads + kvh) & ~3),
                      at + 1024 + R::kBytes);
            codes |= 1u << u;
          }
        }
        const int sh = (t & (kStages - 1)) * 4;
        colds = (colds & ~(15u << sh)) | codes << sh;
      } else if (whole && base + kPos <= len) {
        int at_blk = blk, at_place = place;
#pragma unroll
        for (int c = 0; c < kPos / kWhole; ++c) {
          const char* const k0 = kbase + (page_of(at_blk - blk0) + (int64_t)at_place * a.row_bytes);
#pragma unroll
          for (int j = 0; j < kWhole / R::kGroup; ++j) {
            const int i = c * (kWhole / R::kGroup) + j;
            const char* const k = k0 + (int64_t)j * R::kGroup * a.row_bytes;
            load_lds(k, key_from ^ key_turn(i), k + to_values, value_from ^ value_turn(i), to + i * 1024, R::kBytes);
          }
          at_place += kWhole;
          if (at_place == (int)a.div_page.d) {
            at_place = 0;
            ++at_blk;
          }
        }
      } else {
#pragma unroll 1
        for (int i = 0; i < kLoads; ++i) {
          // past the row's end: its last group again, and in that its last position (never seen by a query)
          const int pos = min(base + i * R::kGroup, (len - 1) / R::kGroup * R::kGroup);
          const int bi = (int)a.div_page.div((uint32_t)pos);
          const char* const k = kbase + (page_of(bi - blk0) + (int64_t)(pos - bi * (int)a.div_page.d) * a.row_bytes);
          const uint32_t back = (uint32_t)(max(lp - (len - 1 - pos), 0) * a.row_bytes);
          load_lds(k, (key_from ^ key_turn(i)) - back, k + to_values, (value_from ^ value_turn(i)) - back, to + i * 1024,
                   R::kBytes);
        }
      }
      blk += block_step;
      place += place_step;
      if (place >= (int)a.div_page.d) {
        place -= (int)a.div_page.d;
        ++blk;
      }
    };

    // The wave's codes of tile t, which have come, as elements in their places.
    const auto decode = [&](int t) __attribute__((always_inline)) {
      const uint32_t codes = colds >> (t & (kStages - 1)) * 4;
      char* const stage = s_ring + 2 * (t & (kStages - 1)) * R::kBytes;
#pragma unroll 1
      for (int u = 0; u < kUnits; ++u) {
        if (!(codes >> u & 1)) continue;
        const int p0 = wave * kPos + u * kUnit;  // of the tile
        char *const kp = stage + p0 * HD * 2, *const vp0 = kp + R::kBytes;
        const int ch = lane * 4 % HD;  // a lane's four channels of keys, of positions HD / 4 lanes apart
        uint32_t kc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) kc[i] = *(const uint32_t*)(kp + lane * 4 + i * 256);
        const uint32_t ks = *(const uint32_t*)(kp + 1024 + ch);
        const u32x4 vc = *(const u32x4*)(vp0 + lane * 16);
        const uint32_t vs = *(const uint32_t*)(vp0 + 1024 + lane * 4);
        const float s0 = scale_of(ks & 255u), s1 = scale_of(ks >> 8 & 255u);
        const float s2 = scale_of(ks >> 16 & 255u), s3 = scale_of(ks >> 24);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t w0 = (scaled2<E, false>(kc[i], s0) & 0xffffu) | (scaled2<E, false>(kc[i], s1) & 0xffff0000u);
          const uint32_t w1 = (scaled2<E, true>(kc[i], s2) & 0xffffu) | (scaled2<E, true>(kc[i], s3) & 0xffff0000u);
          *(u32x2*)(stage + key_at<HD>(p0 + (lane * 4 + i * 256) / HD, ch / 8) + (ch & 4) * 2) = u32x2{w0, w1};
        }
        // values past the row's end are zeros: whatever a page holds there takes no part
        const bool in = code_p < len - (c0 + t - nodes_here) * kTile - p0;
        const float sv = scale_of(vs >> ((code_p * a.kv_heads + kvh) & 3) * 8 & 255u);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const u32x4 w = {scaled2<E, false>(vc[2 * c], sv), scaled2<E, true>(vc[2 * c], sv),
                           scaled2<E, false>(vc[2 * c + 1], sv), scaled2<E, true>(vc[2 * c + 1], sv)};
          *(u32x4*)(stage + R::kBytes + value_at<HD>(p0 + code_p, lane % (HD / 16) * 2 + c)) = in ? w : u32x4{0, 0, 0, 0};
        }
      }
    };

    f32x16 o[kDT], s[kSub];
    u32x4 hi[kSub][2], lo[kSub][2];
#pragma unroll
    for (int d = 0; d < kDT; ++d) o[d] = f32x16{0};
    float m = -INFINITY, l = 0.0f;

    const auto turned = [](const lds_char* p, uint32_t bits) __attribute__((always_inline)) {
      return (lds_char*)(uintptr_t)((uint32_t)(uintptr_t)p ^ bits);
    };
    u32x4 key[2][kKeys];
    const auto read_keys = [&](const lds_char* from, int n, u32x4 (&to)[kKeys]) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kKeys; ++i) {
        const int u = (n * kKeys + i) / kKS, k = (n * kKeys + i) % kKS;
        const lds_char* const at = turned(from, (uint32_t)(k << 5)) + u * 32 * HD * 2;
        to[i] = *(const __attribute__((address_space(3))) u32x4*)at;
      }
    };
    constexpr int kKeyBatches = kSub * kKS / kKeys;

    // ---- V of tile t times its probabilities
    const auto weigh_values = [&](int t) __attribute__((always_inline)) {
      typedef __attribute__((address_space(3))) s16x4 lds4;
      const lds_char* const from = ring + (t & (kStages - 1)) * (2 * R::kBytes) + value_lane;
      constexpr int kVals = 2, kBatches = 2 * kSub * (kDT / kVals);  // batches of 16 positions by 64 dims
      u32x4 val[2][kVals];
      const auto read_values = [&](int n, u32x4 (&to)[kVals]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kVals; ++i) {
          const int d = n % (kDT / kVals) * kVals + i;
          lds_char* const x = turned(from, (uint32_t)(d << 6)) + n / (kDT / kVals) * 16 * HD * 2;
          const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)x);
          const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(x + 8 * HD * 2));
          const u32x2 w0 = __builtin_bit_cast(u32x2, v0), w1 = __builtin_bit_cast(u32x2, v1);
          to[i] = u32x4{w0[0], w0[1], w1[0], w1[1]};
        }
      };
      read_values(0, val[0]);
#pragma unroll
      for (int n = 0; n < kBatches; ++n) {
        if (n + 1 < kBatches) read_values(n + 1, val[(n + 1) & 1]);
        __builtin_amdgcn_sched_barrier(0);  // the next values are on their way while these are multiplied
        const int p = n / (kDT / kVals), d0 = n % (kDT / kVals) * kVals;
#pragma unroll
        for (int i = 0; i < kVals; ++i) o[d0 + i] = mfma<E>(val[n & 1][i], lo[p / 2][p & 1], o[d0 + i]);
#pragma unroll
        for (int i = 0; i < kVals; ++i) o[d0 + i] = mfma<E>(val[n & 1][i], hi[p / 2][p & 1], o[d0 + i]);
      }
      if (t < nodes_here) {
        asm volatile("" : "+s"(rare));  // nodes whose V is not finite, for the rows that see them alone
#pragma unroll 1
        for (int u = 0; u < kSub; ++u) {
          const int jb = (t0 + t) * kTile + (kg * kSub + u) * 32;
          uint32_t bad = jb < rare->nodes ? __builtin_amdgcn_readfirstlane(s_bad[jb / 32]) : 0u;
          while (bad) {
            const int j = __builtin_ctz(bad);
            bad &= bad - 1;
            float p = 0.0f;
#pragma unroll
            for (int w = 0; w < kSub; ++w)
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const uint32_t h = hi[w][i / 8][(i % 8) / 2], r = lo[w][i / 8][(i % 8) / 2];
                const float x = i & 1 ? high_of<E>(h) + high_of<E>(r) : low_of<E>(h) + low_of<E>(r);
                p = w == u && (j >> 3) * 4 + (j & 3) == i ? x : p;
              }
            const f32x2 both = halves(p);
            p = j & 4 ? both[1] : both[0];
            const char* vrow = rare->nv + (int64_t)b * rare->n_sb + (int64_t)kvh * rare->n_sh + (int64_t)(jb + j) * rare->n_st + half * 8;
#pragma unroll
            for (int d = 0; d < kDT; ++d)
#pragma unroll
              for (int w4 = 0; w4 < 4; ++w4) {
                u32x2 w = *(const u32x2*)(vrow + d * 64 + w4 * 16);
                asm volatile("" : "+v"(w));  // waited for here: never outstanding in the tiles' loop
                if (p > 0.0f) {
                  o[d][4 * w4] += p * low_of<E>(w[0]);
                  o[d][4 * w4 + 1] += p * high_of<E>(w[0]);
                  o[d][4 * w4 + 2] += p * low_of<E>(w[1]);
                  o[d][4 * w4 + 3] += p * high_of<E>(w[1]);
                }
              }
          }
        }
      }
    };

    // ---- the running maximum after tile t's scores (masked here); the sums follow it when it grows by 2^8
    const auto raise = [&](int t, f32x16 (&x)[kSub]) __attribute__((always_inline)) {
      const int valid = len - (c0 + t - nodes_here) * kTile;  // cached positions from the tile's first on
      float top = -INFINITY;
#pragma unroll
      for (int u = 0; u < kSub; ++u) {
        const int pb = (kg * kSub + u) * 32;
        if (t < nodes_here || valid < pb + 32) {
          uint32_t seen;
          if (t < nodes_here) {
            asm volatile("" : "+s"(rare));
            const int jb = (t0 + t) * kTile + pb;
            seen = jb < rare->nodes && row < rare->rows ? s_mask[node_row - node_lo][jb / 32] : 0u;
          } else {
            seen = valid <= pb ? 0u : (1u << (valid - pb)) - 1u;
          }
          seen >>= 4 * half;
#pragma unroll
          for (int i = 0; i < 16; ++i) x[u][i] = seen >> (8 * (i / 4) + i % 4) & 1 ? x[u][i] : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, x[u][i]);
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
    };

    // ---- scores of tile t
    const auto score = [&](int t) __attribute__((always_inline)) {
      const lds_char* const keys = ring + (t & (kStages - 1)) * (2 * R::kBytes) + key_lane;
      read_keys(keys, 0, key[0]);
#pragma unroll
      for (int u = 0; u < kSub; ++u) s[u] = f32x16{0};
#pragma unroll
      for (int n = 0; n < kKeyBatches; ++n) {
        if (n + 1 < kKeyBatches) read_keys(keys, n + 1, key[(n + 1) & 1]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < kKeys; ++i) {
          const int u = (n * kKeys + i) / kKS, k = (n * kKeys + i) % kKS;
          s[u] = mfma<E>(key[n & 1][i], q[k], s[u]);
        }
      }
    };

    // ---- probabilities of a tile against the running maximum, as pairs of 16-bit numbers
    const auto weights = [&]() __attribute__((always_inline)) {
      const float shift = m == -INFINITY ? 0.0f : -m;
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float p0 = exp2_(fmaf(s[u][i], a.scale_log2, shift)), p1 = exp2_(fmaf(s[u][i + 1], a.scale_log2, shift));
          l += p0;
          l += p1;
          const uint32_t w = pack2<E>(p0, p1);
          hi[u][i / 8][(i % 8) / 2] = w;
          lo[u][i / 8][(i % 8) / 2] = pack2<E>(p0 - low_of<E>(w), p1 - high_of<E>(w));
        }
    };

    // A stage that step t has read is loaded again, with tile t + kStages, in the step after.
    if (WK > 1 && !first) lds_only_barrier();  // the piece before is joined from the ring
    first = false;
    constexpr int kAhead = kStages - 1;
    const auto load_step = [&](int t) __attribute__((always_inline)) {
      if (t + kAhead >= nodes_here && t + kAhead < count) load_cached(t + kAhead);
    };
    for (int t = nodes_here; t < min(count, kAhead); ++t) load_cached(t);
    // tiles on their way when step t + 1 needs its own
    const auto tiles_after = [&](int t) __attribute__((always_inline)) {
      return max(min(count - 1, t + kAhead) - (t + 1), 0);
    };
    if (nodes_here > 0) {  // the tree's mask as bits
      if (tid < kWords) s_bad[tid] = 0;
      const int rows_here = (int)a.div_group.div((uint32_t)min(rb * kRows + kRows - 1, rare->rows - 1)) - node_lo + 1;
      const int words = (rare->nodes + 63) / 64;  // of 64 nodes
      constexpr int kMany = 4;                    // of them a wave has in flight
      for (int i0 = wave * kMany; i0 < rows_here * words; i0 += kNW * kMany) {
        uint8_t byte[kMany];
#pragma unroll
        for (int u = 0; u < kMany; ++u) {
          const int i = min(i0 + u, rows_here * words - 1), n = node_lo + i / words, j = i % words * 64 + lane;
          byte[u] = j <= n;
          if (rare->mask)
            byte[u] = rare->mask[(int64_t)b * rare->m_sb + (int64_t)n * rare->m_si + (int64_t)min(j, rare->nodes - 1) * rare->m_sj];
        }
#pragma unroll
        for (int u = 0; u < kMany; ++u) {
          const int i = min(i0 + u, rows_here * words - 1), j = i % words * 64 + lane;
          const uint64_t bits = __ballot(byte[u] != 0 && j < rare->nodes);
          if (lane == 0) *(uint64_t*)&s_mask[i / words][i % words * 2] = bits;
        }
      }
      lds_only_barrier();  // s_bad is cleared
    }
    for (int t = 0; t < nodes_here; ++t) {  // at most kStages of them
      load_nodes(t, false);
      load_nodes(t, true);
    }
    const auto step_end = [&](int t) __attribute__((always_inline)) {  // tile t + 1 is there for every wave
      wait_tiles<2 * kLoads, kAhead - 1, !COLD>(tiles_after(t));
      if constexpr (COLD) {
        if (t + 1 >= nodes_here && t + 1 < count) decode(t + 1);
        lds_only_barrier();
      }
    };
    step_end(-1);
    asm volatile("" : "+s"(rare));
    if (!wave_live) {  // no query rows: the loads alone
      for (int t = 0; t < count; ++t) {
        load_step(t);
        step_end(t);
      }
    } else {
      for (int t = 0; t < count; ++t) {
        load_step(t);
        score(t);
        raise(t, s);
        weights();
        weigh_values(t);
        step_end(t);
      }
    }
    asm volatile("" : "+s"(rare));
    const f32x2 ls = halves(l);
    l = ls[0] + ls[1];

    if constexpr (WK > 1) {  // join the groups of positions
      float* s_join = (float*)s_ring;
      if (kg > 0) {
        float* to = s_join + ((kg - 1) * WQ + qg) * kPer * 64;
#pragma unroll
        for (int d = 0; d < kDT; ++d)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *(f32x4*)(to + (d * 4 + g) * 256 + lane * 4) =
                f32x4{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
        to[kDT * 1024 + lane] = m;
        to[kDT * 1024 + 64 + lane] = l;
      }
      lds_only_barrier();
      if (kg == 0) {
        float top = m, scale[WK];
        scale[0] = m;
#pragma unroll
        for (int k = 1; k < WK; ++k) {
          scale[k] = s_join[((k - 1) * WQ + qg) * kPer * 64 + kDT * 1024 + lane];
          top = fmaxf(top, scale[k]);
        }
#pragma unroll
        for (int k = 0; k < WK; ++k) scale[k] = scale[k] == -INFINITY ? 0.0f : exp2_(scale[k] - top);
        m = top;
        l *= scale[0];
#pragma unroll
        for (int d = 0; d < kDT; ++d) o[d] *= scale[0];
#pragma unroll
        for (int k = 1; k < WK; ++k) {
          const float* from = s_join + ((k - 1) * WQ + qg) * kPer * 64;
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
    }
    if (kg > 0 || row >= rare->rows) continue;
    if (t0 == 0 && t1 == tiles) {
      const float by = l > 0.0f || l != l ? 1.0f / l : 0.0f;
      char* op = rare->out + (int64_t)b * rare->o_sb + (int64_t)head * rare->o_sh + (int64_t)node_row * rare->o_st +
                 half * 4 * (int)sizeof(OutT);
#pragma unroll
      for (int d = 0; d < kDT; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          store4<E, OutT>(op + (d * 32 + g * 8) * (int)sizeof(OutT),
                          f32x4{o[d][4 * g] * by, o[d][4 * g + 1] * by, o[d][4 * g + 2] * by, o[d][4 * g + 3] * by});
    } else {
      const int64_t rec = (int64_t)(2 * group + (t0 == 0)) * rare->rows + row;
      float* to = rare->part + rec * HD + half * 4;
#pragma unroll
      for (int d = 0; d < kDT; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *(f32x4*)(to + d * 32 + g * 8) = f32x4{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
      if (half == 0) *(f32x2*)(rare->part_ml + rec * 2) = f32x2{m, l};
    }
  }
}

// Joins the records of a pair: HD / 4 threads a query row, which share the search for the maximum.
template <int E, int HD, int TILE, typename OutT>
__global__ void __launch_bounds__(kThreads) tree_flat_join_kernel(const TreeArgs a) {
  constexpr int kLanes = HD / 4, kPer = kThreads / kLanes, kTile = TILE;
  constexpr int kMany = 8;  // records in flight
  const int pair = (int)blockIdx.x;
  const int b = pair / a.kv_heads, kvh = pair - b * a.kv_heads;
  int before, all;
  count_places<kTile>(a, b, (int)threadIdx.x & 63, &before, &all);
  const int range = range_of(a, all);
  const int tiles = pair_tiles<kTile>(a, row_length(a, b));
  const int start = before * a.kv_heads + kvh * (tiles + kPairCost) + kPairCost;
  const int g0 = start / range, g1 = (start + tiles - 1) / range;
  if (g0 == g1) return;
  const int of_row = (int)threadIdx.x % kLanes, d = of_row * 4;
  for (int row = (int)blockIdx.y * kPer + (int)threadIdx.x / kLanes; row < a.rows; row += (int)gridDim.y * kPer) {
    const auto record = [&](int g) { return (int64_t)(2 * g + (g == g0)) * a.rows + row; };
    float top = -INFINITY;
    for (int g = g0 + of_row; g <= g1; g += kLanes) top = fmaxf(top, a.part_ml[record(g) * 2]);
#pragma unroll
    for (int n = 1; n < kLanes; n *= 2) top = fmaxf(top, __shfl_xor(top, n, kLanes));
    f32x4 sum = {0, 0, 0, 0};
    float l = 0.0f;
    for (int g = g0; g <= g1; g += kMany) {
      f32x2 ml[kMany];
      f32x4 v[kMany];
#pragma unroll
      for (int u = 0; u < kMany; ++u) {
        const int64_t rec = record(min(g + u, g1));
        ml[u] = *(const f32x2*)(a.part_ml + rec * 2);
        v[u] = *(const f32x4*)(a.part + rec * HD + d);
      }
#pragma unroll
      for (int u = 0; u < kMany; ++u) {
        if (g + u > g1) break;
        const float by = ml[u][0] == -INFINITY ? 0.0f : exp2_(ml[u][0] - top);
        sum += by * v[u];
        l += by * ml[u][1];
      }
    }
    const float by = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    const int node = (int)a.div_group.div((uint32_t)row);
    store4<E, OutT>(a.out + (int64_t)b * a.o_sb + (int64_t)(kvh * a.group + row - node * a.group) * a.o_sh +
                        (int64_t)node * a.o_st + d * (int)sizeof(OutT),
                    sum * by);
  }
}

struct Plan {
  bool flat;
  int wq, threads, tile, row_blocks, groups;
  int64_t splits, range, pairs, rows;
};

// How a call is cut: query rows by the fewest blocks, then ranges of tiles so that the launch fills the GPU.
bool plan_of(const barq_kv_pool* p, bool cold, int64_t batch, int64_t q_heads, int64_t nodes, int64_t max_seq,
             int64_t mean_seq, Plan* out) {
  if (!p || p->elem_bytes != 2 || (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256)) return false;
  if (p->kv_heads < 1 || batch < 1 || batch > p->max_batch || q_heads < 1 || q_heads % p->kv_heads || nodes < 1 ||
      nodes > BARQ_TREE_MAX_NODES || max_seq < 0 || mean_seq < 0)
    return false;
  const int64_t cap = p->max_blocks * p->page_size;
  const int64_t longest = max_seq == 0 ? cap : std::min(max_seq, cap);
  const int64_t rows = q_heads / p->kv_heads * nodes;
  if (rows > (int64_t(1) << 17)) return false;
  const int64_t hd = p->head_dim, pairs = batch * p->kv_heads;
  // The flat list wants tiles by asynchronous loads (a load's group of positions in one page, their offsets in 32
  // bits, a tree in its stages at once) and enough work to pay for finding each workgroup's place in it.  Whole calls,
  // pairs cut evenly by the host -> flat list, 8 KV heads of 128, 4 query rows: 1 x 333 positions 13.2 -> 13.5 us,
  // 16 x 333 13.6 -> 19.0, 4 x 2,900 23.6 -> 20.1, 16 x 2,900 42.6 -> 40.2; 192 query rows: 1 x 700 15.1 -> 21.8,
  // 16 x 2,900 91.6 -> 76.7.  fp8 pages are decoded by the flat list's loads alone.
  const int64_t mean_tiles = (std::min(mean_seq ? mean_seq : longest, longest) + 63) / 64 + (nodes + 63) / 64;
  if (cold && hd == 256) return false;
  out->flat = (cold || pairs * mean_tiles > 512) && p->page_size % (cold ? 16 : 512 / hd) == 0 &&
              p->kv_heads * hd * 2 < (int64_t(1) << 27) && nodes <= (hd == 256 ? 128 : 256);
  if (out->flat) {
    // Groups of 32 query rows of a workgroup, and by how many positions of a tile it is cut besides: eight waves,
    // two a SIMD, since one alone issues a vector instruction only every eighth cycle.  (fp8 pages on eight groups
    // spill 27 registers.)
    const int wq = rows > 128 && hd != 256 && !cold ? 8 : rows > 64 ? 4 : rows > 32 ? 2 : 1;
    const int64_t blocks = (rows + 32 * wq - 1) / (32 * wq);
    // 64 positions a tile (32 of head size 256), twice as many with few query rows: a 32-position piece for every
    // wave.  fp8 pages of head size 64 take 128 always, since a load of codes covers 16 of them.
    const int64_t kt = cold && hd == 64 ? 128 : std::min<int64_t>(64, 8192 / hd) * (wq > 2 ? 1 : 2);
    out->wq = wq;
    out->tile = (int)kt;
    out->threads = hd == 256 ? (wq == 1 ? 128 : 256) : wq == 1 ? 256 : 512;
    out->row_blocks = (int)blocks;
    out->groups = (int)std::max<int64_t>(1, 256 / blocks);  // one workgroup a compute unit
    out->pairs = pairs;
    out->rows = rows;
    return pairs * ((longest + kt - 1) / kt + (nodes + kt - 1) / kt + kPairCost) < (int64_t(1) << 30);
  }
  if (cold) return false;
  const int wq = rows > 64 ? 4 : rows > 32 || p->head_dim == 256 ? 2 : 1;
  const int tile = wq == 1 ? 128 : 64;
  const int64_t blocks = (rows + 32 * wq - 1) / (32 * wq);
  const auto tiles_of = [&](int64_t n) { return (n + tile - 1) / tile + (nodes + tile - 1) / tile; };
  const int64_t most = tiles_of(longest), mean = tiles_of(mean_seq ? std::min(mean_seq, longest) : longest);
  const int64_t want = p->head_dim == 256 ? 256 : 512;  // workgroups that are resident at once
  // The mean tiles of a pair over all of the launch's ranges; two tiles a range at least, since a join costs what a
  // tile does, but one of the 128 positions of few query rows where a pair is cut anyhow.  Whole calls, two -> one (us):
  // 4 query rows of head size 128 over 333 / 700 / 1,500 positions 13.5 / 13.6 / 14.6 -> 11.3 / 12.3 / 13.2, over 100
  // (two tiles) 10.6 -> 11.5; 52 query rows over 1,500 14.6 -> 15.9.
  const int64_t least = wq == 1 && most > 2 ? 1 : 2;
  int64_t range = std::max<int64_t>(least, (mean * pairs * blocks + want - 1) / want);
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
  if (p.flat) return 2 * (int64_t)p.groups * p.rows * (hd + 2) * 4;
  return p.splits == 1 ? 0 : p.pairs * p.splits * p.rows * (hd + 2) * 4;
}

using Kernel = const void*;
template <int E, int HD, typename OutT>
Kernel by_shape(int wq) {
  if constexpr (HD != 256)
    if (wq == 1) return (Kernel)&tree_kernel<E, HD, 1, OutT>;
  return wq == 2 ? (Kernel)&tree_kernel<E, HD, 2, OutT> : (Kernel)&tree_kernel<E, HD, 4, OutT>;
}
template <int E, typename OutT>
Kernel by_head(int64_t hd, int wq) {
  return hd == 256 ? by_shape<E, 256, OutT>(wq) : hd == 128 ? by_shape<E, 128, OutT>(wq) : by_shape<E, 64, OutT>(wq);
}
template <int E, typename OutT>
Kernel join_of(int64_t hd) {
  return hd == 256   ? (Kernel)&tree_join_kernel<E, 256, OutT>
         : hd == 128 ? (Kernel)&tree_join_kernel<E, 128, OutT>
                     : (Kernel)&tree_join_kernel<E, 64, OutT>;
}

template <int E, int HD, bool COLD, typename OutT>
Kernel flat_by_shape(const Plan& p) {
  constexpr int kTile = COLD && HD == 64 ? 128 : 64;
  if constexpr (HD == 256) {
    return p.wq == 4   ? (Kernel)&tree_flat_kernel<E, 256, 4, 1, 32, false, OutT>
           : p.wq == 2 ? (Kernel)&tree_flat_kernel<E, 256, 2, 2, 64, false, OutT>
                       : (Kernel)&tree_flat_kernel<E, 256, 1, 2, 64, false, OutT>;
  } else {
    if constexpr (!COLD)
      if (p.wq == 8) return (Kernel)&tree_flat_kernel<E, HD, 8, 1, kTile, false, OutT>;
    return p.wq == 4 ? (Kernel)&tree_flat_kernel<E, HD, 4, 2, kTile, COLD, OutT>
           : p.wq == 2 ? (Kernel)&tree_flat_kernel<E, HD, 2, 4, 128, COLD, OutT>
                       : (Kernel)&tree_flat_kernel<E, HD, 1, 4, 128, COLD, OutT>;
  }
}
template <int E, typename OutT>
Kernel flat_by_head(int64_t hd, bool cold, const Plan& p) {
  if (hd == 256) return flat_by_shape<E, 256, false, OutT>(p);
  if (hd == 128) return cold ? flat_by_shape<E, 128, true, OutT>(p) : flat_by_shape<E, 128, false, OutT>(p);
  return cold ? flat_by_shape<E, 64, true, OutT>(p) : flat_by_shape<E, 64, false, OutT>(p);
}
template <int E, typename OutT>
Kernel flat_join_of(int64_t hd, const Plan& p) {
  if (hd == 256)
    return p.tile == 32 ? (Kernel)&tree_flat_join_kernel<E, 256, 32, OutT> : (Kernel)&tree_flat_join_kernel<E, 256, 64, OutT>;
  if (hd == 128)
    return p.tile == 64 ? (Kernel)&tree_flat_join_kernel<E, 128, 64, OutT> : (Kernel)&tree_flat_join_kernel<E, 128, 128, OutT>;
  return p.tile == 64 ? (Kernel)&tree_flat_join_kernel<E, 64, 64, OutT> : (Kernel)&tree_flat_join_kernel<E, 64, 128, OutT>;
}

int launch(Kernel kernel, dim3 grid, void** args, void* stream, int threads = kThreads) {
  if (hipLaunchKernel(kernel, grid, dim3((uint32_t)threads), args, 0, (hipStream_t)stream) == hipSuccess) return BARQ_KV_OK;
  (void)hipGetLastError();
  return BARQ_KV_ERR_LAUNCH;
}

}  // namespace

extern "C" {

int64_t barq_tree_attention_workspace_bytes(const barq_kv_pool* pool, int64_t cold, int64_t batch, int64_t q_heads, int64_t nodes,
                                            int64_t max_seq, int64_t mean_seq) {
  Plan p;
  return plan_of(pool, cold != 0, batch, q_heads, nodes, max_seq, mean_seq, &p) ? workspace_of(p, pool->head_dim) : -1;
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
      !plan_of(pool, cold != nullptr, batch, q_heads, nodes, max_seq, mean_seq, &plan))
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
               (((uintptr_t)cold->key_codes | (uintptr_t)cold->value_codes | (uintptr_t)cold->key_scales) & 15) ||
               ((uintptr_t)cold->value_scales & 3)))
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
  a.part_ml = a.part + (plan.flat ? 2 * plan.groups : plan.pairs * plan.splits) * plan.rows * hd;
  a.batch = (int32_t)batch;
  a.groups = plan.groups;
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
  if (plan.flat) {
    const Kernel flat = f16 ? (f32 ? flat_by_head<kF16, float>(hd, cold, plan) : flat_by_head<kF16, uint16_t>(hd, cold, plan))
                            : (f32 ? flat_by_head<kBF16, float>(hd, cold, plan) : flat_by_head<kBF16, uint16_t>(hd, cold, plan));
    const Kernel join = f16 ? (f32 ? flat_join_of<kF16, float>(hd, plan) : flat_join_of<kF16, uint16_t>(hd, plan))
                            : (f32 ? flat_join_of<kBF16, float>(hd, plan) : flat_join_of<kBF16, uint16_t>(hd, plan));
    void* args[] = {&a};
    const int64_t per = kThreads / (hd / 4);
    const int rc = launch(flat, dim3((uint32_t)((plan.groups + 7) / 8 * 8 * plan.row_blocks)), args, stream,
                          plan.threads);
    if (rc != BARQ_KV_OK) return rc;
    // Workgroups to fill the GPU once, each with the pair's place in the list found once.
    const int64_t most = std::max<int64_t>(1, 2048 / plan.pairs);
    return launch(join, dim3((uint32_t)plan.pairs, (uint32_t)std::min(most, (plan.rows + per - 1) / per)), args, stream);
  }
  const Kernel kernel = f16 ? (f32 ? by_head<kF16, float>(hd, plan.wq) : by_head<kF16, uint16_t>(hd, plan.wq))
                            : (f32 ? by_head<kBF16, float>(hd, plan.wq) : by_head<kBF16, uint16_t>(hd, plan.wq));
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
