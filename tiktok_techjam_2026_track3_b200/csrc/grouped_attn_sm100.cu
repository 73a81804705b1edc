// Grouped-head attention on the tensor cores: causal attention over packed
// prompts, and attention of a batch of single tokens over a prefix they share.
//
//   o_r = sum_u p_ru v_u,  p_ru = 2^(c q_r.k_u - m_r) / l_r,  c = scale log2(e),
// computed key tile by key tile with a running reference m_r and sum l_r (the
// recurrence of an online softmax; m moves only when a tile exceeds it by 2^8).
//
// The group packs into the tile.  A 128-row query tile holds P = 128 / group
// consecutive positions times the group's heads (row = position * group + head):
// one TMA box [P][group][64 columns] of q lands as exactly these rows, K and V of
// the one key / value head are read once for the whole group, and a prompt of 20
// tokens with 4 heads per group fills 80 of 128 rows instead of 4 tiles of 20.
// (group not dividing 128: the last 128 - P * group rows idle.)  For the shared
// prefix the "positions" are the batch's sequences, so its K and V tiles are read
// once for all of them.
//
// Work item = (key / value head, 2 P consecutive positions of one prompt) = query
// tiles A and B that share every K/V tile (head_dim above 128: one tile), or, for
// the prefix, (head, 2 P sequences, a range of the prefix's keys), whose partial
// result (o, log2 of the sum) a later kernel joins.  One persistent CTA per SM,
// items dealt longest first, all heads of an entry together, in snake order.  (A head's
// entries together, the dense kernel's order when K and V exceed the L2, measured 2 to
// 28% slower on ten batches of 65 to 540 MB of K and V, and 5 and 8% faster on two of
// 2 and 4 prompts of 65536 and 32768 tokens, 8 heads of 128.)
//
// Keys that no row of an item may see (later tokens, the next prompt's, rows past
// the tensor) can sit in its last K/V tile and hold anything: their scores are
// replaced by -inf before any arithmetic, and P.V reads V only up to the last
// visible key rounded up to 16 rows, the rounding's rows zeroed in shared memory
// (0 * NaN would not be 0).  Later tokens of the row's own prompt do meet P = 0 in
// the tiles on the diagonal: an output that comes out NaN although its softmax is
// finite and such a token holds an infinity or NaN is computed again from its row's own
// keys alone once the block's items are done (repair_items; rows that need no repair
// pay one multiply-add per output).
//
// Roles, tensor-memory layouts and schedules are those of the dense kernel
// (flash_attn_sm100.cu), whose measurements chose them:
//   warp 0       TMA: K_j / V_j tiles into rings, item after item
//   warps 1, 3   MMA issue (one lane): S_t = Q_t K_j^T into TMEM, O_t += P_t V_j with
//                P read from TMEM; head_dim 64: warp 1 tile A, warp 3 tile B;
//                above: warp 1 for both
//   warp 2       TMA: the items' Q tiles
//   warps 4..    softmax: head_dim 64, 8 warps per tile with 16 rows each, P in its
//                own TMEM columns; above, 4 warps per tile with 32 rows each, P
//                written over S
//
// Bound by (a call among others, 16384 + 2049 tokens, 32 heads over 4 of 128: 2.20 ms, 1.02
// PFLOP/s; 8 ragged prompts of up to 2048, 16 heads of 64: 91 us, 0.51 PFLOP/s; replayed
// as a graph 2.12 ms and 85 us): at head_dim 128 a step of two tiles takes ~3800 cycles, softmax 2050 plus its products and their hand-offs
// 1740 per tile, alternating, against 2048 of the tensor pipe; at 64 the exponential
// unit (62% busy) and the hand-offs.  Items of one or two key tiles (96 prompts of up
// to 256 tokens: 74 us, 3.3 TB/s) take ~5 us each, their chain of barriers.  The head_dim-64
// kernels spill 16 to 24 bytes of their 96 and 104 registers, the others none.
#include <atomic>

#include "attn_math.cuh"
#include "sm100_ptx.cuh"
#include "ttj_internal.h"

namespace ttj {
namespace {

constexpr int kTile = 128;                  // rows of a query tile, keys of a K/V tile
constexpr int kChunkBytes = 128 * 128;      // [128 rows][64 columns] of 16-bit, swizzled
constexpr uint32_t kTmemCols = 512;

struct GroupedParams {
  void* out;              // prompts: [T, Hq, hd]
  float* lse;             // prompts: [T, Hq] or null
  const int4* plan;       // prompts: PlanEntry records
  float* part_o;          // prefix: [splits][B][Hq][hd]
  float* part_lse;        // prefix: [splits][B][Hq], log2 of the sum of exponentials
  int num_items, num_entries, kv_heads, group, positions;  // positions = 128 / group
  int num_heads, hd;
  int kv_shift;           // log2 of kv_heads, or -1
  int box_store;          // head_dim 64: a softmax warp's rows are whole groups, its output a TMA box
  int wide_store;         // head_dim above: output rows are 32-byte aligned
  int batch, prefix, split_keys, row_items;  // prefix: row_items = ceil(B / (tiles * positions))
  float scale_log2;
  int* status;
  const void *q, *k, *v;  // prompts: for repair_items
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;
};

template <int HD>
struct GroupedSmem {
  static_assert(HD == 64 || HD == 128 || HD == 256, "padded head sizes");
  static constexpr int kNT = HD == 256 ? 1 : 2;
  static constexpr bool kSepP = HD == 64;
  static constexpr int kThreads = kSepP ? 640 : 384;
  static constexpr int kLaunchRegs = kSepP ? 96 : 168;
  static constexpr uint32_t kRegsCtl = kSepP ? 64 : 136;
  static constexpr uint32_t kRegsSoftmax = kSepP ? 104 : 184;
  static_assert(128 * kRegsCtl + (kThreads - 128) * kRegsSoftmax == kThreads * kLaunchRegs,
                "register split must use the launch budget");
  static constexpr int kEpiRows = kSepP ? 16 : 0;    // rows of a softmax warp's staging box
  // K / V ring stages: what fits.  With one K stage more than V stages, K_m may be
  // loaded once V_{m-1} could be, as both wait for step m - 3 or earlier: K needs no
  // release barrier of its own (a commit less for the MMA warp, ~100 cycles a step).
  static constexpr int kStagesK = HD == 64 ? 4 : (HD == 128 ? 3 : 1);
  static constexpr int kStagesV = HD == 64 ? 3 : (HD == 128 ? 2 : 1);
  static constexpr bool kReleaseK = kStagesK != kStagesV + 1;
  static constexpr int kTileBytes = HD * 2 * 128;
  static constexpr int kQBufs = HD == 64 ? 2 : 1;
  static constexpr int kQOff = 0;                    // [kQBufs][Q_A, Q_B]
  static constexpr int kKOff = kNT * kQBufs * kTileBytes;
  static constexpr int kVOff = kKOff + kStagesK * kTileBytes;
  static constexpr int kEpiOff = kVOff + kStagesV * kTileBytes;
  static constexpr int kBarOff = kEpiOff + (kThreads / 32 - 4) * kEpiRows * 128;
  static constexpr int kTotal = 1024 + kBarOff + 512;
  static_assert(kTotal <= 232448, "shared memory budget");
  static constexpr uint32_t kColP = kSepP ? 256 : 0;    // + t*64 (separate) / + t*128 (over S)
  static constexpr uint32_t kPStride = kSepP ? 64 : 128;
  static constexpr uint32_t kColO = kSepP ? 384 : 256;  // + t*HD
};

// One work item: positions q0 .. q0 + nq - 1, keys k0 .. k0 + nk - 1; position
// q0 + i sees keys up to k0 + rel + i (prompts) or all nk of them (prefix).
struct Seg {
  int q0, nq, k0, nk, rel, kvh, part;
};

template <bool PREFIX, int NT>
__device__ __forceinline__ Seg seg_of(int item, const GroupedParams& p) {
  Seg s;
  if constexpr (PREFIX) {
    const int per_head = p.num_entries;  // row items x splits
    s.kvh = item / per_head;
    const int r = item - s.kvh * per_head;
    s.part = r / p.row_items;
    s.q0 = (r - s.part * p.row_items) * NT * p.positions;
    s.nq = min(NT * p.positions, p.batch - s.q0);
    s.k0 = s.part * p.split_keys;
    s.nk = min(p.split_keys, p.prefix - s.k0);
    s.rel = 0;
  } else {
    const int e = p.kv_shift >= 0 ? item >> p.kv_shift : item / p.kv_heads;
    s.kvh = item - e * p.kv_heads;
    const int4 w = __ldg(p.plan + e);
    s.q0 = w.x;
    s.nq = w.y;
    s.k0 = w.z;
    s.rel = w.x - w.z;
    s.nk = s.rel + w.y;
    s.part = 0;
  }
  return s;
}

// Keys that tile t's last position sees (0: the tile has no position).
template <bool PREFIX>
__device__ __forceinline__ int tile_keys(const Seg& s, int t, int positions) {
  const int np = min(positions, s.nq - t * positions);
  if (np <= 0) return 0;
  return PREFIX ? s.nk : s.rel + t * positions + np;
}
__device__ __forceinline__ int key_tiles(int keys) { return (keys + kTile - 1) / kTile; }

// Key tiles the item loads: a second tile that has positions sees at least as
// many as the first.
template <bool PREFIX, int NT>
__device__ __forceinline__ int item_tiles(const Seg& s, int positions) {
  const int a = key_tiles(tile_keys<PREFIX>(s, 0, positions));
  return NT == 2 ? max(a, key_tiles(tile_keys<PREFIX>(s, 1, positions))) : a;
}

// Row r of a tile is position r / group, head r % group; the positions of the rows a
// thread deals with are formed once (row_pos), not per item.
__device__ __forceinline__ int row_pos(int r, const GroupedParams& p) { return r / p.group; }

// Where row r = (pos, head r - pos * group) of tile t goes: its row in [tokens][Hq]
// (or [sequences][Hq]), or -1 for a row that is no position's.
__device__ __forceinline__ int64_t row_index(int r, int pos, int t, const Seg& s, const GroupedParams& p) {
  const int at = t * p.positions + pos;
  if (pos >= p.positions || at >= s.nq) return -1;
  return (int64_t)(s.q0 + at) * p.num_heads + s.kvh * p.group + (r - pos * p.group);
}

// Last key (relative to the item's first) that position pos of tile t sees.
template <bool PREFIX>
__device__ __forceinline__ int row_limit(int pos, int t, const Seg& s, const GroupedParams& p) {
  return PREFIX ? s.nk - 1 : s.rel + t * p.positions + pos;
}

__device__ __forceinline__ void st_global_v8(void* to, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}

// Store a staged box of ROWS rows x 64 columns (16-bit, 128-byte rows, swizzled): as
// one TMA box where all its rows are positions of this prompt, else row by row, 16
// bytes per lane, `at` being the output row of the box's row lane % ROWS.  (The row
// by row form kept a warp ~1500 cycles per box, with its 8 dependent stores.)
template <typename T, int ROWS>
__device__ __forceinline__ void store_box(uint32_t box, int64_t at, int r0, int t, int col0, const Seg& s,
                                          const CUtensorMap* tm_out, const GroupedParams& p) {
  const int lane = threadIdx.x & 31;
  if (p.box_store && __all_sync(0xffffffffu, at >= 0)) {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      tma_store_4d(tm_out, box, col0, 0, s.kvh, s.q0 + t * p.positions + row_pos(r0, p));
      bulk_commit_group();
    }
    return;
  }
  __syncwarp();
  const int col = col0 + 8 * (lane & 7);
#pragma unroll
  for (int i = 0; i < ROWS; i += 4) {
    const int row = i + (lane >> 3);
    const int64_t to = __shfl_sync(0xffffffffu, at, row);
    uint4 w;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                 : "r"(box + row * 128 + (((lane & 7) ^ (row & 7)) << 4)) : "memory");
    if (to >= 0 && col < p.hd) *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + to * p.hd + col) = w;
  }
}
// Before a box is written again: its last store has read it.
__device__ __forceinline__ void box_free() {
  if ((threadIdx.x & 31) == 0) bulk_wait_group_read<0>();
  __syncwarp();
}

// Outputs again that came out NaN or infinite only because of keys that their row does
// not see: the tiles on the diagonal multiply those by P = 0.  Called by all softmax
// warps of a block once its items k_lo .. k_hi are done (some of them have such a row),
// so that no other role waits however long the prompts are; shared memory is free then.
//
// Column c of an output depends on column c of V alone.  Per tile and column: the first
// key whose value is NaN, +inf, -inf (among those its products read), and the last such
// key that some row does not see.  A row is right where it sees that last key, or is NaN
// by keys that it sees (a NaN, infinities of both signs) or by its own sum (which a
// column of finite values tells); infinite by those keys alone it is that infinity, if
// their scores are finite for certain (`vast`); else the block forms it again, the keys
// dealt out over the warps.
// (One NaN at the end of 32768 tokens, 8 heads over 2 of 128: 46 ms; one warp per row, a
// key after the other inside the softmax loop, took 540.)
template <int HD>
struct Repair {
  using L = GroupedSmem<HD>;
  static constexpr int kThreads = L::kThreads - 128;  // every warp but the first four
  static constexpr int kWarps = kThreads / 32;
  static constexpr int kLanes = HD / 8;               // lanes per key, 8 dimensions each
  static constexpr int kKeys = 32 / kLanes;           // keys of a warp's step
  static constexpr int kParts = kWarps * kKeys;
  static constexpr int kRows = HD == 64 ? 2 : 4;      // rows formed together (registers)
  static constexpr int kNone = 0x7fffffff;
  int first[3][HD], last[HD];                         // of NaN, +inf, -inf; of any
  int rows[kTile], count;                             // to be formed again
  int vast;                                           // a key of such a value may score -inf: it weighs 0
  float m[kParts][kRows], l[kParts][kRows], o[kParts][kRows][HD];
};

__device__ __forceinline__ void repair_sync(int threads) { asm volatile("barrier.cta.sync 1, %0;" ::"r"(threads) : "memory"); }
__device__ __forceinline__ bool repair_any(bool mine, int threads) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}\n"
      : "=r"(any) : "r"((uint32_t)mine), "r"(threads) : "memory");
  return any != 0u;
}

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& w, float (&x)[8]) {
  const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = Pack<T>::unpack(ws[j]);
    x[2 * j] = f.x;
    x[2 * j + 1] = f.y;
  }
}

template <typename T, int HD>
__device__ __noinline__ void repair_items(const GroupedParams& p, Repair<HD>& x, int k_lo, int k_hi) {
  using R = Repair<HD>;
  constexpr int NT = GroupedSmem<HD>::kNT;
  const int tid = threadIdx.x - 128, warp = tid >> 5, lane = tid & 31;
  const int piece = lane % R::kLanes;                 // this lane's dimensions, 8 piece ..
  const bool live = piece * 8 < p.hd;
  T* const out = static_cast<T*>(p.out);
  auto put = [&](int64_t at, int col, float v) {
    const uint16_t w = (uint16_t)Pack<T>::two(v, 0.f);
    *reinterpret_cast<uint16_t*>(out + at * p.hd + col) = w;
  };
  for (int k = k_lo; k <= k_hi; ++k) {
    const Seg s = seg_of<false, NT>(item_of(k), p);
    const T* const key = static_cast<const T*>(p.k) + s.k0 * p.k_row + s.kvh * p.k_head;
    const T* const kp = key + piece * 8;
    const T* const vp = static_cast<const T*>(p.v) + s.k0 * p.v_row + s.kvh * p.v_head + piece * 8;
    for (int t = 0; t < NT; ++t) {
      const int keys = tile_keys<false>(s, t, p.positions);
      if (keys == 0) continue;
      const int seen = row_limit<false>(0, t, s, p) + 1;  // keys that every row sees
      const int end = min((keys + 15) & ~15, s.nk);       // P.V reads V up to here
      for (int i = tid; i < HD; i += R::kThreads) {
        x.first[0][i] = x.first[1][i] = x.first[2][i] = R::kNone;
        x.last[i] = -1;
      }
      if (tid == 0) x.count = x.vast = 0;
      repair_sync(R::kThreads);
      auto scan = [&](int from, int to, bool unseen) -> bool {
        constexpr int kStep = R::kThreads / R::kLanes, kAhead = 4;
        bool found = false;
        for (int u0 = from + tid / R::kLanes; u0 < to; u0 += kAhead * kStep) {
          uint4 w[kAhead];
#pragma unroll
          for (int i = 0; i < kAhead; ++i) {
            const int64_t u = u0 + i * kStep;
            w[i] = live && u < to ? __ldg(reinterpret_cast<const uint4*>(vp + u * p.v_row)) : make_uint4(0u, 0u, 0u, 0u);
          }
#pragma unroll
          for (int i = 0; i < kAhead; ++i) {
            float e[8], z = 0.f;
            unpack8<T>(w[i], e);
#pragma unroll
            for (int j = 0; j < 8; ++j) z = fmaf(e[j], 0.f, z);
            if (z == 0.f) continue;                       // all finite
            found = true;
            const int u = u0 + i * kStep;
            for (int c = 0; c < p.hd && !*static_cast<volatile int*>(&x.vast); c += 8) {
              float y[8];
              unpack8<T>(__ldg(reinterpret_cast<const uint4*>(key + u * p.k_row + c)), y);
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (!(fabsf(y[j]) < 1e30f)) x.vast = 1;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              if (e[j] - e[j] == 0.f) continue;
              int* const f = &x.first[e[j] != e[j] ? 0 : (e[j] > 0.f ? 1 : 2)][piece * 8 + j];
              if (u < *static_cast<volatile int*>(f)) atomicMin(f, u);
              if (unseen) atomicMax(&x.last[piece * 8 + j], u);
            }
          }
        }
        return found;
      };
      if (!repair_any(scan(seen, end, true), R::kThreads)) continue;
      scan(0, seen, false);
      repair_sync(R::kThreads);
      for (int r = warp; r < kTile; r += R::kWarps) {     // which rows
        const int pos = row_pos(r, p), limit = row_limit<false>(pos, t, s, p);
        const int64_t at = row_index(r, pos, t, s, p);
        if (at < 0) continue;
        bool form = false, infinite = false;
        int finite = -1;                                  // a column of finite values
        for (int c = lane; c < p.hd; c += 32) {
          const int f0 = x.first[0][c], f1 = x.first[1][c], f2 = x.first[2][c];
          if (min(f0, min(f1, f2)) == R::kNone) finite = c;
          if (x.last[c] <= limit || f0 <= limit || (f1 <= limit && f2 <= limit)) continue;
          (f1 <= limit || f2 <= limit ? infinite : form) = true;
        }
        form = __any_sync(0xffffffffu, form);
        infinite = __any_sync(0xffffffffu, infinite);
        finite = __reduce_max_sync(0xffffffffu, finite);
        if (!form && !infinite) continue;
        if (!form && finite >= 0) {
          const uint16_t w = __ldcg(reinterpret_cast<const uint16_t*>(out + at * p.hd + finite));
          const float v = Pack<T>::unpack(w).x;
          if (v != v) continue;                           // NaN altogether
        }
        if (form || finite < 0 || x.vast) {
          if (lane == 0) x.rows[atomicAdd(&x.count, 1)] = r;
        } else {
          for (int c = lane; c < p.hd; c += 32) {
            const int f0 = x.first[0][c], f1 = x.first[1][c], f2 = x.first[2][c];
            if (x.last[c] <= limit || f0 <= limit || (f1 <= limit) == (f2 <= limit)) continue;
            put(at, c, f1 <= limit ? INFINITY : -INFINITY);
          }
        }
      }
      repair_sync(R::kThreads);
      const int count = x.count;
      for (int r0 = 0; r0 < count; r0 += R::kRows) {
        float q[R::kRows][8], o[R::kRows][8], m[R::kRows], l[R::kRows];
        int limit[R::kRows], most = 0;
#pragma unroll
        for (int i = 0; i < R::kRows; ++i) {
          const int r = x.rows[min(r0 + i, count - 1)], pos = row_pos(r, p);
          limit[i] = row_limit<false>(pos, t, s, p);
          most = max(most, limit[i]);
          const T* from = static_cast<const T*>(p.q) + (int64_t)(s.q0 + t * p.positions + pos) * p.q_row +
                          (s.kvh * p.group + r - pos * p.group) * p.q_head + piece * 8;
          unpack8<T>(live ? __ldg(reinterpret_cast<const uint4*>(from)) : make_uint4(0u, 0u, 0u, 0u), q[i]);
          m[i] = -INFINITY;
          l[i] = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) o[i][j] = 0.f;
        }
        uint4 kw, vw;
        auto load = [&](int64_t u) {
          const bool ok = live && u <= most;
          kw = ok ? __ldg(reinterpret_cast<const uint4*>(kp + u * p.k_row)) : make_uint4(0u, 0u, 0u, 0u);
          vw = ok ? __ldg(reinterpret_cast<const uint4*>(vp + u * p.v_row)) : make_uint4(0u, 0u, 0u, 0u);
        };
        const int mine = lane / R::kLanes;
        load(warp * R::kKeys + mine);
        for (int u0 = warp * R::kKeys; u0 <= most; u0 += R::kParts) {
          float ks[8], vs[8];
          unpack8<T>(kw, ks);
          unpack8<T>(vw, vs);
          load((int64_t)u0 + R::kParts + mine);
#pragma unroll
          for (int i = 0; i < R::kRows; ++i) {
            float c = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) c = fmaf(q[i][j], ks[j], c);
#pragma unroll
            for (int w = R::kLanes / 2; w > 0; w >>= 1) c += __shfl_xor_sync(0xffffffffu, c, w);
            if (u0 + mine > limit[i]) continue;
            c *= p.scale_log2;
            const float mn = fmaxf(m[i], c);
            const float keep = m[i] == -INFINITY ? 0.f : fast_exp2(m[i] - mn), e = c == -INFINITY ? 0.f : fast_exp2(c - mn);
            l[i] = fmaf(l[i], keep, e);
            m[i] = mn;
#pragma unroll
            for (int j = 0; j < 8; ++j) o[i][j] = fmaf(e, vs[j], o[i][j] * keep);
          }
        }
        const int part = warp * R::kKeys + mine;
#pragma unroll
        for (int i = 0; i < R::kRows; ++i) {
          if (piece == 0) x.m[part][i] = m[i], x.l[part][i] = l[i];
#pragma unroll
          for (int j = 0; j < 8; ++j) x.o[part][i][piece * 8 + j] = o[i][j];
        }
        repair_sync(R::kThreads);
        for (int n = tid; n < R::kRows * HD; n += R::kThreads) {
          const int i = n / HD, c = n % HD;
          if (r0 + i >= count || c >= p.hd) continue;
          const int r = x.rows[r0 + i], pos = row_pos(r, p), lim = row_limit<false>(pos, t, s, p);
          const int f0 = x.first[0][c], f1 = x.first[1][c], f2 = x.first[2][c];
          if (x.last[c] <= lim || f0 <= lim || (f1 <= lim && f2 <= lim)) continue;
          float top = -INFINITY, sum = 0.f, v = 0.f;
          for (int w = 0; w < R::kParts; ++w) top = fmaxf(top, x.m[w][i]);
          for (int w = 0; w < R::kParts; ++w) {
            const float f = x.m[w][i] == -INFINITY ? 0.f : fast_exp2(x.m[w][i] - top);
            sum = x.l[w][i] == 0.f ? sum : fmaf(x.l[w][i], f, sum);
            v = fmaf(x.o[w][i][c], f, v);
          }
          v /= sum;
          if (!x.vast && (f1 <= lim || f2 <= lim)) v = sum - sum != 0.f || sum == 0.f ? NAN : (f1 <= lim ? INFINITY : -INFINITY);
          put(row_index(r, pos, t, s, p), c, v);
        }
        repair_sync(R::kThreads);
      }
      repair_sync(R::kThreads);
    }
  }
}

// Item k of this block has an output that repair_items must look at (the first and the
// last of them follow the abort flag).
__device__ __forceinline__ void note_repair(volatile int* abort_flag, int k) {
  if ((threadIdx.x & 31) == 0) {
    int* const redo = const_cast<int*>(abort_flag) + 1;
    atomicMin(&redo[0], k);
    atomicMax(&redo[1], k);
  }
}

// Softmax, two warps per tile and TMEM lane quarter (head_dim 64): warp w serves
// tile (w - 4) / 8 and 16 rows; lane 4g + k holds rows g and g + 8 of them and of
// each 8-key group n keys 8n + 2k and 8n + 2k + 1 (the 16-lane TMEM shapes).
template <typename T, int HD, bool PREFIX>
__device__ __forceinline__ void softmax_pairs(const GroupedParams& p, uint8_t* epi_base, uint32_t tmem,
                                              const CUtensorMap* tm_out,
                                              uint64_t* s_full, uint64_t* s_free, uint64_t* p_full,
                                              uint64_t* o_done, volatile int* abort_flag) {
  using L = GroupedSmem<HD>;
  static_assert(HD == 64 && L::kSepP, "separate P, one 64-column output");
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int t = (warp - 4) >> 3;
  const int g = lane >> 2, kq = lane & 3;
  const int r0 = (warp & 3) * 32 + (((warp - 4) >> 2) & 1) * 16;  // this warp's first row of the tile
  const uint32_t t_lane = tmem + (static_cast<uint32_t>(r0) << 16);
  const uint32_t t_s = t_lane + t * 128;
  const uint32_t t_p = t_lane + L::kColP + t * 64;
  const uint32_t t_o = t_lane + L::kColO + t * HD;
  const uint32_t box = smem_u32(epi_base) + (warp - 4) * (L::kEpiRows * 128);
  // positions of this lane's rows g, g + 8 and of the box's row lane % 16, a byte each
  const uint32_t pos3 = (uint32_t)row_pos(r0 + g, p) | (uint32_t)row_pos(r0 + g + 8, p) << 8 |
                        (uint32_t)row_pos(r0 + (lane & 15), p) << 16;
  uint32_t sf_phase = 0, od_phase = 0;
  auto row_max4 = [](float v) {  // over the four threads of a row
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
  };
  auto row_sum4 = [](float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    return v + __shfl_xor_sync(0xffffffffu, v, 2);
  };
  bool ok = true;
  for (int k = 0; ok; ++k) {
    const int item = item_of(k);
    if (item >= p.num_items) break;
    int n_kv, lim_a, lim_b, lim_first;
    {
      const Seg s = seg_of<PREFIX, L::kNT>(item, p);
      n_kv = key_tiles(tile_keys<PREFIX>(s, t, p.positions));
      lim_a = row_limit<PREFIX>(pos3 & 255, t, s, p) - 2 * kq;
      lim_b = row_limit<PREFIX>((pos3 >> 8) & 255, t, s, p) - 2 * kq;
      lim_first = row_limit<PREFIX>(0, t, s, p);
    }
    if (n_kv == 0) continue;
    float m_a = -INFINITY, m_b = -INFINITY;  // exponent references (log2 units), moved lazily
    float l_a = 0.f, l_b = 0.f;              // this thread's part of each row's sum
    for (int j = 0; j < n_kv; ++j) {
      if (!mbar_wait_warp(&s_full[t], sf_phase, p.status, kDevTimeoutSoftmax, abort_flag)) { ok = false; break; }
      sf_phase ^= 1u;
      tc_fence_after();
      float s[64];  // s[4n + e]: row (e < 2 ? a : b), key 8n + 2k + (e & 1)
      {
        uint32_t u[64];
        tmem_ld_16x256b_x16(t_s, u);
#pragma unroll
        for (int i = 0; i < 64; ++i) s[i] = __uint_as_float(u[i]);
      }
      tc_fence_before();
      mbar_arrive(&s_free[t]);  // the tensor core may overwrite S_t now
      const int k0 = j * kTile;
      if (k0 + kTile - 1 > lim_first) {
        // key k0 + 8n + 2k + (e & 1) is visible iff 8n + (e & 1) <= limit - k0 - 2k
        const int da = lim_a - k0, db = lim_b - k0;
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          s[4 * n + 0] = 8 * n <= da ? s[4 * n + 0] : -INFINITY;
          s[4 * n + 1] = 8 * n + 1 <= da ? s[4 * n + 1] : -INFINITY;
          s[4 * n + 2] = 8 * n <= db ? s[4 * n + 2] : -INFINITY;
          s[4 * n + 3] = 8 * n + 1 <= db ? s[4 * n + 3] : -INFINITY;
        }
      }
      float ma[4], mb[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        ma[c] = fmaxf(s[16 * c + 0], s[16 * c + 1]);
        mb[c] = fmaxf(s[16 * c + 2], s[16 * c + 3]);
#pragma unroll
        for (int n = 4 * c + 1; n < 4 * c + 4; ++n) {
          ma[c] = fmax3(ma[c], s[4 * n], s[4 * n + 1]);
          mb[c] = fmax3(mb[c], s[4 * n + 2], s[4 * n + 3]);
        }
      }
      const float mxa = row_max4(fmaxf(fmaxf(ma[0], ma[1]), fmaxf(ma[2], ma[3])));
      const float mxb = row_max4(fmaxf(fmaxf(mb[0], mb[1]), fmaxf(mb[2], mb[3])));
      const float mta = mxa * p.scale_log2, mtb = mxb * p.scale_log2;
      const float mna = (mta > m_a + 8.f) ? mta : m_a;
      const float mnb = (mtb > m_b + 8.f) ? mtb : m_b;
      const float mua = mna == -INFINITY ? 0.f : mna;
      const float mub = mnb == -INFINITY ? 0.f : mnb;
      const float alpha_a = fast_exp2(m_a - mua);
      const float alpha_b = fast_exp2(m_b - mub);
      const uint64_t c2 = f2_pack(p.scale_log2, p.scale_log2);
      const uint64_t nma = f2_pack(-mua, -mua), nmb = f2_pack(-mub, -mub);
      uint32_t pk[32];  // P words: pk[2n] row a, pk[2n + 1] row b, word column 4n + k
      uint64_t sa2[2] = {0ull, 0ull}, sb2[2] = {0ull, 0ull};
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        float x0, x1;
        f2_unpack(ffma2(f2_pack(s[4 * n], s[4 * n + 1]), c2, nma), x0, x1);
        const float e0 = fast_exp2(x0), e1 = fast_exp2(x1);
        pk[2 * n] = Pack<T>::two(e0, e1);
        sa2[n & 1] = fadd2(sa2[n & 1], f2_pack(e0, e1));
        f2_unpack(ffma2(f2_pack(s[4 * n + 2], s[4 * n + 3]), c2, nmb), x0, x1);
        const float e2 = fast_exp2(x0), e3 = fast_exp2(x1);
        pk[2 * n + 1] = Pack<T>::two(e2, e3);
        sb2[n & 1] = fadd2(sb2[n & 1], f2_pack(e2, e3));
      }
      float a0, a1, b0, b1;
      f2_unpack(fadd2(sa2[0], sa2[1]), a0, a1);
      f2_unpack(fadd2(sb2[0], sb2[1]), b0, b1);
      l_a = l_a * alpha_a + (a0 + a1);
      l_b = l_b * alpha_b + (b0 + b1);
      m_a = mna;
      m_b = mnb;
      if (j > 0) {
        // P_t(j-1) V must have completed: it reads the P buffer written here and
        // is the last write to O_t before a rescale.
        if (!mbar_wait_warp(&o_done[t], od_phase, p.status, kDevTimeoutSoftmax, abort_flag)) { ok = false; break; }
        od_phase ^= 1u;
        tc_fence_after();
      }
      tmem_st_16x128b_x16(t_p, pk);
      if (j > 0 && __any_sync(0xffffffffu, alpha_a != 1.f || alpha_b != 1.f)) {
        uint32_t o[32];
        tmem_ld_16x256b_x8(t_o, o);
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          o[4 * n + 0] = __float_as_uint(__uint_as_float(o[4 * n + 0]) * alpha_a);
          o[4 * n + 1] = __float_as_uint(__uint_as_float(o[4 * n + 1]) * alpha_a);
          o[4 * n + 2] = __float_as_uint(__uint_as_float(o[4 * n + 2]) * alpha_b);
          o[4 * n + 3] = __float_as_uint(__uint_as_float(o[4 * n + 3]) * alpha_b);
        }
        tmem_st_16x256b_x8(t_o, o);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_full[t]);
    }
    if (!ok) break;
    l_a = row_sum4(l_a);
    l_b = row_sum4(l_b);
    // (of the prefix's keys all may score -inf and others count: that part is zeros)
    const float inv_a = PREFIX && l_a == 0.f ? 0.f : 1.f / l_a, inv_b = PREFIX && l_b == 0.f ? 0.f : 1.f / l_b;
    const Seg s = seg_of<PREFIX, L::kNT>(item, p);
    float* lse = PREFIX ? p.part_lse + (int64_t)s.part * p.batch * p.num_heads : p.lse;
    if (lse != nullptr && kq < 2) {  // one thread per row
      const int64_t at = row_index(r0 + g + 8 * kq, (pos3 >> (8 * kq)) & 255, t, s, p);
      const float v = kq == 0 ? m_a + log2f(l_a) : m_b + log2f(l_b);
      if (at >= 0) lse[at] = PREFIX ? v : v * 0.69314718055994531f;
    }
    if (!mbar_wait_warp(&o_done[t], od_phase, p.status, kDevTimeoutSoftmax, abort_flag)) break;
    od_phase ^= 1u;
    tc_fence_after();
    uint32_t o[32];  // o[4n + e]: row (e < 2 ? a : b), column 8n + 2k + (e & 1)
    tmem_ld_16x256b_x8(t_o, o);
    if constexpr (PREFIX) {
      const int64_t ra = row_index(r0 + g, pos3 & 255, t, s, p), rb = row_index(r0 + g + 8, (pos3 >> 8) & 255, t, s, p);
      float* part = p.part_o + (int64_t)s.part * p.batch * p.num_heads * p.hd;
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const int col = 8 * n + 2 * kq;
        if (col >= p.hd) break;
        if (ra >= 0) *reinterpret_cast<float2*>(part + ra * p.hd + col) =
            make_float2(__uint_as_float(o[4 * n]) * inv_a, __uint_as_float(o[4 * n + 1]) * inv_a);
        if (rb >= 0) *reinterpret_cast<float2*>(part + rb * p.hd + col) =
            make_float2(__uint_as_float(o[4 * n + 2]) * inv_b, __uint_as_float(o[4 * n + 3]) * inv_b);
      }
    } else {
      box_free();
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        // 128-byte rows, 16-byte chunk n holds columns 8n..8n+7, swizzled by row & 7
        const uint32_t wa = Pack<T>::two(__uint_as_float(o[4 * n]) * inv_a, __uint_as_float(o[4 * n + 1]) * inv_a);
        const uint32_t wb = Pack<T>::two(__uint_as_float(o[4 * n + 2]) * inv_b, __uint_as_float(o[4 * n + 3]) * inv_b);
        st_shared_u32(box + g * 128 + ((n ^ (g & 7)) << 4) + 4 * kq, wa);
        st_shared_u32(box + (g + 8) * 128 + ((n ^ (g & 7)) << 4) + 4 * kq, wb);
      }
      store_box<T, 16>(box, row_index(r0 + (lane & 15), pos3 >> 16, t, s, p), r0, t, 0, s, tm_out, p);
      uint64_t za = 0ull, zb = 0ull;  // NaN where a row's output is (or infinite)
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        za = ffma2(f2_pack(__uint_as_float(o[4 * n]), __uint_as_float(o[4 * n + 1])), 0ull, za);
        zb = ffma2(f2_pack(__uint_as_float(o[4 * n + 2]), __uint_as_float(o[4 * n + 3])), 0ull, zb);
      }
      float a0, a1, b0, b1;
      f2_unpack(za, a0, a1);
      f2_unpack(zb, b0, b1);
      uint32_t bad_a = __ballot_sync(0xffffffffu, a0 + a1 != 0.f && l_a - l_a == 0.f);
      uint32_t bad_b = __ballot_sync(0xffffffffu, b0 + b1 != 0.f && l_b - l_b == 0.f);
      if ((bad_a | bad_b) != 0u) note_repair(abort_flag, k);
    }
    // The next item's first P.V overwrites O_t only after this thread's next
    // p_full arrival, which follows these TMEM loads.
  }
  if (lane == 0) bulk_wait_group_all();  // output boxes complete before exit
}

// Softmax, one warp per tile and TMEM lane quarter, thread = row, P over S
// (head_dim 128 and 256).
template <typename T, int HD, bool PREFIX>
__device__ __forceinline__ void softmax_rows(const GroupedParams& p, uint32_t tmem, uint64_t* s_full, uint64_t* p_full, uint64_t* o_done,
                                             volatile int* abort_flag) {
  using L = GroupedSmem<HD>;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int t = warp >= 8 ? 1 : 0;
  if (t >= L::kNT) return;  // one tile per item: warps 8..11 have no work
  const int r0 = (warp & 3) * 32;
  const int r = r0 + lane;  // row within the tile
  const uint32_t t_lane = tmem + (static_cast<uint32_t>(r0) << 16);
  const uint32_t t_s = t_lane + t * 128;
  const uint32_t t_p = t_lane + L::kColP + t * L::kPStride;
  const uint32_t t_o = t_lane + L::kColO + t * HD;
  const int pos = row_pos(r, p);
  uint32_t sf_phase = 0, od_phase = 0;
  bool ok = true;
  Seg next = seg_of<PREFIX, L::kNT>(item_of(0), p);  // (every block has an item)
  for (int k = 0; ok; ++k) {
    if (item_of(k) >= p.num_items) break;
    const Seg sg = next;
    if (item_of(k + 1) < p.num_items) next = seg_of<PREFIX, L::kNT>(item_of(k + 1), p);
    const int keys = tile_keys<PREFIX>(sg, t, p.positions), n_kv = key_tiles(keys);
    if (n_kv == 0) continue;
    const int limit = row_limit<PREFIX>(pos, t, sg, p), lim_first = row_limit<PREFIX>(0, t, sg, p);
    float m_run = -INFINITY;  // exponent reference (log2 units), moved lazily
    float l_run = 0.f;        // running sum of P in fp32
    for (int j = 0; j < n_kv; ++j) {
      if (!mbar_wait_warp(&s_full[t], sf_phase, p.status, kDevTimeoutSoftmax, abort_flag)) { ok = false; break; }
      sf_phase ^= 1u;
      tc_fence_after();
      float s[kTile];
      {
        uint32_t u[kTile];
        tmem_ld128(t_s, u);
#pragma unroll
        for (int i = 0; i < kTile; ++i) s[i] = __uint_as_float(u[i]);
      }
      const int k0 = j * kTile;
      if (k0 + kTile - 1 > lim_first) {
        const int lim = limit - k0;
#pragma unroll
        for (int i = 0; i < kTile; ++i) s[i] = i <= lim ? s[i] : -INFINITY;
      }
      // Keys past the tile's last visible one are computed neither by Q.K nor read by
      // P.V; the softmax skips them 32 at a time.
      const int chunks = (min(keys - k0, kTile) + 31) >> 5;
      // row max: eight independent chains of 3-input max per half
      auto half_max = [&](int i0) {
        float mx8[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) mx8[q] = fmaxf(s[i0 + q], s[i0 + 8 + q]);
#pragma unroll
        for (int i = 16; i < 64; i += 16)
#pragma unroll
          for (int q = 0; q < 8; ++q) mx8[q] = fmax3(mx8[q], s[i0 + i + q], s[i0 + i + 8 + q]);
        return fmax3(fmax3(mx8[0], mx8[1], mx8[2]), fmax3(mx8[3], mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7]));
      };
      float mx = half_max(0);
      if (chunks > 2) mx = fmaxf(mx, half_max(64));
      const float m_tile = mx * p.scale_log2;
      const float m_new = (m_tile > m_run + 8.f) ? m_tile : m_run;
      const float m_use = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = fast_exp2(m_run - m_use);  // 1 unchanged, 0 from -inf
      const uint64_t c2 = f2_pack(p.scale_log2, p.scale_log2);
      const uint64_t nm2 = f2_pack(-m_use, -m_use);
      uint32_t pk[2][32];
      uint64_t sum2[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
      for (int c = 0; c < kTile / 32; ++c) {
        if (c >= chunks) break;  // uniform
        uint32_t (&pc)[16] = *reinterpret_cast<uint32_t(*)[16]>(&pk[c >> 1][(c & 1) * 16]);
#pragma unroll
        for (int ii = 0; ii < 16; ++ii) {
          const int i = c * 16 + ii;
          float x0, x1;
          f2_unpack(ffma2(f2_pack(s[2 * i], s[2 * i + 1]), c2, nm2), x0, x1);
          const float e0 = fast_exp2(x0);
          const float e1 = fast_exp2(x1);
          pc[ii] = Pack<T>::two(e0, e1);
          sum2[i & 3] = fadd2(sum2[i & 3], f2_pack(e0, e1));
        }
        tmem_st16(t_p + c * 16, pc);  // over the S columns already read
      }
      float a0, a1;
      f2_unpack(fadd2(fadd2(sum2[0], sum2[1]), fadd2(sum2[2], sum2[3])), a0, a1);
      l_run = l_run * alpha + (a0 + a1);
      m_run = m_new;
      // S_t(j) being ready means P_t(j-1) V has completed: O_t may be rescaled
      if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(t_o + c * 32, o);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
          tmem_st32(t_o + c * 32, o);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_full[t]);
    }
    if (!ok) break;
    const int64_t at = row_index(r, pos, t, sg, p);
    float* lse = PREFIX ? p.part_lse + (int64_t)sg.part * p.batch * p.num_heads : p.lse;
    if (lse != nullptr && at >= 0) {
      const float v = m_run + log2f(l_run);
      lse[at] = PREFIX ? v : v * 0.69314718055994531f;
    }
    if (!mbar_wait_warp(&o_done[t], od_phase, p.status, kDevTimeoutSoftmax, abort_flag)) break;
    od_phase ^= 1u;
    tc_fence_after();
    const float inv_l = PREFIX && l_run == 0.f ? 0.f : 1.f / l_run;  // (as above: a part of zeros)
    if constexpr (PREFIX) {
      float* part = p.part_o + ((int64_t)sg.part * p.batch * p.num_heads + at) * p.hd;
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        if (32 * c >= p.hd) break;  // uniform
        uint32_t o[32];
        __syncwarp();
        tmem_ld32(t_o + c * 32, o);
        if (at >= 0) {
          // (hd is a multiple of 8: every row of the workspace is 32-byte aligned)
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = __float_as_uint(__uint_as_float(o[i + e]) * inv_l);
            if (32 * c + i < p.hd) st_global_v8(part + 32 * c + i, w);
          }
        }
      }
    } else {
      // A thread's row goes out as whole 32-byte sectors straight from its registers.
      // (Staging 64 columns in shared memory for a TMA box took ~2300 cycles of an
      // item's ~7000 with one key tile: two proxy fences and a wait for the box.)
      T* out = static_cast<T*>(p.out) + at * p.hd;
      uint64_t z = 0ull;  // NaN where the row's output is (or infinite)
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        if (32 * c >= p.hd) break;  // uniform
        uint32_t o[32];
        __syncwarp();  // (rows of no position stored nothing in the last round)
        tmem_ld32(t_o + c * 32, o);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          z = ffma2(f2_pack(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1])), 0ull, z);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          if (at < 0) break;
          uint32_t w[8];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            w[i] = Pack<T>::two(__uint_as_float(o[16 * q + 2 * i]) * inv_l, __uint_as_float(o[16 * q + 2 * i + 1]) * inv_l);
          const int col = 32 * c + 16 * q;
          if (p.wide_store && col + 16 <= p.hd) {
            st_global_v8(out + col, w);
          } else {
            if (col < p.hd) *reinterpret_cast<uint4*>(out + col) = make_uint4(w[0], w[1], w[2], w[3]);
            if (col + 8 < p.hd) *reinterpret_cast<uint4*>(out + col + 8) = make_uint4(w[4], w[5], w[6], w[7]);
          }
        }
      }
      float z0, z1;
      f2_unpack(z, z0, z1);
      const uint32_t bad = __ballot_sync(0xffffffffu, at >= 0 && z0 + z1 != 0.f && l_run - l_run == 0.f);
      if (bad != 0u) note_repair(abort_flag, k);
    }
  }
}

template <typename T, int HD, bool PREFIX>
__global__ void __launch_bounds__(GroupedSmem<HD>::kThreads, 1)
grouped_attn_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                    const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_out,
                    const __grid_constant__ GroupedParams p) {
  using L = GroupedSmem<HD>;
  constexpr int SK = L::kStagesK, SV = L::kStagesV;
  constexpr int NT = L::kNT;
  constexpr bool kSepP = L::kSepP;
  constexpr int kChunks = HD / 64;
  constexpr int kBf16 = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
  constexpr uint32_t kIdescPV = idesc_f16(kTile, HD, kBf16, 1);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = smem + L::kQOff;
  uint8_t* sK = smem + L::kKOff;
  uint8_t* sV = smem + L::kVOff;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* q_full = bars;              // [kQBufs][2] per tile: Q_t loaded
  uint64_t* q_empty = q_full + 4;       // [kQBufs][2] per tile: last Q_t K^T of the item done
  uint64_t* k_full = q_empty + 4;       // [SK]
  uint64_t* k_empty = k_full + SK;      // [2][SK] per tile: its Q_t K^T done with the stage
  uint64_t* v_full = k_empty + 2 * SK;  // [SV]
  uint64_t* v_empty = v_full + SV;      // [2][SV] per tile: its P_t V done with the stage
  uint64_t* s_full = v_empty + 2 * SV;  // [2] per tile: S_t written
  uint64_t* s_free = s_full + 2;        // [2] per tile: S_t read by the softmax (separate P)
  uint64_t* p_full = s_free + 2;        // [2] per tile: P_t written
  uint64_t* o_done = p_full + 2;        // [2] per tile: one phase per completed P_t V (separate P) or item
  uint64_t* drain = o_done + 2;         // [2] per issuer: every MMA completed
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* redo = abort_flag + 1;  // [2] first and last of the items to repair

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  constexpr int kSoftmaxThreads = kSepP ? 256 : 128;  // per tile

  if (threadIdx.x == 0) {
    for (int s = 0; s < SK; ++s) {
      mbar_init(&k_full[s], 1);
      for (int t = 0; t < 2; ++t) mbar_init(&k_empty[t * SK + s], 1);
    }
    for (int s = 0; s < SV; ++s) {
      mbar_init(&v_full[s], 1);
      for (int t = 0; t < 2; ++t) mbar_init(&v_empty[t * SV + s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      for (int b = 0; b < 2; ++b) {
        mbar_init(&q_full[b * 2 + t], 1);
        mbar_init(&q_empty[b * 2 + t], 1);
      }
      mbar_init(&s_full[t], 1);
      mbar_init(&s_free[t], kSoftmaxThreads);
      mbar_init(&p_full[t], kSoftmaxThreads);
      mbar_init(&o_done[t], 1);
      mbar_init(&drain[t], 1);
    }
    *abort_flag = 0;
    redo[0] = 0x7fffffff;
    redo[1] = -1;
    fence_mbar_init();
  }
  if (p.positions * p.group < kTile) {
    // rows of the Q tiles that no box ever writes: zeros, so that no stale bits
    // make their (unused) softmax rescale at every step
    const int first = p.positions * p.group * 128;
    for (int c = 0; c < NT * L::kQBufs * kChunks; ++c)
      for (int i = first + threadIdx.x * 16; i < kChunkBytes; i += L::kThreads * 16)
        *reinterpret_cast<uint4*>(sQ + c * kChunkBytes + i) = make_uint4(0u, 0u, 0u, 0u);
    fence_proxy_async_smem();
  }
  if (warp == 0) {
    __syncwarp();
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_dependency_wait();  // the previous kernel's writes are visible from here
  grid_launch_dependents();

  if (warp < 4) {
    setmaxnreg_dec<L::kRegsCtl>();
    if (warp == 0 && lane == 0) {
      // ------------------------------------------------------------ K/V producer
      // A stage is refilled once every issuer has released its previous key tile
      // (with P over S one warp issues both tiles' products and releases through
      // tile B's barriers).
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
      auto reclaim = [&](uint64_t* empty, int stages, int kv) -> bool {
        const int st = kv % stages;
        const uint32_t phase = ((kv / stages) & 1) ^ 1;  // passes on the first round
        return (!kSepP || mbar_wait(&empty[st], phase, p.status, kDevTimeoutSmemEmpty, abort_flag)) &&
               mbar_wait(&empty[stages + st], phase, p.status, kDevTimeoutSmemEmpty, abort_flag);
      };
      int kv = 0;  // running K/V tile counter across items
      bool ok = true;
      for (int k = 0; ok; ++k) {
        const int item = item_of(k);
        if (item >= p.num_items) break;
        const Seg s = seg_of<PREFIX, NT>(item, p);
        const int n_kv = item_tiles<PREFIX, NT>(s, p.positions);
        for (int j = 0; j < n_kv; ++j, ++kv) {
          const int sk = kv % SK, sv = kv % SV;
          if (L::kReleaseK && !reclaim(k_empty, SK, kv)) { ok = false; break; }
          mbar_arrive_expect_tx(&k_full[sk], L::kTileBytes);
          for (int c = 0; c < kChunks; ++c)
            tma_load_3d(sK + sk * L::kTileBytes + c * kChunkBytes, &tm_k, &k_full[sk], 64 * c, s.kvh, s.k0 + j * kTile);
          if (!reclaim(v_empty, SV, kv)) { ok = false; break; }
          mbar_arrive_expect_tx(&v_full[sv], L::kTileBytes);
          for (int c = 0; c < kChunks; ++c)
            tma_load_3d(sV + sv * L::kTileBytes + c * kChunkBytes, &tm_v, &v_full[sv], 64 * c, s.kvh, s.k0 + j * kTile);
        }
      }
    } else if (warp == 2 && lane == 0) {
      // ------------------------------------------------------------ Q producer
      tma_prefetch_desc(&tm_q);
      const uint32_t bytes = (uint32_t)(p.positions * p.group) * 128u * kChunks;
      int cnt[2] = {0, 0};  // Q_t tiles loaded so far
      bool ok = true;
      for (int k = 0; ok; ++k) {
        const int item = item_of(k);
        if (item >= p.num_items) break;
        const Seg s = seg_of<PREFIX, NT>(item, p);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if (!ok || t * p.positions >= s.nq) continue;
          const int qb = cnt[t] % L::kQBufs;
          const uint32_t qph = (cnt[t] / L::kQBufs) & 1;
          ++cnt[t];
          ok = mbar_wait(&q_empty[qb * 2 + t], qph ^ 1u, p.status, kDevTimeoutSmemEmpty, abort_flag);
          if (!ok) continue;
          mbar_arrive_expect_tx(&q_full[qb * 2 + t], bytes);
          for (int c = 0; c < kChunks; ++c)
            tma_load_4d(sQ + (qb * NT + t) * L::kTileBytes + c * kChunkBytes, &tm_q, &q_full[qb * 2 + t], 64 * c, 0,
                        s.kvh, s.q0 + t * p.positions);
        }
      }
    } else if (warp == 1 || (kSepP && warp == 3)) {
      // ------------------------------------------------------------ MMA issue
      // The whole warp waits (it zeroes V rows together), lane 0 issues.
      // S_t columns of keys past the tile's last visible one are not computed:
      // n = keys of this tile rounded up to 16 (the softmax masks the rest).
      auto qk = [&](int t, int st, int qb, int keys) {
        const uint32_t n = (uint32_t)min(kTile, (keys + 15) & ~15);
        const uint32_t idesc = idesc_f16(kTile, 0, kBf16, 0) | ((n >> 3) << 17);
        const uint32_t q_addr = smem_u32(sQ + (qb * NT + t) * L::kTileBytes);
        const uint32_t k_addr = smem_u32(sK + st * L::kTileBytes);
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const uint32_t off = (kk >> 2) * kChunkBytes + (kk & 3) * 32;
          umma_f16_ss(tmem + t * 128, smem_desc_sw128(q_addr + off, 16, 1024),
                      smem_desc_sw128(k_addr + off, 16, 1024), idesc, kk > 0 ? 1u : 0u);
        }
      };
      auto pv = [&](int t, int st, bool accumulate, int keys) {
        const uint32_t v_addr = smem_u32(sV + st * L::kTileBytes);
#pragma unroll
        for (int kk = 0; kk < kTile / 16; ++kk) {
          // V is MN-major: 16 keys = 16 rows of 128 bytes; next 64-column chunk at +16 KB.
          if (16 * kk < keys)
            umma_f16_ts(tmem + L::kColO + t * HD, tmem + L::kColP + t * L::kPStride + kk * 8,
                        smem_desc_sw128(v_addr + kk * 16 * 128, kChunkBytes, 1024), kIdescPV,
                        (accumulate || kk > 0) ? 1u : 0u);
        }
      };
      // V rows `valid` .. up to the next multiple of 16 of a stage become zeros:
      // P.V reads them (with P = 0 in every row that counts).
      auto zero_v_tail = [&](int st, int valid) {
        if ((valid & 15) == 0) return;
        const int rows = 16 - (valid & 15);
        for (int i = lane; i < rows * 8 * kChunks; i += 32) {
          const int c = i / (rows * 8), w = i - c * rows * 8;
          *reinterpret_cast<uint4*>(sV + st * L::kTileBytes + c * kChunkBytes + valid * 128 + w * 16) =
              make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
        __syncwarp();
      };
      if constexpr (kSepP) {
        // One issuing warp per tile; the Q.K cursor runs one key tile ahead of the
        // P.V cursor, across items: S_t(j+1) is issued once the softmax has read
        // S_t(j) (s_free), then O_t += P_t(j) V_j once P_t(j) is written.  Key tiles
        // that only the other query tile uses are waited for and released too: a
        // barrier's parity can only be followed phase by phase.
        const int t = warp == 3 ? 1 : 0;
        int qk_k = -1, qk_j = 0, qk_kv = 0, qk_keys = 0, qk_n = 0, qk_cnt = 0;
        bool qk_first = true;
        auto qk_open = [&]() -> bool {
          const int item = item_of(++qk_k);
          if (item >= p.num_items) return false;
          const Seg s = seg_of<PREFIX, NT>(item, p);
          qk_keys = tile_keys<PREFIX>(s, t, p.positions);
          qk_n = item_tiles<PREFIX, NT>(s, p.positions);
          qk_j = 0;
          return true;
        };
        bool qk_live = qk_open();
        uint32_t sfree_ph = 0u, pf_ph = 0u;
        auto issue_qk = [&]() -> bool {
          if (!qk_live) return true;
          const int keys = qk_keys - qk_j * kTile;  // this tile's keys from here on
          const int qb = qk_cnt % L::kQBufs;
          // the barriers of this product, polled together (a completed wait costs this
          // warp ~125 cycles)
          const int st = qk_kv % SK;
          const uint32_t q_phase = (qk_cnt / L::kQBufs) & 1, k_phase = (qk_kv / SK) & 1;
          const bool need_q = keys > 0 && qk_j == 0, need_s = keys > 0 && !qk_first;
          const bool ready = (!need_q || mbar_try_wait(smem_u32(&q_full[qb * 2 + t]), q_phase)) &
                             (!need_s || mbar_try_wait(smem_u32(&s_free[t]), sfree_ph)) &
                             mbar_try_wait(smem_u32(&k_full[st]), k_phase);
          if (!__all_sync(0xffffffffu, ready)) {
            if (need_q && !mbar_wait_warp(&q_full[qb * 2 + t], q_phase, p.status, kDevTimeoutTmaFull, abort_flag)) return false;
            if (need_s && !mbar_wait_warp(&s_free[t], sfree_ph, p.status, kDevTimeoutSoftmax, abort_flag)) return false;
            if (!mbar_wait_warp(&k_full[st], k_phase, p.status, kDevTimeoutTmaFull, abort_flag)) return false;
          }
          if (need_s) sfree_ph ^= 1u;
          ++qk_kv;
          const bool last = keys > 0 && keys <= kTile;  // the last S_t of the item: Q_t may be replaced
          if (keys > 0) {
            tc_fence_after();
            if (lane == 0) {
              qk(t, st, qb, keys);
              umma_commit(&s_full[t]);
              if constexpr (L::kReleaseK) umma_commit(&k_empty[t * SK + st]);
              if (last) umma_commit(&q_empty[qb * 2 + t]);
            }
            qk_first = false;
          } else if (L::kReleaseK && lane == 0) {
            mbar_arrive(&k_empty[t * SK + st]);
          }
          __syncwarp();
          if (last) ++qk_cnt;
          if (++qk_j == qk_n) qk_live = qk_open();
          return true;
        };
        bool ok = issue_qk();
        int kv = 0;
        for (int k = 0; ok; ++k) {
          const int item = item_of(k);
          if (item >= p.num_items) break;
          const Seg s = seg_of<PREFIX, NT>(item, p);
          const int keys = tile_keys<PREFIX>(s, t, p.positions), nk = s.nk;
          const int n = item_tiles<PREFIX, NT>(s, p.positions);
          for (int j = 0; j < n; ++j, ++kv) {
            if (!issue_qk()) { ok = false; break; }
            const bool active = j * kTile < keys;
            const int st = kv % SV;
            const uint32_t v_phase = (kv / SV) & 1;
            const bool ready = (!active || mbar_try_wait(smem_u32(&p_full[t]), pf_ph)) &
                               mbar_try_wait(smem_u32(&v_full[st]), v_phase);
            if (!__all_sync(0xffffffffu, ready)) {
              if (active && !mbar_wait_warp(&p_full[t], pf_ph, p.status, kDevTimeoutSoftmax, abort_flag)) { ok = false; break; }
              if (!mbar_wait_warp(&v_full[st], v_phase, p.status, kDevTimeoutTmaFull, abort_flag)) { ok = false; break; }
            }
            if (active) pf_ph ^= 1u;
            if (active) {
              // both tiles' issuers may write these zeros; a product that already
              // reads them reads zeros either way
              if (nk - j * kTile < kTile) zero_v_tail(st, nk - j * kTile);
              tc_fence_after();
              if (lane == 0) {
                pv(t, st, j > 0, keys - j * kTile);
                umma_commit(&o_done[t]);
                umma_commit(&v_empty[t * SV + st]);
              }
            } else if (lane == 0) {
              mbar_arrive(&v_empty[t * SV + st]);
            }
            __syncwarp();
          }
        }
        // Nothing of this warp's may still run on the tensor core when TMEM is
        // released (matters only after an abort).
        if (lane == 0) {
          umma_commit(&drain[t]);
          mbar_wait(&drain[t], 0, p.status, kDevTimeoutSoftmax, nullptr);
        }
        __syncwarp();
      } else {
        static_assert(L::kQBufs == 1, "the single-issuer schedule uses one Q buffer per tile");
        // P over S: one warp issues both tiles, PV_A(j) QK_A(j+1) PV_B(j) QK_B(j+1).
        // Stages are released through tile B's barriers, once every earlier
        // product of this thread has completed.
        int kv = 0;
        uint32_t pf_phase[2] = {0u, 0u}, q_phase[2] = {0u, 0u};
        bool ok = true;
        Seg next = seg_of<PREFIX, NT>(item_of(0), p);
        for (int k = 0; ok; ++k) {
          if (item_of(k) >= p.num_items) break;
          const Seg s = next;
          const int keys_a = tile_keys<PREFIX>(s, 0, p.positions);
          const int keys_b = NT == 2 ? tile_keys<PREFIX>(s, 1, p.positions) : 0;
          const int n_a = key_tiles(keys_a), n_b = key_tiles(keys_b), n = max(n_a, n_b);
          const int nk = s.nk;
          const int kv0 = kv;
          {
            const int st = kv0 % SK;
            const uint32_t k_phase = (kv0 / SK) & 1;
            const bool ready = mbar_try_wait(smem_u32(&q_full[0]), q_phase[0]) &
                               (n_b == 0 || mbar_try_wait(smem_u32(&q_full[1]), q_phase[1])) &
                               mbar_try_wait(smem_u32(&k_full[st]), k_phase);
            if (!__all_sync(0xffffffffu, ready)) {
              if (!mbar_wait_warp(&q_full[0], q_phase[0], p.status, kDevTimeoutTmaFull, abort_flag)) break;
              if (n_b > 0 && !mbar_wait_warp(&q_full[1], q_phase[1], p.status, kDevTimeoutTmaFull, abort_flag)) break;
              if (!mbar_wait_warp(&k_full[st], k_phase, p.status, kDevTimeoutTmaFull, abort_flag)) break;
            }
            q_phase[0] ^= 1u;
            if (n_b > 0) q_phase[1] ^= 1u;
            tc_fence_after();
            if (lane == 0) {
              qk(0, st, 0, keys_a);
              umma_commit(&s_full[0]);
              if (n_a == 1) umma_commit(&q_empty[0]);
              if (n_b > 0) {
                qk(1, st, 0, keys_b);
                umma_commit(&s_full[1]);
                if (n_b == 1) umma_commit(&q_empty[1]);
              }
              if constexpr (L::kReleaseK) umma_commit(&k_empty[SK + st]);
            }
            __syncwarp();
          }
          // the next item's place, while this one's first softmax runs
          if (item_of(k + 1) < p.num_items) next = seg_of<PREFIX, NT>(item_of(k + 1), p);
          for (int j = 0; j < n; ++j) {
            const int st = (kv0 + j) % SV;
            const int st_n = (kv0 + j + 1) % SK;
            const int left = nk - j * kTile;  // keys of the item from this tile on
            // The three barriers this step starts on, polled together: one after the
            // other, each completed wait costs this warp ~125 cycles of its ~3600.
            uint64_t* const p_first = n_a > j ? &p_full[0] : &p_full[1];
            const uint32_t p_phase = n_a > j ? pf_phase[0] : pf_phase[1];
            const bool ready = (j + 1 == n || mbar_try_wait(smem_u32(&k_full[st_n]), ((kv0 + j + 1) / SK) & 1)) &
                               mbar_try_wait(smem_u32(&v_full[st]), ((kv0 + j) / SV) & 1) &
                               mbar_try_wait(smem_u32(p_first), p_phase);
            if (!__all_sync(0xffffffffu, ready)) {
              if (j + 1 < n && !mbar_wait_warp(&k_full[st_n], ((kv0 + j + 1) / SK) & 1, p.status, kDevTimeoutTmaFull,
                                               abort_flag)) { ok = false; break; }
              if (!mbar_wait_warp(&v_full[st], ((kv0 + j) / SV) & 1, p.status, kDevTimeoutTmaFull, abort_flag)) { ok = false; break; }
              if (!mbar_wait_warp(p_first, p_phase, p.status, kDevTimeoutSoftmax, abort_flag)) { ok = false; break; }
            }
            if (left < kTile) zero_v_tail(st, left);
            if (j < n_a) {
              pf_phase[0] ^= 1u;
              tc_fence_after();
              if (lane == 0) {
                pv(0, st, j > 0, keys_a - j * kTile);
                if (j + 1 < n_a) {
                  qk(0, st_n, 0, keys_a - (j + 1) * kTile);
                  umma_commit(&s_full[0]);
                  if (j + 2 == n_a) umma_commit(&q_empty[0]);
                } else {
                  umma_commit(&o_done[0]);
                }
              }
              __syncwarp();
            }
            if (j < n_b) {
              if (j < n_a && !mbar_wait_warp(&p_full[1], pf_phase[1], p.status, kDevTimeoutSoftmax, abort_flag)) { ok = false; break; }
              pf_phase[1] ^= 1u;
              tc_fence_after();
            }
            if (lane == 0) {
              if (j < n_b) pv(1, st, j > 0, keys_b - j * kTile);
              umma_commit(&v_empty[SV + st]);
              if (j + 1 < n_b) {
                qk(1, st_n, 0, keys_b - (j + 1) * kTile);
                umma_commit(&s_full[1]);
                if (j + 2 == n_b) umma_commit(&q_empty[1]);
              } else if (j < n_b) {
                umma_commit(&o_done[1]);
              }
              if (L::kReleaseK && j + 1 < n) umma_commit(&k_empty[SK + st_n]);
            }
            __syncwarp();
          }
          kv = kv0 + n;
        }
        if (lane == 0) {
          umma_commit(&drain[0]);
          mbar_wait(&drain[0], 0, p.status, kDevTimeoutSoftmax, nullptr);
        }
        __syncwarp();
      }
    }
  } else {
    setmaxnreg_inc<L::kRegsSoftmax>();
    if constexpr (kSepP)
      softmax_pairs<T, HD, PREFIX>(p, smem + L::kEpiOff, tmem, &tm_out, s_full, s_free, p_full, o_done, abort_flag);
    else
      softmax_rows<T, HD, PREFIX>(p, tmem, s_full, p_full, o_done, abort_flag);
    if constexpr (!PREFIX) {
      using R = Repair<HD>;
      static_assert(sizeof(R) <= L::kBarOff, "the Q, K and V buffers hold it");
      repair_sync(R::kThreads);  // every item of the block is done (or a wait ran out)
      if (redo[0] <= redo[1] && !*abort_flag) repair_items<T, HD>(p, *reinterpret_cast<R*>(smem), redo[0], redo[1]);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, kTmemCols);
}

// Check the register count the kernel's setmaxnreg split assumes (with another
// the softmax warps' increase could never complete) and opt in to its shared
// memory, once per kernel and device.
template <typename Kernel>
int prepare_kernel(Kernel kern, int launch_regs, int smem, std::atomic<uint64_t>& done) {
  int dev = 0;
  TTJ_CUDA_TRY(cudaGetDevice(&dev));
  const uint64_t bit = (uint64_t)1 << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_acquire) & bit)) return TTJ_OK;
  cudaFuncAttributes fa;
  TTJ_CUDA_TRY(cudaFuncGetAttributes(&fa, kern));
  if (fa.numRegs != launch_regs)
    return fail(TTJ_ERR_UNSUPPORTED, "attention kernel register count differs from its register split");
  TTJ_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  done.fetch_or(bit, std::memory_order_release);
  return TTJ_OK;
}

struct GroupedTensors {
  const void *q, *k, *v;
  int64_t q_rows, kv_rows;                  // tokens or sequences; tokens or prefix rows
  int64_t q_row_stride, q_head_stride, k_row_stride, k_head_stride, v_row_stride, v_head_stride;
};

template <typename T, int HD, bool PREFIX>
int launch_grouped(const GroupedTensors& x, const GroupedParams& p, int max_blocks, cudaStream_t stream) {
  using L = GroupedSmem<HD>;
  const CUtensorMapDataType dt = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const uint64_t hd = (uint64_t)p.hd, g = (uint64_t)p.group, hkv = (uint64_t)p.kv_heads;
  CUtensorMap tm_q, tm_k, tm_v, tm_out;
  {
    const uint64_t dims[4] = {hd, g, hkv, (uint64_t)x.q_rows};
    const uint64_t strides[3] = {(uint64_t)x.q_head_stride * 2, (uint64_t)x.q_head_stride * 2 * g,
                                 (uint64_t)x.q_row_stride * 2};
    const uint32_t box[4] = {64, (uint32_t)p.group, 1, (uint32_t)p.positions};
    if (int rc = encode_tmap(&tm_q, dt, 4, x.q, dims, strides, box)) return rc;
  }
  const uint64_t dims[3] = {hd, hkv, (uint64_t)x.kv_rows};
  const uint32_t box[3] = {64, 1, kTile};
  const uint64_t ks[2] = {(uint64_t)x.k_head_stride * 2, (uint64_t)x.k_row_stride * 2};
  const uint64_t vs[2] = {(uint64_t)x.v_head_stride * 2, (uint64_t)x.v_row_stride * 2};
  if (int rc = encode_tmap(&tm_k, dt, 3, x.k, dims, ks, box)) return rc;
  if (int rc = encode_tmap(&tm_v, dt, 3, x.v, dims, vs, box)) return rc;
  if (p.box_store) {
    // out [T][Hq][hd] as [T][kv heads][group][hd]: a softmax warp's rows, 64 columns
    const uint64_t odims[4] = {hd, g, hkv, (uint64_t)x.q_rows};
    const uint64_t ostr[3] = {hd * 2, hd * 2 * g, hd * 2 * g * hkv};
    const uint32_t obox[4] = {64, (uint32_t)p.group, 1, (uint32_t)(16 / p.group)};
    if (int rc = encode_tmap(&tm_out, dt, 4, p.out, odims, ostr, obox)) return rc;
  } else {
    tm_out = tm_q;  // not used
  }
  auto kern = grouped_attn_kernel<T, HD, PREFIX>;
  static std::atomic<uint64_t> done{0};
  if (int rc = prepare_kernel(kern, L::kLaunchRegs, L::kTotal, done)) return rc;
  const int grid = p.num_items < max_blocks ? p.num_items : max_blocks;
  TTJ_CUDA_TRY(launch_pdl(kern, dim3(grid), dim3(L::kThreads), L::kTotal, stream, tm_q, tm_k, tm_v, tm_out, p));
  return TTJ_OK;
}

template <bool PREFIX>
int dispatch(int dtype, const GroupedTensors& x, const GroupedParams& p, int max_blocks, cudaStream_t stream) {
  if (dtype == TTJ_F16) {
    if (p.hd <= 64) return launch_grouped<__half, 64, PREFIX>(x, p, max_blocks, stream);
    if (p.hd <= 128) return launch_grouped<__half, 128, PREFIX>(x, p, max_blocks, stream);
    return launch_grouped<__half, 256, PREFIX>(x, p, max_blocks, stream);
  }
  if (p.hd <= 64) return launch_grouped<__nv_bfloat16, 64, PREFIX>(x, p, max_blocks, stream);
  if (p.hd <= 128) return launch_grouped<__nv_bfloat16, 128, PREFIX>(x, p, max_blocks, stream);
  return launch_grouped<__nv_bfloat16, 256, PREFIX>(x, p, max_blocks, stream);
}

}  // namespace

int launch_prompt_attn(const ttj_prompt_attn_args& a, cudaStream_t stream) {
  GroupedTensors x{a.q, a.k, a.v, a.tokens, a.tokens, a.q_token_stride, a.q_head_stride,
                   a.k_token_stride, a.k_head_stride, a.v_token_stride, a.v_head_stride};
  GroupedParams p{};
  p.out = a.out;
  p.lse = a.lse;
  p.plan = reinterpret_cast<const int4*>(a.plan);
  p.num_entries = (int)a.plan_entries;
  p.kv_heads = (int)a.num_kv_heads;
  p.num_items = (int)(a.plan_entries * a.num_kv_heads);
  p.num_heads = (int)a.num_heads;
  p.group = (int)(a.num_heads / a.num_kv_heads);
  p.positions = kTile / p.group;
  p.hd = (int)a.head_dim;
  p.kv_shift = (p.kv_heads & (p.kv_heads - 1)) == 0 ? __builtin_ctz((unsigned)p.kv_heads) : -1;
  p.box_store = p.hd <= 64 && 16 % p.group == 0;
  p.wide_store = p.hd % 16 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 31) == 0;
  p.scale_log2 = (float)((double)a.scale * 1.4426950408889634);
  p.status = a.status;
  p.q = a.q;
  p.k = a.k;
  p.v = a.v;
  p.q_row = a.q_token_stride, p.q_head = a.q_head_stride;
  p.k_row = a.k_token_stride, p.k_head = a.k_head_stride;
  p.v_row = a.v_token_stride, p.v_head = a.v_head_stride;
  return dispatch<false>(a.dtype, x, p, sm_count(), stream);
}

int launch_prefix_parts(const ttj_shared_prefix_attn_args& a, float* part_o, float* part_lse, int parts,
                        int part_keys, int max_blocks, cudaStream_t stream) {
  GroupedTensors x{a.q, a.prefix_k, a.prefix_v, a.batch, a.prefix_len, a.q_seq_stride, a.q_head_stride,
                   a.prefix_k_row_stride, a.prefix_k_head_stride, a.prefix_v_row_stride, a.prefix_v_head_stride};
  GroupedParams p{};
  p.part_o = part_o;
  p.part_lse = part_lse;
  p.kv_heads = (int)a.num_kv_heads;
  p.num_heads = (int)a.num_heads;
  p.group = (int)(a.num_heads / a.num_kv_heads);
  p.positions = kTile / p.group;
  p.hd = (int)a.head_dim;
  p.batch = (int)a.batch;
  p.prefix = (int)a.prefix_len;
  p.split_keys = part_keys;
  const int64_t per_item = plan_positions(p.group, a.head_dim);
  p.row_items = (int)((a.batch + per_item - 1) / per_item);
  const int64_t items = (int64_t)p.row_items * parts * a.num_kv_heads;
  if (items >= ((int64_t)1 << 31) - 65536) return fail(TTJ_ERR_UNSUPPORTED, "too many attention work items");
  p.num_entries = p.row_items * parts;
  p.num_items = (int)items;
  p.scale_log2 = (float)((double)a.scale * 1.4426950408889634);
  p.status = a.status;
  return dispatch<true>(a.dtype, x, p, max_blocks, stream);
}

}  // namespace ttj
