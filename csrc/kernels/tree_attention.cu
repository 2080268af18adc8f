// Attention of drafted trees over the paged KV cache.  A sequence's keys are its committed context, base = kv_len - tree_len
// of them, followed by its tree's nodes; its query rows are the last q_len nodes.  Row i (node n = tree_len - q_len + i)
// sees every context key (with a sliding window those at positions > base + depth_n - window) and the nodes whose bit is
// set in masks[n]:
//     o_n = sum_j exp(s_nj - m_n) v_j / sum_j exp(s_nj - m_n),   s_nj = scale q_n . k_j,   m_n = max_j s_nj;
// a row that sees nothing is zero.
#include "../common/ptx.cuh"
#include "../common/tmap.cuh"

namespace afb {

struct TreeAttnParams {
  const __nv_bfloat16* q;
  long q_stride;
  const void* k_cache;
  const void* v_cache;       // [num_blocks, page, Hkv, D]
  const int* tables;
  long table_stride;
  int max_blocks, page, num_blocks;
  const int* q_starts;
  const int* q_lens;
  const int* kv_lens;
  const int* tree_lens;
  const int* masks;          // [B, nodes, words]
  long mask_stride;          // between sequences (0: one tree for all)
  int nodes, words;
  const int* depths;         // [B, nodes], read when window > 0
  long depth_stride;
  __nv_bfloat16* out;
  long out_stride;
  int T, Hq, Hkv, D;
  int window;                // 0: none, also for one that reaches every key of max_kv
  int max_kv;                // what the caller says that no kv_len passes
  int zero_rest;             // rows of no sequence become zero
  float scale_log2;
  int B, max_q, box_rows, page_shift;         // log2(page), -1 when page is no power of two
  int row_tiles;             // of a KV head
  int splits, chunk;         // chunks of a sequence at most; 64-key tiles of a chunk
  int groups;                // tcgen05: pieces of the line of tiles
  int heads, blocks;         // KV heads of a block, blocks
  uint32_t g_magic;          // r / (Hq / Hkv) = umulhi(r, g_magic), 0 when that is r
  float* part_o;             // [splits, T * Hq, D]; tcgen05: [CTAs, 2, D / 8, 128, 8]
  float* part_lse;           // base 2, a value per row of part_o
  long part_rows;            // T * Hq
};

struct TreeSeq {
  int q_start, q_len, kv_len, tree_len, base;
};

// Lengths of one sequence, brought into the ranges that every access below relies on; what had to be changed is reported.
__device__ __forceinline__ TreeSeq tree_seq(const TreeAttnParams& p, int b) {
  TreeSeq s;
  const int q0 = p.q_starts[b], ql = p.q_lens[b], kv = p.kv_lens[b], tl = p.tree_lens[b];
  s.q_start = max(q0, 0);
  s.q_len = max(min(ql, p.T - s.q_start), 0);
  s.kv_len = max(0, static_cast<int>(min(static_cast<long>(kv), static_cast<long>(p.max_blocks) * p.page)));
  s.tree_len = max(0, min(min(tl, s.kv_len), p.nodes));
  s.q_len = min(min(s.q_len, s.tree_len), p.max_q);
  s.base = s.kv_len - s.tree_len;
  if (s.q_start != q0 || s.q_len != ql || s.kv_len != kv || s.tree_len != tl || kv > p.max_kv) status_set(kStatusBadIndex);
  return s;
}

constexpr int kKeys = 64;      // keys of a tile

// Range of 64-key tiles that some row of the sequence sees, and the first key that none of them masks by the window.
struct TreeTiles {
  int lo_key, lo, hi;
};
__device__ __forceinline__ TreeTiles tree_tiles(const TreeAttnParams& p, const TreeSeq& s) {
  TreeTiles t;
  t.lo_key = p.window > 0 ? max(0, s.base - p.window + 1) : 0;   // of a root; deeper nodes start later
  t.lo = t.lo_key / kKeys;
  t.hi = (s.kv_len + kKeys - 1) / kKeys;
  if (t.hi - t.lo > static_cast<long>(p.splits) * p.chunk) {                        // more keys than the caller said
    t.hi = t.lo + p.splits * p.chunk;
    status_set(kStatusBadIndex);
  }
  return t;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Zeros in the rows that belong to no sequence and follow those of sequence b (for the first also in front of all), columns
// col .. col + n - 1 (multiples of 8): this thread's, of `threads`.  Starts may be in any order.  Where every sequence begins
// at the end of the one before it and the last ends at T, there is nothing to do and that shows from one more load (`next`,
// which is best on its way with the others); otherwise the next start is looked up.
__device__ __forceinline__ int next_start(const TreeAttnParams& p, int b) { return b + 1 < p.B ? p.q_starts[b + 1] : p.T; }
__device__ __forceinline__ void zero_gap(const TreeAttnParams& p, const TreeSeq& s, int next, int b, int col, int n,
                                         int threads, int me) {
  const int end = s.q_start + s.q_len;
  const bool front = b == 0 && (s.q_start > 0 || s.q_len == 0), behind = s.q_len > 0 && next != end;
  if (!front && !behind) return;
  int first = p.T, after = p.T;                    // start of all rows that sequences have, of those from `end` on
  for (int c = threadIdx.x & 31; c < p.B; c += 32) {
    const TreeSeq t = tree_seq(p, c);
    if (t.q_len == 0) continue;
    first = min(first, t.q_start);
    if (t.q_start >= end) after = min(after, t.q_start);
  }
  first = front ? __reduce_min_sync(0xffffffffu, first) : 0;
  after = behind ? __reduce_min_sync(0xffffffffu, after) : end;
  const int cols = n / 8;
  for (long x = me; x < static_cast<long>(first + after - end) * cols; x += threads) {
    const long row = x / cols;
    *reinterpret_cast<uint4*>(p.out + (row < first ? row : row - first + end) * p.out_stride + col + x % cols * 8) =
        make_uint4(0, 0, 0, 0);
  }
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(valid ? 8 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Cache row of key j, or -1 where there is none (outside [lo, kv_len), or a block id that is not one).
__device__ __forceinline__ long tree_slot(const TreeAttnParams& p, const int* table, int j, int lo, int kv_len) {
  if (j < lo || j >= kv_len) return -1;
  const int blk = p.page_shift >= 0 ? j >> p.page_shift : j / p.page;
  const int id = table[blk];
  if (static_cast<unsigned>(id) >= static_cast<unsigned>(p.num_blocks)) {
    status_set(kStatusBadIndex);
    return -1;
  }
  return static_cast<long>(id) * p.page + (j - blk * p.page);
}

// Brings keys k0 .. k0 + 63 of one KV head to shared memory, zeros where there is no key and behind column D.  bf16: rows
// of DP elements whose 16-byte columns are XORed with the row's low three bits (conflict-free ldmatrix); e4m3: plain
// rows of DP bytes, expanded later by the threads that loaded them.
template <int DP, bool KV8>
__device__ __forceinline__ void load_tile(uint32_t sk, uint32_t sv, const TreeAttnParams& p, const int* table, int hk,
                                          int k0, int lo, int kv_len) {
  constexpr int ROW = DP * (KV8 ? 1 : 2);       // bytes
  constexpr int CH = ROW / 16, PASS = 128 / CH;  // 16-byte columns; rows per pass of the CTA
  const int ch = threadIdx.x % CH, r0 = threadIdx.x / CH;
  const int el = KV8 ? 1 : 2;
  const long row_bytes = static_cast<long>(p.Hkv) * p.D * el;
  const long col = static_cast<long>(hk) * p.D * el + ch * 16;
  const uint8_t* k = static_cast<const uint8_t*>(p.k_cache);
  const uint8_t* v = static_cast<const uint8_t*>(p.v_cache);
  const bool in_row = ch * 16 < p.D * el;
#pragma unroll
  for (int i = 0; i < kKeys / PASS; ++i) {
    const int row = r0 + i * PASS;
    const long slot = tree_slot(p, table, k0 + row, lo, kv_len);
    const bool ok = slot >= 0 && in_row;
    const long off = ok ? slot * row_bytes + col : 0;
    if (KV8) {
      const uint32_t d = row * ROW + ch * 16;
      if (p.D % 16 == 0) {
        cp_async16(sk + d, k + off, ok);
        cp_async16(sv + d, v + off, ok);
      } else {                                   // rows of an odd number of 8-byte units
        const bool second = ok && ch * 16 + 8 < p.D;
        const long off2 = second ? off + 8 : 0;
        cp_async8(sk + d, k + off, ok);
        cp_async8(sk + d + 8, k + off2, second);
        cp_async8(sv + d, v + off, ok);
        cp_async8(sv + d + 8, v + off2, second);
      }
    } else {
      const uint32_t d = row * ROW + ((ch ^ (row & 7)) << 4);
      cp_async16(sk + d, k + off, ok);
      cp_async16(sv + d, v + off, ok);
    }
  }
}

// Four e4m3 bytes -> four bf16, NaN codes (all seven low bits set) as NaN.
__device__ __forceinline__ uint2 e4m3_to_bf16(uint32_t w) {
  uint2 o;
  e4m3x4_to_bf16x4(w, kE4m3ToBf16Unit, o.x, o.y);
  const uint32_t nan = __vcmpeq4(w & 0x7F7F7F7Fu, 0x7F7F7F7Fu);
  if (nan) {
    o.x |= __byte_perm(nan, 0u, 0x1100) & 0x7FFF7FFFu;
    o.y |= __byte_perm(nan, 0u, 0x3322) & 0x7FFF7FFFu;
  }
  return o;
}

template <int DP>
__device__ __forceinline__ void expand_tile(uint32_t raw, uint32_t work) {
  constexpr int CH = DP / 16, PASS = 128 / CH;
  const int ch = threadIdx.x % CH, r0 = threadIdx.x / CH;
#pragma unroll
  for (int i = 0; i < kKeys / PASS; ++i) {
    const int row = r0 + i * PASS;
    uint4 w;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                 : "r"(raw + row * DP + ch * 16));
    const uint2 a = e4m3_to_bf16(w.x), b = e4m3_to_bf16(w.y), c = e4m3_to_bf16(w.z), d = e4m3_to_bf16(w.w);
    const uint32_t base = work + row * DP * 2;
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(base + (((2 * ch) ^ (row & 7)) << 4)), "r"(a.x),
                 "r"(a.y), "r"(b.x), "r"(b.y)
                 : "memory");
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(base + (((2 * ch + 1) ^ (row & 7)) << 4)), "r"(c.x),
                 "r"(c.y), "r"(d.x), "r"(d.y)
                 : "memory");
  }
}

// Bits of the keys k0 .. k0 + 63 that tree node `node` sees.
__device__ __forceinline__ uint64_t tree_bits(const TreeAttnParams& p, const TreeSeq& s, int b, int node, int k0) {
  const int ctx = min(max(s.base - k0, 0), kKeys);              // context keys of the tile
  uint64_t see = ctx == kKeys ? ~0ull : (1ull << ctx) - 1;
  const int* depths = p.depths + b * p.depth_stride;
  int first = 0;
  if (p.window > 0) {
    first = s.base + depths[node] - p.window + 1;               // context keys in front of it are too far
    const int gone = min(max(first - k0, 0), kKeys);
    see &= gone == kKeys ? 0ull : ~0ull << gone;
  }
  if (ctx < kKeys) {
    const int x0 = k0 - s.base;                                 // tree node at bit 0 (may be negative)
    const uint32_t* m = reinterpret_cast<const uint32_t*>(p.masks) + b * p.mask_stride + static_cast<long>(node) * p.words;
    const auto word = [&](int w) -> uint64_t { return w >= 0 && w < p.words ? m[w] : 0u; };
    const int at = max(x0, 0), w = at >> 5, sh = at & 31;
    uint64_t t = (word(w) | word(w + 1) << 32) >> sh;
    if (sh) t |= word(w + 2) << (64 - sh);
    const int left = s.tree_len - at;                           // nodes from there on
    t &= left >= 64 ? ~0ull : left <= 0 ? 0ull : (1ull << left) - 1;
    if (p.window > 0 && p.window <= p.nodes) {                  // ancestors may be too far as well
      for (uint64_t r = t; r; r &= r - 1) {
        const int x = at + __ffsll(static_cast<long long>(r)) - 1;
        if (depths[x] <= depths[node] - p.window) t &= ~(1ull << (x - at));
      }
    }
    see |= x0 < 0 ? t << -x0 : t;
  }
  return see;
}

// Few rows, little work, windows, wide heads, pages that are no multiple of 8: row tiles of 16 * WR (position,
// head-in-group) rows of one KV head against one chunk of its keys, on mma.sync with a three-stage cp.async ring.  Four
// warps: WR of them own 16 rows each, and 4 / WR groups share the 64 keys of a tile.  Bound by memory up to some 16 rows (64 x
// 2000 keys, 12 rows, 32 / 8 heads of 128: 174 us cold, 3.0 TB/s), by the four warps' instructions above.  One request of 8192
// keys and a tree of 26: 37 us; 12 x 5000 keys, a window of 1024, 256-wide heads, pages of 24: 45 us, where the 208 KiB of the
// ring and Q leave one CTA of four warps on an SM.  Weights are rounded to bf16 for the product with V, their sum is not.
template <int DP, int WR, bool KV8>
struct MmaShape {
  static constexpr int kRow = DP * (KV8 ? 1 : 2);
  static constexpr int kStage = 2 * kKeys * kRow;
  static constexpr int kStages = 3;
  static constexpr int kWork = KV8 ? 2 * kKeys * DP * 2 : 0;    // the bf16 tiles that codes are expanded to
  static constexpr bool kQShared = DP > 128;                    // wider heads: Q fragments would not fit the registers
  static constexpr int kQ = kQShared ? 16 * WR * DP * 2 : 0;
  static constexpr int kSmem = kStages * kStage + kWork + kQ;
  static constexpr int kMerge = WR < 4 ? kKeys * DP * 4 + 512 : 0;   // 4 warps x 16 rows of fp32, maxima, sums
  static constexpr int kTotal = kSmem > kMerge ? kSmem : kMerge;
};

template <int DP, int WR, bool KV8>
__global__ void __launch_bounds__(128) tree_attn_mma_kernel(const TreeAttnParams p) {
  using L = MmaShape<DP, WR, KV8>;
  constexpr int WK = 4 / WR;                // key groups
  constexpr int NKB = 8 / WK;               // 8-key blocks of a warp
  constexpr int ND = DP / 8, KSTEPS = DP / 16;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t s0 = smem_u32(smem);
  const uint32_t s_work = s0 + L::kStages * L::kStage, s_q = s_work + L::kWork;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wr = warp % WR, wk = warp / WR;
  griddep_launch();
  griddep_wait();
  // row tiles of one head next to one another: they share the keys in L2
  int idx = blockIdx.x;
  const int rt = idx % p.row_tiles; idx /= p.row_tiles;
  const int hk = idx % p.Hkv; idx /= p.Hkv;
  const int split = idx % p.splits, b = idx / p.splits;
  const int G = p.Hq / p.Hkv;
  const int next = next_start(p, b);
  const TreeSeq s = tree_seq(p, b);
  const int rows = s.q_len * G, row0 = rt * 16 * WR;
  if (p.zero_rest && split == 0 && rt == 0) zero_gap(p, s, next, b, hk * G * p.D, G * p.D, 128, threadIdx.x);
  const TreeTiles tt = tree_tiles(p, s);
  const int t0 = tt.lo + split * p.chunk, t1 = min(tt.hi, t0 + p.chunk);
  const int ntiles = t1 - t0;
  if (row0 >= rows || (ntiles <= 0 && split > 0)) return;
  const bool whole = tt.hi - tt.lo <= p.chunk;       // this CTA has all keys of the sequence
  const int* table = p.tables + b * p.table_stride;

  int r_tok[2], r_head[2], r_node[2];
  bool r_ok[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = row0 + wr * 16 + (lane >> 2) + 8 * h;
    r_ok[h] = r < rows;
    const int i = r_ok[h] ? r / G : 0;
    r_tok[h] = s.q_start + i;
    r_head[h] = hk * G + (r_ok[h] ? r % G : 0);
    r_node[h] = s.tree_len - s.q_len + i;
  }
  // Q: fragments straight from global memory, or (wide heads) staged once in the tiles' swizzled layout.
  uint32_t qf[L::kQShared ? 1 : KSTEPS][4];
  if constexpr (!L::kQShared) {
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = kk * 16 + 2 * (lane & 3);
        const __nv_bfloat16* qp = p.q + r_tok[h] * p.q_stride + r_head[h] * p.D + c;
        qf[kk][h] = r_ok[h] && c < p.D ? *reinterpret_cast<const uint32_t*>(qp) : 0u;
        qf[kk][2 + h] = r_ok[h] && c + 8 < p.D ? *reinterpret_cast<const uint32_t*>(qp + 8) : 0u;
      }
  } else {
    for (int x = threadIdx.x; x < 16 * WR * (DP / 8); x += 128) {
      const int r = x / (DP / 8), ch = x % (DP / 8);
      const int g = row0 + r;
      const bool ok = g < rows && ch * 8 < p.D;
      const __nv_bfloat16* qp = p.q + (s.q_start + (ok ? g / G : 0)) * p.q_stride + (hk * G + (ok ? g % G : 0)) * p.D + (ok ? ch * 8 : 0);
      cp_async16(s_q + r * DP * 2 + ((ch ^ (r & 7)) << 4), qp, ok);
    }
  }

  float o[ND][4];
#pragma unroll
  for (int i = 0; i < ND; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.0f, 0.0f};

#pragma unroll
  for (int st = 0; st < L::kStages - 1; ++st) {
    if (st < ntiles) {
      const uint32_t a = s0 + st * L::kStage;
      load_tile<DP, KV8>(a, a + L::kStage / 2, p, table, hk, (t0 + st) * kKeys, tt.lo_key, s.kv_len);
    }
    cp_async_commit();
  }
  for (int it = 0; it < ntiles; ++it) {
    const uint32_t stage = s0 + (it % L::kStages) * L::kStage;
    if (it + L::kStages - 1 < ntiles) {
      const uint32_t a = s0 + ((it + L::kStages - 1) % L::kStages) * L::kStage;
      load_tile<DP, KV8>(a, a + L::kStage / 2, p, table, hk, (t0 + it + L::kStages - 1) * kKeys, tt.lo_key, s.kv_len);
    }
    cp_async_commit();
    cp_async_wait<L::kStages - 1>();
    uint32_t sk = stage, sv = stage + L::kStage / 2;
    if constexpr (KV8) {                    // each thread expands what it loaded: only its own copies must have landed
      expand_tile<DP>(sk, s_work);
      expand_tile<DP>(sv, s_work + kKeys * DP * 2);
      sk = s_work;
      sv = s_work + kKeys * DP * 2;
    }
    __syncthreads();
    const int k0 = (t0 + it) * kKeys, wkey = wk * (kKeys / WK);

    float sc[NKB][4];
#pragma unroll
    for (int nb = 0; nb < NKB; ++nb) sc[nb][0] = sc[nb][1] = sc[nb][2] = sc[nb][3] = 0.0f;
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk) {
      uint32_t qx[4];
      if constexpr (L::kQShared) {
        const int r = wr * 16 + (lane & 15), ch = kk * 2 + (lane >> 4);
        ldsm4(qx, s_q + r * DP * 2 + ((ch ^ (r & 7)) << 4));
      }
      const uint32_t(&a)[4] = L::kQShared ? qx : qf[L::kQShared ? 0 : kk];
#pragma unroll
      for (int nb = 0; nb < NKB; nb += 2) {
        const int key = wkey + nb * 8 + ((lane >> 4) << 3) + (lane & 7), ch = kk * 2 + ((lane >> 3) & 1);
        uint32_t kb[4];
        ldsm4(kb, sk + key * DP * 2 + ((ch ^ (key & 7)) << 4));
        mma16816(sc[nb], a, kb[0], kb[1]);
        mma16816(sc[nb + 1], a, kb[2], kb[3]);
      }
    }
    // Tiles that lie wholly in every row's context are not masked.  In the others a masked key's weight is zero, and since
    // 0 times an infinity or a NaN is no zero, a tile whose values are not all finite is looked at key by key.
    const bool mixed = k0 + kKeys > s.base || (p.window > 0 && k0 <= s.base + s.tree_len - p.window);
    uint64_t see[2] = {~0ull, ~0ull};
    bool careful = false;
    if (mixed) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        see[h] = r_ok[h] ? tree_bits(p, s, b, r_node[h], k0) : 0ull;
#pragma unroll
        for (int nb = 0; nb < NKB; ++nb)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (!((see[h] >> (wkey + nb * 8 + 2 * (lane & 3) + e)) & 1)) sc[nb][2 * h + e] = -INFINITY;
      }
      uint32_t odd = 0;
      for (int x = threadIdx.x; x < kKeys * DP / 2; x += 128) {
        uint32_t w;
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(sv + x * 4));
        odd |= __vcmpeq2(w & 0x7F807F80u, 0x7F807F80u);
      }
      careful = __syncthreads_or(odd != 0);
    }
    float neg[2];
    float alpha[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float mx = -INFINITY;
#pragma unroll
      for (int nb = 0; nb < NKB; ++nb) mx = fmaxf(mx, fmaxf(sc[nb][2 * h], sc[nb][2 * h + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float m_new = fmaxf(m_run[h], mx * p.scale_log2);
      const float m_use = m_new == -INFINITY ? 0.0f : m_new;
      alpha[h] = exp2f(m_run[h] - m_use);
      m_run[h] = m_new;
      l_run[h] *= alpha[h];
      neg[h] = -m_use;
    }
    uint32_t pf[NKB / 2][4];
#pragma unroll
    for (int nb = 0; nb < NKB; ++nb) {
      float w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        w[e] = ex2(fmaf(sc[nb][e], p.scale_log2, neg[e >> 1]));
        l_run[e >> 1] += w[e];
      }
      // weights are rounded to bf16 for the tensor cores, their sum is not: 2^-8 of each weight, below the output's own
      // rounding once they are summed
      pf[nb >> 1][(nb & 1) * 2 + 0] = pack_bf16x2(w[0], w[1]);
      pf[nb >> 1][(nb & 1) * 2 + 1] = pack_bf16x2(w[2], w[3]);
    }
    if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        o[i][0] *= alpha[0]; o[i][1] *= alpha[0];
        o[i][2] *= alpha[1]; o[i][3] *= alpha[1];
      }
    }
    if (careful) {
      // Add what is not finite to the rows that see it, then take it out of the tile.
#pragma unroll
      for (int i = 0; i < ND; ++i)
        for (int key = wkey; key < wkey + kKeys / WK; ++key) {
          uint32_t w;
          asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(sv + key * DP * 2 + ((i ^ (key & 7)) << 4) + (lane & 3) * 4));
          if (!__vcmpeq2(w & 0x7F807F80u, 0x7F807F80u)) continue;
          const float2 v = unpack_bf16x2(w);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (!((see[h] >> key) & 1)) continue;
            if (!isfinite(v.x)) o[i][2 * h] += v.x;
            if (!isfinite(v.y)) o[i][2 * h + 1] += v.y;
          }
        }
      __syncthreads();
      for (int x = threadIdx.x; x < kKeys * DP / 2; x += 128) {
        uint32_t w;
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(sv + x * 4));
        w &= ~__vcmpeq2(w & 0x7F807F80u, 0x7F807F80u);
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(sv + x * 4), "r"(w) : "memory");
      }
      __syncthreads();
    }
#pragma unroll
    for (int ks = 0; ks < NKB / 2; ++ks)
#pragma unroll
      for (int db = 0; db < ND / 2; ++db) {
        const int key = wkey + ks * 16 + (((lane >> 3) & 1) << 3) + (lane & 7), ch = db * 2 + (lane >> 4);
        uint32_t vb[4];
        ldsm4_t(vb, sv + key * DP * 2 + ((ch ^ (key & 7)) << 4));
        mma16816(o[2 * db], pf[ks], vb[0], vb[1]);
        mma16816(o[2 * db + 1], pf[ks], vb[2], vb[3]);
      }
    __syncthreads();
  }
  cp_async_wait<0>();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 1);
    l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 2);
  }
  if constexpr (WK == 1) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (!r_ok[h]) continue;
      const float inv = l_run[h] != 0.0f ? 1.0f / l_run[h] : 0.0f;
      const long row = static_cast<long>(r_tok[h]) * p.Hq + r_head[h];
      __nv_bfloat16* op = p.out + r_tok[h] * p.out_stride + r_head[h] * p.D + 2 * (lane & 3);
      float* po = p.part_o + (split * p.part_rows + row) * p.D + 2 * (lane & 3);
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        if (i * 8 >= p.D) break;
        const float x = o[i][2 * h] * inv, y = o[i][2 * h + 1] * inv;
        if (whole) *reinterpret_cast<uint32_t*>(op + i * 8) = pack_bf16x2(x, y);
        else *reinterpret_cast<float2*>(po + i * 8) = make_float2(x, y);
      }
      if (!whole && (lane & 3) == 0)
        p.part_lse[split * p.part_rows + row] = l_run[h] != 0.0f ? m_run[h] + log2f(l_run[h]) : -INFINITY;
    }
  } else {
    // join the key groups through shared memory
    float* sO = reinterpret_cast<float*>(smem);           // [4 warps][16][DP]
    float* sM = sO + 4 * 16 * DP;
    float* sL = sM + 64;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<float2*>(sO + (warp * 16 + (lane >> 2) + 8 * h) * DP + i * 8 + 2 * (lane & 3)) =
            make_float2(o[i][2 * h], o[i][2 * h + 1]);
    if ((lane & 3) == 0)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        sM[warp * 16 + (lane >> 2) + 8 * h] = m_run[h];
        sL[warp * 16 + (lane >> 2) + 8 * h] = l_run[h];
      }
    __syncthreads();
    for (int x = threadIdx.x; x < 16 * WR * (DP / 4); x += 128) {
      const int r = x / (DP / 4), c = (x % (DP / 4)) * 4;
      const int g = row0 + r;
      if (g >= rows || c >= p.D) continue;
      float M = -INFINITY, l = 0.0f;
#pragma unroll
      for (int k = 0; k < WK; ++k) M = fmaxf(M, sM[(k * WR + r / 16) * 16 + r % 16]);
      const float use = M == -INFINITY ? 0.0f : M;
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int k = 0; k < WK; ++k) {
        const int at = (k * WR + r / 16) * 16 + r % 16;
        // a group that saw nothing has no say (and 0 times a value that is not finite must not come of it)
        if (sL[at] == 0.0f) continue;
        const float f = exp2f(sM[at] - use);
        const float4 v = *reinterpret_cast<const float4*>(sO + at * DP + c);
        l += f * sL[at];
        acc.x += f * v.x; acc.y += f * v.y; acc.z += f * v.z; acc.w += f * v.w;
      }
      const float inv = l != 0.0f ? 1.0f / l : 0.0f;
      const int tok = s.q_start + g / G, head = hk * G + g % G;
      if (whole) {
        *reinterpret_cast<uint2*>(p.out + tok * p.out_stride + head * p.D + c) =
            make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
      } else {
        const long row = split * p.part_rows + static_cast<long>(tok) * p.Hq + head;
        *reinterpret_cast<float4*>(p.part_o + row * p.D + c) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
        if (c == 0) p.part_lse[row] = l != 0.0f ? M + log2f(l) : -INFINITY;
      }
    }
  }
}


// ---------------------------------------------------------------------------------------------------------
// Many rows per KV head (a tree of 16 nodes with a group of 4 has 64): the same computation on tcgen05, over keys in tiles
// of 128 and row tiles of 128 (position, head-in-group) rows.
//
// Work split.  The batch's tiles (sequence, block of KV heads, key tile) form one line, cut into as many equal pieces as the
// GPU has groups of `heads x row_tiles` CTAs; the CTAs of a group take one KV head of the block and one row tile each
// over the same piece.  So the heads of a token, which lie next to one another in a page, are read at about the same time
// (DRAM rows are opened once), and K and V come from L2 for all row tiles but one.
// A piece ends anywhere in a sequence: a CTA has at most two segments that are not a whole (sequence,
// head), stores those in 32 bits with their log-sum, and a second kernel joins them.  Sequences of any mix of lengths keep
// every SM busy until the end, and the partial rows take 2 x 128 rows per CTA whatever the lengths.
//
// Fifteen warps:
//   0-7  softmax: two threads per row (a row is a lane of tensor memory, which two warps may read), 64 keys each, who tell
//        each other their maxima.  A thread reads its scores into registers and writes the weights as packed 16-bit
//        numbers over scores that both have read.  O is rescaled only when a row's maximum grew by more than 2^8 over the
//        one in use: weights then reach 2^8 at most, which the 32-bit sums do not mind.  bf16 caches take bf16 weights
//        (A and B of a product have one type): 2^-9 of a weight on average, of the largest too, which would be exactly 1
//        under its own maximum.  Against 64 bits the output is off by 2.3e-3 of its spread, 1.7e-3 of which is its own
//        rounding to bf16; the mma.sync kernel, whose maximum never lags, by 1.8e-3, and fp16 weights by 1.7e-3.
//   8-11 Q to shared memory, and what TMA cannot do: e4m3 tiles are expanded, and values that are no numbers are taken out
//        of V tiles with masked keys (0 times such a value is no zero), see `careful` below.
//   12   one thread issues S = Q K^T (both K-major) and O += P V (P from tensor memory, V as it lies: MN-major) as their
//        operands come in.
//   13, 14  TMA of K and of V, one box per piece of a page (the largest power of two of rows that divides the page size,
//        at most 128) and 128 bytes of columns; zeros come from outside the tensor for D that fills no box and for block
//        ids that are none.  K tiles are free again once their scores are there, long before the V tile of the same keys.
// Tensor memory: three score tiles (the next scores are there before this tile's weights are) and O.
//
// e4m3 caches are expanded to fp16, which holds every e4m3 value exactly and takes one conversion instruction per two
// values (bf16 took five).  Q is brought to fp16 by a power of two per row (2^-114 to 2^100), to a largest magnitude in
// [2^14, 2^15): 11 bits for the 8 of bf16, and elements under 2^-28 of their row's largest round to multiples of 2^-39 of
// it, far below what a sum of 32-bit products keeps.  The weights become fp16 as 2^7 times themselves: full 11 bits down to
// 2^-21 of the maximum.
// ---------------------------------------------------------------------------------------------------------
//
// Measured (B200, in the order of a program's calls): 64 sequences of up to 2048 keys, trees of up to 16, 32 / 8 heads of 128:
// 98 us (3.6 TB/s); 16 x 8192 keys, trees of 21, 64 / 8 heads: 211 us (2.6 TB/s, 428 TFLOP/s); one of 131072 keys, a tree of
// 64 (two row tiles): 212 us (2.5 TB/s, 646 TFLOP/s); 32 x 4096 keys of e4m3, trees of 13: 156 us.  One level of a tree, 8 rows
// of 21 nodes over 64 x 2048 keys: 113 us, e4m3 186 us (4 rows, on mma.sync: 162 and 210).  bf16 with one row tile is bound by
// memory in its steady state (a 64 KiB pair of tiles per SM and 1.76 us: 5.5 TB/s over the 148 SMs), by 7 to 9 us to its
// first weights and by the ends of its segments, some 2 us each; e4m3 by the expansion (1500 cycles of four warps a tile, two
// tiles a step).  Both 64-wide kernels spill 16 to 32 bytes, the 128-wide ones nothing.
// What was tried and lost, in the first case: cp.async instead of TMA (105 us), one softmax group with all 128 scores in
// registers (124 us: it spills, and spills miss an L1 of 28 KiB), two groups on alternate tiles with an O each (141 us: no
// room for a third score tile, so each waits for its own product).
constexpr int kTcKeys = 128;
constexpr int kTcThreads = 480;
constexpr int kMaxTcNodes = 256;

template <int DP, bool KV8>
struct TcShape {
  static constexpr int kPanels = DP / 64;
  static constexpr int kTile = kTcKeys * DP * 2;             // a K tile, a V tile, the Q tile (16-bit)
  static constexpr int kStages = (KV8 ? 2 : 3) * (128 / DP); // of K and of V
  static constexpr int kRawTile = KV8 ? kTcKeys * DP : 0;    // e4m3
  static constexpr int kRaw = kStages;
  static constexpr int kQOff = kStages * 2 * kTile;
  static constexpr int kRawOff = kQOff + kTile;
  static constexpr int kBars = kRawOff + kRaw * 2 * kRawTile;
  static constexpr int kWords = kBars + (DP == 64 ? 512 : 288);   // what a row's two threads tell [2][2][128], scan
  static constexpr int kTotal = kWords + 2048 + 80 + 512;    // Q's powers of two [4][128] bytes
  static constexpr int kTmem = 512;                          // 3 x 128 scores, DP of O
  static_assert(2 * kTotal > 228 * 1024, "one CTA per SM: it takes all of tensor memory");
  static_assert(kTotal <= 227 * 1024, "shared memory of a CTA");
};

__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
// Halves that are infinite or NaN as bf16, as 0xFFFF.
__device__ __forceinline__ uint32_t no_number(uint32_t w) { return __vcmpeq2(w & 0x7F807F80u, 0x7F807F80u); }
// Shared-memory offset of 16-byte column ch of row r in a bf16 tile of 64-column panels with the 128-byte swizzle.
__device__ __forceinline__ uint32_t tc_at(int r, int ch) {
  return (ch >> 3) * (kTcKeys * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
}


__device__ __forceinline__ void tmem_st_x8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// max(a, b, c) and the packed 32-bit pairs of sm_100.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  // volatile: kept in front of the next loads, whose registers it frees
  asm volatile("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ uint64_t pair(uint32_t lo, uint32_t hi) {
  uint64_t y;
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "r"(lo), "r"(hi));
  return y;
}
__device__ __forceinline__ float2 unpair(uint64_t x) {
  float2 y;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(y.x), "=f"(y.y) : "l"(x));
  return y;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t y;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(a), "l"(b), "l"(c));
  return y;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t y;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
  return y;
}

// Four e4m3 bytes -> four fp16 (exact; a NaN code becomes a NaN).
__device__ __forceinline__ void e4m3x4_to_f16x4(uint32_t w, uint32_t& lo01, uint32_t& hi23) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo01), "=r"(hi23)
      : "r"(w));
}

// Key tiles of one KV head of a sequence; none when it has no rows.
__device__ __forceinline__ int tc_tiles(const TreeSeq& s) { return s.q_len > 0 ? (s.kv_len + kTcKeys - 1) / kTcKeys : 0; }

// Sum over the block of v, and the sum of the threads in front of this one.
__device__ __forceinline__ int block_scan(int v, int* red, int* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) red[warp] = x;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) {
    if (w < warp) before += red[w];
    all += red[w];
  }
  __syncthreads();
  *total = all;
  return before + x - v;
}

// A piece of the line of tiles, walked segment by segment: tiles t0 .. t1 of (sequence b, head hk of this CTA).
struct TcWalk {
  int at, end, b, start, tiles;     // position, end of the piece; sequence, its first tile on the line, tiles of a block
  int hk, t0, t1;
  int sub;                          // this CTA's head of a block
  __device__ __forceinline__ bool next(const TreeAttnParams& p) {
    if (at >= end) return false;
    while (at >= start + tiles * p.blocks) {
      start += tiles * p.blocks;
      if (++b >= p.B) return false;
      tiles = tc_tiles(tree_seq(p, b));
    }
    const int off = at - start;
    const int block = off / tiles;
    t0 = off - block * tiles;
    hk = block * p.heads + sub;
    t1 = min(tiles, t0 + end - at);
    at += t1 - t0;
    return true;
  }
  __device__ __forceinline__ bool whole() const { return t1 - t0 == tiles; }
};

template <int DP, bool KV8>
__global__ void __launch_bounds__(kTcThreads, 1)
    tree_attn_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                        const __grid_constant__ TreeAttnParams p) {
  using L = TcShape<DP, KV8>;
  constexpr float kOffset = KV8 ? 7.0f : 0.0f;      // weights are 2^kOffset times themselves
  extern __shared__ __align__(1024) uint8_t smem_tiles[];     // (the swizzle goes by address bits)
  uint8_t* smem = smem_tiles;
  const uint32_t s_ring = smem_u32(smem), s_q = s_ring + L::kQOff;   // K tiles, V tiles, Q, raw K tiles, raw V tiles
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBars);
  // of K (v = 0) and V tiles: TMA has landed (raw tiles if e4m3), raw tile is free, expanded or cleaned, its product is done
  const auto full = [&](int v, int i) { return bars + v * L::kRaw + i; };
  const auto raw_empty = [&](int v, int i) { return bars + (2 + v) * L::kRaw + i; };
  const auto ready = [&](int v, int i) { return bars + 4 * L::kRaw + v * L::kStages + i; };
  const auto empty = [&](int v, int i) { return bars + 4 * L::kRaw + (2 + v) * L::kStages + i; };
  uint64_t* q_full = bars + 4 * L::kRaw + 4 * L::kStages;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_empty + 1;                   // [3], one per score tile
  uint64_t* p_full = s_full + 3;
  uint64_t* pv_done = p_full + 1;
  uint64_t* drained = pv_done + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  int* s_careful = reinterpret_cast<int*>(tmem_slot + 1);
  static_assert(L::kBars + (4 * L::kRaw + 4 * L::kStages + 8) * 8 + 8 <= L::kWords, "barriers");
  float* s_tell = reinterpret_cast<float*>(smem + L::kWords);       // [2][2][128]
  int* s_walk = reinterpret_cast<int*>(s_tell + 512);              // b, start
  int* red = s_walk + 2;                                            // [16]
  int8_t* s_power = reinterpret_cast<int8_t*>(s_tell + 532);       // [4][128]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int v = 0; v < 2; ++v) {
      for (int i = 0; i < L::kRaw; ++i) {
        mbar_init(full(v, i), 1);
        mbar_init(raw_empty(v, i), 4);
      }
      for (int i = 0; i < L::kStages; ++i) {
        mbar_init(ready(v, i), 128);
        mbar_init(empty(v, i), 1);
      }
    }
    for (int i = 0; i < 3; ++i) mbar_init(&s_full[i], 1);
    mbar_init(p_full, 256);
    mbar_init(pv_done, 1);
    mbar_init(q_full, 128);
    mbar_init(q_empty, 1);
    mbar_init(drained, 1);
    mbar_fence_init();
    *s_careful = 0;
  }
  griddep_wait();
  if (s_ring & 1023) {
    if (threadIdx.x == 0) status_set(kStatusBadIndex);
    return;
  }
  const int G = p.Hq / p.Hkv;
  const int rt = blockIdx.x % p.row_tiles, group = blockIdx.x / (p.row_tiles * p.heads);
  // the line of tiles: its length, then the sequence in which this piece begins
  int line = 0, per = 0;
  for (int pass = 0; pass < 2; ++pass) {
    int before = 0;
    for (int b0 = 0; b0 < p.B; b0 += kTcThreads) {
      const int b = b0 + threadIdx.x;
      const int mine = b < p.B ? tc_tiles(tree_seq(p, b)) * p.blocks : 0;
      int total;
      const int front = before + block_scan(mine, red, &total);
      if ((pass == 1 || p.B <= kTcThreads) && mine > 0) {
        if (pass == 0) per = (total + p.groups - 1) / p.groups;
        const int begin = group * per;
        if (begin >= front && begin < front + mine) {
          s_walk[0] = b;
          s_walk[1] = front;
        }
      }
      before += total;
    }
    line = before;
    per = max(1, (line + p.groups - 1) / p.groups);
    if (p.B <= kTcThreads) break;
  }
  TcWalk walk;
  walk.sub = blockIdx.x / p.row_tiles % p.heads;
  walk.at = group * per;
  walk.end = min(line, walk.at + per);
  if (walk.at >= line) return;                    // whole CTA, nothing allocated
  if (warp == 12) {
    tmem_alloc(tmem_slot, L::kTmem);
    tmem_relinquish();
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  // Not before the allocation: a successor that takes tensor memory ahead of its own wait must find this CTA served.
  griddep_launch();
  walk.b = s_walk[0];
  walk.start = s_walk[1];
  walk.tiles = tc_tiles(tree_seq(p, walk.b));
  const uint32_t tmem = *tmem_slot, tmem_o = tmem + 3 * kTcKeys;
  const int row0 = rt * 128;
  // the next segment that has rows in this CTA's row tile
  const auto step = [&](TcWalk& w) -> bool {
    while (w.next(p))
      if (row0 == 0 || row0 < tree_seq(p, w.b).q_len * G) return true;
    return false;
  };

  if (warp < 8) {
    const int half = warp >> 2, row = threadIdx.x & 127, r = row0 + row;
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;   // this warp's 32 lanes, in bits 16 and up
    int j = 0, told = 0;                          // tiles so far, over all segments; times the pairs have met
    // A row's two threads tell each other a value: their warps meet in a barrier of their own.
    const auto tell = [&](float x) -> float {
      float* at = s_tell + (told & 1) * 256;
      ++told;
      at[half * 128 + row] = x;
      tcgen05_fence_before();
      asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory");
      tcgen05_fence_after();
      return at[(half ^ 1) * 128 + row];
    };
    // A wait that gave up is in the status word and makes the others give up at once; every thread still walks all
    // segments to their end, because the pairs of warps meet on the way.
    for (int seg = 0; step(walk); ++seg) {
      // Lengths are read again where they are needed, rather than kept in registers through the loop.
      int mixed_from;                             // first tile with a key that some row does not see
      bool row_ok, warp_ok;                       // !warp_ok: no row of this warp is real, its lanes may hold anything
      {
        const TreeSeq s = tree_seq(p, walk.b);
        mixed_from = s.base / kTcKeys;
        row_ok = r < s.q_len * G;
        warp_ok = row0 + (warp & 3) * 32 < s.q_len * G;
      }
      float m_use = -INFINITY, l = 0.0f, scale = p.scale_log2;
#pragma unroll 1
      for (int t = walk.t0; t < walk.t1; ++t, ++j) {
        mbar_wait(&s_full[j % 3], (j / 3) & 1, kStatusMmaWaitTimeout);
        __syncwarp();
        tcgen05_fence_after();
        float alpha = 1.0f;
        if (warp_ok) {
          const uint32_t ts = tmem + (j % 3) * kTcKeys + lanes;
          uint32_t sc[2][32];
          tmem_ld_32x32b_x32(ts + half * 64, sc[0]);
          tmem_ld_32x32b_x32(ts + half * 64 + 32, sc[1]);
          if (KV8 && t == walk.t0) scale = p.scale_log2 * __int_as_float((127 - s_power[(seg & 3) * 128 + row]) << 23);
          tmem_ld_wait();
          if (t >= mixed_from) {
            const TreeSeq s = tree_seq(p, walk.b);
            const uint64_t see = row_ok ? tree_bits(p, s, walk.b, s.tree_len - s.q_len + r / G, t * kTcKeys + half * 64) : 0ull;
#pragma unroll
            for (int k = 0; k < 64; ++k)
              if (!((see >> k) & 1)) sc[k / 32][k % 32] = 0xff800000u;
            __syncwarp();
          }
          float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int k = 0; k < 32; k += 2)
#pragma unroll
            for (int c = 0; c < 2; ++c) top[c] = max3(top[c], __uint_as_float(sc[c][k]), __uint_as_float(sc[c][k + 1]));
          const float mine = fmaxf(top[0], top[1]);
          const float m_new = fmaxf(mine, tell(mine)) * scale;
          if (m_new > m_use + 8.0f || (m_use == -INFINITY && m_new > m_use)) {
            alpha = ex2(m_use - m_new);
            m_use = m_new;
            l *= alpha;
          }
          const float neg = m_use == -INFINITY ? 0.0f : kOffset - m_use;
          const uint64_t scale2 = pair(__float_as_uint(scale), __float_as_uint(scale));
          const uint64_t neg2 = pair(__float_as_uint(neg), __float_as_uint(neg));
          uint64_t sum[2] = {0, 0};
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const float2 e = unpair(fma2(pair(sc[c][2 * k], sc[c][2 * k + 1]), scale2, neg2));
              const float w0 = ex2(e.x), w1 = ex2(e.y);
              sum[k & 1] = add2(sum[k & 1], pair(__float_as_uint(w0), __float_as_uint(w1)));
              if constexpr (KV8) {
                const __half2 h = __floats2half2_rn(w0, w1);
                pk[k] = *reinterpret_cast<const uint32_t*>(&h);
              } else {
                pk[k] = pack_bf16x2(w0, w1);
              }
            }
            tmem_st_32x32b_x16(ts + half * 32 + c * 16, pk);
          }
          const float2 total = unpair(add2(sum[0], sum[1]));
          l += total.x + total.y;
        }
        // The last product must be in before O is touched, and before p_full moves on by one more phase.
        if (j > 0) {
          mbar_wait(pv_done, (j - 1) & 1, kStatusMmaWaitTimeout);
          __syncwarp();
          tcgen05_fence_after();
          if (t > walk.t0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
#pragma unroll 1
            for (int c = half * (DP / 2); c < (half + 1) * (DP / 2); c += 16) {   // half of the columns
              uint32_t x[16];
              tmem_ld_32x32b_x16(tmem_o + lanes + c, x);
              tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 16; ++k) x[k] = __float_as_uint(__uint_as_float(x[k]) * alpha);
              tmem_st_32x32b_x16(tmem_o + lanes + c, x);
            }
          }
        }
        tmem_st_wait();
        tcgen05_fence_before();
        mbar_arrive(p_full);
      }
      // ------------------------------------------------------------- the segment's rows, half of the columns a thread
      mbar_wait(pv_done, (j - 1) & 1, kStatusMmaWaitTimeout);
      __syncwarp();
      tcgen05_fence_after();
      if (!warp_ok) continue;
      const float sum = l + tell(l);
      const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
      const TreeSeq s = tree_seq(p, walk.b);
      const bool whole = walk.whole();
      const int node = s.tree_len - s.q_len + (row_ok ? r / G : 0);
      const int tok = s.q_start + (row_ok ? r / G : 0), head = walk.hk * G + (row_ok ? r % G : 0);
      const long part = blockIdx.x * 2l + (walk.t0 > 0 ? 0 : 1);
      if (row_ok && half == 0 && !whole)
        p.part_lse[part * 128 + row] = sum != 0.0f ? (m_use == -INFINITY ? 0.0f : m_use) + log2f(sum) - kOffset : -INFINITY;
      const bool careful = *reinterpret_cast<volatile int*>(s_careful) != 0;
#pragma unroll 1
      for (int c = half * (DP / 2); c < (half + 1) * (DP / 2) && c < p.D; c += 32) {
        uint32_t x[32];
        __syncwarp();
        tmem_ld_32x32b_x32(tmem_o + lanes + c, x);
        tmem_ld_wait();
        if (!row_ok) continue;
        float o[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = sum != 0.0f ? __uint_as_float(x[k]) * inv : 0.0f;
        if (careful) {
          const int* table = p.tables + walk.b * p.table_stride;
#pragma unroll 1
          for (int k0 = max(walk.t0, s.base / kTcKeys) * kTcKeys; k0 < walk.t1 * kTcKeys; k0 += 64) {
#pragma unroll 1
            for (uint64_t see = tree_bits(p, s, walk.b, node, k0); see; see &= see - 1) {
              const int key = k0 + __ffsll(static_cast<long long>(see)) - 1;
              const long slot = tree_slot(p, table, key, 0, s.kv_len);
              if (slot < 0) continue;
              const long at = (slot * p.Hkv + walk.hk) * p.D + c;
#pragma unroll
              for (int k = 0; k < 32; ++k) {
                if (c + k >= p.D) break;
                float v;
                if (KV8) {
                  const uint8_t code = static_cast<const uint8_t*>(p.v_cache)[at + k];
                  v = (code & 0x7F) == 0x7F ? __int_as_float(0x7fffffff) : 0.0f;
                } else {
                  v = __bfloat162float(static_cast<const __nv_bfloat16*>(p.v_cache)[at + k]);
                }
                if (!isfinite(v)) o[k] += v;
              }
            }
          }
        }
#pragma unroll
        for (int k = 0; k < 32; k += 8) {
          if (c + k >= p.D) break;
          if (whole) {
            *reinterpret_cast<uint4*>(p.out + tok * p.out_stride + head * p.D + c + k) =
                make_uint4(pack_bf16x2(o[k], o[k + 1]), pack_bf16x2(o[k + 2], o[k + 3]), pack_bf16x2(o[k + 4], o[k + 5]),
                           pack_bf16x2(o[k + 6], o[k + 7]));
          } else {                                // [D / 8][128 rows][8]: the lanes' 32 bytes lie next to one another
            float* po = p.part_o + (part * (p.D / 8) + (c + k) / 8) * 1024 + row * 8;
            *reinterpret_cast<float4*>(po) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
            *reinterpret_cast<float4*>(po + 4) = make_float4(o[k + 4], o[k + 5], o[k + 6], o[k + 7]);
          }
        }
      }
    }
  } else {
    bool alive = true;
    int j = 0;                                    // tiles so far, over all segments: the phases of every ring
    if (warp < 12) {
      // -------------------------------------------------------------- Q; expand / clean: warp w has keys and rows 32 w .. 32 w + 31
      const int w = warp - 8;
      TreeSeq s = tree_seq(p, walk.b);             // of the segment
      const auto put_q = [&](const TcWalk& wk, int seg) {
        constexpr int CH = DP / 8, PASS = 32 / CH, BATCH = CH;
        const int ch = lane % CH, rows = s.q_len * G;
        for (int i0 = 0; i0 < CH; i0 += BATCH) {
          uint4 v[BATCH];
#pragma unroll
          for (int i = 0; i < BATCH; ++i) {
            const int qr = w * 32 + (i0 + i) * PASS + lane / CH, gr = row0 + qr;
            v[i] = make_uint4(0, 0, 0, 0);
            const int tok = p.g_magic ? __umulhi(gr, p.g_magic) : gr;
            if (gr < rows && ch * 8 < p.D)
              v[i] = *reinterpret_cast<const uint4*>(p.q + (s.q_start + tok) * p.q_stride + (wk.hk * G + gr - tok * G) * p.D + ch * 8);
          }
#pragma unroll
          for (int i = 0; i < BATCH; ++i) {
            const int qr = w * 32 + (i0 + i) * PASS + lane / CH;
            if constexpr (KV8) {
              const float2 x0 = unpack_bf16x2(v[i].x), x1 = unpack_bf16x2(v[i].y), x2 = unpack_bf16x2(v[i].z), x3 = unpack_bf16x2(v[i].w);
              float top = fmaxf(fmaxf(fmaxf(fabsf(x0.x), fabsf(x0.y)), fmaxf(fabsf(x1.x), fabsf(x1.y))),
                                fmaxf(fmaxf(fabsf(x2.x), fabsf(x2.y)), fmaxf(fabsf(x3.x), fabsf(x3.y))));
#pragma unroll
              for (int o = CH / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
              // 2^e with top 2^e in [2^14, 2^15); rows of zeros, and rows with an infinity (which stays one), as they are
              const int ex = top > 0.0f && top < INFINITY ? max(-114, min(100, 14 - ilogbf(top))) : 0;
              const float up = __int_as_float((ex + 127) << 23);
              if (ch == 0) s_power[(seg & 3) * 128 + qr] = static_cast<int8_t>(ex);
              const __half2 h0 = __floats2half2_rn(x0.x * up, x0.y * up), h1 = __floats2half2_rn(x1.x * up, x1.y * up);
              const __half2 h2 = __floats2half2_rn(x2.x * up, x2.y * up), h3 = __floats2half2_rn(x3.x * up, x3.y * up);
              v[i] = make_uint4(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1),
                                *reinterpret_cast<const uint32_t*>(&h2), *reinterpret_cast<const uint32_t*>(&h3));
            }
            sts128(s_q + tc_at(qr, ch), v[i].x, v[i].y, v[i].z, v[i].w);
          }
        }
        fence_proxy_async_smem();
        mbar_arrive(q_full);
      };
      // V values that are no numbers must not meet a weight of zero: they are taken out of tiles with masked keys, and the
      // rows that do see such a key get it back at the end (s_careful).
      const auto clean = [&](int t) {              // V tile j, the segment's tile t
        constexpr int CH = DP / 8, PASS = 32 / CH;
        const int st = j % L::kStages;
        if (!__all_sync(0xffffffffu, mbar_wait(full(1, st), (j / L::kStages) & 1, kStatusTmaWaitTimeout))) return false;
        if ((t + 1) * kTcKeys > s.base) {
          const uint32_t sv = s_ring + (L::kStages + st) * L::kTile;
          for (int i = 0; i < CH; ++i) {
            const int key = w * 32 + i * PASS + lane / CH;
            const uint32_t at = sv + tc_at(key, lane % CH);
            const uint4 v = lds128(at);
            const uint32_t m0 = no_number(v.x), m1 = no_number(v.y), m2 = no_number(v.z), m3 = no_number(v.w);
            if (m0 | m1 | m2 | m3) {
              sts128(at, v.x & ~m0, v.y & ~m1, v.z & ~m2, v.w & ~m3);
              // (behind the last key lies whatever the ring held before)
              if (t * kTcKeys + key < s.kv_len) *reinterpret_cast<volatile int*>(s_careful) = 1;
            }
          }
          fence_proxy_async_smem();
        }
        mbar_arrive(ready(1, st));
        return true;
      };
      const auto widen = [&](int v, int n, int keys) -> bool {       // tile n of K (v = 0) or V; keys: clean it, it has so many
        constexpr int CH = DP / 16, PASS = 32 / CH, BATCH = CH;
        const int ch = lane % CH, sub = lane / CH;
        const int first = (ch >> 2) & 1;           // columns 2 ch and 2 ch + 1, in the order that spreads over the banks
        const int st = n % L::kStages, rs = n % L::kRaw;
        bool ok = mbar_wait(full(v, rs), (n / L::kRaw) & 1, kStatusTmaWaitTimeout);
        if (n >= L::kStages) ok = ok && mbar_wait(empty(v, st), ((n / L::kStages) & 1) ^ 1, kStatusEmptyWaitTimeout);
        if (!__all_sync(0xffffffffu, ok)) return false;
        const uint32_t from = s_ring + L::kRawOff + (v * L::kRaw + rs) * L::kRawTile + (w * 32 + sub) * DP + ch * 16;
        const uint32_t to = s_ring + (v * L::kStages + st) * L::kTile;
#pragma unroll
        for (int i0 = 0; i0 < CH; i0 += BATCH) {
          uint4 x[BATCH];
#pragma unroll
          for (int i = 0; i < BATCH; ++i) x[i] = lds128(from + (i0 + i) * PASS * DP);
#pragma unroll
          for (int i = 0; i < BATCH; ++i) {
            const int row = w * 32 + (i0 + i) * PASS + sub;
            uint32_t o[8];
            e4m3x4_to_f16x4(x[i].x, o[0], o[1]);
            e4m3x4_to_f16x4(x[i].y, o[2], o[3]);
            e4m3x4_to_f16x4(x[i].z, o[4], o[5]);
            e4m3x4_to_f16x4(x[i].w, o[6], o[7]);
            if (keys) {
              uint32_t had = 0;
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const uint32_t nan = __vcmpeq2(o[k] & 0x7C007C00u, 0x7C007C00u);
                had |= nan;
                o[k] &= ~nan;
              }
              if (had && row < keys) *reinterpret_cast<volatile int*>(s_careful) = 1;   // (behind the last key lies anything)
            }
            const uint32_t at0 = to + tc_at(row, 2 * ch + first), at1 = to + tc_at(row, 2 * ch + 1 - first);
            sts128(at0, first ? o[4] : o[0], first ? o[5] : o[1], first ? o[6] : o[2], first ? o[7] : o[3]);
            sts128(at1, first ? o[0] : o[4], first ? o[1] : o[5], first ? o[2] : o[6], first ? o[3] : o[7]);
          }
        }
        fence_proxy_async_smem();
        mbar_arrive(ready(v, st));
        __syncwarp();
        if (lane == 0) mbar_arrive(raw_empty(v, rs));
        return true;
      };
      for (int seg = 0; alive && step(walk); ++seg) {
        // Q is one tile: the scores that read the last one must be there
        if (seg > 0) alive = __all_sync(0xffffffffu, mbar_wait(q_empty, (seg - 1) & 1, kStatusMmaWaitTimeout));
        if (!alive) break;
        s = tree_seq(p, walk.b);
        put_q(walk, seg);
        for (int t = walk.t0; t < walk.t1 && alive; ++t, ++j) {
          if constexpr (KV8) {                     // K a tile ahead of V, as the scores are ahead of the products
            const int keys = s.kv_len - (t - 1) * kTcKeys;
            alive = widen(0, j, 0) && (t == walk.t0 || widen(1, j - 1, t * kTcKeys > s.base ? keys : 0));
          } else {
            alive = clean(t);
          }
        }
        if constexpr (KV8) {
          const int keys = s.kv_len - (walk.t1 - 1) * kTcKeys;
          if (alive) alive = widen(1, j - 1, walk.t1 * kTcKeys > s.base ? keys : 0);
        }
      }
    } else if (warp == 13 || warp == 14) {
      // -------------------------------------------------------------- TMA: K (warp 13), V (warp 14)
      const int v = warp - 13;
      constexpr int PANELS = KV8 ? 1 : L::kPanels; // boxes of 128 bytes of columns (e4m3: the whole head)
      constexpr int PANEL_COLS = KV8 ? DP : 64, ROW = KV8 ? DP : 128;
      const CUtensorMap* map = v ? &map_v : &map_k;
      uint64_t* freed = KV8 ? raw_empty(v, 0) : empty(v, 0);
      uint8_t* ring = smem + (KV8 ? L::kRawOff + v * L::kRaw * L::kRawTile : v * L::kStages * L::kTile);
      const int box = p.box_rows, nowhere = p.num_blocks * p.page;
      while (alive && step(walk)) {
        const int* table = p.tables + walk.b * p.table_stride;
        const int kv_len = tree_seq(p, walk.b).kv_len;
        for (int t = walk.t0; t < walk.t1; ++t, ++j) {
          const int st = j % L::kRaw;
          if (j >= L::kRaw) {
            alive = __all_sync(0xffffffffu, mbar_wait(&freed[st], ((j / L::kRaw) & 1) ^ 1, kStatusEmptyWaitTimeout));
            if (!alive) break;
          }
          const int k0 = t * kTcKeys;
          const int pieces = (min(kTcKeys, kv_len - k0) + box - 1) / box;
          if (lane == 0) mbar_expect_tx(full(v, st), pieces * box * ROW * PANELS);
          __syncwarp();
          for (int x = lane; x < pieces * PANELS; x += 32) {
            const int gp = x / PANELS, pn = x % PANELS;
            const int key = k0 + gp * box, blk = p.page_shift >= 0 ? key >> p.page_shift : key / p.page;
            const int id = table[blk];
            int at = nowhere;                      // outside the tensor: zeros
            if (static_cast<unsigned>(id) < static_cast<unsigned>(p.num_blocks)) at = id * p.page + (key - blk * p.page);
            else status_set(kStatusBadIndex);
            tma_load_3d(ring + st * (KV8 ? L::kRawTile : L::kTile) + pn * (kTcKeys * 128) + gp * box * ROW, map, full(v, st),
                        pn * PANEL_COLS, walk.hk, at);
          }
        }
      }
      if (!alive)                                  // nothing may land in this CTA's shared memory after it has gone
        for (int i = max(0, j - L::kRaw); i < j; ++i)
          mbar_wait(full(v, i % L::kRaw), (i / L::kRaw) & 1, kStatusTmaWaitTimeout);
    } else if (warp == 12 && lane == 0) {
      // -------------------------------------------------------------- the MMAs
      constexpr uint32_t kind = KV8 ? ~((1u << 7) | (1u << 10)) : ~0u;     // operands fp16 or bf16
      constexpr uint32_t idesc_s = umma_idesc_bf16(128, kTcKeys) & kind, idesc_o = umma_idesc_bf16(128, DP, 0, 1) & kind;
      const auto has = [&](uint64_t* bar, int n) { return mbar_test(&bar[n % L::kStages], (n / L::kStages) & 1); };
      uint64_t* k_in = KV8 ? ready(0, 0) : full(0, 0);
      int seg = -1, left = 0, o = 0;               // j: next tile of scores; o: next tile of the products
      uint32_t fresh = 0;                          // bit n % 4: tile n is the first of its segment
      bool more = true;
      const auto advance = [&]() {                 // to the next tile in line
        if (left == 0) {
          more = step(walk);
          left = walk.t1 - walk.t0;
          ++seg;
        }
      };
      advance();
      uint64_t since = 0;
      for (uint32_t it = 0; more || o < j;) {
        bool moved = false;
        // scores of tile j go where tile j - 3 had its weights
        if (more && j < o + 3 && (j < 3 || mbar_test(pv_done, (j - 3) & 1) || o > j - 2) &&
            (left < walk.t1 - walk.t0 || mbar_test(q_full, seg & 1)) && has(k_in, j)) {
          tcgen05_fence_after();
          const int st = j % L::kStages;
          const uint32_t sk = s_ring + st * L::kTile;
#pragma unroll
          for (int k = 0; k < DP / 16; ++k)        // 16 columns: 32 bytes within a panel
            umma_bf16(tmem + (j % 3) * kTcKeys, umma_desc_k_sw128(s_q + (k / 4) * (kTcKeys * 128)) + 2 * (k % 4),
                      umma_desc_k_sw128(sk + (k / 4) * (kTcKeys * 128)) + 2 * (k % 4), idesc_s, k != 0);
          umma_commit(&s_full[j % 3]);
          umma_commit(empty(0, st));
          fresh = (fresh & ~(1u << (j & 3))) | (left == walk.t1 - walk.t0 ? 1u << (j & 3) : 0u);
          ++j;
          if (--left == 0) umma_commit(q_empty);
          advance();
          moved = true;
        }
        if (o < j && mbar_test(p_full, o & 1) && has(ready(1, 0), o)) {
          tcgen05_fence_after();
          const int st = o % L::kStages;
          const uint32_t sv = s_ring + (L::kStages + st) * L::kTile;
#pragma unroll
          for (int k = 0; k < kTcKeys / 16; ++k)   // 16 keys: two groups of eight 128-byte rows; panels of 64 columns apart
            umma_bf16_ts(tmem_o, tmem + (o % 3) * kTcKeys + k * 8, umma_desc_mn_sw128(sv + k * 2048, kTcKeys * 128), idesc_o,
                         k != 0 || !((fresh >> (o & 3)) & 1));
          umma_commit(empty(1, st));
          umma_commit(pv_done);
          ++o;
          moved = true;
        }
        if (moved) {
          it = 0;
          since = 0;
        } else if ((++it & 63u) == 0u) {           // bounded as every wait: by polls, by time, by an earlier failure
          const uint64_t now = globaltimer_ns();
          if (since == 0) since = now | 1ull;
          if (it > AFB_SPIN_LIMIT || static_cast<int64_t>(now - since) > static_cast<int64_t>(AFB_LOCAL_WAIT_NS) ||
              (status_peek() & kStatusAnyWaitTimeout)) {
            status_set(kStatusTmaWaitTimeout);
            alive = false;
            break;
          }
        }
      }
      if (!alive) {                                // let what was issued finish before tensor memory is given back
        umma_commit(drained);
        mbar_wait(drained, 0, kStatusMmaWaitTimeout);
      }
    }
  }
  __syncwarp();
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 12) {
    tcgen05_fence_after();
    tmem_dealloc(tmem, L::kTmem);
  }
}

// Joins the (sequence, head)s of the kernel above that lie on several pieces of the line.  A thread takes eight columns of
// rows of one sequence; the sequence's place on the line is summed up by the block.  It has the zeros of the rows that no
// sequence has, too.
__global__ void __launch_bounds__(256) tree_attn_tc_join_kernel(const __grid_constant__ TreeAttnParams p) {
  __shared__ int red[8];
  griddep_launch();
  griddep_wait();
  const int b = blockIdx.y;
  const int next = next_start(p, b);
  const TreeSeq s = tree_seq(p, b);
  __shared__ int s_start;
  int start = 0, line = 0;
  for (int b0 = 0; b0 < p.B; b0 += 256) {
    const int c = b0 + threadIdx.x;
    const int mine = c < p.B ? tc_tiles(tree_seq(p, c)) * p.blocks : 0;
    int total;
    const int front = line + block_scan(mine, red, &total);
    if (c == b) s_start = front;
    line += total;
  }
  __syncthreads();
  start = s_start;
  const int per = max(1, (line + p.groups - 1) / p.groups);
  if (p.zero_rest) zero_gap(p, s, next, b, 0, p.Hq * p.D, gridDim.x * 256, blockIdx.x * 256 + threadIdx.x);
  const int tiles = tc_tiles(s), G = p.Hq / p.Hkv, chunks = p.D / 8;
  for (int y = blockIdx.x * 256 + threadIdx.x; y < s.q_len * p.Hq * chunks; y += gridDim.x * 256) {
    const int x = y / chunks, ch = y - x * chunks;
    const int i = x / p.Hq, head = x - i * p.Hq, hk = head / G, r = i * G + head - hk * G, rt = r / 128;
    const int u0 = start + hk / p.heads * tiles, c0 = u0 / per, c1 = (u0 + tiles - 1) / per;
    if (c0 == c1) continue;                        // stored whole
    const auto part = [&](int c) { return ((static_cast<long>(c) * p.heads + hk % p.heads) * p.row_tiles + rt) * 2 + (c == c0 ? 1 : 0); };
    float M = -INFINITY;
#pragma unroll 8
    for (int c = c0; c <= c1; ++c) M = fmaxf(M, p.part_lse[part(c) * 128 + (r & 127)]);
    const float use = M == -INFINITY ? 0.0f : M;
    float acc[8] = {}, l = 0.0f;
#pragma unroll 4
    for (int c = c0; c <= c1; ++c) {
      const float lse = p.part_lse[part(c) * 128 + (r & 127)];
      const float* po = p.part_o + (part(c) * chunks + ch) * 1024 + (r & 127) * 8;
      const float4 v0 = *reinterpret_cast<const float4*>(po), v1 = *reinterpret_cast<const float4*>(po + 4);
      const float f = ex2(lse - use);              // (a row that saw nothing there: zeros and -inf)
      l += f;
      acc[0] += f * v0.x; acc[1] += f * v0.y; acc[2] += f * v0.z; acc[3] += f * v0.w;
      acc[4] += f * v1.x; acc[5] += f * v1.y; acc[6] += f * v1.z; acc[7] += f * v1.w;
    }
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    *reinterpret_cast<uint4*>(p.out + (s.q_start + i) * p.out_stride + head * p.D + ch * 8) =
        make_uint4(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv),
                   pack_bf16x2(acc[4] * inv, acc[5] * inv), pack_bf16x2(acc[6] * inv, acc[7] * inv));
  }
}

// Joins the chunks of a sequence that has more than one: o = sum_c 2^(lse_c - max) o_c / sum_c 2^(lse_c - max).  A thread
// takes four columns of a row.  Chunks in which a row saw nothing hold zeros and a log-sum of -inf, so that no branch stands
// between the loads of different chunks.
__global__ void __launch_bounds__(128) tree_attn_join_kernel(const TreeAttnParams p) {
  griddep_launch();
  griddep_wait();
  const int b = blockIdx.y;
  const TreeSeq s = tree_seq(p, b);
  const TreeTiles tt = tree_tiles(p, s);
  const int n = (tt.hi - tt.lo + p.chunk - 1) / p.chunk, chunks = p.D / 4;
  const int y = blockIdx.x * 128 + threadIdx.x, x = y / chunks, d = (y - x * chunks) * 4;
  if (n <= 1 || x >= s.q_len * p.Hq) return;
  const long row = static_cast<long>(s.q_start) * p.Hq + x;
  float M = -INFINITY;
#pragma unroll 8
  for (int c = 0; c < n; ++c) M = fmaxf(M, p.part_lse[c * p.part_rows + row]);
  const float use = M == -INFINITY ? 0.0f : M;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float l = 0.0f;
#pragma unroll 8
  for (int c = 0; c < n; ++c) {
    const float f = ex2(p.part_lse[c * p.part_rows + row] - use);
    const float4 v = *reinterpret_cast<const float4*>(p.part_o + (c * p.part_rows + row) * p.D + d);
    l += f;
    acc.x += f * v.x; acc.y += f * v.y; acc.z += f * v.z; acc.w += f * v.w;
  }
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;
  *reinterpret_cast<uint2*>(p.out + (row / p.Hq) * p.out_stride + (row % p.Hq) * p.D + d) =
      make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
}

// How many 64-key tiles a CTA takes.  Every CTA costs about one tile's time besides its tiles (filling its ring, storing
// its rows), and CTAs run in waves of `slots`: the number of chunks with the least total is taken.
inline int pick_chunk(long units, int tiles, int slots) {
  if (tiles < 1) return 1;
  long best = -1;
  int chunk = tiles;
  for (int s = 1; s <= 64 && s <= tiles; ++s) {
    const int c = (tiles + s - 1) / s;
    const long n = (tiles + c - 1) / c;
    const long cost = (units * n + slots - 1) / slots * (c + 1) + (n > 1 ? 2 : 0);
    if (best < 0 || cost < best) { best = cost; chunk = c; }
  }
  return chunk;
}

// Which kernel takes a call.  The tcgen05 one needs pages that TMA can bring, 16-byte rows, no window, and enough work to
// pay for its start (locating its piece, Q, the first tile: some 9 us, e4m3 a few more) and for its join.  Work is counted
// in (row, key, KV head) triples at D = 128.  It also has a fixed cost for every (sequence, head) that a CTA comes to, which
// up to 64 rows, one row tile of the other kernel, takes several tiles of keys to pay for.  Measured, mma.sync against
// tcgen05 in us, cold, replayed from a graph, Hkv = 8, D = 128 (* where the rule takes the slower one):
//   bf16   1 x 8192, 128 rows (8 M): 43 / 49       1 x 32768, 64 rows (17 M): 68 / 68    1 x 8192, 256 rows (17 M): 64 / 43
//          4 x 1000, 128 rows (4 M): 33 / 35       4 x 4000, 32 rows (4 M): 41 / 39 *    4 x 1000, 256 rows (8 M): 45 / 37
//          16 x 500, 20 rows (1 M): 27 / 27        16 x 500, 64 rows (4 M): 33 / 29      16 x 2000, 20 rows (5 M): 61 / 51
//          64 x 250, 64 rows (8 M): 51 / 64        64 x 250, 128 rows (16 M): 90 / 77    64 x 500, 20 rows (5 M): 59 / 61 *
//          64 x 1000, 20 rows (10 M): 102 / 80     64 x 2000, 64 rows (66 M): 246 / 131  200 x 500, 64 rows (51 M): 209 / 172
//   e4m3   1 x 8192, 128 rows (8 M): 47 / 64       1 x 32768, 64 rows (17 M): 76 / 84    1 x 8192, 256 rows (17 M): 76 / 61
//          4 x 4000, 64 rows (8 M): 45 / 53        4 x 4000, 128 rows (16 M): 78 / 56    16 x 500, 128 rows (8 M): 49 / 49
//          16 x 2000, 32 rows (8 M): 72 / 76       16 x 2000, 48 rows (12 M): 80 / 75 *  64 x 250, 128 rows (16 M): 103 / 113 *
//          1 x 65536, 20 rows (10 M): 113 / 107    4 x 8192, 64 rows (17 M): 78 / 78     8 x 8192, 20 rows (10 M): 125 / 110
//          64 x 500, 64 rows (16 M): 90 / 113      64 x 500, 128 rows (33 M): 160 / 127  64 x 1000, 32 rows (16 M): 129 / 127
//          64 x 2000, 20 rows (20 M): 242 / 182    200 x 500, 64 rows (51 M): 240 / 291  200 x 500, 128 rows (102 M): 453 / 307
// Few (sequence, head)s favour mma.sync, whose chunks of 64 keys spread them over more CTAs with less to begin with.  On
// e4m3 both times go by the keys alone up to 64 rows: mma.sync has its one row tile, tcgen05 its expansion.
inline bool use_tc(long units, int rows, int D, int kv8, int window, int page, int max_kv) {
  if (window > 0 || D > 128 || (kv8 && D % 16) || page % 8 || rows <= 16) return false;
  const double work = static_cast<double>(units) * rows * max_kv * D / 128;
  if (kv8) return rows > 64 ? work >= 16e6 : max_kv >= 1000 && work >= 4e5 * rows;
  return (rows > 64 || max_kv >= 500) && work >= (units < 32 ? 14e6 : units < 128 ? 5e6 : 2e6);
}

template <int DP, bool KV8>
int launch_tc(TreeAttnParams& p, long ctas, cudaStream_t stream) {
  using L = TcShape<DP, KV8>;
  auto kernel = tree_attn_tc_kernel<DP, KV8>;
  AFB_CONFIGURE_KERNEL(kernel, L::kTotal, kTcThreads, L::kTmem);
  p.box_rows = 8;
  while (p.box_rows < kTcKeys && p.page % (2 * p.box_rows) == 0) p.box_rows *= 2;
  CUtensorMap mk, mv;
  const uint64_t el = KV8 ? 1 : 2, head = p.D * el, row = head * p.Hkv, slots = static_cast<uint64_t>(p.num_blocks) * p.page;
  const uint32_t cols = KV8 ? DP : 64;
  if (make_tmap_3d(&mk, p.k_cache, el, p.D, p.Hkv, slots, head, row, cols, 1, p.box_rows, KV8 ? 0 : 3) ||
      make_tmap_3d(&mv, p.v_cache, el, p.D, p.Hkv, slots, head, row, cols, 1, p.box_rows, KV8 ? 0 : 3))
    return -1;
  AFB_CHECK_CUDA(launch_pdl(kernel, dim3(static_cast<unsigned>(ctas)), dim3(kTcThreads), L::kTotal, stream, mk, mv, p));
  return 0;
}

template <int DP, int WR, bool KV8>
int launch_mma(const TreeAttnParams& p, long ctas, cudaStream_t stream) {
  using L = MmaShape<DP, WR, KV8>;
  auto kernel = tree_attn_mma_kernel<DP, WR, KV8>;
  AFB_CONFIGURE_KERNEL(kernel, L::kTotal, 128, 0);
  AFB_CHECK_CUDA(launch_pdl(kernel, dim3(static_cast<unsigned>(ctas)), dim3(128), L::kTotal, stream, p));
  return 0;
}
template <int DP, bool KV8>
int launch_mma(const TreeAttnParams& p, int wr, long ctas, cudaStream_t stream) {
  return wr == 1 ? launch_mma<DP, 1, KV8>(p, ctas, stream)
                 : wr == 2 ? launch_mma<DP, 2, KV8>(p, ctas, stream) : launch_mma<DP, 4, KV8>(p, ctas, stream);
}

// A window that reaches the first key of the longest sequence masks nothing: positions lie below max_kv.
inline int real_window(int window, int max_kv) { return window > 0 && window < max_kv ? window : 0; }

// Sizes of a launch: what follows from the shapes alone, so that the caller can provide the partial rows.
struct TreeLaunch {
  bool tc;
  int wr, row_tiles, splits, chunk, groups, heads;
  long part_rows, scratch;   // rows and floats of the partial rows
};
inline TreeLaunch tree_launch(int B, int T, int Hq, int Hkv, int D, int kv8, int page, int nodes, int window, int max_q_len,
                              int max_kv) {
  TreeLaunch t = {};
  const int rows = max_q_len * (Hq / Hkv);
  t.tc = use_tc(static_cast<long>(B) * Hkv, rows, D, kv8, window, page, max_kv);
  t.splits = t.chunk = t.groups = t.heads = 1;
  if (t.tc) {
    t.row_tiles = (rows + 127) / 128;
    // The largest block of at most eight heads (2 KiB of a token in bf16 at D = 128) that leaves no more than one in
    // sixteen of the SMs without a CTA; one head where there is none.
    const int sms = device_sm_count();
    t.heads = 1;
    for (int h = 2; h <= 8; ++h)
      if (Hkv % h == 0 && sms / (h * t.row_tiles) * h * t.row_tiles >= sms - sms / 16) t.heads = h;
    const long line = static_cast<long>(B) * (Hkv / t.heads) * ((max_kv + kTcKeys - 1) / kTcKeys);
    const long most = sms / (t.row_tiles * t.heads);
    t.groups = static_cast<int>(line < most ? line : most);
    if (t.groups < 1) t.groups = 1;
    t.part_rows = static_cast<long>(t.groups) * t.heads * t.row_tiles * 2 * 128;
    t.scratch = t.part_rows * (D + 1);
    return t;
  }
  t.wr = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  t.row_tiles = rows > 0 ? (rows + 16 * t.wr - 1) / (16 * t.wr) : 1;
  const long reach = window > 0 ? static_cast<long>(window) + nodes + 63 : max_kv;     // (64 bits: the sum may pass 2^31)
  const int tiles = static_cast<int>(reach < max_kv ? reach : max_kv) / kKeys + 1;
  t.chunk = pick_chunk(static_cast<long>(B) * Hkv * t.row_tiles, tiles, device_sm_count() * (D <= 64 ? 3 : D <= 128 ? 2 : 1));
  t.splits = (tiles + t.chunk - 1) / t.chunk;
  t.part_rows = static_cast<long>(T) * Hq;
  t.scratch = t.splits > 1 ? t.splits * t.part_rows * (D + 1) : 0;
  return t;
}

}  // namespace afb

extern "C" {

// Floats of scratch that afb_tree_attention needs for these sizes.
long afb_tree_attention_scratch(int B, int T, int Hq, int Hkv, int D, int kv8, int page, int nodes, int window,
                                int max_q_len, int max_kv) {
  using namespace afb;
  if (B <= 0 || Hkv <= 0 || Hq < Hkv || page <= 0 || max_q_len < 0 || max_kv < 0) return 0;
  return tree_launch(B, T, Hq, Hkv, D, kv8, page, nodes, real_window(window, max_kv), max_q_len, max_kv).scratch;
}

int afb_tree_attention(const void* q, long q_stride, const void* k_cache, const void* v_cache, int kv8, int num_blocks,
                       int page, const int* tables, long table_stride, int max_blocks, const int* q_starts,
                       const int* q_lens, const int* kv_lens, const int* tree_lens, const int* masks, long mask_stride,
                       int nodes, int words, const int* depths, long depth_stride, void* out, long out_stride, int B,
                       int T, int Hq, int Hkv, int D, int max_q_len, int max_kv, int window, int zero_rest, float scale,
                       float* scratch, long scratch_floats, cudaStream_t stream) {
  using namespace afb;
  if (B <= 0 || T <= 0) return 0;
  if (D < 8 || D > 256 || D % 8 || Hkv <= 0 || Hq % Hkv || page <= 0 || nodes < 1 || nodes > kMaxTcNodes ||
      words != (nodes + 31) / 32 || (window > 0 && !depths) || B > 65535 || static_cast<long>(max_q_len) * (Hq / Hkv) > 65535 || max_q_len < 0 || max_kv < 0 ||
      static_cast<long>(num_blocks) * page > 0x7fffffffl) {
    set_last_error("afb_tree_attention: bad arguments (B=%d Hq=%d Hkv=%d D=%d blocks=%d page=%d nodes=%d words=%d window=%d)",
                   B, Hq, Hkv, D, num_blocks, page, nodes, words, window);
    return -1;
  }
  // Masked scores are -inf before they are scaled and maxima are taken before it too, so the scale has to be positive; it
  // stays a normal number after the e4m3 path's powers of two, 2^-100 to 2^114.
  if (!(scale >= 0.99e-7f && scale <= 1.01e4f)) {
    set_last_error("afb_tree_attention: the scale is a positive number from 1e-7 to 1e4, not %g", static_cast<double>(scale));
    return -1;
  }
  const auto odd = [](const void* x, int to) { return (reinterpret_cast<uintptr_t>(x) & (to - 1)) != 0; };
  if (odd(q, 16) || odd(out, 16) || odd(k_cache, 16) || odd(v_cache, 16) || odd(scratch, 16) || q_stride % 8 || out_stride % 8) {
    set_last_error("afb_tree_attention: q, out and the caches start on 16 bytes, token strides are multiples of 8 elements");
    return -1;
  }
  window = real_window(window, max_kv);
  const TreeLaunch t = tree_launch(B, T, Hq, Hkv, D, kv8, page, nodes, window, max_q_len, max_kv);
  const long ctas = t.tc ? static_cast<long>(t.groups) * t.heads * t.row_tiles : static_cast<long>(B) * t.splits * Hkv * t.row_tiles;
  // tiles are counted in 32 bits on the device
  const long line = (static_cast<long>(max_blocks) * page / kKeys + 1) * B * Hkv;
  if (t.scratch > scratch_floats || (t.scratch && !scratch) || ctas > 0x7fffffffl || line > 0x7fffffffl) {
    set_last_error("afb_tree_attention: %ld floats of scratch are needed, %ld given (or too many tiles: %ld)", t.scratch,
                   scratch_floats, line);
    return -1;
  }
  TreeAttnParams p{static_cast<const __nv_bfloat16*>(q), q_stride, k_cache, v_cache, tables, table_stride, max_blocks, page,
                   num_blocks, q_starts, q_lens, kv_lens, tree_lens, masks, mask_stride, nodes, words, depths, depth_stride,
                   static_cast<__nv_bfloat16*>(out), out_stride, T, Hq, Hkv, D, window, max_kv, zero_rest,
                   scale * 1.4426950408889634f};
  p.B = B;
  p.max_q = max_q_len;
  p.page_shift = -1;
  for (int sh = 0; sh < 31; ++sh)
    if (page == 1 << sh) p.page_shift = sh;
  p.row_tiles = t.row_tiles;
  p.splits = t.tc ? 1 << 20 : t.splits;
  p.chunk = t.tc ? 1 << 20 : t.chunk;
  p.groups = t.groups;
  p.heads = t.heads;
  p.blocks = Hkv / t.heads;
  p.g_magic = Hq == Hkv ? 0 : static_cast<uint32_t>(((1ull << 32) + Hq / Hkv - 1) / (Hq / Hkv));   // exact for rows under 2^16
  p.part_rows = t.part_rows;
  p.part_o = scratch;
  p.part_lse = scratch + (t.scratch / (D + 1)) * D;
  int rc;
  if (t.tc)
    rc = D <= 64 ? (kv8 ? launch_tc<64, true>(p, ctas, stream) : launch_tc<64, false>(p, ctas, stream))
                 : kv8 ? launch_tc<128, true>(p, ctas, stream) : launch_tc<128, false>(p, ctas, stream);
  else if (kv8)
    rc = D <= 64 ? launch_mma<64, true>(p, t.wr, ctas, stream)
                 : D <= 128 ? launch_mma<128, true>(p, t.wr, ctas, stream) : launch_mma<256, true>(p, t.wr, ctas, stream);
  else
    rc = D <= 64 ? launch_mma<64, false>(p, t.wr, ctas, stream)
                 : D <= 128 ? launch_mma<128, false>(p, t.wr, ctas, stream) : launch_mma<256, false>(p, t.wr, ctas, stream);
  if (rc) return rc;
  const long out_rows = static_cast<long>(max_q_len) * Hq;
  if (t.tc && (t.groups > 1 || zero_rest))
    AFB_CHECK_CUDA(launch_pdl(tree_attn_tc_join_kernel, dim3(static_cast<unsigned>((out_rows * (D / 8) + 255) / 256), B),
                              dim3(256), 0, stream, p));
  else if (!t.tc && t.splits > 1 && out_rows > 0)
    AFB_CHECK_CUDA(launch_pdl(tree_attn_join_kernel, dim3(static_cast<unsigned>((out_rows * (D / 4) + 127) / 128), B), dim3(128), 0,
                              stream, p));
  return 0;
}

}  // extern "C"
