// The integer side of a speculative round over trees of drafted tokens, and of any packed step:
//   * step_maps    block tables, KV slots, rotary positions, packed starts of a step from the requests' lengths and the
//                  block ids that belong to them;
//   * tree_plan    ancestor bit masks and depths of drafted trees from their parent links;
//   * tree_accept  the walk along the drafts that the target model agrees with, and the move of the accepted nodes' cache
//                  rows to the front of their tree.
// The reference keeps its block tables on the host and verifies one chain of drafts per round
// (zig/pkg/inference/src/runtime/kv/block_table.zig:18-107, zig/pkg/inference/src/pipelines/generation.zig:3228).
#include "../common/ptx.cuh"
#include "../common/tmap.cuh"

namespace afb {

constexpr int kMaxTreeNodes = 256;
constexpr int kMaxTreeWords = kMaxTreeNodes / 32;

// ---------------------------------------------------------------------------------------------------------
// step_maps.  With s_b = sum of q over the sequences before b, n_b = ceil((kv_b + q_b) / page) and o_b the sum of n:
//   table[b][j] = blocks[o_b + j] for j < n_b, 0 behind;   slot of row s_b + i = table[b][(kv_b + i) / page] * page
//   + (kv_b + i) % page;   position = kv_b + i, or with depths kv_b - (tree_b - q_b) + depth of node tree_b - q_b + i.
// A CTA owns `per_cta` sequences (and one of gridDim.y slices of their rows): it sums the lengths in front of them
// itself, so there is one launch and no pass over the lengths before it.  4.2 us in a graph for 64 sequences, 10.3 us with
// the plan of 512 trees of 64 nodes and tables of 4160 entries (14.5 MB): latency, the tables' stores at 1.4 TB/s.
// ---------------------------------------------------------------------------------------------------------
struct StepMapsParams {
  const int* kv_before;
  const int* q_lens;
  const int* blocks;
  int num_ids;
  const int* depths;     // [B, depth_stride] or null
  long depth_stride;
  int depth_nodes;       // nodes a depth row holds
  const int* tree_lens;  // null: q_lens
  const int* shift;      // null: 0
  int B, page, max_blocks, T, per_cta;
  int* q_starts;
  int* kv_lens;
  int* logit_rows;
  int* positions;
  int* slots;
  int* tables;           // [B, max_blocks]
};

__device__ __forceinline__ long block_sum(long v, long* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  long s = 0;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) s += red[w];
  __syncthreads();
  return s;
}

__global__ void __launch_bounds__(256) step_maps_kernel(const StepMapsParams p) {
  __shared__ long red[8];
  griddep_launch();
  griddep_wait();
  const int b0 = blockIdx.x * p.per_cta, b1 = min(p.B, b0 + p.per_cta);
  long rows = 0, ids = 0;
  for (int c = threadIdx.x; c < b0; c += blockDim.x) {
    const int q = max(p.q_lens[c], 0);
    rows += q;
    ids += (static_cast<long>(max(p.kv_before[c], 0)) + q + p.page - 1) / p.page;
  }
  rows = block_sum(rows, red);
  ids = block_sum(ids, red);
  const int lane0 = blockIdx.y * blockDim.x + threadIdx.x, step = gridDim.y * blockDim.x;
  for (int b = b0; b < b1; ++b) {
    const int q = max(p.q_lens[b], 0), kv = max(p.kv_before[b], 0);
    const long need_l = (static_cast<long>(kv) + q + p.page - 1) / p.page;
    const bool bad = p.q_lens[b] < 0 || p.kv_before[b] < 0 || need_l > p.max_blocks || ids + need_l > p.num_ids ||
                     rows + q > p.T;
    if (lane0 == 0) {
      // what does not fit stays inside the step's rows: whoever indexes by these may rely on it
      if (bad) status_set(kStatusBadIndex);
      p.q_starts[b] = static_cast<int>(min(rows, static_cast<long>(p.T)));
      p.kv_lens[b] = static_cast<int>(min(static_cast<long>(kv) + q, 0x7fffffffl));
      p.logit_rows[b] = static_cast<int>(min(rows + q, static_cast<long>(p.T))) - 1;
    }
    const int need = static_cast<int>(min(min(need_l, static_cast<long>(p.max_blocks)), max(0l, p.num_ids - ids)));
    const int* mine = p.blocks + ids;
    int* table = p.tables + static_cast<long>(b) * p.max_blocks;
    for (int j = lane0; j < p.max_blocks; j += step) table[j] = j < need ? mine[j] : 0;
    const int tree = p.tree_lens ? p.tree_lens[b] : q;
    const int shift = p.shift ? p.shift[b] : 0;
    for (int i = lane0; i < q; i += step) {
      const long t = rows + i;
      if (t >= p.T) break;
      // unsigned, and slots in 64 bits: a length near 2^31 must not become a key in front of the table, nor a block id
      // that is none the slot of another one
      const uint32_t key = static_cast<uint32_t>(kv) + i, page = p.page, blk = key / page;
      const bool held = blk < static_cast<uint32_t>(need);
      const long slot = held ? static_cast<long>(mine[blk]) * p.page + key % page : -1;
      if (held && (slot < 0 || slot > 0x7fffffffl)) status_set(kStatusBadIndex);
      p.slots[t] = slot < 0 || slot > 0x7fffffffl ? -1 : static_cast<int>(slot);
      int pos = static_cast<int>(key);
      if (p.depths) {
        const int node = tree - q + i;
        const bool inside = node >= 0 && node < p.depth_nodes;
        if (!inside) status_set(kStatusBadIndex);
        pos = kv - (tree - q) + (inside ? p.depths[b * p.depth_stride + node] : 0);
      }
      p.positions[t] = pos + shift;
    }
    rows += q;
    ids += need_l;
  }
  if (b1 == p.B) {  // rows behind the last sequence
    for (long t = rows + lane0; t < p.T; t += step) {
      p.slots[t] = -1;
      p.positions[t] = 0;
    }
  }
}

// ---------------------------------------------------------------------------------------------------------
// tree_plan: node i sees itself and every node on its way to a root.  One thread follows one node's links; a tree of 64
// drafts is rarely deeper than 16.  A link that does not point to an earlier node makes the node a root and is reported.
// ---------------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256) tree_plan_kernel(const int* parents, long parent_stride, const int* lens, int N,
                                                        int W, int* masks, int* depths) {
  __shared__ int up[kMaxTreeNodes];
  griddep_launch();
  griddep_wait();
  const int b = blockIdx.x;
  const int n = lens ? min(max(lens[b], 0), N) : N;
  if (lens && threadIdx.x == 0 && lens[b] != n) status_set(kStatusBadIndex);
  for (int i = threadIdx.x; i < N; i += blockDim.x) {
    int u = i < n ? parents[b * parent_stride + i] : -1;
    if (u < -1 || u >= i) {
      status_set(kStatusBadIndex);
      u = -1;
    }
    up[i] = u;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < N; i += blockDim.x) {
    uint32_t m[kMaxTreeWords];
#pragma unroll
    for (int w = 0; w < kMaxTreeWords; ++w) m[w] = 0;
    int depth = -1;
    for (int c = i < n ? i : -1; c >= 0; c = up[c]) {
      ++depth;
#pragma unroll
      for (int w = 0; w < kMaxTreeWords; ++w) m[w] |= (c >> 5) == w ? 1u << (c & 31) : 0u;
    }
    int* row = masks + (static_cast<long>(b) * N + i) * W;
#pragma unroll
    for (int w = 0; w < kMaxTreeWords; ++w)
      if (w < W) row[w] = static_cast<int>(m[w]);
    depths[static_cast<long>(b) * N + i] = max(depth, 0);
  }
}

// ---------------------------------------------------------------------------------------------------------
// tree_accept.  The walk starts at node 0 and goes to the child (the lowest, if two are alike) whose token is the
// target's choice at the current node; path[i] is the i-th node on it.  Links point to earlier nodes, so path[i] >= i and
// the path ascends: a thread that owns one 16-byte column of the rows may move row path[i] to row i for i = 1, 2, ...
// in place, several loads ahead of their stores, without ever overwriting a row that is still to be read.  Every CTA walks
// its tree itself (a warp, a ballot per step), which takes less than a second launch.  4.8 us in a graph for one tree; 12 us for
// 64 trees of 64 nodes over 32 layers of 2 KiB rows (about 50 MB moved, 4.2 TB/s).
// ---------------------------------------------------------------------------------------------------------
struct AcceptCache {
  uint8_t* data[2];       // keys, values: [layers][num_slots][row_bytes]
  long row_bytes[2];
  long layer_bytes[2];
  long num_slots;
  const int* slots;       // [B, slot_stride]
  long slot_stride;
  int layers;
  int nodes;              // nodes whose rows this cache holds (a draft model has none for its last level)
};
struct AcceptParams {
  const int* tokens;
  const int* parents;
  const int* target;
  const int* lens;        // null: N
  long token_stride, parent_stride, target_stride;
  int N, num_caches;
  int* path;              // [B, N]
  int* count;
  int* next;
  AcceptCache cache[2];
};

template <typename V>
__device__ __forceinline__ void move_rows(const AcceptCache& c, int which, const int* src, const int* dst, int moves,
                                          int first, int step) {
  const long cols = c.row_bytes[which] / static_cast<long>(sizeof(V));
  const long total = cols * c.layers;
  for (long x = first; x < total; x += step) {
    V* base = reinterpret_cast<V*>(c.data[which] + (x / cols) * c.layer_bytes[which]) + x % cols;
    for (int i = 0; i < moves; i += 4) {
      V v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + j < moves) v[j] = base[src[i + j] * cols];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + j < moves) base[dst[i + j] * cols] = v[j];
    }
  }
}

__global__ void __launch_bounds__(256) tree_accept_kernel(const AcceptParams p) {
  __shared__ int path[kMaxTreeNodes];
  __shared__ int src[2][kMaxTreeNodes], dst[2][kMaxTreeNodes];
  __shared__ int s_count, s_moves[2];
  griddep_launch();
  griddep_wait();
  const int b = blockIdx.x, N = p.N;
  const int n = p.lens ? min(max(p.lens[b], 1), N) : N;
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    const int* tokens = p.tokens + b * p.token_stride;
    const int* parents = p.parents + b * p.parent_stride;
    const int* target = p.target + b * p.target_stride;
    // candidates: nodes whose token is what the target chose at their parent
    int up[kMaxTreeWords];
#pragma unroll
    for (int w = 0; w < kMaxTreeWords; ++w) {
      const int i = w * 32 + lane;
      int u = i > 0 && i < n ? parents[i] : -1;
      if (u >= i) {
        status_set(kStatusBadIndex);
        u = -1;
      }
      up[w] = u >= 0 && tokens[i] == target[u] ? u : -1;
    }
    int cur = 0, count = 1;
    if (lane == 0) path[0] = 0;
    for (;;) {
      int child = -1;
#pragma unroll
      for (int w = 0; w < kMaxTreeWords; ++w) {
        if (w * 32 >= n) break;
        const uint32_t hit = __ballot_sync(0xffffffffu, up[w] == cur);
        if (child < 0 && hit) child = w * 32 + __ffs(hit) - 1;
      }
      if (child < 0) break;
      cur = child;
      if (lane == 0) path[count] = child;
      ++count;
    }
    if (lane == 0) {
      s_count = count;
      if (blockIdx.y == 0) {
        p.count[b] = count;
        p.next[b] = target[cur];
        if (p.lens && p.lens[b] != n) status_set(kStatusBadIndex);
      }
    }
    __syncwarp();
    // the moves of each cache: rows that the path does not leave where they are
    for (int c = 0; c < p.num_caches; ++c) {
      const AcceptCache& ca = p.cache[c];
      const int* slots = ca.slots + b * ca.slot_stride;
      int moves = 0;
      for (int i0 = 0; i0 < count; i0 += 32) {
        const int i = i0 + lane;
        int from = 0, to = 0;
        bool take = i < count && path[i] != i && path[i] < ca.nodes;
        if (take) {
          from = slots[path[i]];
          to = slots[i];
          if (from < 0 || to < 0 || from >= ca.num_slots || to >= ca.num_slots) {
            status_set(kStatusBadIndex);
            take = false;
          }
        }
        const uint32_t who = __ballot_sync(0xffffffffu, take);
        const int at = moves + __popc(who & ((1u << lane) - 1u));
        if (take) {
          src[c][at] = from;
          dst[c][at] = to;
        }
        moves += __popc(who);
      }
      if (lane == 0) s_moves[c] = moves;
    }
  }
  __syncthreads();
  if (blockIdx.y == 0)
    for (int i = threadIdx.x; i < N; i += blockDim.x) p.path[static_cast<long>(b) * N + i] = i < s_count ? path[i] : -1;
  const int first = blockIdx.y * blockDim.x + threadIdx.x, step = gridDim.y * blockDim.x;
  for (int c = 0; c < p.num_caches; ++c) {
    const int moves = s_moves[c];
    if (moves == 0) continue;
    for (int which = 0; which < 2; ++which) {
      const AcceptCache& ca = p.cache[c];
      const uintptr_t align = reinterpret_cast<uintptr_t>(ca.data[which]) | ca.row_bytes[which] | ca.layer_bytes[which];
      if ((align & 15) == 0)
        move_rows<uint4>(ca, which, src[c], dst[c], moves, first, step);
      else if ((align & 3) == 0)
        move_rows<uint32_t>(ca, which, src[c], dst[c], moves, first, step);
      else
        move_rows<uint8_t>(ca, which, src[c], dst[c], moves, first, step);
    }
  }
}

}  // namespace afb

extern "C" {

int afb_step_maps(const int* kv_before, const int* q_lens, const int* blocks, int num_ids, const int* depths,
                  long depth_stride, int depth_nodes, const int* tree_lens, const int* shift, int B, int page,
                  int max_blocks, int T, int* q_starts, int* kv_lens, int* logit_rows, int* positions, int* slots,
                  int* tables, cudaStream_t stream) {
  using namespace afb;
  if (B <= 0 || page <= 0 || max_blocks < 0 || T < 0 || num_ids < 0) {
    set_last_error("afb_step_maps: bad sizes (B=%d page=%d max_blocks=%d T=%d ids=%d)", B, page, max_blocks, T, num_ids);
    return -1;
  }
  StepMapsParams p{kv_before, q_lens, blocks, num_ids, depths, depth_stride, depth_nodes, tree_lens, shift, B, page,
                   max_blocks, T, 1, q_starts, kv_lens, logit_rows, positions, slots, tables};
  p.per_cta = (B + 591) / 592;
  const int groups = (B + p.per_cta - 1) / p.per_cta;
  const long items = max_blocks > T / B ? max_blocks : T / B;
  long slices = (items + 511) / 512;
  if (slices > 592 / groups) slices = 592 / groups;
  if (slices < 1) slices = 1;
  AFB_CHECK_CUDA(launch_pdl(step_maps_kernel, dim3(groups, static_cast<unsigned>(slices)), dim3(256), 0, stream, p));
  return 0;
}

int afb_tree_plan(const int* parents, long parent_stride, const int* lens, int B, int N, int* masks, int* depths,
                  cudaStream_t stream) {
  using namespace afb;
  if (B <= 0) return 0;
  if (N < 1 || N > kMaxTreeNodes) {
    set_last_error("afb_tree_plan: a tree has 1 to %d nodes (N=%d)", kMaxTreeNodes, N);
    return -1;
  }
  const int threads = N <= 32 ? 32 : N <= 64 ? 64 : N <= 128 ? 128 : 256;
  AFB_CHECK_CUDA(launch_pdl(tree_plan_kernel, dim3(B), dim3(threads), 0, stream, parents, parent_stride, lens, N,
                            (N + 31) / 32, masks, depths));
  return 0;
}

// Up to two caches (pass null pointers for those that are not there); row and layer pitches in bytes.
int afb_tree_accept(const int* tokens, long token_stride, const int* parents, long parent_stride, const int* target,
                    long target_stride, const int* lens, int B, int N, int* path, int* count, int* next, void* k0,
                    void* v0, long k0_row, long v0_row, int layers0, long slots0, const int* slot_ids0, long stride0,
                    int nodes0, void* k1, void* v1, long k1_row, long v1_row, int layers1, long slots1,
                    const int* slot_ids1, long stride1, int nodes1, cudaStream_t stream) {
  using namespace afb;
  if (B <= 0) return 0;
  if (N < 1 || N > kMaxTreeNodes) {
    set_last_error("afb_tree_accept: a tree has 1 to %d nodes (N=%d)", kMaxTreeNodes, N);
    return -1;
  }
  AcceptParams p{tokens, parents, target, lens, token_stride, parent_stride, target_stride, N, 0, path, count, next, {}};
  long columns = 0;
  const auto add = [&](void* k, void* v, long kr, long vr, int layers, long slots, const int* ids, long stride, int nodes) {
    if (!k || layers <= 0) return;
    AcceptCache& c = p.cache[p.num_caches++];
    c.data[0] = static_cast<uint8_t*>(k); c.data[1] = static_cast<uint8_t*>(v);
    c.row_bytes[0] = kr; c.row_bytes[1] = vr;
    c.layer_bytes[0] = kr * slots; c.layer_bytes[1] = vr * slots;
    c.num_slots = slots; c.slots = ids; c.slot_stride = stride; c.layers = layers; c.nodes = nodes;
    columns += layers * (kr + vr) / 32;   // 16-byte columns of one of the two tensors
  };
  add(k0, v0, k0_row, v0_row, layers0, slots0, slot_ids0, stride0, nodes0);
  add(k1, v1, k1_row, v1_row, layers1, slots1, slot_ids1, stride1, nodes1);
  long slices = (columns + 255) / 256;
  const long most = B < 1184 ? 1184 / B : 1;
  if (slices > most) slices = most;
  if (slices < 1) slices = 1;
  AFB_CHECK_CUDA(launch_pdl(tree_accept_kernel, dim3(B, static_cast<unsigned>(slices)), dim3(256), 0, stream, p));
  return 0;
}

}  // extern "C"
