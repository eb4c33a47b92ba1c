// Drafted trees over a KV cache kept in pages (gfx950): attention of every
// node over the past and its own ancestors, and the acceptance of the nodes
// that the drawn tokens follow, with the move of their K and V rows.
//
// Tree b holds n <= 64 nodes, rows starts[b] .. of the step, and sits at the
// last n of the lengths[row] positions of its sequence: "past" below is what
// lies before it.  As everywhere over pages, device-held indices are checked
// before they form an address.
#include "paged_device.h"

namespace cascade {

constexpr int kTreeNodes = 64;  // one mask word, one node a lane

struct TreeArgs : PagedAttnArgs {
  const int32_t *starts;
  const int64_t *masks;
  int64_t tokens;
  int32_t max_tree;
};

struct Tree {
  int64_t row;  // < 0: nothing to do
  int32_t first;  // of its q rows
  int32_t nodes;
};

// Tree b's place among the step's rows, if it has any.
__device__ __forceinline__ Tree tree_of(const int32_t *starts, const int32_t *rows,
                                        int64_t tokens, int max_tree, int64_t b,
                                        int32_t *error) {
  Tree t{-1, 0, 0};
  const int64_t row = rows != nullptr ? rows[b] : b;
  if (row < 0) return t;
  const int64_t first = starts[b], end = starts[b + 1];
  if (first < 0 || end < first || end > tokens || end - first > max_tree) {
    flag_range(error);
    return t;
  }
  t.row = row;
  t.first = static_cast<int32_t>(first);
  t.nodes = static_cast<int32_t>(end - first);
  return t;
}

// ------------------------------------------------------------- attention
// One wave a (node, query head): an online softmax, one position at a time.
template <int D>
__global__ __launch_bounds__(kWave) void tree_attention_kernel(TreeArgs a) {
  constexpr int E = D / kWave;
  const int64_t b = blockIdx.z;
  const int node = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
  Tree t = tree_of(a.starts, a.rows, a.tokens, a.max_tree, b, lane == 0 ? a.error : nullptr);
  if (t.row < 0 || node >= t.nodes) return;
  if (t.row >= a.sequences) {
    if (lane == 0) flag_range(a.error);
    return;
  }
  const int len = a.lengths[t.row];
  if (len < t.nodes || len > a.max_length) {
    if (lane == 0) flag_range(a.error);
    return;
  }
  const int past = len - t.nodes;
  const int64_t token = t.first + node;
  const uint64_t mask = static_cast<uint64_t>(a.masks[token]);
  const int64_t kv = h / a.group;
  float q[E], acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = bf16_to_f32(a.q[token * a.q_token + h * a.q_head + E * lane + e]);
    acc[e] = 0.0f;
  }
  float m = -FLT_MAX, l = 0.0f;
  for (int p = 0; p < len; ++p) {
    if (p >= past && !((mask >> (p - past)) & 1)) continue;
    const int page = a.table[t.row * a.table_stride + (p >> a.page_shift)];
    if (page < 0 || page >= a.num_pages) {
      if (lane == 0) flag_range(a.error);
      continue;
    }
    const int64_t at = page * a.page_stride + kv * a.head_stride +
                       static_cast<int64_t>(p & ((1 << a.page_shift) - 1)) * D + E * lane;
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(q[e], bf16_to_f32(a.k_pages[at + e]), s);
    s = wave_sum(s) * a.scale_log2;
    const float mnew = fmaxf(m, s);
    const float keep = paged_exp2(m - mnew), w = paged_exp2(s - mnew);
    m = mnew;
    l = fmaf(l, keep, w);
#pragma unroll
    for (int e = 0; e < E; ++e)
      acc[e] = fmaf(w, bf16_to_f32(a.v_pages[at + e]), acc[e] * keep);
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
    a.out[token * a.out_token + h * a.out_head + E * lane + e] =
        f32_to_bf16(l == 0.0f ? 0.0f : acc[e] / l);
}

// ------------------------------------------------------------ acceptance
struct AcceptArgs {
  const int32_t *starts;
  const int64_t *ids;
  const int32_t *parents;
  const int64_t *targets;
  int64_t tokens;
  int32_t max_tree;
  int32_t *path, *counts;
  int64_t *next_ids;
  unsigned char *pages;  // null: no rows to move
  int64_t plane_bytes, page_bytes, row_bytes;
  int32_t num_pages;
  int32_t page_shift;
  const int32_t *table;
  int64_t table_stride;
  int64_t sequences;
  int64_t max_length;
  const int32_t *lengths;
  const int32_t *rows;
  int64_t vectors;  // 16-byte pieces that a position has in all planes
  int32_t row_vectors, head_vectors;  // of one row, of a position in one plane
  int32_t *error;
};

constexpr int kAcceptThreads = 256;

// Workgroup (tree, piece of the planes).  Every wave follows the path for
// itself, a node a lane: the children that fit are one ballot, and since a
// child lies behind its parent the path is an ascending set of bits and the
// walk ends.  A thread owns one 16-byte column of the rows and moves it for
// all nodes of the path, in order: the j-th goes to slot j, which lies before
// its own and before those of all later ones.
__global__ __launch_bounds__(kAcceptThreads) void tree_accept_kernel(AcceptArgs a) {
  const int64_t b = blockIdx.x;
  const int lane = threadIdx.x & (kWave - 1);
  const bool writes = blockIdx.y == 0 && threadIdx.x < kWave;
  const Tree t = tree_of(a.starts, a.rows, a.tokens, a.max_tree, b,
                         writes && lane == 0 ? a.error : nullptr);
  const int n = t.row < 0 ? 0 : t.nodes;
  int64_t id = 0, target = -1;
  int parent = -1;
  if (lane < n) {
    id = a.ids[t.first + lane];
    parent = a.parents[t.first + lane];
    target = a.targets[t.first + lane];
  }
  uint64_t on = n > 0 ? 1 : 0;
  int64_t next = -1;
  for (int cur = 0; n > 0;) {
    next = static_cast<int64_t>(lane_u64(static_cast<uint64_t>(target), cur));
    const uint64_t fits = __ballot(lane > cur && lane < n && parent == cur && id == next);
    if (next < 0 || fits == 0) break;
    cur = __ffsll(static_cast<unsigned long long>(fits)) - 1;
    on |= uint64_t{1} << cur;
  }
  const int count = __popcll(on);
  if (writes) {
    const int place = __popcll(on & ((uint64_t{1} << lane) - 1));
    if ((on >> lane) & 1) a.path[b * a.max_tree + place] = lane;
    if (lane >= count && lane < a.max_tree) a.path[b * a.max_tree + lane] = -1;
    if (lane == 0) {
      a.counts[b] = count;
      a.next_ids[b] = next;
    }
  }
  if (a.pages == nullptr || n == 0) return;
  if (t.row >= a.sequences) {
    if (writes && lane == 0) flag_range(a.error);
    return;
  }
  const int64_t len = a.lengths[t.row];
  if (len < n || len > a.max_length) {
    if (writes && lane == 0) flag_range(a.error);
    return;
  }
  const int64_t v = static_cast<int64_t>(blockIdx.y) * kAcceptThreads + threadIdx.x;
  const int64_t plane = v / a.head_vectors;
  const int in_plane = static_cast<int>(v % a.head_vectors);
  const int64_t head = in_plane / a.row_vectors;
  const int64_t page_size = int64_t{1} << a.page_shift;
  unsigned char *base = a.pages + plane * a.plane_bytes + head * page_size * a.row_bytes +
                        (in_plane % a.row_vectors) * 16;
  const int32_t *table = a.table + t.row * a.table_stride;
  int j = 0;
  for (uint64_t left = on; left != 0; left &= left - 1, ++j) {
    const int node = __ffsll(static_cast<unsigned long long>(left)) - 1;
    if (node == j) continue;
    const int64_t from = len - n + node, to = len - n + j;
    const int from_page = table[from >> a.page_shift], to_page = table[to >> a.page_shift];
    if (from_page < 0 || from_page >= a.num_pages || to_page < 0 || to_page >= a.num_pages) {
      if (writes && lane == 0) flag_range(a.error);
      continue;
    }
    if (v >= a.vectors) continue;
    *reinterpret_cast<u32x4 *>(base + to_page * a.page_bytes + (to & (page_size - 1)) * a.row_bytes) =
        *reinterpret_cast<const u32x4 *>(base + from_page * a.page_bytes +
                                         (from & (page_size - 1)) * a.row_bytes);
  }
}

static bool int32_ok(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }
static bool int64_ok(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 7) == 0; }

}  // namespace cascade

using namespace cascade;

extern "C" size_t cascade_paged_tree_attention_workspace_bytes(
    int64_t trees, int64_t max_tree, int64_t n_q_heads, int64_t n_kv_heads,
    int64_t head_dim, int64_t max_length) {
  if (trees <= 0 || trees > 0xffff || max_tree <= 0 || max_tree > kTreeNodes ||
      n_kv_heads <= 0 || n_q_heads <= 0 || n_q_heads % n_kv_heads ||
      n_q_heads / n_kv_heads > kPagedGroup || n_q_heads > 0xffff ||
      (head_dim != 64 && head_dim != 128) || max_length <= 0 || max_length > 0x7fffffff - 64)
    return 0;
  return kPagedAlign;
}

extern "C" int cascade_paged_tree_attention_bf16(
    const void *q, int64_t q_token_stride, int64_t q_head_stride, int64_t tokens,
    const int32_t *starts, const int64_t *masks, int64_t trees, int64_t max_tree,
    const void *k_pages, const void *v_pages, int64_t page_stride,
    int64_t page_head_stride, int64_t num_pages, int64_t page_size,
    const int32_t *page_table, int64_t table_stride, int64_t sequences,
    const int32_t *lengths, const int32_t *rows, int64_t max_length,
    int64_t n_q_heads, int64_t n_kv_heads, int64_t head_dim, float scale,
    void *out, int64_t out_token_stride, int64_t out_head_stride, void *workspace,
    size_t workspace_bytes, int32_t *error_flag, void *stream) {
  if (q == nullptr || starts == nullptr || masks == nullptr || k_pages == nullptr ||
      v_pages == nullptr || page_table == nullptr || lengths == nullptr || out == nullptr ||
      workspace == nullptr)
    return CASCADE_EINVAL;
  if (tokens <= 0 || tokens > 0x7fffffff || trees <= 0 || max_tree <= 0 || n_kv_heads <= 0 ||
      sequences <= 0 || num_pages <= 0 || num_pages > 0x7fffffff || max_length <= 0)
    return CASCADE_EINVAL;
  TreeArgs a{};
  const size_t need = cascade_paged_tree_attention_workspace_bytes(
      trees, max_tree, n_q_heads, n_kv_heads, head_dim, max_length);
  if (need == 0 || !page_shift_of(page_size, &a.page_shift)) return CASCADE_ESHAPE;
  if (table_stride < (max_length + page_size - 1) / page_size ||
      page_head_stride < page_size * head_dim ||
      page_stride < (n_kv_heads - 1) * page_head_stride + page_size * head_dim)
    return CASCADE_EINVAL;
  if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(out) ||
      !aligned16(workspace) || !int32_ok(starts) || !int64_ok(masks) ||
      !int32_ok(page_table) || !int32_ok(lengths) || !int32_ok(rows) ||
      !int32_ok(error_flag))
    return CASCADE_EALIGN;
  const int64_t strides[] = {q_token_stride, q_head_stride, page_stride,
                             page_head_stride, out_token_stride, out_head_stride};
  for (int64_t s : strides)
    if (!stride_ok(s)) return CASCADE_EALIGN;
  if (workspace_bytes < need) return CASCADE_EWORKSPACE;
  a.q = static_cast<const uint16_t *>(q);
  a.q_token = q_token_stride;
  a.q_head = q_head_stride;
  a.k_pages = static_cast<const uint16_t *>(k_pages);
  a.v_pages = static_cast<const uint16_t *>(v_pages);
  a.page_stride = page_stride;
  a.head_stride = page_head_stride;
  a.num_pages = static_cast<int32_t>(num_pages);
  a.table = page_table;
  a.table_stride = table_stride;
  a.sequences = sequences;
  a.lengths = lengths;
  a.rows = rows;
  a.max_length = static_cast<int32_t>(max_length);
  a.group = static_cast<int32_t>(n_q_heads / n_kv_heads);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.out = static_cast<uint16_t *>(out);
  a.out_token = out_token_stride;
  a.out_head = out_head_stride;
  a.error = error_flag;
  a.batch = static_cast<int32_t>(trees);
  a.kv_heads = static_cast<int32_t>(n_kv_heads);
  a.starts = starts;
  a.masks = masks;
  a.tokens = tokens;
  a.max_tree = static_cast<int32_t>(max_tree);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(max_tree), static_cast<unsigned>(n_q_heads),
                  static_cast<unsigned>(trees));
  return head_dim == 128
             ? launch_kernel(tree_attention_kernel<128>, grid, dim3(kWave), 0, s, a)
             : launch_kernel(tree_attention_kernel<64>, grid, dim3(kWave), 0, s, a);
}

extern "C" int cascade_paged_tree_accept(
    const int32_t *starts, const int64_t *ids, const int32_t *parents,
    const int64_t *targets, int64_t tokens, int64_t trees, int64_t max_tree,
    int32_t *path, int32_t *counts, int64_t *next_ids, void *pages,
    int64_t planes, int64_t plane_bytes, int64_t num_pages, int64_t n_kv_heads,
    int64_t page_size, int64_t row_bytes, const int32_t *page_table,
    int64_t table_stride, int64_t sequences, int64_t max_pages,
    const int32_t *lengths, const int32_t *rows, int32_t *error_flag,
    void *stream) {
  if (starts == nullptr || ids == nullptr || parents == nullptr || targets == nullptr ||
      path == nullptr || counts == nullptr || next_ids == nullptr)
    return CASCADE_EINVAL;
  if (tokens <= 0 || tokens > 0x7fffffff || trees <= 0 || max_tree <= 0)
    return CASCADE_EINVAL;
  if (max_tree > kTreeNodes || trees > kMaxThreads / kAcceptThreads) return CASCADE_ESHAPE;
  if (!int32_ok(starts) || !int64_ok(ids) || !int32_ok(parents) || !int64_ok(targets) ||
      !int32_ok(path) || !int32_ok(counts) || !int64_ok(next_ids) || !int32_ok(rows) ||
      !int32_ok(error_flag))
    return CASCADE_EALIGN;
  AcceptArgs a{};
  a.starts = starts;
  a.ids = ids;
  a.parents = parents;
  a.targets = targets;
  a.tokens = tokens;
  a.max_tree = static_cast<int32_t>(max_tree);
  a.path = path;
  a.counts = counts;
  a.next_ids = next_ids;
  a.rows = rows;
  a.error = error_flag;
  int64_t pieces = 1;
  if (pages != nullptr) {
    if (page_table == nullptr || lengths == nullptr || planes <= 0 || num_pages <= 0 ||
        num_pages > 0x7fffffff || n_kv_heads <= 0 || row_bytes <= 0 || sequences <= 0 ||
        max_pages <= 0 || table_stride < max_pages || plane_bytes < 0)
      return CASCADE_EINVAL;
    if (n_kv_heads > 1024 || row_bytes > 2048 || planes > 0xffff ||
        !page_shift_of(page_size, &a.page_shift) || max_pages > 0x7fffffff / page_size)
      return CASCADE_ESHAPE;
    if (!aligned16(pages) || (plane_bytes & 15) || (row_bytes & 15) || !int32_ok(page_table) ||
        !int32_ok(lengths))
      return CASCADE_EALIGN;
    a.page_bytes = n_kv_heads * page_size * row_bytes;
    if (planes > 1 && plane_bytes / num_pages < a.page_bytes) return CASCADE_EINVAL;
    a.pages = static_cast<unsigned char *>(pages);
    a.plane_bytes = plane_bytes;
    a.row_bytes = row_bytes;
    a.num_pages = static_cast<int32_t>(num_pages);
    a.table = page_table;
    a.table_stride = table_stride;
    a.sequences = sequences;
    a.max_length = max_pages * page_size;
    a.lengths = lengths;
    a.row_vectors = static_cast<int32_t>(row_bytes / 16);
    a.head_vectors = static_cast<int32_t>(n_kv_heads) * a.row_vectors;
    a.vectors = planes * a.head_vectors;
    pieces = (a.vectors + kAcceptThreads - 1) / kAcceptThreads;
    if (pieces > 0xffff) return CASCADE_ESHAPE;
  }
  const dim3 grid(static_cast<unsigned>(trees), static_cast<unsigned>(pieces));
  return launch_kernel(tree_accept_kernel, grid, dim3(kAcceptThreads), 0,
                       static_cast<hipStream_t>(stream), a);
}
