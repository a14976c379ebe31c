// Attention of sequences with a shared beginning over the paged key/value cache: one query row a sequence, the merge of partial
// results, and the entry point.
//
// Sequence r of group g has n_r stored tokens, its own among them.  Its key and value j lie at place j of the pages of the group's
// first sequence where j < P_g, else of its own.  Head h of its row:
//     o = sum_j w_j v_j / sum_j w_j,   w_j = exp(scale q . k_j),   max(0, n_r - W) <= j < n_r   (W: the window, if there is one)
// A sum over keys may be taken in parts: with m the largest score of a part, l = sum exp(s_j - m) and a = sum exp(s_j - m) v_j, parts
// join as  M = max m,  o = sum a exp(m - M) / sum l exp(m - M).  So the shared keys are read once for all sequences of a group,
// whose rows fill the tiles of a matrix product, and each sequence's own keys once for its G rows.  A row that sees nothing gives 0.
// The work is cut as shared_schedule.cuh says; the kernels: shared_attn_few.cuh, shared_attn_many.cuh where many rows share keys,
// rows_attn.cuh in 32-bit arithmetic, which bfloat16 heads without a tensor-core kernel take too (8 groups of 5 behind 4,096 tokens
// with 130 of their own, 28 heads on 4: of 96 222 us, of 128 on the tensor cores 43, each call behind a flushed L2).
#include "merge_parts.cuh"
#include "rows_attn.cuh"
#include "shared_schedule.cuh"
#include "tensor_checks.cuh"

namespace {
using namespace shared;

constexpr int FEW_CTAS = 2;                                 // an SM (shared_attn_few.cuh)
constexpr long FEW_ROWS_OF_A_TILE = 1 << ROW_SHIFT_FEW;
// What an item's beginning and end cost, in key tiles; rows of a tile of which all takes twice as long (64 rows 2 us a key tile and CTA
// where 16 take 0.6).  8 groups of 5 behind 4,101 tokens with 130 of their own, 28 heads of 128 on 4, and 7 groups of 50 behind 56 with
// 97, 16 on 4, with 0 to 5: 48.5, 42.6, 39.3, 35.8, 37.0, 36.4 us and 72.6, 61.0, 54.9, 50.6, 50.4, 49.3; with 3, and twice from above 16
// rows, 32, and never: 35.5, 35.8, 38.8 and 50.5, 50.6, 70.5.  (In 32 bits a key tile takes 8 us, and nothing is small beside it: 2 groups
// of 5 behind 701, 12 heads on 2, with 0 to 2: 21.6, 25.2, 32.2.)
// A kernel more is some 7 us more, which so many of its tiles an SM repay.  One group of 16 and 64 sequences of 28 heads on 4, and of
// 40 of 64 on 8, heads of 128, with both kernels and with the one for few alone: shared parts of 4,000 tokens (3.4, 11.9 and 17.0 tiles
// an SM) 25.2, 39.7 and 43.0 us and 21.3, 39.2 and 48.6; of 8,000 26.2, 43.6 and 50.6 and 28.1, 65.1 and 72.1; of 32,000 39.3, 69.8
// and 94.2 and 55.2, 160.5 and 211.9.  8 groups of 16 with 28 heads: 1,000 tokens (6.1) 37.3 and 35.2, 2,000 (12.1) 39.1 and 43.5.
// Groups and lengths are the device's, so the rule goes by rows a group on average and by the pages that a sequence may have: one
// group of many rows among many of one goes to the kernel for few, in tiles of 64 that each read the shared keys, and short
// beginnings in wide page tables pay for the kernel more.
constexpr long MANY_UNITS = 12;
constexpr int EXTRA_FEW = 3, HEAVY_FEW = 32, EXTRA_32BIT = 0, EXTRA_MANY = 5;

// Joins a row's partial results: `quads` neighbouring threads have four columns each of a row and head, and where rows are few, so many
// threads more (`share`) divide the partial results of a row among them, up to one for each CTA (8 rows behind 16,384 tokens, 12 heads
// of 128 on 2: 150 parts; a layer of a step 41 us where one thread a row took 75).
// Groups and lengths were there before the kernels in front began, and are looked at before their results are waited for; then two
// latencies are left, the records' and the partial results'.
constexpr int COMBINE_THREADS = 256;
template <typename T>
__global__ void __launch_bounds__(COMBINE_THREADS, 3)
shared_combine_kernel(const Shape sh, const Shape sh_many, const SharedScratch scratch, const SharedScratch scratch_many,
                      T* __restrict__ out, long out_stride, int D, int ctas, int ctas_many, int share) {
  __shared__ Starts starts;
  __shared__ float4 sums[COMBINE_THREADS];
  __shared__ float2 mls[COMBINE_THREADS];
  const int H = sh.KVH * sh.G, quads = D / 4, per_row = quads * share, tid = threadIdx.x;
  const int of_block = COMBINE_THREADS / per_row, in_block = tid / per_row, in_row = tid - in_block * per_row;
  const long row_head = (long)blockIdx.x * of_block + in_block;
  const int mine = in_row / quads, d = (in_row - mine * quads) * 4;  // which of the row's parts; its columns
  const int row = in_block < of_block ? (int)min(row_head / H, (long)sh.rows) : sh.rows, h = (int)(row_head % H);
  const int head = h / sh.G, of_head = h - head * sh.G;
  const int length = row < sh.rows ? sh.length(row) : 0;  // (asked for with the groups)
  starts.bring(sh, Starts::ask(sh));
  const int g = row < sh.rows ? group_of(starts, sh.groups, row) : -1;
  bool many = false, sees[2] = {false, false};  // the shared part was the other kernel's
  int of_tile[2] = {0, 0};
  long item[2] = {0, 0};
  if (g >= 0) {
    const int first = starts.start[g], n = starts.start[g + 1] - first;
    const int prefix = n > 1 ? min(max(0, sh.prefix_len[g]), sh.most_ctx) : 0, lo = sh.window > 0 ? max(0, length - sh.window) : 0;
    many = (long)n * sh.G > sh.many;
    // an item of which the row sees a key is there, and has a record
    sees[0] = lo < min(prefix, length);
    sees[1] = max(prefix, lo) < length;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const Shape& of = part == 0 && many ? sh_many : sh;
      const int rr = (part == 0 ? (row - first) * sh.G : 0) + of_head;
      of_tile[part] = rr & (of.rows_per_tile() - 1);
      item[part] = of.item(part, g, part == 0 ? first : row, rr >> of.row_shift, head);
    }
  }
  pdl_launch_dependents();
  pdl_wait();
  // asked for with the records, which say whether they are wanted
  Record rec[2];
  float2 ml[2];
  float4 o[2];
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    const bool of_many = part == 0 && many;
    const size_t at = ((size_t)part * sh.rows + row) * H + h;
    rec[part] = {0, 0, 1};
    ml[part] = make_float2(-INFINITY, 0.f);
    o[part] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (sees[part]) {
      rec[part] = (of_many ? scratch_many : scratch).records[item[part]];
      ml[part] = reinterpret_cast<const float2*>(scratch.rows_ml)[at];
      o[part] = *reinterpret_cast<const float4*>(scratch.rows_o + at * D + d);
    }
    // (a record that a CTA whose wait ran out did not write is none)
    const Record x = rec[part];
    if (x.cta < 0 || x.parts < 0 || x.stride < 1 || (x.parts > 0 && x.cta + (x.parts - 1) * x.stride >= (of_many ? ctas_many : ctas)))
      rec[part] = {0, 0, 1};
  }
  auto load = [&](int k, float2& a, float4& b) {
    const int part = k >= rec[0].parts;
    if (part) k -= rec[0].parts;
    const Record x = part ? rec[1] : rec[0];
    if (x.parts <= 1) {
      a = part ? ml[1] : ml[0];
      b = part ? o[1] : o[0];
    } else {
      const bool of_many = part == 0 && many;
      const SharedScratch& of = of_many ? scratch_many : scratch;
      const size_t slot = 2 * (size_t)(x.cta + k * x.stride) + (k == 0);
      const size_t at = (slot << (of_many ? sh_many.row_shift : sh.row_shift)) + (part ? of_tile[1] : of_tile[0]);
      a = reinterpret_cast<const float2*>(of.part_ml)[at];
      b = *reinterpret_cast<const float4*>(of.part_o + at * D + d);
    }
  };
  const int parts = rec[0].parts + rec[1].parts;
  // thread `mine` has the parts mine, mine + share, ...
  const int own = parts > mine ? (parts - mine + share - 1) / share : 0;
  const Merged x = merge_parts<4>(own, [&](int k, float2& a, float4& b) { load(mine + k * share, a, b); });
  float4 v = merged(x);
  if (share > 1) {
    sums[tid] = x.sum;
    mls[tid] = make_float2(x.top, x.total);
    __syncthreads();
    if (mine > 0) return;
    v = merged(merge_parts<2>(min(parts, share), [&](int k, float2& a, float4& b) {
      a = mls[tid + k * quads];
      b = sums[tid + k * quads];
    }));
  }
  if (g >= 0) store4(out + (size_t)row * out_stride + (size_t)h * D + d, v);  // (a row in no group is left as it is)
}

// A kernel's scratch of its own, laid out from `at` on.
long layout(SharedScratch& x, float* at, const Shape& sh, long ctas, long D) {
  const long rows = sh.rows_per_tile();
  x.part_o = at;
  x.part_ml = x.part_o + 2 * ctas * rows * D;
  x.records = reinterpret_cast<Record*>(x.part_ml + 4 * ctas * rows);
  return 2 * ctas * rows * (D + 2) + 2 * ((sh.items() + 1) / 2 * 2);
}
}  // namespace

struct DspSharedOptions {  // as ops/beams.py packs them
  long window, sms, few, many;
  double scale;
};

// Addresses of the tensor-core kernels' entry points for this head size, or 0: `few`, `many` (heads of 32 have none).
// tensors: q, key pool, value pool, page table, ctx_len, group_start, prefix_len, out, scratch.
extern "C" int dsp_shared_attention(const DspTensor* t, const DspSharedOptions* o, cudaStream_t stream) {
  const DspTensor &q = t[0], &k = t[1], &v = t[2], &table = t[3], &ctx = t[4], &start = t[5], &prefix = t[6], &out = t[7], &scratch = t[8];
#define SHARED_REQUIRE(cond, ...) DSP_REQUIRE(cond, "shared_prefix_attention: " __VA_ARGS__)
  SHARED_REQUIRE(q.device >= 0, "CUDA tensors only (there is no CPU path)");
  SHARED_REQUIRE(q.dims == 2 && k.dims == 4 && v.dims == 4, "q [R, H * D] and two pools [pages, heads, page_size, D] expected");
  const long R = q.size[0], columns = q.size[1], pages = k.size[0], KVH = k.size[1], page = k.size[2], D = k.size[3];
  SHARED_REQUIRE(q.dtype == DSP_T_F32 || q.dtype == DSP_T_BF16, "kernels exist for float32 and bfloat16");
  SHARED_REQUIRE(k.dtype == q.dtype && v.dtype == q.dtype && k.device == q.device && v.device == q.device && k.contiguous && v.contiguous &&
                     v.size[0] == pages && v.size[1] == KVH && v.size[2] == page && v.size[3] == D,
                 "the pools must be contiguous, alike, and of the type and on the device of q");
  SHARED_REQUIRE(R == 0 || q.stride[1] == 1 || columns == 1, "the columns of q must be neighbours");
  SHARED_REQUIRE(D % 8 == 0 && D >= 8 && D <= 256 && KVH > 0 && columns > 0 && columns % D == 0 && columns / D % KVH == 0,
                 "%ld query columns on %ld heads of %ld (a multiple of 8 up to 256)", columns, KVH, D);
  SHARED_REQUIRE(is_scale(o->scale) && o->window >= 0 && o->window <= 0x7fffffff,
                 "scale %g must be positive and finite in 32 bits, window %ld not negative", o->scale, o->window);
  SHARED_REQUIRE(prefix.dims == 1 && prefix.size[0] <= MAX_GROUPS, "prefix_len must be one-dimensional, of at most %d groups", MAX_GROUPS);
  const long groups = prefix.size[0];
  SHARED_REQUIRE(tensor_is(ctx, DSP_T_I32, q.device, 1, R) && tensor_is(start, DSP_T_I32, q.device, 1, groups + 1) &&
                     tensor_is(prefix, DSP_T_I32, q.device, 1, groups),
                 "ctx_len [%ld], group_start [%ld] and prefix_len [%ld] must be contiguous int32 on the device of q", R, groups + 1, groups);
  SHARED_REQUIRE(is_page_table(table, q.device, R), "page_table must be int32 [%ld, pages], neighbouring pages side by side", R);
  SHARED_REQUIRE(out.dtype == q.dtype && out.device == q.device && out.dims == 2 && out.size[0] == R && out.size[1] == columns &&
                     (R == 0 || out.stride[1] == 1 || columns == 1) && (R <= 1 || out.stride[0] >= columns),
                 "out must be like the queries [%ld, %ld] with neighbouring columns, no two rows in one place", R, columns);
  SHARED_REQUIRE(R <= 0x7fffffff && pages <= 0x7fffffff && page >= 1 && page <= 0x7fffffff && o->sms >= 1 && table.stride[0] <= 0x7fffffff,
                 "sizes out of range");
  if (R == 0 || groups == 0) return 0;
  const uintptr_t bits = (uintptr_t)q.data | (uintptr_t)k.data | (uintptr_t)v.data | (uintptr_t)out.data;
  const long piece = q.dtype == DSP_T_F32 ? 4 : 8;  // elements of 16 bytes
  SHARED_REQUIRE(bits % 16 == 0 && (R == 1 || (q.stride[0] % piece == 0 && out.stride[0] % piece == 0)), "rows must begin on 16 bytes");
  // the tensor-core kernels are built for these page sizes; everything else takes the 32-bit kernel
  const bool tensor_cores = o->few != 0 && q.dtype == DSP_T_BF16 && (D == 32 || D == 64 || D == 128) &&
                            (page == 8 || page == 16 || page == 32 || page == 64) && pages > 0;
  const long ctas = o->sms * (tensor_cores ? FEW_CTAS : D > 128 ? 1 : 2);  // (by shared memory two CTAs an SM)
  DspSharedAttention a = {};
  a.sh.group_start = (const int*)start.data;
  a.sh.prefix_len = (const int*)prefix.data;
  a.sh.ctx_len = (const int*)ctx.data;
  a.sh.groups = (int)groups;
  a.sh.KVH = (int)KVH;
  a.sh.G = (int)(columns / D / KVH);
  a.sh.window = (int)o->window;
  a.sh.rows = (int)R;
  a.sh.row_shift = tensor_cores ? ROW_SHIFT_FEW : ROW_SHIFT_32BIT;
  a.sh.extra = tensor_cores ? EXTRA_FEW : EXTRA_32BIT;
  a.sh.heavy = tensor_cores ? HEAVY_FEW : 0x7fffffff;
  a.sh.min_units = 1 + a.sh.extra;
  // Where groups have more rows a head on average than a tile of the kernel for few, and their shared parts may be so long (as long
  // as their pages) that each SM has MANY_UNITS of its tiles or more, the shared parts of those that do are the other kernel's.
  const long units = (R * a.sh.G + FEW_ROWS_OF_A_TILE - 1) / FEW_ROWS_OF_A_TILE * KVH * (table.size[1] * page / KEYS_PER_TILE + 1);
  const bool use_many = tensor_cores && o->many != 0 && R * a.sh.G > groups * FEW_ROWS_OF_A_TILE && units > MANY_UNITS * o->sms;
  a.sh.many = use_many ? FEW_ROWS_OF_A_TILE : 0x7fffffff;
  // places are counted in 32 bits, a tile of keys beyond the last among them
  a.sh.most_ctx = (int)min(table.size[1] * page, 1L << 30);
  // Units are counted in 32 bits: those of all items, each over as many tokens as a sequence's pages hold.
  SHARED_REQUIRE(R * a.sh.G <= 0x7fffffff && a.sh.items() <= 0x7fffffff / (2 * (a.sh.most_ctx / KEYS_PER_TILE + 1 + EXTRA_MANY)),
                 "%ld rows of %ld heads over pages for %d tokens a sequence are too many for one call", R, columns / D, a.sh.most_ctx);
  DspSharedAttention many = a;
  many.sh.is_many = 1;
  many.sh.row_shift = ROW_SHIFT_MANY;
  many.sh.heavy = 0x7fffffff;
  many.sh.extra = EXTRA_MANY;
  many.sh.min_units = 2 + EXTRA_MANY;
  a.ctas = (int)ctas;
  many.ctas = use_many ? (int)o->sms : 0;
  const long of_rows = 2 * R * columns / D;
  a.scratch.rows_o = many.scratch.rows_o = (float*)scratch.data;
  a.scratch.rows_ml = many.scratch.rows_ml = a.scratch.rows_o + of_rows * D;
  long floats = of_rows * (D + 2);
  floats += layout(a.scratch, (float*)scratch.data + floats, a.sh, a.ctas, D);
  if (use_many) floats += layout(many.scratch, (float*)scratch.data + floats, many.sh, many.ctas, D);
  SHARED_REQUIRE(scratch.contiguous && scratch.device == q.device && scratch.dims == 1 && (uintptr_t)scratch.data % 16 == 0 &&
                     scratch.size[0] >= floats,
                 "scratch is too small: %ld of %ld", scratch.size[0], floats);
  SHARED_REQUIRE(current_device() == q.device, "the tensors are on device %d, the current device is %d", q.device, current_device());
  a.q = q.data;
  a.k_pool = k.data;
  a.v_pool = v.data;
  a.page_table = (const int*)table.data;
  a.out = out.data;
  a.q_stride = q.stride[0];
  a.out_stride = out.stride[0];
  a.pt_stride = (int)table.stride[0];
  a.table_width = (int)min(table.size[1], 0x7fffffffL);
  a.D = (int)D;
  a.page_size = (int)page;
  a.num_pages = (int)pages;
  a.scale = (float)o->scale;
  a.err = a.sh.err = dsp_device_error_ptr();
  SHARED_REQUIRE(a.err != nullptr, "no device error word");
  if (tensor_cores) {
    typedef int (*Kernel)(const DspSharedAttention*, cudaStream_t);
    int rc = 0;
    a.beside = use_many;
    if (use_many) {
      DspSharedAttention x = a;
      x.sh = many.sh;
      x.scratch = many.scratch;
      x.ctas = many.ctas;
      x.sh.err = a.err;
      rc = reinterpret_cast<Kernel>(o->many)(&x, stream);
    }
    if (rc == 0) rc = reinterpret_cast<Kernel>(o->few)(&a, stream);
    SHARED_REQUIRE(rc == 0, "%s", rc == 4 ? "shared memory opt-in or tensor map creation failed" : "launch failed");
  } else {
    const int rc = q.dtype == DSP_T_F32 ? launch_rows_attn<SharedWork, float>(a, stream) : launch_rows_attn<SharedWork, bf16>(a, stream);
    if (rc != 0) return rc;
  }
  // threads that share a row and head: one for eight of the parts that a shared part's item may have, by the CTAs that there are for
  // each and by its key tiles
  const long quads = D / 4, row_heads = R * columns / D, of_part = use_many ? many.ctas : ctas,
             parts = min(of_part / min(groups * KVH, of_part), (long)a.sh.most_ctx / KEYS_PER_TILE);
  int share = 1;
  while (quads * share * 2 <= COMBINE_THREADS && share * 16 <= parts) share *= 2;
  const long of_block = COMBINE_THREADS / (quads * share);
  const dim3 grid((unsigned)((row_heads + of_block - 1) / of_block));
  if (q.dtype == DSP_T_F32)
    DSP_CUDA(launch_pdl(shared_combine_kernel<float>, grid, dim3(COMBINE_THREADS), 0, stream, a.sh, many.sh, a.scratch, many.scratch,
                        (float*)a.out, a.out_stride, a.D, a.ctas, many.ctas, share));
  else
    DSP_CUDA(launch_pdl(shared_combine_kernel<bf16>, grid, dim3(COMBINE_THREADS), 0, stream, a.sh, many.sh, a.scratch, many.scratch,
                        (bf16*)a.out, a.out_stride, a.D, a.ctas, many.ctas, share));
  DSP_CHECK_LAUNCH("shared_prefix_attention");
  return 0;
}
