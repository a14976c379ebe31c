"""The kernels of the choice of continuations (csrc/beam_select.cu) run on the host, with copies that never arrive: what the groups'
kernel reads of a CTA that left, it reads where something was written, and says nothing of rows that it does not know."""
import re
import subprocess

import pytest
import torch

import host_block
from beams_util import plain_select

# What the kernels take from other headers.  A copy into shared memory is there at once; the waits of one CTA run out from a turn on.
STUBS = {
    "packed2.cuh": r"""
inline float2 add2(float2 a, float2 b) { return {a.x + b.x, a.y + b.y}; }
inline float2 mul2(float2 a, float2 b) { return {a.x * b.x, a.y * b.y}; }
inline float max3(float a, float b, float c) { return fmaxf(a, fmaxf(b, c)); }
""",
    "tcgen05_common.cuh": r"""
inline int lost_cta = -1, lost_turn = 0;
inline int waits[4096];
namespace tc {
inline uint32_t smem_u32(const void*) { return 0; }
inline void mbar_init(uint64_t* bar, int) { *bar = 0; }
inline void mbar_expect_tx(uint64_t* bar, uint32_t) { ++*bar; }  // (phases that are complete)
inline bool mbar_wait(uint64_t* bar, uint32_t parity) {
  if (blockIdx.x == lost_cta && waits[threadIdx.x]++ >= lost_turn) return false;
  while ((*bar & 1) == parity) Block::current()->give_way();
  return true;
}
}
inline float to_f32(float x) { return x; }
""",
    "tensor_checks.cuh": ""}

# The scratch is as long as it has to be and full of ones, so that what was not written names a row and entries that are not there.
PROGRAM = r"""
#include <sys/mman.h>
#include "common.cuh"
#include "kernels.cu"
// An array with nothing behind it that can be read.
template <typename T> T* guarded(size_t n) {
  const size_t page = 4096, size = (n * sizeof(T) + page - 1) / page * page, behind = 1 << 26;
  char* at = (char*)mmap(nullptr, size + behind, PROT_NONE, MAP_PRIVATE | MAP_ANONYMOUS | MAP_NORESERVE, -1, 0);
  if (at == MAP_FAILED || mprotect(at, size, PROT_READ | PROT_WRITE) != 0) exit(4);
  return (T*)(at + size - n * sizeof(T));
}
int main() {
  int rows, vocab, groups, n, ctas;
  if (scanf("%d %d %d %d %d %d %d", &rows, &vocab, &groups, &n, &ctas, &lost_cta, &lost_turn) != 7) return 4;
  std::vector<int> start(groups + 1), parent(groups * n), token(groups * n);
  std::vector<float> score(groups * n);
  float *logits = guarded<float>((size_t)rows * vocab), *scores = guarded<float>(rows);
  for (int& x : start) if (scanf("%d", &x) != 1) return 4;
  for (int i = 0; i < rows; ++i) if (scanf("%f", scores + i) != 1) return 4;
  for (int i = 0; i < rows * vocab; ++i) if (scanf("%f", logits + i) != 1) return 4;
  int err = 0;
  Args a = {};
  const int pieces = (vocab + PIECE - 1) / PIECE;
  a.run = (rows * pieces + ctas - 1) / ctas;
  ctas = (rows * pieces + a.run - 1) / a.run;
  const long need = layout(a, nullptr, rows, pieces, ctas, n);
  float* scratch = guarded<float>((need + 3) / 4 * 4);
  memset(scratch, 0xff, need * 4);
  layout(a, scratch, rows, pieces, ctas, n);
  a.logits = logits, a.scores = scores, a.group_start = start.data();
  a.parent = parent.data(), a.token = token.data(), a.score = score.data();
  a.stride = vocab, a.rows = rows, a.groups = groups, a.vocab = vocab, a.pieces = pieces, a.n = n, a.bulk = 1, a.err = &err;
  Block block;
  gridDim.x = ctas;
  for (blockIdx.x = 0; blockIdx.x < ctas; ++blockIdx.x) {
    memset(waits, 0, sizeof waits);
    block.run(THREADS, [&] { beam_pieces_kernel<float>(a); });
  }
  for (blockIdx.x = 0; blockIdx.x < groups; ++blockIdx.x) block.run(THREADS, [&] { beam_groups_kernel(a); });
  printf("%d\n", err);
  for (int i = 0; i < groups * n; ++i) printf("%d %d %.9g\n", parent[i], token[i], score[i]);
}
"""


@pytest.fixture(scope="module")
def select(tmp_path_factory):
    kernels = host_block.source("beam_select.cu")
    kernels = kernels[:kernels.index("// tensors: logits, scores")]  # (what comes behind is the entry point)
    kernels, copies = re.subn(r'asm volatile\("cp\.async\.bulk.*?"memory"\);',
                              "memcpy(stage_bytes + (size_t)k * PIECE * sizeof(T), (const T*)a.logits + (size_t)row * a.stride + first, bytes);",
                              kernels, flags=re.S)
    kernels, powers = re.subn(r'asm\("ex2.*?\(x\)\);', "y = exp2f(x);", kernels)
    kernels = re.sub(r'asm volatile\("fence[^;]*;[^;]*;', "", kernels)
    kernels, stages = re.subn(r"extern __shared__ __align__\(128\) unsigned char stage_bytes\[\];", "static unsigned char stage_bytes[STAGES * PIECE * 4];",
                              kernels)
    assert (copies, powers, stages) == (1, 1, 1) and "asm" not in re.sub(r"//.*", "", kernels)
    program = host_block.compiled(tmp_path_factory.mktemp("select"), {**STUBS, "kernels.cu": kernels}, PROGRAM)

    def of(logits, scores, starts, n, ctas, lost_cta=-1, lost_turn=0):
        rows, vocab = logits.shape
        numbers = [rows, vocab, len(starts) - 1, n, ctas, lost_cta, lost_turn, *starts, *scores.tolist(), *logits.flatten().tolist()]
        done = subprocess.run([program], input=" ".join(map(repr, numbers)), capture_output=True, text=True, timeout=300)
        assert done.returncode == 0, (done.returncode, done.stderr)
        error, *lines = done.stdout.splitlines()
        found = [line.split() for line in lines]
        as_groups = lambda k, kind: torch.tensor([kind(f[k]) for f in found]).view(-1, n)
        return int(error), as_groups(0, int), as_groups(1, int), as_groups(2, float)

    return of


def inputs(rows, vocab, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return 2.5 * torch.randn(rows, vocab, generator=gen), -10 * torch.rand(rows, generator=gen)


@pytest.mark.parametrize("rows,vocab,starts,n,ctas", [(4, 20000, [0, 2, 4], 8, 5), (6, 8192, [0, 1, 6], 12, 3), (5, 30000, [0, 5], 40, 20)])
def test_as_the_plain_form(select, rows, vocab, starts, n, ctas):
    logits, scores = inputs(rows, vocab)
    error, parent, token, _ = select(logits, scores, starts, n, ctas)
    want_parent, want_token, _ = plain_select(logits, scores, starts, n)
    assert error == 0 and torch.equal(parent, want_parent) and torch.equal(token, want_token)


@pytest.mark.parametrize("lost_turn", [0, 1, 3])
@pytest.mark.parametrize("rows,vocab,starts,n,ctas,lost_cta", [
    (4, 20000, [0, 2, 4], 8, 3, 1), (6, 8192, [0, 1, 6], 12, 1, 0), (6, 8192, [0, 2, 4, 6], 12, 2, 0), (5, 30000, [0, 2, 5], 40, 4, 3),
    (300, 100, [0, 100, 300], 5, 3, 2)])
def test_copies_that_never_arrive(select, rows, vocab, starts, n, ctas, lost_cta, lost_turn):
    logits, scores = inputs(rows, vocab, seed=1)
    error, parent, token, score = select(logits, scores, starts, n, ctas, lost_cta, lost_turn)
    # rows of which a CTA that left had a piece
    pieces = -(-vocab // 8192)
    run = -(-rows * pieces // ctas)
    lost = {p // pieces for p in range(lost_cta * run + lost_turn, min((lost_cta + 1) * run, rows * pieces))}
    assert error == (4 if lost else 0)
    want_parent, want_token, _ = plain_select(logits, scores, starts, n)
    for g, (a, b) in enumerate(zip(starts, starts[1:])):
        if not lost & set(range(a, b)):
            assert torch.equal(parent[g], want_parent[g]) and torch.equal(token[g], want_token[g])
        there = parent[g] >= 0
        assert ((parent[g] >= a) & (parent[g] < b))[there].all() and ((token[g] >= 0) & (token[g] < vocab))[there].all()
        assert (parent[g][~there] == -1).all() and (token[g][~there] == -1).all()
