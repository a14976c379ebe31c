"""How the attention of sequences with a shared beginning is cut, run on the host: csrc/shared_schedule.cuh compiled by the C++ compiler,
a block's threads as coroutines that meet where its threads do.  Every key tile that a row of a group sees is walked once, no other
is, and every walk ends."""
import random
import subprocess

import pytest

import host_block

# Reads a call, walks every CTA's run, and writes the shares.
PROGRAM = r"""
#include "shared_schedule.cuh"
static std::vector<int> numbers(int n) { std::vector<int> v(n); for (int& x : v) if (scanf("%d", &x) != 1) exit(4); return v; }
int main() {
  const std::vector<int> h = numbers(12);
  shared::Shape sh = {};
  const int ctas = h[10], threads = h[11];
  sh.groups = h[0], sh.rows = h[1], sh.KVH = h[2], sh.G = h[3], sh.window = h[4], sh.most_ctx = h[5], sh.row_shift = h[6], sh.extra = h[7];
  sh.heavy = h[8], sh.is_many = h[9] < 0, sh.many = abs(h[9]), sh.min_units = 1 + sh.extra + sh.is_many;
  const std::vector<int> start = numbers(sh.groups + 1), prefix = numbers(sh.groups), ctx = numbers(sh.rows);
  int err = 0;
  sh.group_start = start.data(), sh.prefix_len = prefix.data(), sh.ctx_len = ctx.data(), sh.err = &err;
  static shared::Groups groups;
  static shared::Run run;
  Block block;
  for (int cta = 0; cta < ctas; ++cta) {
    memset((void*)&run, 0x5a, sizeof run);  // (what is not written is not read)
    block.run(threads, [&] {
      shared::make_plan(sh, groups, run, cta, ctas);
      __syncthreads();
      if (threadIdx.x == 0) memset((void*)&groups, 0x5a, sizeof groups);  // (its place is used for something else while the run is walked)
      __syncthreads();
      if (threadIdx.x >= 32) return;
      shared::Walk w;
      int steps = 0;
      for (bool more = w.begin(sh, run, cta); more;) {
        const shared::Share t = w.at;
        const shared::Note note = w.split(sh);
        if (threadIdx.x == 0)
          printf("%d %d %d %d %d %d %d %d %d %d %ld %d %d\n", cta, t.part, t.group, t.first, t.n, t.head, t.row_tile, t.kt_begin, t.kt_end, t.slot,
                 note.item, (int)note.record.parts, (int)note.record.stride);
        if (++steps > 100000) fprintf(stderr, "a walk does not end\n"), exit(5);
        more = w.next(sh);
      }
    });
  }
  printf("error %d items %ld\n", err, sh.items());
}
"""


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    names = ("shared_schedule.cuh", "rows_schedule.cuh")
    program = host_block.compiled(tmp_path_factory.mktemp("cut"), {name: host_block.source(name) for name in names}, PROGRAM)

    def of(starts, prefix, ctx, kv_heads=2, group=4, window=0, most_ctx=1 << 20, row_shift=6, extra=3, heavy=32, many=1 << 20, is_many=False,
           ctas=24, threads=160):
        numbers = [len(prefix), len(ctx), kv_heads, group, window, most_ctx, row_shift, extra, heavy, -many if is_many else many, ctas, threads]
        done = subprocess.run([program], input=" ".join(map(str, numbers + starts + prefix + ctx)), capture_output=True, text=True, timeout=120)
        assert done.returncode == 0, (done.returncode, done.stderr)
        *lines, last = done.stdout.splitlines()
        shares = [tuple(map(int, line.split())) for line in lines]
        _, error, _, items = last.split()
        check(shares, int(error), int(items), starts, prefix, ctx, kv_heads, group, window, most_ctx, row_shift, many, is_many, ctas)

    return of


def groups_there(starts, rows):
    """Groups that are among the rows and begin behind those before them."""
    there, at = [], 0
    for g, (a, b) in enumerate(zip(starts, starts[1:])):
        if 0 <= a <= b <= rows and a >= at:
            there.append(g)
            at = b
    return there


def check(shares, error, items, starts, prefix, ctx, kv_heads, group, window, most_ctx, row_shift, many, is_many, ctas):
    rows, tile = len(ctx), 1 << row_shift
    there = groups_there(starts, rows)
    assert error == (0 if len(there) == len(prefix) else 16)
    length = [min(max(0, n), most_ctx) for n in ctx]
    low = lambda r: max(0, length[r] - window) if window else 0
    want = {}  # (part, group, first row, row tile, head) -> key tiles
    for g in there:
        a, b = starts[g], starts[g + 1]
        p = min(max(0, prefix[g]), most_ctx) if b - a > 1 else 0
        segments = []
        if b - a > 1 and ((b - a) * group > many) == is_many:
            seen = [(low(r), min(p, length[r])) for r in range(a, b)]
            segments.append((0, a, b - a, min(x for x, _ in seen), max(y for _, y in seen)))
        if not is_many:
            segments += [(1, r, 1, max(p, low(r)), length[r]) for r in range(a, b)]
        for part, first, n, begin, end in segments:
            if begin < end:
                for row_tile in range(-(-n * group // tile)):
                    for head in range(kv_heads):
                        want[part, g, first, row_tile, head] = range(begin // 64, -(-end // 64))
    got, parts = {}, {}
    for cta, part, g, first, n, head, row_tile, kt_begin, kt_end, slot, item, of_item, stride in shares:
        key = part, g, first, row_tile, head
        assert key in want and kt_begin < kt_end and n == (1 if part else starts[g + 1] - starts[g])
        got.setdefault(key, []).append((kt_begin, kt_end))
        assert slot in (-1, 2 * cta, 2 * cta + 1)
        if item >= 0:  # it begins here; its parts are in these CTAs
            assert item < items and key not in parts and (slot == -1) == (of_item == 1)
            parts[key] = [cta + k * stride for k in range(of_item)]
        else:
            assert slot == 2 * cta
    assert got.keys() == want.keys() == parts.keys()
    ctas_of = {}
    for cta, part, g, first, n, head, row_tile, *_ in shares:
        ctas_of.setdefault((part, g, first, row_tile, head), []).append(cta)
    for key, tiles in want.items():
        ranges = sorted(got[key])
        assert ranges[0][0] == tiles.start and ranges[-1][1] == tiles.stop and all(x[1] == y[0] for x, y in zip(ranges, ranges[1:]))
        assert ctas_of[key] == parts[key]
    records = [share[10] for share in shares if share[10] >= 0]
    assert len(set(records)) == len(records)


SHAPES = [dict(), dict(window=200), dict(row_shift=5, extra=0, heavy=1 << 30, threads=256), dict(many=64),
          dict(many=64, is_many=True, row_shift=8, extra=5, heavy=1 << 30, threads=384)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("seed", range(6))
def test_every_key_tile_is_walked_once(walk, shape, seed):
    rng = random.Random(seed)
    starts, prefix, ctx = [0], [], []
    for _ in range(rng.choice([1, 3, 40, 200])):
        n, p = rng.choice([0, 1, 2, 5, 30]), rng.choice([0, 1, 63, 64, 500, 3000])
        starts.append(starts[-1] + n)
        prefix.append(p)
        ctx += [rng.choice([0, p, p + rng.randrange(1, 300)]) for _ in range(n)]
    ctx += [5] * rng.randrange(3)  # rows of no group
    walk(starts, prefix, ctx, ctas=rng.choice([3, 11, 24]), **shape)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("ctas", [4, 24])
@pytest.mark.parametrize("starts,prefix,rows", [
    ([0, 301, 299, 301, 301], [0, 0, 4000, 0], 301),   # the third has two rows of the first
    ([0, 301, 100, 301, 301], [500, 0, 4000, 0], 301),
    ([0, 40, 20, 60, 50, 90, 90], [64, 0, 64, 0, 64, 0], 90),
    ([-1, 100, 200, 300, 400], [100] * 4, 300),
    ([0, 2 ** 31 - 1, 4, 200, -2 ** 31, 200, 260], [70, 70, 70, 70, 70, 70], 300),
    ([300, 300, 10, 280, 280, 5], [70, 70, 70, 70, 70], 300),
    ([9, 5, 1], [70, 70], 300)])
def test_groups_that_overlap_or_lie_outside_are_left_out(walk, shape, ctas, starts, prefix, rows):
    rng = random.Random(rows)
    walk(starts, prefix, [rng.choice([0, 64, 65, 200, 4100]) for _ in range(rows)], ctas=ctas, **shape)


def test_many_groups_of_which_every_other_is_left_out(walk):
    starts = [x for g in range(512) for x in (3 * g, 1 << 30)] + [1600]
    walk(starts, [100] * 1024, [130] * 1600, ctas=5)
