"""Device code on the host: what a block's threads call, for threads that are coroutines and meet where a block's threads do.  A test
writes ``COMMON`` in the place of csrc/common.cuh and compiles the code that it looks at with the C++ compiler."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dispec_b200", "csrc")

COMMON = r"""
#pragma once
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <math.h>
#include <ucontext.h>
#include <algorithm>
#include <functional>
#include <vector>
using std::max;
using std::min;
#define __device__
#define __host__
#define __global__
#define __shared__ static
#define __forceinline__ inline
#define __noinline__
#define __launch_bounds__(...)
#define __align__(n) __attribute__((aligned(n)))
struct float2 { float x, y; };
struct uint2 { unsigned x, y; };
struct uint4 { unsigned x, y, z, w; };
inline float2 make_float2(float x, float y) { return {x, y}; }
inline uint2 make_uint2(unsigned x, unsigned y) { return {x, y}; }
struct Dim { int x; };
enum { DSP_ERR_WAIT_LIMIT = 4, DSP_ERR_BAD_GROUP = 16 };
inline Dim threadIdx, blockIdx, blockDim, gridDim;

// A block of coroutines.  A thread that meets others gives way until all of them have come.
struct Block {
  struct Thread { ucontext_t at; std::vector<char> stack; bool done; };
  struct Meeting { int expected = 0, come = 0; long turn = 0; int any = 0, result = 0; long long values[1024]; long long out[1024]; };
  std::vector<Thread> threads;
  std::vector<Meeting> warps;
  Meeting all;
  ucontext_t home;
  int now = 0;
  std::function<void()> work;
  static Block*& current() { static Block* b; return b; }
  static void enter() { Block* b = current(); b->work(); b->threads[b->now].done = true; }
  void run(int n, std::function<void()> f) {
    work = f, current() = this, blockDim.x = n;
    threads.resize(n), warps.resize((n + 31) / 32);
    all.expected = n, all.come = 0;
    for (auto& w : warps) w.expected = 32, w.come = 0;
    for (auto& t : threads) {
      t.stack.resize(1 << 16), t.done = false;
      getcontext(&t.at);
      t.at.uc_stack.ss_sp = t.stack.data(), t.at.uc_stack.ss_size = t.stack.size(), t.at.uc_link = &home;
      makecontext(&t.at, enter, 0);
    }
    for (long idle = 0; idle < 1000000; ++idle) {
      bool left = false;
      for (now = 0; now < n; ++now)
        if (!threads[now].done) left = true, threadIdx.x = now, swapcontext(&home, &threads[now].at);
      if (!left) return;
    }
    fprintf(stderr, "threads wait for one another\n"), exit(3);
  }
  void give_way() { swapcontext(&threads[now].at, &home); }
  void meet(Meeting& m, int place, long long value) {
    const long turn = m.turn;
    m.values[place] = value;
    if (++m.come == m.expected) {
      std::copy(m.values, m.values + m.expected, m.out);
      m.come = 0, ++m.turn;
      return;
    }
    while (m.turn == turn) give_way();
  }
};
inline long long* meet_all(long long value = 0) { Block* b = Block::current(); b->meet(b->all, threadIdx.x, value); return b->all.out; }
// (what the others bring is there until all have come again)
inline long long* meet_warp(long long value) {
  Block* b = Block::current();
  Block::Meeting& w = b->warps[threadIdx.x / 32];
  b->meet(w, threadIdx.x % 32, value);
  return w.out;
}
template <typename T> long long bits_of(T x) { long long v = 0; memcpy(&v, &x, sizeof x); return v; }
template <typename T> T of_bits(long long v) { T x; memcpy(&x, &v, sizeof x); return x; }
template <typename T, typename F> T over_warp(T x, F f) {
  const long long* v = meet_warp(bits_of(x));
  T r = of_bits<T>(v[0]);
  for (int i = 1; i < 32; ++i) r = f(r, of_bits<T>(v[i]));
  return r;
}
inline void __syncthreads() { meet_all(); }
inline int __syncthreads_or(int x) { const long long* v = meet_all(x != 0); int any = 0; for (int i = 0; i < blockDim.x; ++i) any |= v[i] != 0; return any; }
inline void __syncwarp() { meet_warp(0); }
template <typename T> T __reduce_max_sync(unsigned, T x) { return over_warp(x, [](T a, T b) { return max(a, b); }); }
template <typename T> T __reduce_min_sync(unsigned, T x) { return over_warp(x, [](T a, T b) { return min(a, b); }); }
template <typename T> T __reduce_add_sync(unsigned, T x) { return over_warp(x, [](T a, T b) { return a + b; }); }
inline unsigned __ballot_sync(unsigned, int x) { const long long* v = meet_warp(x != 0); unsigned r = 0; for (int i = 0; i < 32; ++i) r |= (unsigned)(v[i] != 0) << i; return r; }
template <typename T> T __shfl_sync(unsigned, T x, int l) { return of_bits<T>(meet_warp(bits_of(x))[l]); }
template <typename T> T __shfl_xor_sync(unsigned, T x, int o) { return of_bits<T>(meet_warp(bits_of(x))[(threadIdx.x % 32) ^ o]); }
template <typename T> T __shfl_up_sync(unsigned, T x, int o) { const int l = threadIdx.x % 32; return of_bits<T>(meet_warp(bits_of(x))[l < o ? l : l - o]); }
inline int __ffs(unsigned x) { return __builtin_ffs((int)x); }
inline unsigned __float_as_uint(float x) { return (unsigned)bits_of(x); }
inline float __uint_as_float(unsigned x) { return of_bits<float>(x); }
inline long long __double_as_longlong(double x) { return bits_of(x); }
inline double __longlong_as_double(long long x) { return of_bits<double>(x); }
inline void __nanosleep(unsigned) {}
inline int atomicAdd(int* p, int x) { const int old = *p; *p += x; return old; }
inline void atomicOr(int* p, int x) { *p |= x; }
inline void atomicMin(int* p, int x) { *p = min(*p, x); }
inline void atomicMax(int* p, int x) { *p = max(*p, x); }
inline void pdl_wait() {}
inline void pdl_launch_dependents() {}
"""


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return f.read()


def compiled(folder, files, program, *flags):
    """Writes ``files`` {name: text} beside COMMON and compiles ``program``, which includes them."""
    cxx = os.environ.get("CXX") or shutil.which("g++")
    if not cxx:
        pytest.skip("no C++ compiler")
    for name, text in {"common.cuh": COMMON, **files, "program.cpp": program}.items():
        (folder / name).write_text(text)
    subprocess.run([cxx, "-std=c++20", "-O2", "-w", *flags, "-I", str(folder), str(folder / "program.cpp"), "-o", str(folder / "program")], check=True)
    return str(folder / "program")
