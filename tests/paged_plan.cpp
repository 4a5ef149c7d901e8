// Runs the paged prefill's plan and every workgroup's search for its piece on
// the CPU: a wave's 64 lanes are coroutines that meet at each operation across
// lanes.  Reads one call from stdin -- dtype (0 fp32, 1 bf16), batch, n_rows,
// n_heads, n_kv_heads, cap, workgroups to run at most, then batch lengths and batch + 1 row starts -- and
// prints the plan (rows of a unit, workgroups, pieces, slots, bytes of records) and a
// line per piece found: workgroup b g unit part parts row0 rows slot tok0 rem0.
#include <setjmp.h>
#include <ucontext.h>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <vector>

namespace {

constexpr int LANES = 64;
struct Lane {  // entered through its context once, then by jumps (a context's switch is two system calls)
  ucontext_t first;
  jmp_buf at;
  std::vector<char> stack;
  bool begun = false, done = false;
};
Lane lanes[LANES];
jmp_buf scheduler;
int current = 0;
int64_t board[2][LANES];  // what the lanes gave to an operation, and to the one before it
int turn[LANES];          // of each lane: operations so far

// All lanes' x: returns when every lane has given its own.
const int64_t *meet(int64_t x) {
  const int slot = turn[current] & 1;
  board[slot][current] = x;
  ++turn[current];
  if (_setjmp(lanes[current].at) == 0) _longjmp(scheduler, 1);
  return board[slot];
}
int as_int(float x) {
  int i;
  __builtin_memcpy(&i, &x, 4);
  return i;
}
float as_float(int i) {
  float x;
  __builtin_memcpy(&x, &i, 4);
  return x;
}

int wave_scan(int x) {
  const int64_t *v = meet(x);
  int64_t s = 0;
  for (int l = 0; l <= current; ++l) s += v[l];
  if (s < INT32_MIN || s > UINT32_MAX) {
    fprintf(stderr, "a scan passes 32 bits: %lld\n", (long long)s);
    exit(2);
  }
  return (int)(uint32_t)s;
}
int wave_min(int x) {
  const int64_t *v = meet(x);
  int64_t m = v[0];
  for (int l = 1; l < LANES; ++l) m = v[l] < m ? v[l] : m;
  return (int)m;
}
float wave_total(float x) {
  const int64_t *v = meet(as_int(x));
  float s = 0.f;
  for (int l = 0; l < LANES; ++l) s += as_float((int)v[l]);
  return s;
}
int __builtin_amdgcn_readlane(int x, int lane) {
  const int64_t *v = meet(x);
  if (lane < 0 || lane >= LANES) {
    fprintf(stderr, "a value of lane %d is read\n", lane);
    exit(2);
  }
  return (int)v[lane];
}
int __builtin_amdgcn_readfirstlane(int x) { return (int)meet(x)[0]; }
unsigned long long __builtin_amdgcn_ballot_w64(bool x) {
  const int64_t *v = meet(x);
  unsigned long long b = 0;
  for (int l = 0; l < LANES; ++l) b |= (unsigned long long)(v[l] != 0) << l;
  return b;
}

struct ThreadIndex {
  struct {
    operator int() const { return current; }
  } x;
} threadIdx;

}  // namespace

#define __device__
#define __forceinline__ inline
using std::max;
using std::min;
#include <algorithm>
#include "bn_paged_plan.hpp"

using namespace bn;

namespace {

PrefillParams params;
int block, rows_of_unit;
bool found[LANES];
Piece pieces[LANES];

void lane_main() {
  const int l = current;
  Piece w{};
  found[l] = rows_of_unit == 32    ? find_piece<32>(params, block, w)
             : rows_of_unit == 128 ? find_piece<128>(params, block, w)
                                   : find_piece<256>(params, block, w);
  pieces[l] = w;
  lanes[l].done = true;
  _longjmp(scheduler, 1);
}

void resume(int l) {
  current = l;
  if (_setjmp(scheduler) != 0) return;
  if (lanes[l].begun) _longjmp(lanes[l].at, 1);
  lanes[l].begun = true;
  setcontext(&lanes[l].first);
}

void run_wave() {
  for (int l = 0; l < LANES; ++l) {
    Lane &x = lanes[l];
    x.begun = x.done = false;
    turn[l] = 0;
    x.stack.resize(64 << 10);
    getcontext(&x.first);
    x.first.uc_stack.ss_sp = x.stack.data();
    x.first.uc_stack.ss_size = x.stack.size();
    x.first.uc_link = nullptr;
    makecontext(&x.first, lane_main, 0);
  }
  for (;;) {
    int left = 0;
    for (int l = 0; l < LANES; ++l) {
      if (lanes[l].done) continue;
      resume(l);
      left += !lanes[l].done;
    }
    if (left == 0) return;
    if (left != LANES) {
      fprintf(stderr, "the lanes part ways\n");
      exit(2);
    }
  }
}

}  // namespace

int main() {
  int dtype, batch, n_rows, n_heads, hkv, cap, most;
  if (scanf("%d %d %d %d %d %d %d", &dtype, &batch, &n_rows, &n_heads, &hkv, &cap, &most) != 7) return 1;
  std::vector<int32_t> lens(batch), starts(batch + 1);
  for (auto &x : lens)
    if (scanf("%d", &x) != 1) return 1;
  for (auto &x : starts)
    if (scanf("%d", &x) != 1) return 1;
  const PrefillPlan d = plan_prefill(dtype ? BN_BF16 : BN_F32, batch, n_rows, n_heads, hkv, cap);
  params.a.c.lens = lens.data();
  params.a.c.batch = batch;
  params.a.c.n_kv_heads = hkv;
  params.a.c.cap = cap;
  params.a.starts = starts.data();
  params.a.n_rows = n_rows;
  params.a.n_heads = n_heads;
  params.a.group = n_heads / hkv;
  params.a.inv_group = 1.0f / (float)params.a.group;
  params.a.prefix_len = 0;
  params.slots = (int)d.slots;
  params.parts_all = d.parts_all;
  params.pieces = (int)d.pieces;
  params.prefix_parts = 0;
  rows_of_unit = 32 * d.hw;
  printf("%d %lld %lld %lld %lld\n", rows_of_unit, (long long)d.groups, (long long)d.pieces, (long long)d.slots,
         (long long)d.records);
  for (block = 0; block < std::min<int64_t>(d.groups, most); ++block) {
    run_wave();
    for (int l = 1; l < LANES; ++l)
      if (found[l] != found[0] || (found[0] && __builtin_memcmp(&pieces[l], &pieces[0], sizeof(Piece)))) {
        fprintf(stderr, "the lanes disagree in workgroup %d\n", block);
        return 2;
      }
    const Piece &w = pieces[0];
    if (found[0])
      printf("%d %d %d %d %d %d %d %d %d %d %d\n", block, w.b, w.g, w.unit, w.part, w.parts, w.row0, w.rows, w.slot,
             w.tok0, w.rem0);
  }
  return 0;
}
