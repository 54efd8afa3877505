// Runs a kernel's blocks one after another on the CPU, each thread a fiber.  A fiber gives
// way where it waits for its wave (wave_exchange) or its block (block_barrier).  LANE_ORDER
// says who goes next: 0 the next thread, 1 the one before, 2 mostly the same wave, at times
// any other.  Dynamic shared memory is filled with junk before every block.
#include "hip/hip_runtime.h"

#include <sys/mman.h>

Index threadIdx, blockIdx, gridDim, blockDim;
char* dynamic_lds;

extern "C" void switch_fiber(void** from, void* to);
asm(R"(
.text
.globl switch_fiber
switch_fiber:
  push %rbx
  push %rbp
  push %r12
  push %r13
  push %r14
  push %r15
  mov %rsp,(%rdi)
  mov %rsi,%rsp
  pop %r15
  pop %r14
  pop %r13
  pop %r12
  pop %rbp
  pop %rbx
  ret
)");

namespace {
constexpr int MAX_THREADS = 1024;
constexpr size_t STACK = 256 << 10, MAX_LDS = 160 << 10;
constexpr long MAX_WAIT = 100000000;  // turns without progress: a wait that never ends

struct Wave {
  uint64_t slot[2][64], live_at[2], mask;
  int arrived, live;
  unsigned round;
  void step() {
    live_at[round & 1] = mask;
    arrived = 0;
    ++round;
  }
};
Wave waves[MAX_THREADS / 64];
void *stacks[MAX_THREADS], *saved[MAX_THREADS], *main_saved;
bool ended[MAX_THREADS];
int threads, current, live_threads, at_barrier;
unsigned barrier_round;
const std::function<void()>* kernel_body;
const char* kernel_name;
const int order = getenv("LANE_ORDER") ? atoi(getenv("LANE_ORDER")) : 0;
uint64_t random_state = 12345;

[[noreturn]] void fail(const char* what) {
  fprintf(stderr, "%s: %s (thread %d of block %u, %u)\n", kernel_name, what, current, blockIdx.x, blockIdx.y);
  abort();
}
void set_current(int t) {
  current = t;
  threadIdx = {static_cast<unsigned>(t), 0, 0};
}
int next_live(int from, int step) {
  int n = from;
  do n = (n + threads + step) % threads;
  while (ended[n] && n != from);
  return n;
}
int next_thread() {
  if (order == 0) return next_live(current, 1);
  if (order == 1) return next_live(current, -1);
  random_state = random_state * 6364136223846793005ull + 1442695040888963407ull;
  int n = (random_state >> 60) == 0 ? static_cast<int>((random_state >> 33) % threads) : current;
  const int first = n & ~63, count = threads - first < 64 ? threads - first : 64, start = n;
  do n = first + (n - first + 1) % count;
  while ((ended[n] || n == current) && n != start);
  return ended[n] || n == current ? next_live(current, 1) : n;
}
void give_way() {
  const int me = current, n = next_thread();
  if (n == me) {
    if (ended[me]) switch_fiber(&saved[me], main_saved);
    return;
  }
  set_current(n);
  switch_fiber(&saved[me], saved[n]);
  set_current(me);
}
void fiber() {
  (*kernel_body)();
  ended[current] = true;
  Wave& w = waves[current >> 6];
  w.mask &= ~(uint64_t(1) << (current & 63));
  if (--w.live && w.arrived == w.live) w.step();
  if (--live_threads && at_barrier == live_threads) {
    at_barrier = 0;
    ++barrier_round;
  }
  give_way();
  fail("a thread that has ended was resumed");
}
}  // namespace

void wave_exchange(uint64_t v, uint64_t* all, uint64_t* live) {
  Wave& w = waves[current >> 6];
  const unsigned round = w.round;
  w.slot[round & 1][current & 63] = v;
  if (++w.arrived == w.live) w.step();
  for (long i = 0; w.round == round; ++i) {
    give_way();
    if (i > MAX_WAIT) fail("a wave waits for a lane that does not come");
  }
  memcpy(all, w.slot[round & 1], sizeof w.slot[0]);
  *live = w.live_at[round & 1];
}

void block_barrier() {
  const unsigned round = barrier_round;
  if (++at_barrier == live_threads) {
    at_barrier = 0;
    ++barrier_round;
  }
  for (long i = 0; barrier_round == round; ++i) {
    give_way();
    if (i > MAX_WAIT) fail("a barrier that not every thread reaches");
  }
}

void run_grid(dim3 grid, dim3 block, size_t lds, const std::function<void()>& kernel, const char* name) {
  kernel_name = name;
  kernel_body = &kernel;
  threads = block.x;
  if (threads < 1 || threads > MAX_THREADS || block.y * block.z != 1 || !grid.x || !grid.y || grid.z != 1 ||
      static_cast<uint64_t>(grid.x) * threads >= uint64_t(1) << 32 || lds > MAX_LDS)
    fail("a launch that the device refuses");
  gridDim = {grid.x, grid.y, grid.z};
  blockDim = {block.x, 1, 1};
  for (unsigned y = 0; y < grid.y; ++y)
    for (unsigned x = 0; x < grid.x; ++x) {
      blockIdx = {x, y, 0};
      dynamic_lds = static_cast<char*>(malloc(lds ? lds : 1));
      memset(dynamic_lds, 0x5a, lds);
      memset(waves, 0, sizeof waves);
      live_threads = threads;
      at_barrier = 0;
      for (int t = 0; t < threads; ++t) {
        if (!stacks[t])
          stacks[t] = mmap(nullptr, STACK, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0);
        void** top = reinterpret_cast<void**>(static_cast<char*>(stacks[t]) + STACK);
        *--top = nullptr;  // alignment
        *--top = reinterpret_cast<void*>(fiber);
        for (int i = 0; i < 6; ++i) *--top = nullptr;  // the registers that switch_fiber restores
        saved[t] = top;
        ended[t] = false;
        ++waves[t >> 6].live;
        waves[t >> 6].mask |= uint64_t(1) << (t & 63);
      }
      const int first = order == 1 ? threads - 1 : 0;
      set_current(first);
      switch_fiber(&main_saved, saved[first]);
      free(dynamic_lds);
    }
}

static char error_text[512];
void ghm_set_error(const char* text, const char*, int) { snprintf(error_text, sizeof error_text, "%s", text); }
int ghm_launch_status() { return 0; }
extern "C" const char* ghm_last_error_string() { return error_text; }
extern "C" int ghm_device_ok() { return 1; }
