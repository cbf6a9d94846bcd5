// Runs a kernel compiled for the CPU lane by lane: one workgroup after the other, each lane a context of its own.  A lane runs until it meets its wave
// (a builtin that looks at other lanes) or its workgroup (a barrier), or ends; a wave goes on when all its lanes that have not ended wait at the same
// place, a workgroup when all its waves do.  Lanes that meet in different numbers end the process.  Waves run one after the other between barriers, so
// a missing barrier is not found here.  Test infrastructure only.
#include <hip/hip_runtime.h>

#include <setjmp.h>
#include <stdio.h>
#include <stdlib.h>
#include <sys/mman.h>
#include <ucontext.h>

#include <vector>

namespace lanes {

dim3 thread, block, threads, blocks;
alignas(16) char dynamic_memory[160 << 10];

enum State { kRuns, kMeetsWave, kMeetsBlock, kEnded };
constexpr size_t kStack = 256 << 10;

struct Lane {
    jmp_buf at;  // (ucontext's own switch is a system call each time)
    char* stack;
    State state;
    unsigned meetings;  // with its wave
};
struct Wave {
    Words given[2][64];  // of this meeting and the one before, which some lanes may not have read yet
    uint64_t arrived[2];
    unsigned meeting[2];
};

static std::vector<Lane> all;
static std::vector<Wave> waves;
static jmp_buf scheduler;
static int current;
static const std::function<void()>* body;

static void wait(State state) {
    Lane& lane = all[current];
    lane.state = state;
    if (_setjmp(lane.at) == 0) _longjmp(scheduler, 1);
}

Seen meet_wave(const Words& mine) {
    const int me = current;
    Wave& wave = waves[me / 64];
    const unsigned meeting = ++all[me].meetings;
    const int now = meeting & 1;
    if (wave.meeting[now] != meeting) {
        wave.meeting[now] = meeting;
        wave.arrived[now] = 0;
        memset(wave.given[now], 0xee, sizeof wave.given[now]);  // lanes that have ended give nothing sensible
    }
    wave.given[now][me % 64] = mine;
    wave.arrived[now] |= 1ull << me % 64;
    wait(kMeetsWave);
    return {wave.given[now], wave.arrived[now], me % 64};
}

void meet_block() { wait(kMeetsBlock); }

// A lane's context is made once; it runs one workgroup's lane after the other.
static ucontext_t maker, made;

static void entry() {
    Lane& lane = all[current];
    if (_setjmp(lane.at) == 0) swapcontext(&made, &maker);
    for (;;) {
        (*body)();
        wait(kEnded);
    }
}

static void fail(const char* why) {
    fprintf(stderr, "workgroup %u, %u: %s\n", block.x, block.y, why);
    abort();
}

// Until all the wave's lanes wait for the workgroup or have ended.
static void run_wave(int first, int last) {
    for (;;) {
        for (current = first; current < last; ++current) {
            if (all[current].state != kRuns) continue;
            thread = dim3(current % threads.x, current / threads.x);
            if (_setjmp(scheduler) == 0) _longjmp(all[current].at, 1);
        }
        bool meets = false, waits = false;
        unsigned meeting = 0;
        for (int i = first; i < last; ++i) {
            waits |= all[i].state == kMeetsBlock;
            if (all[i].state != kMeetsWave) continue;
            if (meets && all[i].meetings != meeting) fail("lanes of a wave in different meetings");
            meets = true;
            meeting = all[i].meetings;
        }
        if (!meets) return;
        if (waits) fail("lanes of a wave at a barrier while others meet");
        for (int i = first; i < last; ++i)
            if (all[i].state == kMeetsWave) all[i].state = kRuns;
    }
}

void launch(dim3 grid, dim3 group, const std::function<void()>& kernel) {
    const int n = group.x * group.y;
    threads = group;
    blocks = grid;
    body = &kernel;
    all.reserve(1024);  // (a workgroup's most: lanes keep their place)
    while ((int)all.size() < n) {
        current = (int)all.size();
        all.push_back(Lane());
        all.back().stack = static_cast<char*>(mmap(nullptr, kStack, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0));
        getcontext(&made);
        made.uc_stack.ss_sp = all.back().stack;
        made.uc_stack.ss_size = kStack;
        made.uc_link = nullptr;
        makecontext(&made, entry, 0);
        swapcontext(&maker, &made);
    }
    for (unsigned y = 0; y < grid.y; ++y)
        for (unsigned x = 0; x < grid.x; ++x) {
            block = dim3(x, y);
            waves.assign((n + 63) / 64, Wave());
            for (int i = 0; i < n; ++i) {
                all[i].state = kRuns;
                all[i].meetings = 0;
            }
            for (bool ended = false; !ended;) {
                ended = true;
                for (int first = 0; first < n; first += 64) run_wave(first, std::min(n, first + 64));
                for (int i = 0; i < n; ++i) {
                    ended &= all[i].state == kEnded;
                    if (all[i].state == kMeetsBlock) all[i].state = kRuns;
                }
            }
        }
}

}  // namespace lanes

namespace hfrk {
void set_last_hip_error(hipError_t) {}
}  // namespace hfrk
