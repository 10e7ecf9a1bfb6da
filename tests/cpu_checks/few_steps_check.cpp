// The teams of the one-token kernels, with waits that only some threads of a team see run out: the whole team leaves, and the kernel ends.
//
//   few_steps_check <thread of the team> <step> <both>
//
// from that thread on, threads of team 1 give up at that step; both: those of team 4 do so at their next one, as they find that a wait has run out.
#include "fake_warp.hpp"

#include <mutex>

static const int TEAMS = 6, PER_TEAM = 128, STEPS = 40;
static int from_thread, bad_step, both;
static fake::Barrier named[TEAMS];
static thread_local unsigned long long waits;
static std::atomic<int> agreed[TEAMS][1024];        // threads that said yes to a vote
static thread_local int votes;

static void bar_init(uint32_t, unsigned) {}
static uint32_t smem_at(const void *) { return 0; }
static void team_sync(int team) { named[team].wait(PER_TEAM * ++waits); }
CB_UNUSED static bool team_all(int team, bool v)
{
    std::atomic<int> &n = agreed[team][votes++];
    n += v;
    team_sync(team);
    return n.load() == PER_TEAM;
}
static thread_local int waited;
static bool bar_wait(uint32_t, unsigned, volatile int *broken)
{
    const int team = (int)threadIdx.x / PER_TEAM, step = waited++;
    if (team == 1 && step == bad_step && (int)threadIdx.x % PER_TEAM >= from_thread) {
        *broken = 1;
        return false;
    }
    if (both && team == 4 && step > bad_step && (int)threadIdx.x % 3 == 0) return false;
    return true;
}
#include "kernels.inc"

static std::mutex mu;
static std::vector<int> taken[TEAMS];

int main(int argc, char **argv)
{
    if (argc != 4) return 2;
    from_thread = atoi(argv[1]);
    bad_step = atoi(argv[2]);
    both = atoi(argv[3]);
    static unsigned char ring[1];
    static int head[16];
    fake::run_block(TEAMS * PER_TEAM, 0, 1, [&] {
        int now = -1;
        few_steps(
            STEPS, ring, head, [](int, uint32_t, uint32_t) {}, [&](int step) { now = step; },
            [&](const unsigned char *) {
                __shfl_xor_sync(0xffffffffu, 1.0f, 1);          // all lanes of the warp have come
                team_sync((int)threadIdx.x / PER_TEAM);
                std::lock_guard<std::mutex> lk(mu);
                taken[threadIdx.x / PER_TEAM].push_back(now);
            });
    });
    for (int t = 0; t < TEAMS; t++) {
        // all of a team's threads have worked on the same steps
        const int gives_up = t == 1 ? bad_step : t == 4 && both ? bad_step + 1 : 1000, own = (STEPS - t + TEAMS - 1) / TEAMS, want = own < gives_up ? own : gives_up;
        if ((int)taken[t].size() != want * PER_TEAM) {
            printf("team %d: %d steps of threads instead of %d\n", t, (int)taken[t].size(), want * PER_TEAM);
            return 1;
        }
    }
    if (head[2] != 1) {
        printf("not told\n");
        return 1;
    }
    printf("ok\n");
    return 0;
}
