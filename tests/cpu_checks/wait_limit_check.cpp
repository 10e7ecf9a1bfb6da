// How long a wait for the products of a tile lasts: `ns` nanoseconds for each of `steps` steps (negative: they never come).  Prints whether they were waited for, and
// after how many seconds.
#include "fake_warp.hpp"

static double now_ns, each_ns, done_ns;
static bool bar_try(uint32_t, unsigned)
{
    now_ns += each_ns;                              // a look takes a while
    return done_ns >= 0 && now_ns >= done_ns;
}
static unsigned long long global_timer() { return 5000000000000ull + (unsigned long long)now_ns; }
#include "kernels.inc"

int main(int argc, char **argv)
{
    if (argc != 3) return 2;
    const double steps = atof(argv[1]), ns = atof(argv[2]);
    done_ns = ns < 0 ? -1 : steps * ns;
    each_ns = 1e5;
    volatile int broken = 0;
    const bool came = bar_wait(0, 0, &broken, (int)steps);
    printf("%d %d %.3f\n", (int)came, broken, now_ns * 1e-9);
    return 0;
}
