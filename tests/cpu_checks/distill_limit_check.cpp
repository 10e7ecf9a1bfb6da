// The limits that calls of distill_loss set for their kernels' shared memory.  Arguments: numbers of columns, a call for each, with and
// without lse and gradient.  Prints each kernel's smallest and largest limit.
#include "fake_launch.hpp"

namespace cb200 {
unsigned *next_counter() { static unsigned c; return &c; }
}  // namespace cb200

int main(int argc, char **argv)
{
    std::map<std::string, std::pair<int, int>> limits;
    fake::on_shared_limit = [&](const std::string &name, int v) {
        auto &l = limits.insert({name, {v, v}}).first->second;
        l = {v < l.first ? v : l.first, v > l.second ? v : l.second};
    };
    const double options[2] = {1.0, 1.0};
    int64_t pos[1001] = {};
    float word[1000] = {};
    for (int i = 1; i < argc; i++)
        for (int form = 0; form < 4; form++) {
            const int64_t n = atoll(argv[i]);
            if (comet_b200_dev_distill_loss_f32_i64(1000, n, pos, pos, word, 4, form & 1 ? word : nullptr, nullptr, word, n, form & 2 ? word : nullptr, n, options,
                                                    word, word, nullptr) ||
                comet_b200_dev_distill_loss_bf16_i64(1000, n, pos, pos, word, 4, form & 1 ? word : nullptr, nullptr, word, n, form & 2 ? word : nullptr, n, options,
                                                     word, word, nullptr)) {
                printf("%s\n", cb200::g_err);
                return 1;
            }
        }
    for (auto &l : limits) printf("%d %d\n", l.second.first, l.second.second);
    return 0;
}
