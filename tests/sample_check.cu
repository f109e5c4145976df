// Host-only driver for tests/test_sample_split.py: prints how sampling cuts n rows of vocab words over CTAs, by the library's own
// rule (sample_split in serve.h), for every vocab of a range.
#include "../nunchi_b200/csrc/serve.h"

#include <cstdio>
#include <cstdlib>

int main(int argc, char **argv) {
    if (argc != 5) return 2;
    const int n = atoi(argv[1]), lo = atoi(argv[2]), hi = atoi(argv[3]), step = atoi(argv[4]);
    for (int v = lo; v <= hi; v += step) {
        const imi::SampleSplit s = imi::sample_split(n, v);
        printf("%d %d %d %d %d\n", v, s.ctas, s.seg, s.share, s.rank);
    }
    return 0;
}
