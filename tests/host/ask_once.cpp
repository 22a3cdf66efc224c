// ask_once (vc_cluster.h): answers are kept, failures are not.
#include "vc_cluster.h"

#include <stdio.h>

static int fails = 0;
#define CHECK(x) \
    if (!(x)) { \
        printf("line %d: %s\n", __LINE__, #x); \
        fails++; \
    }

int main() {
    std::atomic<int> known{0};
    int n = 7, asked = 0;
    auto answer = [&](int value, cudaError_t e) {
        return [&asked, value, e](int *out) {
            asked++;
            *out = value;
            return e;
        };
    };
    CHECK(vc::ask_once(known, &n, answer(5, cudaErrorUnknown)) == cudaErrorUnknown && known.load() == 0);
    CHECK(vc::ask_once(known, &n, answer(9, cudaSuccess)) == cudaSuccess && n == 9 && asked == 2);
    CHECK(vc::ask_once(known, &n, answer(3, cudaErrorUnknown)) == cudaSuccess && n == 9 && asked == 2);
    std::atomic<int> none{0};
    CHECK(vc::ask_once(none, &n, answer(0, cudaSuccess)) == cudaSuccess && n == -1);
    CHECK(vc::ask_once(none, &n, answer(4, cudaSuccess)) == cudaSuccess && n == -1 && asked == 3);
    std::atomic<int> large{0};
    CHECK(vc::ask_once(large, &n, answer(2, cudaErrorInvalidClusterSize)) == cudaSuccess && n == -1);
    return fails;
}
