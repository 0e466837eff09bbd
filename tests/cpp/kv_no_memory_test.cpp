// kv_no_memory_test.cpp -- the cache and attention calls where the host's memory runs out while a message is made: the
// exception stays inside, the status says failure and ns_last_error() says why.  No GPU is needed.  Exit status 0 = pass.
// Built by __graft_entry__.build() and run by tests/test_kv_host.py.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <new>

#include "ns_ffn.h"

namespace {
bool none_left = false;
}
void *operator new(std::size_t n) {
    void *p = none_left ? nullptr : std::malloc(n);
    if (!p) throw std::bad_alloc();
    return p;
}
void operator delete(void *p) noexcept { std::free(p); }
void operator delete(void *p, std::size_t) noexcept { std::free(p); }

int main() {
    int failures = 0;
    for (int op = 0; op < 3; ++op) {
        auto call = [&] {
            if (op == 0)
                return ns_kv_append(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 1, nullptr, nullptr, nullptr, 0.f, nullptr, 0, 0, nullptr, nullptr);
            if (op == 1) return ns_paged_attention(nullptr, nullptr, nullptr, nullptr, 1, 1.f, 0, nullptr, 1, nullptr);
            return ns_shared_prefix_attention(nullptr, nullptr, nullptr, 0, nullptr, 1, 1.f, nullptr, 1, nullptr);
        };
        none_left = true;
        const int rc = call();
        const bool said = std::strcmp(ns_last_error(), "no host memory") == 0;
        none_left = false;
        const int rc2 = call();
        const bool again = std::strstr(ns_last_error(), "null context") != nullptr;
        std::printf("call %d: status %d, message %s; with memory %d, message %s\n", op, rc, said ? "right" : "wrong", rc2, again ? "right" : "wrong");
        failures += !(rc == NS_ERR_HIP && said && rc2 == NS_ERR_ARG && again);
    }
    std::printf(failures ? "FAILED\n" : "PASSED\n");
    return failures;
}
