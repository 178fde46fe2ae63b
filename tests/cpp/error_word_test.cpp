// The words for the sticky device error word, on the host.  Prints "error word ok".
#include "host_logic.h"

#include <cstdio>
#include <cstdlib>

static void expect(bool ok, const char *what) {
    if (ok) return;
    std::fprintf(stderr, "expected %s\n", what);
    std::exit(1);
}
static bool has(unsigned word, const char *text) { return lcu::describe_error_word(word).find(text) != std::string::npos; }

int main() {
    for (unsigned w = 1; w < 16; ++w) {
        expect(has(w, ("device error word " + std::to_string(w)).c_str()), "the word itself");
        expect(has(w, "bounded wait") == ((w & 3) != 0), "a wait for bits 0 and 1 only");
        expect(has(w, "out of range") == ((w & 4) != 0), "an index for bit 2 only");
        expect(has(w, "unknown") == ((w & 8) != 0), "unknown bits to be named");
    }
    std::puts("error word ok");
    return 0;
}
