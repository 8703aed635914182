// The current device around a call, with stand-ins for the two CUDA functions.
#include <cstdio>
#include <vector>

#include "rg_device_scope.h"

static int current = 0, get_fails = 0, set_fails = 0;
static std::vector<int> sets;
struct fake {
    static int get(int* d) { return get_fails ? 1 : (*d = current, 0); }
    static int set(int d) { return sets.push_back(d), set_fails ? 7 : (current = d, 0); }
};
typedef rg_device_scope<fake> scope;

#define EXPECT(c) do { if (!(c)) return printf("line %d: %s\n", __LINE__, #c), 1; } while (0)

int main() {
    { scope s(0, true); EXPECT(current == 0 && sets.empty() && s.failed() == 0); }
    EXPECT(sets.empty());  // nothing to do, nothing done
    { scope s(2, true); EXPECT(current == 2); }
    EXPECT(current == 0 && (sets == std::vector<int>{2, 0}));
    { scope s(2, true); { scope t(3, true); EXPECT(current == 3); } EXPECT(current == 2); }
    EXPECT(current == 0);
    { scope s(2, false); EXPECT(current == 2); }
    EXPECT(current == 2);
    sets.clear(), current = 0, set_fails = 1;
    { scope s(9, true); EXPECT(s.failed() == 7 && current == 0); }
    set_fails = 0, get_fails = 1, sets.clear();
    { scope s(1, true); EXPECT(current == 1); }
    EXPECT(current == 1 && sets.size() == 1);  // what was current is not known: nothing to put back
    puts("OK");
}
