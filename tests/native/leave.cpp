// The sanitized drivers' entry: the driver's own main is compiled as driver_main, and
// the program leaves without the exit handlers.  The GPU runtime's free memory there,
// which can make the sanitizer give device memory out of its quarantine back to that
// runtime, gone by then, and it fails for that after every check has passed.
#include <cstdio>
#include <cstdlib>

int driver_main();

int main() {
    const int rc = driver_main();
    fflush(stdout);
    fflush(stderr);
    std::_Exit(rc);
}
