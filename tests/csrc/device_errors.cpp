// Prints status and text of al_device_errors for the recorded words given as
// arguments (index=value).
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "../../arclight_amd/csrc/device_errors.hpp"

int main(int argc, char ** argv) {
    int w[kErrWords] = {};
    for (int i = 1; i < argc; ++i) w[atoi(argv[i])] = atoi(strchr(argv[i], '=') + 1);
    std::string text;
    const int status = device_error_status(w, text);
    printf("%d %s\n", status, text.c_str());
    return 0;
}
