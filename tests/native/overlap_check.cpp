// Host build of opfoundry_amd/csrc/dsa_overlap.h for tests/test_overlap.py.
#include "../../opfoundry_amd/csrc/dsa_overlap.h"

extern "C" {

int rows_within(int64_t T, int64_t H, int64_t st, int64_t sh, int64_t w) {
    return dsa_overlap::within({T, H, st, sh, w});
}
int rows_between(int64_t T, int64_t Ha, int64_t sta, int64_t sha, int64_t Hb, int64_t stb, int64_t shb, int64_t w,
                 int64_t delta) {
    return dsa_overlap::between({T, Ha, sta, sha, w}, {T, Hb, stb, shb, w}, delta);
}

}  // extern "C"
