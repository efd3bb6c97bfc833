// Test support: the head's losses' argument check compiled for the host, so that the refusals are tested without a GPU.
#include "../../presk_b200/csrc/psk_head_shape.h"
#include <cstring>

extern "C" int head_shape_check(const psk_launch *l, char *err, size_t cap)
{
    psk::HeadShape h;
    std::string e;
    const int rc = psk::head_shape(l, h, e);
    strncpy(err, e.c_str(), cap - 1);
    err[cap - 1] = 0;
    return rc;
}
