"""The registry of plans in workspace buffers, compiled by itself: operators that keep no plan push none out, and a
program without memory gets no exception out of a C function."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA = "/usr/local/cuda/include"

MAIN = r"""
#include <cassert>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <new>

#include "internal.h"

static bool gNoMemory = false;
void* operator new(std::size_t n)
{
    if (gNoMemory) {
        throw std::bad_alloc();
    }
    return std::malloc(n);
}
void operator delete(void* p) noexcept { std::free(p); }
void operator delete(void* p, std::size_t) noexcept { std::free(p); }

#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)

static const void* At(uintptr_t i) { return reinterpret_cast<const void*>(0x10000 + 64 * i); }

int main()
{
    // nothing is recorded before there is memory for the registry itself
    gNoMemory = true;
    CHECK(AclspPublishPlan(At(0)) == 0);
    CHECK(!AclspPlanIsCurrent(At(0), 1));
    AclspForgetPlan(At(0));
    gNoMemory = false;

    const uint64_t plan = AclspPublishPlan(At(0));
    CHECK(plan != 0 && AclspPlanIsCurrent(At(0), plan) && !AclspPlanIsCurrent(At(1), plan));
    for (uintptr_t i = 1; i < 5000; ++i) {  // buffers without plans: as many as there may be
        AclspForgetPlan(At(i));
    }
    CHECK(AclspPlanIsCurrent(At(0), plan));
    AclspForgetPlan(At(0));
    CHECK(!AclspPlanIsCurrent(At(0), plan));

    // 1024 plans, and the oldest one goes
    uint64_t serial[1025];
    for (uintptr_t i = 0; i < 1024; ++i) {
        serial[i] = AclspPublishPlan(At(i));
    }
    for (uintptr_t i = 0; i < 1024; ++i) {
        CHECK(AclspPlanIsCurrent(At(i), serial[i]));
    }
    const uint64_t newer = AclspPublishPlan(At(0));  // the oldest becomes the newest
    CHECK(newer > serial[0] && !AclspPlanIsCurrent(At(0), serial[0]) && AclspPlanIsCurrent(At(0), newer));
    serial[1024] = AclspPublishPlan(At(1024));
    CHECK(AclspPlanIsCurrent(At(1024), serial[1024]) && !AclspPlanIsCurrent(At(1), serial[1]));
    CHECK(AclspPlanIsCurrent(At(2), serial[2]) && AclspPlanIsCurrent(At(0), newer));

    // no memory: a known buffer's plan is renewed, an unknown buffer has none, nothing else changes
    gNoMemory = true;
    const uint64_t last = AclspPublishPlan(At(0));
    CHECK(last > newer && AclspPlanIsCurrent(At(0), last) && !AclspPlanIsCurrent(At(0), newer));
    CHECK(AclspPublishPlan(At(9000)) == 0 && !AclspPlanIsCurrent(At(9000), 0));
    CHECK(AclspPlanIsCurrent(At(2), serial[2]));
    AclspForgetPlan(At(2));
    CHECK(!AclspPlanIsCurrent(At(2), serial[2]));
    gNoMemory = false;
    CHECK(AclspPlanIsCurrent(At(3), serial[3]));
    CHECK(AclspPlanIsCurrent(At(9000), AclspPublishPlan(At(9000))));
    std::puts("ok");
    return 0;
}
"""


def test_registry_forgets_and_never_throws(tmp_path):
    if shutil.which("g++") is None or not os.path.exists(CUDA):
        pytest.skip("no C++ compiler or CUDA headers")
    (tmp_path / "main.cpp").write_text(MAIN)
    src = os.path.join(ROOT, "ops_sparse_b200", "csrc")
    exe = tmp_path / "registry"
    subprocess.run(["g++", "-std=c++17", "-I", src, "-I", os.path.join(ROOT, "include"), "-I", CUDA, str(tmp_path / "main.cpp"),
                    os.path.join(src, "plan_registry.cpp"), "-o", str(exe), "-lpthread"], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout + done.stderr
