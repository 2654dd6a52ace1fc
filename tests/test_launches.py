"""Which kernels the 8-bit path launches, and what it does where clusters are refused (contexts with restricted SM sets): host code,
run here against a runtime that launches nothing."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "backpack_b200", "csrc")
OBJ = os.path.join(os.path.dirname(HERE), "backpack_b200", "lib", "obj")
CUDA = os.path.dirname(os.path.dirname(shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"))


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    objects = [os.path.join(OBJ, name) for name in ("bpq4k_logprobs.o", "i8_matmul.o")]
    if not all(map(os.path.exists, objects)):
        subprocess.run(["make", "-C", CSRC], check=True, capture_output=True)
    so = str(tmp_path_factory.mktemp("fake") / "libfake.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-fvisibility=hidden", "-I", os.path.join(CUDA, "include"), "-o", so,
                    os.path.join(HERE, "fake_cudart.cpp"), *objects,
                    "-Wl,-Bsymbolic", "-Wl,--no-undefined", "-lpthread"], check=True)
    lib = C.CDLL(so)
    lib.fake_launch.restype = C.c_char_p
    return lib


def launches(fake):
    out, found = (C.c_uint * 4)(), []
    for i in range(fake.fake_count()):
        name = fake.fake_launch(i, out).decode()
        found.append(dict(name=name, grid=out[0], block=out[1], cluster=out[2], refused=bool(out[3])))
    return found


@pytest.mark.parametrize("ftype", [0, 1, 30])
@pytest.mark.parametrize("M,V,top,group", [(1, 128256, 20, 8), (1, 128256, 0, 8), (48, 32003, 5, 4), (130, 32000, 20, 4), (8, 8192, 32, 2), (700, 128256, 5, 1), (1, 70, 1, 1)])
def test_log_probabilities_without_clusters(fake, ftype, M, V, top, group):
    fake.fake_reset(16, 0, 148)
    assert fake.fake_logprobs(ftype, M, V, top, 148) == 0
    (one,) = launches(fake)
    assert one["cluster"] == group and one["grid"] == M * group
    # the same where no cluster may be launched: a CTA to a row, the error is gone
    fake.fake_reset(1, 0, 148)
    assert fake.fake_logprobs(ftype, M, V, top, 148) == 0
    *refused, last = launches(fake)
    assert len(refused) == (group > 1) and all(r["refused"] for r in refused)
    assert not last["refused"] and last["cluster"] == 1 and last["grid"] == M and fake.fake_last_error() == 0


# ---- the 8-bit matmul: (M, N, K), CTAs of a cluster on a whole device ---------------------------------------------------------

PRODUCTS = [(13, 6144, 4096, 2), (64, 1024, 8192, 8), (100, 2048, 14336, 8), (2048, 28672, 8192, 2), (16, 128256, 4096, 1), (1, 1024, 4096, 1)]


@pytest.mark.parametrize("ftype", [0, 1, 30])
@pytest.mark.parametrize("M,N,K,cluster", PRODUCTS)
def test_products_where_clusters_are_refused(fake, ftype, M, N, K, cluster):
    fake.fake_reset(16, 0, 148)
    assert fake.fake_matmul(1, ftype, M, N, K, 148) == 0
    (one,) = launches(fake)
    assert one["cluster"] == cluster
    # a context that says so when it is asked: no launch with a cluster is tried
    fake.fake_reset(1, 0, 148)
    assert fake.fake_matmul(1, ftype, M, N, K, 148) == 0
    (alone,) = launches(fake)
    assert alone["cluster"] == 1 and not alone["refused"] and alone["grid"] >= 1
    # a handle that has asked in a whole context, called in one that refuses
    fake.fake_reset(16, 0, 148)
    assert fake.fake_matmul(1, ftype, M, N, K, 148) == 0
    fake.fake_reset(1, 0, 148)
    assert fake.fake_matmul(0, ftype, M, N, K, 148) == 0
    *refused, last = launches(fake)
    assert len(refused) == (cluster > 1) and all(r["refused"] for r in refused)
    assert last["cluster"] == 1 and not last["refused"] and last["name"] == alone["name"] and last["grid"] == alone["grid"] and fake.fake_last_error() == 0


def test_what_a_restricted_context_answers_is_not_kept_for_others(fake):
    fake.fake_reset(1, 0, 148)
    assert fake.fake_matmul(1, 0, 2048, 28672, 8192, 148) == 0
    fake.fake_reset(16, 0, 148)
    assert fake.fake_matmul(1, 0, 2048, 28672, 8192, 148) == 0       # another handle
    assert [l["cluster"] for l in launches(fake)] == [2]


def test_a_failed_question_is_asked_again(fake):
    fake.fake_reset(16, 2, 148)
    assert fake.fake_matmul(1, 0, 2048, 28672, 8192, 148) == 0
    assert [l["cluster"] for l in launches(fake)] == [1] and fake.fake_last_error() == 0
    fake.fake_reset(16, 0, 148)
    assert fake.fake_matmul(0, 0, 2048, 28672, 8192, 148) == 0
    assert [l["cluster"] for l in launches(fake)] == [2]
    asked = fake.fake_queries()
    assert fake.fake_matmul(0, 0, 2048, 28672, 8192, 148) == 0 and fake.fake_queries() == asked      # and an answer is kept
