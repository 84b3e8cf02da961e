"""Which kernel a product of 4-bit blocks goes to (csrc/gemm_tiles.h, compiled here as host code)."""
import pytest

from test_gemm_tiles import host_program

# (M, N, K): us of the ring tiles 32 x 64, 64 x 64, 128 x 64, 128 x 128 and of 128 x 128 and 256 x 256 tiles on
# MI355X, weights from HBM
TIMES = {
    (64, 9216, 3072): (10.4, 9.1, 9.6, 11.9, 17.0, None),
    (128, 3072, 12288): (20.2, 20.7, 26.4, 36.0, 59.7, None),
    (256, 9216, 3072): (24.1, 16.9, 15.7, 13.6, 18.3, 26.8),
    (513, 3072, 3072): (15.3, 9.8, 9.3, 11.6, 15.3, 22.6),
    (513, 12288, 3072): (51.9, 32.8, 26.9, 26.5, 22.6, 27.0),
    (1024, 3072, 12288): (67.3, 47.3, 42.4, 38.0, 56.6, 91.8),
    (2048, 3072, 3072): (46.9, 28.9, 22.1, 26.1, 20.0, 24.1),
    (2048, 9216, 3072): (131.2, 78.0, 57.5, 63.3, 57.7, 53.0),
    (4096, 1024, 1024): (16.8, 11.1, 8.2, 8.3, 8.9, 11.8),
    (4096, 12288, 3072): (314.2, 197.8, 144.6, 152.8, 132.2, 95.8),
}
# kernels that the GPU tests' shapes are meant to reach
SHAPES = {(1, 9216, 3072): 0, (7, 1001, 288): 1, (3, 64, 8224): 2, (17, 130, 512): 3, (33, 2100, 96): 10,
          (200, 2100, 800): 4, (130, 4100, 800): 5, (300, 4100, 320): 6, (256, 9216, 2080): 7, (513, 12288, 800): 8, (2100, 1001, 768): 6,
          (4100, 4104, 256): 8, (6000, 4100, 288): 9}


@pytest.fixture(scope="module")
def pick(tmp_path_factory):
    run = host_program(tmp_path_factory.mktemp("mx"), """
int main() {
  long long m, n, k, c;
  while (std::scanf("%lld %lld %lld %lld", &m, &n, &k, &c) == 4)
    std::printf("%d\\n", mxf8::mxfp4_pick(m, n, k, (int)c));
}""")
    return lambda shapes, cus=256: [r[0] for r in run([(*s, cus) for s in shapes])]


def test_the_choice_is_close_to_the_fastest(pick):
    for (shape, times), p in zip(TIMES.items(), pick(TIMES)):
        t = times[p - 4]
        assert t is not None and t <= 1.08 * min(x for x in times if x), (shape, p)


def test_few_tokens_go_to_the_rows_kernel(pick):
    assert pick([(m, n, 3072) for m in (1, 16) for n in (1, 3072, 12288)]) == [2, 2, 0, 2, 2, 0]
    assert pick([(1, 3072, 12288), (1, 12288, 12288), (32, 3072, 3072), (32, 9216, 3072), (64, 2048, 512)])[:3] == [2, 1, 3]
    assert pick([(32, 9216, 3072)])[0] >= 4 and pick([(64, 2048, 512)]) == [3] and pick([(65, 2048, 512)])[0] >= 4


@pytest.mark.parametrize("cus", [1, 8, 256])
def test_every_size_has_a_kernel(pick, cus):
    sizes = [(m, n, k) for m in (1, 17, 65, 5000, 1 << 27) for n in (1, 70, 5000, 1 << 27) for k in (32, 12288, 1 << 22)]
    assert all(0 <= p <= 10 for p in pick(sizes, cus))


def test_gpu_test_shapes_of_whole_stages_reach_every_tile_kernel(pick):
    """The shapes of tests/test_gpu_mxfp4.py's test of that name, and those whose slices it compares bit for bit."""
    shapes = {(200, 2100, 768): 4, (130, 4100, 768): 5, (300, 4100, 768): 6, (256, 9216, 2048): 7, (513, 12288, 768): 8,
              (8200, 4100, 768): 9, (4097, 8200, 1024): 9, (2100, 4100, 1536): 9}
    assert dict(zip(shapes, pick(shapes))) == shapes
    for k in (768, 800, 1280):
        slices = [(m, 4100, k) for m in (60, 130, 300, 700, 1100, 2100, 4200, 8200)]
        assert min(pick(slices)) == 4 and max(pick(slices)) == 9 and 10 not in pick(slices)
        assert len(set(pick([(m, 4100, k) for m in range(1, 17)]))) == 1


def test_gpu_test_shapes_reach_every_kernel(pick):
    assert dict(zip(SHAPES, pick(SHAPES))) == SHAPES and set(SHAPES.values()) == set(range(11))
