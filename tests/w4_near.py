"""How near the products with 4-bit weights have to be on average, beside the
worst case that w4_cases.product gives."""

# A group's fp32 sum has terms of up to 111 |x| (w4_cases.product).  For rows x
# without a common sign its partial sums are 111 times the root of the sum of
# x^2 or less in the mean, and each of the 2 group / 32 matrix instructions
# rounds eight times at most, each 2^-23 off: together (independent) 8 * 2^-23 *
# 111 for a group of 128.  The result is that root times what q - zero is in the
# mean, 6.5 (with 55 and 4.6 where the zero is 8 everywhere): 1.6e-5 of it.
FP32_SUMS = 2e-5


def far(out, y):
    """||out - y|| / ||y||, in 64 bits."""

    return float((out.double() - y).norm() / y.norm())


def near_sums(out, y):
    """fp32 rows are as near y as fp32 sums are."""

    return far(out, y) <= FP32_SUMS


def near_rounded(out, y):
    """bf16 rows are as near y as its rounding is: a sum that is off by FP32_SUMS
    moves the rounding of few results, which stay one step of bf16 away."""

    nearest = y.float().to(out.dtype)
    return far(out, y) <= 1.02 * far(nearest, y) + FP32_SUMS
