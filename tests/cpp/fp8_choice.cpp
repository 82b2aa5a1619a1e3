// The choice of a kernel for products in block-scaled 8-bit floating point, product by product.  Reads lines of `experts M N K gate` and prints the name's
// place in the list of kernels that is chosen for each on 256 CUs.
#include "../../nnfusion_amd/csrc/nnf_fp8_plan.h"

#include <cstdio>

int main()
{
    int experts, m, n, k, gate;
    while (scanf("%d %d %d %d %d", &experts, &m, &n, &k, &gate) == 5)
        printf("%d\n", (int)nnf::fp8::choose(m, n, k, gate != 0, experts, 256));
    return 0;
}
