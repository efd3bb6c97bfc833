// What kernels on pairs of CTAs (tcgen05 cta_group::2) share: the cluster's addresses and barriers, a pair's loads,
// products and commits. The division of the work between the two is described where it is used (psk_gemm_tc2.cuh,
// psk_head.cuh). No load is multicast.
#pragma once
#include "psk_gemm_tc.cuh"

namespace psk {
namespace tc2 {

PSK_DEV uint32_t cluster_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

// The address, in the cluster's shared-memory window, of the same offset in CTA `rank`.
PSK_DEV uint32_t map_to_rank(uint32_t local, uint32_t rank)
{
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(local), "r"(rank));
    return a;
}

PSK_DEV void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

PSK_DEV void mbar_arrive_cluster(uint32_t cluster_addr)
{
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// A load of one CTA of the pair, its completion counted on a barrier given by its cluster address (the leader's).
PSK_DEV void tma_load_4d_pair(uint32_t dst, const CUtensorMap *map, uint32_t bar_cluster, int c0, int c1, int c2, int c3)
{
    asm volatile(
        "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar_cluster), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
}

PSK_DEV void umma_pair(uint32_t tmem_c, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_c), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Arrives, once the products issued so far are complete, on the barrier at this offset in both CTAs of the pair.
PSK_DEV void umma_commit_pair(uint32_t bar)
{
    const uint16_t mask = 3;
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"(mask) : "memory");
}

PSK_DEV uint32_t instr_desc_pair(int in_f16, int b_n_major)
{
    uint32_t d = 0;
    d |= 1u << 4;
    d |= (in_f16 ? 0u : 1u) << 7;
    d |= (in_f16 ? 0u : 1u) << 10;
    d |= (b_n_major ? 1u : 0u) << 16;
    d |= (uint32_t)(256 >> 3) << 17; // N of the pair
    d |= (uint32_t)(256 >> 4) << 24; // M of the pair
    return d;
}

} // namespace tc2
} // namespace psk
