/* host_fork.c - lmc_model_fork_seq's page accounting on a machine without a
 * GPU (tests/test_host_fork.py): the model runtime linked with the host
 * stand-ins of host_shard_fakes.c, whose main is put aside.  A forward takes
 * its pages and stops at its first kernel launch, so the pool's count shows
 * what it took; a page's copy is a host memcpy.  One line per step:
 * "F <rc> <free pages>". */
#define main shards_main
#include "host_shard_fakes.c"
#undef main
int lmc_model_fork_seq(lmc_model *m, int src, int dst);

static void step(lmc_model *m, int rc) {
    int ps = 0, np = 0, nf = -1;
    lmc_model_kv_pages(m, &ps, &np, &nf);
    printf("F %d %d\n", rc, nf);
}

int main(int argc, char **argv) {
    if (argc < 2) return 2;
    lmc_model *m = NULL;
    int rc = lmc_model_load_paged(argv[1], 3, 8, LMC_KV_F16, 16, 8, 0, 1, NULL, &m);
    printf("rc %d %s\n", rc, rc ? lmc_last_error() : "");
    if (rc) return 0;
    int tok[8] = {1, 2, 3, 1, 2, 3, 1, 2}, pos[3] = {39, 0, 0}, ids[3];
    step(m, lmc_model_forward(m, tok, pos, 1, NULL, NULL)); /* sequence 0: 3 pages, 5 free */
    step(m, lmc_model_fork_seq(m, 0, 1));                   /* shared: 5 free */
    step(m, lmc_model_fork_seq(m, 1, 2));                   /* three holders of each page */
    step(m, lmc_model_fork_seq(m, 2, 2));                   /* nothing */
    pos[0] = 40, pos[1] = 41, pos[2] = 42;
    step(m, lmc_model_forward(m, tok, pos, 3, NULL, NULL)); /* page 3 of each: two copies, the third keeps it: 3 free */
    step(m, lmc_model_forward(m, tok, pos, 3, NULL, NULL)); /* writable already: 3 free */
    step(m, lmc_model_prefill(m, 1, tok, 8, 12, NULL, NULL)); /* positions 12-19 of sequence 1: pages 1 and 2 copied: 1 free */
    step(m, lmc_model_release_seq(m, 0));                   /* its copy of page 3 only: 2 free */
    pos[0] = 0;
    step(m, lmc_model_prefill(m, 2, tok, 1, 0, NULL, NULL)); /* sequence 2 alone holds page 1 now: nothing taken */
    step(m, lmc_model_fork_seq(m, 1, 0));                   /* sequence 0 shares sequence 1's three */
    step(m, lmc_model_generate(m, tok, 2, 2, 40, 1, ids));  /* positions 0-40 of 0 and 1: three copies wanted, 2 free */
    step(m, lmc_model_fork_seq(m, 2, 1));                   /* sequence 1's pages stay with 0 */
    step(m, lmc_model_release_seq(m, 0));                   /* the last holder of those: 5 free */
    step(m, lmc_model_release_seq(m, 1));                   /* shared with 2 */
    step(m, lmc_model_release_seq(m, 2));                   /* all 8 */
    step(m, lmc_model_fork_seq(m, 0, 1));                   /* an empty sequence */
    step(m, lmc_model_fork_seq(m, 0, 3));                   /* no such sequence */
    step(m, lmc_model_fork_seq(m, -1, 0));
    step(m, lmc_model_fork_seq(NULL, 0, 1));
    lmc_model_free(m);
    rc = lmc_model_load(argv[1], 2, LMC_KV_F16, &m);
    printf("rc %d\n", rc);
    printf("C %d %s\n", lmc_model_fork_seq(m, 0, 1), lmc_last_error());
    lmc_model_free(m);
    return 0;
}
